// Decode attention over a KV cache held in 8 bits.
//
// Mathematics.  With K = ck * sk, V = cv * sv (codes and per-block scales) a row j contributes, to one query head,
//     x_j = (q . ck_j) * sk_j * scale * log2(e)          l = sum_j 2^(x_j - m)
//     y_j = x_j + log2(sv_j)                              o = sum_j 2^(y_j - M + 11) cv_j
//     out = o / l * 2^(M - m - 11)
// with references m, M near the running maxima of x and y: they follow only when a value has outgrown them (x by 2^32, y
// by 2^4, so that a weight stays below fp16's 2^16), which spares most tiles the reduction over the warp and the scaling
// of o.  The V scale rides in the exponent, so the weights that meet the codes have one range whatever the scales: they
// round to fp16 (11 bits, three more than the bf16 weights of a 16-bit cache) and one that is 2^-35 of the largest still
// counts.
//
// The codes are fp16 numbers exactly (e4m3: the conversion instruction; int8: a byte permutation and a subtraction), the
// queries too after a power of two per head, but for elements more than 2^27 below the head's largest, which fp16's subnormals
// round to 2^-38 of it.  Sums are fp32, in the MMA and outside.
//
// Layout.  A warp works alone: its own ring of 32-row tiles, its own mbarriers, no CTA barrier until the end of a segment.
// Rows are the M side of both products (S^T = K q^T and O^T = V^T P^T with m16n8k16), the query heads of a KV head the N
// side, so up to 8 heads cost one MMA column block, and a K row's 16-byte pieces are A fragments as they lie in shared
// memory: the order of the 128 dimensions inside a product is free as long as q follows it.  V rows are interleaved in
// pairs (byte permutations), P^T comes from S^T by movmatrix.
//
// Work.  The 32-row tiles of all (sequence, KV head) segments form one list that is cut into equal pieces, one per CTA
// (one CTA of twelve warps per SM), whatever the lengths: a CTA may end one segment and begin the next.  Every CTA leaves
// one partial (o, M, m, l) per segment that it touches, and the one that arrives last at a segment merges.  Where segments are
// short (ctas_per_segment below) each gets CTAs of its own instead: one, or a cluster whose CTAs send their partials straight
// into the shared memory of the one that finishes the head, which spares the merge three trips to L2.
//
// Bound: HBM, 256 bytes of codes and 8 / block bytes of scales per (row, KV head).
#include "kv8.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace omnikv {
namespace {

constexpr int MAX_G = 16;
// Warps of a CTA by column blocks: 168 and 255 registers a thread (of the 168, six instantiations of 32 spill one or two).
constexpr int kWarps[3] = {0, 12, 8};
constexpr int TILE = 32;                     // rows per tile: one lane per row when rows are fetched one by one
constexpr int STAGES = 2;
constexpr int BOX = TILE * kHeadDim;         // bytes of a K or V tile
constexpr int PITCH = 2 * kHeadDim + 16;     // row pitch of a tile fetched row by row (K | V | pad): conflict-free
constexpr int ROWS_STAGE = TILE * PITCH, TMA_STAGE = 2 * BOX;
constexpr int OS_PITCH = kHeadDim + 4;       // floats per head in the CTA's merge buffer

struct A8Args {
  const unsigned char *k, *v;
  int64_t sb, sh, sr;
  const float *ks, *vs;
  int64_t ssb, ssh;
  int shift, rows;
  const void* q;
  int64_t q_sb, q_sh;
  void* out;
  int64_t o_sb, o_sh;
  const int* idx;
  int64_t idx_stride;
  int idx_cap;
  const int *len, *tail_start, *tail_len;
  float* score_out;
  int64_t score_stride;
  const int* score_len;
  float* ws_o;      // [slot][G][128]
  float4* ws_ml;    // [slot][G] {M, m, l, -}
  unsigned* ws_cnt; // [B * KVH] arrivals, zero between launches
  int* status;
  int B, H, KVH, G, pair;
  int cluster;      // CTAs per segment where each has CTAs of its own
  float scale;
};

// The rows of a sequence: nA listed ones, then the tail [t0, t0 + nB).
struct RowList {
  int nA, nB, t0;
  __device__ __forceinline__ int n() const { return nA + nB; }
  __device__ __forceinline__ int tiles() const { return ceil_div(nA + nB, TILE); }
};
__device__ __forceinline__ RowList row_list(const A8Args& a, int b) {
  RowList r;
  r.nA = max(0, min(a.len[b], a.idx ? a.idx_cap : a.rows));
  r.t0 = 0;
  r.nB = 0;
  if (a.tail_len) {
    r.t0 = max(0, min(a.tail_start[b], a.rows));
    r.nB = max(0, min(a.tail_len[b], a.rows - r.t0));
  }
  return r;
}

// A place in the list of tiles.
struct Cursor {
  int b, kvh, tile, nt;
  RowList list;
  __device__ __forceinline__ void load(const A8Args& a) {
    list = row_list(a, b);
    nt = list.tiles();
  }
  // false: still in the same segment
  __device__ __forceinline__ bool forward(const A8Args& a, int by) {
    tile += by;
    if (tile < nt) return false;
    do {
      tile -= nt;
      if (++kvh == a.KVH) {
        kvh = 0;
        if (++b >= a.B) return true;
        load(a);
      }
    } while (tile >= nt);
    return true;
  }
};
// Where a segment's codes, scales and index list begin.
struct Sources {
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int* idx;
  __device__ __forceinline__ void of(const A8Args& a, int b, int kvh) {
    const int64_t at = (int64_t)b * a.sb + (int64_t)kvh * a.sh, sat = (int64_t)b * a.ssb + (int64_t)kvh * a.ssh;
    k = a.k + at;
    v = a.v + at;
    ks = a.ks + sat;
    vs = a.vs + sat;
    idx = a.idx ? a.idx + (int64_t)b * a.idx_stride : nullptr;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ unsigned movmatrix_trans(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ unsigned sub_h2(unsigned a, unsigned b) {
  unsigned y;
  asm("sub.f16x2 %0, %1, %2;\n" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

// Bytes 0, 1 (hi = false) or 2, 3 of w as two fp16 numbers, exactly.  int8: w ^ 0x80808080 holds code + 128, which under the
// exponent byte 0x64 is the number 1024 + 128 + code.
template <int FMT>
__device__ __forceinline__ unsigned prepare_word(unsigned w) {
  return FMT == kInt8 ? w ^ 0x80808080u : w;
}
template <int FMT, bool HI>
__device__ __forceinline__ unsigned half2_of(unsigned w) {
  if constexpr (FMT == kInt8) {
    return sub_h2(__byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140), 0x64806480u);
  } else {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(HI ? w >> 16 : w & 0xffffu), __NV_E4M3);
    return (unsigned)h.x | (unsigned)h.y << 16;
  }
}

__device__ __forceinline__ void st_cluster4(unsigned addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void cp_async4(void* smem_dst, const void* gmem_src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(smem_dst)), "l"(gmem_src) : "memory");
}

template <int NW>
struct Shared {
  uint64_t full[NW][STAGES];
  float scale[NW][STAGES][2][TILE];  // K and V scale of each row of a tile
  unsigned valid[NW][STAGES];        // rows of the tile that exist
  float ml[NW][MAX_G][3];            // M, m, l of the warps
  int last;
};

// COLS: n8 column blocks of query heads (1: up to 8 heads per KV head, 2: up to 16).  TMA: tiles as boxes of a tensor map
// (rows that follow one another), else rows fetched one by one.  CLUSTER: a cluster of a.cluster CTAs per segment.
template <typename T, int FMT, int COLS, bool TMA, bool CLUSTER>
__global__ void __launch_bounds__(kWarps[COLS] * 32, 1)
decode_attn_kv8_kernel(const A8Args a, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  constexpr int NW = kWarps[COLS], NT = NW * 32;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ Shared<NW> sh;
  constexpr int STAGE_BYTES = TMA ? TMA_STAGE : ROWS_STAGE;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + warp * STAGES * STAGE_BYTES;
  float* o_s = reinterpret_cast<float*>(smem + NW * STAGES * STAGE_BYTES);
  const int G = a.G;
  const float factor = a.scale * kLog2e;

  if (lane < STAGES) mbar_init(&sh.full[warp][lane], 1);
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  if (TMA && tid == 0) {
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(&tm_k) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(&tm_v) : "memory");
  }
  __syncwarp();
  pdl_wait();

  Cursor seg;  // the segment being worked on; tile = 0
  int seg_lo, w0, w1, W = 0, C = 1, each = 0, more = 0;
  bool own = CLUSTER;  // the segment is this CTA's (or its cluster's) alone
  const int c = blockIdx.x, rank = CLUSTER ? (int)cluster_rank() : 0;
  const auto piece_lo = [&](int i) { return i * each + i * more / C; };  // i * more < 2^30
  const auto owner = [&](int tile) {  // the CTA that has this tile
    int i = min(C - 1, (int)(((float)tile + 0.5f) * (float)C / (float)W));
    while (piece_lo(i) > tile) --i;
    while (piece_lo(i + 1) <= tile) ++i;
    return i;
  };
  if constexpr (CLUSTER) {
    seg.b = c / a.cluster / a.KVH;
    seg.kvh = c / a.cluster % a.KVH;
    seg.tile = seg_lo = 0;
    seg.load(a);
    if (seg.nt == 0) {
      if (rank == 0)
        for (int i = tid; i < G * (kHeadDim / 2); i += NT)
          reinterpret_cast<unsigned*>(static_cast<T*>(a.out) + (size_t)seg.b * a.o_sb + (size_t)(seg.kvh * G + (i >> 6)) * a.o_sh)[i & 63] = 0u;
      return;
    }
    cluster_arrive();  // this CTA runs: its shared memory may be written
    w0 = (int)((long long)rank * seg.nt / a.cluster);
    w1 = (int)((long long)(rank + 1) * seg.nt / a.cluster);
  } else {
    // ---- this CTA's piece of the list: tiles [w0, w1) of W ----
    int per_head = 0, filled = 0, longest = 0;  // tiles of all sequences, per KV head; sequences that have any; most tiles
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      const int mine = b0 + lane < a.B ? row_list(a, b0 + lane).tiles() : 0;
      per_head += __reduce_add_sync(0xffffffffu, mine);
      filled += __popc(__ballot_sync(0xffffffffu, mine > 0));
      longest = max(longest, __reduce_max_sync(0xffffffffu, mine));
  }
    if (filled < a.B) {  // a sequence without rows: zeros, written by one CTA
      for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
        if (row_list(a, b).n() > 0) continue;
        for (int i = tid; i < a.H * (kHeadDim / 2); i += NT)
          reinterpret_cast<unsigned*>(static_cast<T*>(a.out) + (size_t)b * a.o_sb + (size_t)(i >> 6) * a.o_sh)[i & 63] = 0u;
      }
      if (filled == 0) return;
  }
    // Pieces.  Segments of different lengths, no more than there are CTAs and none much longer than a CTA's share: one CTA for
    // each.  One piece per segment too when four tiles per warp do a segment: a merge across CTAs costs more than it saves
    // then.  Else as many as there are CTAs; with segments of one length a multiple of them, so that pieces end where segments
    // end, where the CTAs that leaves idle cost less than that spares (5 us, or 2.3 tiles per warp; 12 x 3000 rows of 8 heads:
    // 29.7 us with 148 pieces, 23.3 with 96).
    const int segs = filled * a.KVH, grid = gridDim.x;
    const bool even = longest * filled == per_head;
    W = per_head * a.KVH;
    own = !even && segs <= grid && longest <= W / grid + 32 + segs / 6;
    C = min(grid, own || W <= segs * NW * 4 ? segs : max(W / NW, segs));
    C = min(C, max(segs, (int)sqrtf(12.8f * (float)W * (float)segs / (float)G)));  // a tile costs 190 ns, a partial's head 15 in the merge
    if (C > segs && even && (float)(C % segs) * (float)W <= 2.3f * NW * (float)C * (float)C) C -= C % segs;
    if (c >= C) return;
    int found = -1;
    if (own) {
      int at = c / a.KVH;  // among the sequences that have rows
      for (int b0 = 0; found < 0; b0 += 32) {
        const unsigned some = __ballot_sync(0xffffffffu, b0 + lane < a.B && row_list(a, min(b0 + lane, a.B - 1)).n() > 0);
        if (at < __popc(some)) found = b0 + (int)__fns(some, 0, at + 1);
        at -= __popc(some);
      }
      seg.kvh = c % a.KVH;
      seg.b = found;
      seg.load(a);
      seg_lo = w0 = 0;
      w1 = seg.nt;
    } else {
      each = W / C;
      more = W - each * C;
      w0 = piece_lo(c);
      w1 = piece_lo(c + 1);
      int before = 0;  // tiles per KV head of the sequences in front
      for (int b0 = 0; found < 0; b0 += 32) {
        const int mine = b0 + lane < a.B ? row_list(a, b0 + lane).tiles() : 0;
        int sum = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, sum, off);
          if (lane >= off) sum += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, (before + sum) * a.KVH > w0);
        const int at = hit ? __ffs(hit) - 1 : 31;
        before += __shfl_sync(0xffffffffu, hit ? sum - mine : sum, at);
        if (hit) found = b0 + at;
      }
      seg.b = found;
      seg.load(a);
      seg.kvh = (w0 - before * a.KVH) / seg.nt;
      seg_lo = before * a.KVH + seg.kvh * seg.nt;
    }
    seg.tile = 0;
  }

  // ---- the warp's stream of tiles: every NW-th of the piece ----
  Cursor ahead = seg;  // the next tile to ask for
  Sources from;
  int ahead_w = w0 + warp;
  int asked = 0, pos = -1;
  const auto find_row = [&]() {  // the cache position of this lane's row in the tile to ask for, -1: none
    pos = -1;
    if (ahead_w < w1) {
      const int r = ahead.tile * TILE + lane;
      if (r < ahead.list.nA) pos = from.idx ? from.idx[r] : r;
      else if (r < ahead.list.n()) pos = ahead.list.t0 + (r - ahead.list.nA);
    }
  };
  bool dead = false;  // a wait for a tile has run out: nothing more is asked for
  const auto ask = [&]() {  // copies of one tile, and of its rows' scales
    if (ahead_w < w1 && !dead) {
      const int s = asked % STAGES;
      unsigned char* dst = ring + s * STAGE_BYTES;
      const bool ok = (unsigned)pos < (unsigned)a.rows;
      const unsigned valid = __ballot_sync(0xffffffffu, ok);
      if (lane == 0) {
        sh.valid[warp][s] = valid;
        mbar_expect_tx(&sh.full[warp][s], TMA ? TMA_STAGE : __popc(valid) * 2 * kHeadDim);
        if constexpr (TMA) {
          tma_load_4d(dst, &tm_k, 0, ahead.tile * TILE, ahead.kvh, ahead.b, &sh.full[warp][s]);
          tma_load_4d(dst + BOX, &tm_v, 0, ahead.tile * TILE, ahead.kvh, ahead.b, &sh.full[warp][s]);
        }
      }
      __syncwarp();
      if (ok) {
        if constexpr (!TMA) {
          const int64_t at = (int64_t)pos * a.sr;
          if (a.pair) {
            tma_bulk_g2s(dst + lane * PITCH, from.k + at, 2 * kHeadDim, &sh.full[warp][s]);
          } else {
            tma_bulk_g2s(dst + lane * PITCH, from.k + at, kHeadDim, &sh.full[warp][s]);
            tma_bulk_g2s(dst + lane * PITCH + kHeadDim, from.v + at, kHeadDim, &sh.full[warp][s]);
          }
        }
        cp_async4(&sh.scale[warp][s][0][lane], from.ks + (pos >> a.shift));
        cp_async4(&sh.scale[warp][s][1][lane], from.vs + (pos >> a.shift));
      }
      ++asked;
      ahead_w += NW;
      if (ahead_w < w1 && ahead.forward(a, NW)) from.of(a, ahead.b, ahead.kvh);
    }
    cp_async_commit();
    find_row();
  };
  ahead.tile = w0 - seg_lo;
  if (ahead_w < w1) ahead.forward(a, warp);
  from.of(a, min(ahead.b, a.B - 1), ahead.kvh);
  find_row();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) ask();

  int used = 0;
  int next_w = w0 + warp;  // the warp's next tile
  for (int lo = w0; CLUSTER || lo < w1;) {
    const int seg_hi = seg_lo + seg.nt, hi = min(w1, seg_hi);  // this CTA's tiles of the segment: [lo, hi)
    const int b = seg.b, kvh = seg.kvh, seg_no = b * a.KVH + kvh;
    const int c_lo = own ? 0 : owner(seg_lo), parts = own ? 1 : owner(seg_hi - 1) - c_lo + 1;  // the CTAs that share it

    // ---- queries: fragments of q * 2^e (largest element in [2^13, 2^14)); a logit is z (ks 2^-e) scale log2(e) ----
    unsigned qf[COLS][8][2];
    float qs[COLS][2];  // 2^-e
#pragma unroll
    for (int cb = 0; cb < COLS; ++cb) {
      const int h = cb * 8 + g;
      uint2 raw[8];
      unsigned top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        raw[j] = make_uint2(0, 0);
        if (h < G)
          raw[j] = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.q) + (size_t)b * a.q_sb + (size_t)(kvh * G + h) * a.q_sh +
                                                   16 * (2 * t + (j >> 2)) + 4 * (j & 3));
        const float2 x = unpack16<T>(raw[j].x), y = unpack16<T>(raw[j].y);
        top = max(top, max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(y.x), abs_bits(y.y))));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(13 - ((int)(top >> 23) - 127), 126);
      const float up = __uint_as_float((unsigned)(e + 127) << 23), down = exp2f((float)-e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 x = unpack16<T>(raw[j].x), y = unpack16<T>(raw[j].y);
        qf[cb][j][0] = pack2<__half>(x.x * up, x.y * up);
        qf[cb][j][1] = pack2<__half>(y.x * up, y.y * up);
      }
      qs[cb][0] = __shfl_sync(0xffffffffu, down, 8 * t);
      qs[cb][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
    }
    const int score_lim = a.score_out ? (int)min((int64_t)min(a.score_len[b], seg.list.nA), a.score_stride) : 0;
    float* score_row = a.score_out ? a.score_out + ((size_t)kvh * a.B + b) * a.score_stride : nullptr;

    float m[COLS][2], M[COLS][2], l[COLS][2], o[COLS][8][4];
#pragma unroll
    for (int cb = 0; cb < COLS; ++cb) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m[cb][e] = M[cb][e] = -INFINITY, l[cb][e] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[cb][i][0] = o[cb][i][1] = o[cb][i][2] = o[cb][i][3] = 0.f;
    }

    for (; next_w < hi; next_w += NW) {
      const int s = used % STAGES;
      __syncwarp();  // all lanes are done with the tile whose stage is refilled now
      ask();
      cp_async_wait<STAGES - 1>();
      if (__any_sync(0xffffffffu, !dead && !mbar_wait(&sh.full[warp][s], (used / STAGES) & 1))) {
        // The warp goes on, so that others get the partials and arrivals they count on, with what lies in its ring; the
        // copies that it has asked for land first (a bounded wait each): the ring becomes a merge buffer, then another CTA's.
        dead = true;
        if (lane == 0 && a.status) atomicExch(a.status, 5);
        for (int i = used; i < asked; ++i) mbar_wait(&sh.full[warp][i % STAGES], (i / STAGES) & 1);
        __syncwarp();
      }
      const unsigned char* tile = ring + s * STAGE_BYTES;
      // the 16-byte piece c of row r of the tile's K or V rows
      const auto piece = [&](int v, int r, int cc) {
        if constexpr (TMA) return *reinterpret_cast<const uint4*>(tile + v * BOX + r * kHeadDim + ((cc ^ (r & 7)) << 4));
        else return *reinterpret_cast<const uint4*>(tile + r * PITCH + v * kHeadDim + (cc << 4));
      };
      const unsigned valid = sh.valid[warp][s];
      const float my_ks = sh.scale[warp][s][0][lane], my_lv = log2f(sh.scale[warp][s][1][lane]);

      // ---- S^T = K q^T ----
      float x[2][COLS][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int cb = 0; cb < COLS; ++cb) x[i][cb][0] = x[i][cb][1] = x[i][cb][2] = x[i][cb][3] = 0.f;
        uint4 r0[2], r1[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          r0[u] = piece(0, 16 * i + g, 2 * t + u);
          r1[u] = piece(0, 16 * i + 8 + g, 2 * t + u);
        }
        const unsigned* p0 = reinterpret_cast<const unsigned*>(r0);
        const unsigned* p1 = reinterpret_cast<const unsigned*>(r1);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned u0 = prepare_word<FMT>(p0[j]), u1 = prepare_word<FMT>(p1[j]);
          const unsigned af[4] = {half2_of<FMT, false>(u0), half2_of<FMT, false>(u1), half2_of<FMT, true>(u0), half2_of<FMT, true>(u1)};
#pragma unroll
          for (int cb = 0; cb < COLS; ++cb) mma_16816<__half>(x[i][cb], af, qf[cb][j][0], qf[cb][j][1]);
        }
      }
      // ---- scales, mask, scores ----
      const int row0 = (next_w - seg_lo) * TILE;
      float lv[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // rows 16 i + 8 u + g
          const int r = 16 * i + 8 * u + g;
          const float ks = __shfl_sync(0xffffffffu, my_ks, r);
          lv[i][u] = __shfl_sync(0xffffffffu, my_lv, r);
          const bool ok = (valid >> r) & 1u;
          if (!ok) lv[i][u] = 0.f;  // a scale that was not read
#pragma unroll
          for (int cb = 0; cb < COLS; ++cb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& z = x[i][cb][2 * u + e];
              z = ok ? z * (ks * qs[cb][e]) * factor : -INFINITY;  // (z * ks may leave fp32's range where the logit is in it)
            }
        }
      if (a.score_out) {
        // largest over the heads: a thread holds two heads of four rows (8 j + g); the four threads of a row group trade
        // halves twice, after which thread t has row 8 t + g
        float best[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          best[j] = -INFINITY;
#pragma unroll
          for (int cb = 0; cb < COLS; ++cb)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (cb * 8 + 2 * t + e < G) best[j] = max_nan(best[j], x[j >> 1][cb][2 * (j & 1) + e]);
        }
        const float s0 = (t & 2) ? best[0] : best[2], s1 = (t & 2) ? best[1] : best[3];
        const float k0 = max_nan((t & 2) ? best[2] : best[0], __shfl_xor_sync(0xffffffffu, s0, 2));
        const float k1 = max_nan((t & 2) ? best[3] : best[1], __shfl_xor_sync(0xffffffffu, s1, 2));
        const float mine = max_nan((t & 1) ? k1 : k0, __shfl_xor_sync(0xffffffffu, (t & 1) ? k0 : k1, 1));
        if (row0 + 8 * t + g < score_lim) score_row[row0 + 8 * t + g] = mine * (1.f / kLog2e);
      }
      // ---- weights ----
      unsigned pb[2][COLS][2];
#pragma unroll
      for (int cb = 0; cb < COLS; ++cb) {
        float mx[2], My[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = My[e] = -INFINITY;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              mx[e] = fmaxf(mx[e], x[i][cb][2 * u + e]);
              My[e] = fmaxf(My[e], x[i][cb][2 * u + e] + lv[i][u]);
            }
        }
        const bool outgrown = mx[0] > m[cb][0] + 32.f || mx[1] > m[cb][1] + 32.f || My[0] > M[cb][0] + 4.f || My[1] > M[cb][1] + 4.f;
        if (__any_sync(0xffffffffu, outgrown)) {
          float corr[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
              mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], off));
              My[e] = fmaxf(My[e], __shfl_xor_sync(0xffffffffu, My[e], off));
            }
            mx[e] = fmaxf(m[cb][e], mx[e]);
            My[e] = fmaxf(M[cb][e], My[e]);
            l[cb][e] *= m[cb][e] == mx[e] ? 1.f : ex2(m[cb][e] - mx[e]);
            corr[e] = M[cb][e] == My[e] ? 1.f : ex2(M[cb][e] - My[e]);
            m[cb][e] = mx[e];
            M[cb][e] = My[e];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o[cb][i][0] *= corr[0];
            o[cb][i][1] *= corr[1];
            o[cb][i][2] *= corr[0];
            o[cb][i][3] *= corr[1];
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float mu = m[cb][e] == -INFINITY ? 0.f : m[cb][e], Mu = M[cb][e] == -INFINITY ? 0.f : M[cb][e] - 11.f;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              float& z = x[i][cb][2 * u + e];
              l[cb][e] += ex2(z - mu);
              z = ex2(z + lv[i][u] - Mu);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          pb[i][cb][0] = movmatrix_trans(pack2<__half>(x[i][cb][0], x[i][cb][1]));
          pb[i][cb][1] = movmatrix_trans(pack2<__half>(x[i][cb][2], x[i][cb][3]));
        }
      }
      // ---- O^T += V^T P^T: thread (g, t) holds dimensions 16 g .. 16 g + 15 of four rows ----
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4 v0 = piece(1, 16 * i + 2 * t, g), v1 = piece(1, 16 * i + 2 * t + 1, g);
        uint4 v2 = piece(1, 16 * i + 8 + 2 * t, g), v3 = piece(1, 16 * i + 9 + 2 * t, g);
        if (FMT == kE4m3 && valid != 0xffffffffu) {  // what lies in the place of a missing row may be a NaN code
          const auto keep = [&](uint4& v, int r) {
            if (!((valid >> r) & 1u)) v = make_uint4(0, 0, 0, 0);
          };
          keep(v0, 16 * i + 2 * t);
          keep(v1, 16 * i + 2 * t + 1);
          keep(v2, 16 * i + 8 + 2 * t);
          keep(v3, 16 * i + 9 + 2 * t);
        }
        const unsigned* w0p = reinterpret_cast<const unsigned*>(&v0);
        const unsigned* w1p = reinterpret_cast<const unsigned*>(&v1);
        const unsigned* w2p = reinterpret_cast<const unsigned*>(&v2);
        const unsigned* w3p = reinterpret_cast<const unsigned*>(&v3);
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const unsigned sel = half ? 0x7362 : 0x5140;  // bytes 2 half, 2 half + 1 of two rows, interleaved
            const unsigned ab = prepare_word<FMT>(__byte_perm(w0p[w], w1p[w], sel));
            const unsigned cd = prepare_word<FMT>(__byte_perm(w2p[w], w3p[w], sel));
            const unsigned af[4] = {half2_of<FMT, false>(ab), half2_of<FMT, true>(ab), half2_of<FMT, false>(cd), half2_of<FMT, true>(cd)};
#pragma unroll
            for (int cb = 0; cb < COLS; ++cb) mma_16816<__half>(o[cb][2 * w + half], af, pb[i][cb][0], pb[i][cb][1]);
          }
      }
      ++used;
    }

    // ---- the CTA's partial of the segment ----
    // Behind the CTA's last segment the rings are free and every warp leaves its sums in its own; before that the warps add
    // theirs up in turns in the few buffers that o_s holds (next tiles are on their way into the rings meanwhile).
    const bool last_seg = hi == w1;
    const int bufs = min(NW, MAX_G / G);
    if (last_seg) pdl_trigger();
#pragma unroll
    for (int cb = 0; cb < COLS; ++cb)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[cb][e] += __shfl_xor_sync(0xffffffffu, l[cb][e], off);
        const int h = cb * 8 + 2 * t + e;
        if (g == 0) {
          sh.ml[warp][h][0] = M[cb][e];
          sh.ml[warp][h][1] = m[cb][e];
          sh.ml[warp][h][2] = l[cb][e];
        }
      }
    const auto leave = [&](float* to, bool add, bool scaled) {
#pragma unroll
      for (int cb = 0; cb < COLS; ++cb)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int h = cb * 8 + 2 * t + e;
          if (h >= G) continue;
          float f = 1.f;
          if (scaled) {
            float Ms = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; ++w) Ms = fmaxf(Ms, sh.ml[w][h][0]);
            f = M[cb][e] == Ms ? 1.f : ex2(M[cb][e] - Ms);
          }
          float4* dst = reinterpret_cast<float4*>(to + h * OS_PITCH + 16 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float4 y = make_float4(o[cb][2 * i][e] * f, o[cb][2 * i][2 + e] * f, o[cb][2 * i + 1][e] * f, o[cb][2 * i + 1][2 + e] * f);
            if (add) {
              const float4 old = dst[i];
              y.x += old.x, y.y += old.y, y.z += old.z, y.w += old.w;
            }
            dst[i] = y;
          }
        }
    };
    if (last_seg) {
      __syncwarp();
      leave(reinterpret_cast<float*>(ring), false, false);
      __syncthreads();
    } else {
      __syncthreads();
#pragma unroll 1
      for (int turn = 0; turn * bufs < NW; ++turn) {
        const int buf = warp - turn * bufs;
        if (buf >= 0 && buf < bufs) leave(o_s + buf * G * OS_PITCH, turn > 0, true);
        __syncthreads();
      }
    }
    const auto write_out = [&](int h, const float4& acc, float Ms, float ms, float L) {  // a head without rows: zero
      const float f = L == 0.f ? 0.f : exp2f(Ms - ms - 11.f) / L;
      T* dst = static_cast<T*>(a.out) + (size_t)b * a.o_sb + (size_t)(kvh * G + h) * a.o_sh + lane * 4;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * f, acc.y * f), pack2<T>(acc.z * f, acc.w * f));
    };
    const int hp = CLUSTER ? ceil_div(G, a.cluster) : 0;  // heads that a CTA of the cluster finishes: head h, CTA h % cluster
    if constexpr (CLUSTER) cluster_wait();
    for (int h = warp; h < G; h += NW) {  // a head per warp: lane w holds the factors of warp w's sums
      float Mw = -INFINITY, mw = -INFINITY, L = 0.f;
      if (lane < NW) {
        Mw = sh.ml[lane][h][0];
        mw = sh.ml[lane][h][1];
        L = sh.ml[lane][h][2];
      }
      float Ms = Mw, ms = mw;
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) {
        Ms = fmaxf(Ms, __shfl_xor_sync(0xffffffffu, Ms, off));
        ms = fmaxf(ms, __shfl_xor_sync(0xffffffffu, ms, off));
      }
      Ms = __shfl_sync(0xffffffffu, Ms, 0);
      ms = __shfl_sync(0xffffffffu, ms, 0);
      if (L != 0.f && mw != ms) L *= ex2(mw - ms);
      const float f = Mw == Ms ? 1.f : ex2(Mw - Ms);
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (last_seg) {
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * STAGES * STAGE_BYTES) + h * OS_PITCH + lane * 4);
          const float fw = __shfl_sync(0xffffffffu, f, w);
          acc.x = fmaf(v.x, fw, acc.x), acc.y = fmaf(v.y, fw, acc.y), acc.z = fmaf(v.z, fw, acc.z), acc.w = fmaf(v.w, fw, acc.w);
        }
      } else {
        for (int buf = 0; buf < bufs; ++buf) {
          const float4 v = *reinterpret_cast<const float4*>(o_s + (buf * G + h) * OS_PITCH + lane * 4);
          acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
        }
      }
      if constexpr (CLUSTER) {
        const unsigned to = in_cta(smem_u32(o_s + (rank * hp + h / a.cluster) * OS_PITCH), h % a.cluster);
        st_cluster4(to + lane * 16, acc);
        if (lane == 0) st_cluster4(to + kHeadDim * 4, make_float4(Ms, ms, L, 0.f));
      } else if (parts == 1) {
        write_out(h, acc, Ms, ms, __shfl_sync(0xffffffffu, L, 0));
      } else {
        const size_t slot = (size_t)(c + seg_no) * G + h;  // (CTA, segment) pairs walk a staircase: their sum is unique
        *reinterpret_cast<float4*>(a.ws_o + slot * kHeadDim + lane * 4) = acc;
        if (lane == 0) a.ws_ml[slot] = make_float4(Ms, ms, L, 0.f);
      }
    }
    if constexpr (CLUSTER) {
      __syncwarp();
      cluster_sync_all();  // the partials of every CTA are where they are merged
      for (int i = warp; i * a.cluster + rank < G; i += NW) {
        const float* part = o_s + i * OS_PITCH;
        float4 mine = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);  // lane p: M, m, l of CTA p
        if (lane < a.cluster) mine = *reinterpret_cast<const float4*>(part + lane * hp * OS_PITCH + kHeadDim);
        float Ms = mine.x, ms = mine.y;
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) {
          Ms = fmaxf(Ms, __shfl_xor_sync(0xffffffffu, Ms, off));
          ms = fmaxf(ms, __shfl_xor_sync(0xffffffffu, ms, off));
        }
        Ms = __shfl_sync(0xffffffffu, Ms, 0);
        ms = __shfl_sync(0xffffffffu, ms, 0);
        float L = mine.z != 0.f && mine.y != ms ? mine.z * ex2(mine.y - ms) : mine.z;
        const float f = mine.x == Ms ? 1.f : ex2(mine.x - Ms);
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < a.cluster; ++p) {
          const float4 v = *reinterpret_cast<const float4*>(part + p * hp * OS_PITCH + lane * 4);
          const float fp = __shfl_sync(0xffffffffu, f, p);
          acc.x = fmaf(v.x, fp, acc.x), acc.y = fmaf(v.y, fp, acc.y), acc.z = fmaf(v.z, fp, acc.z), acc.w = fmaf(v.w, fp, acc.w);
        }
        write_out(i * a.cluster + rank, acc, Ms, ms, __shfl_sync(0xffffffffu, L, 0));
      }
      break;
    }
    if (parts > 1) {
      __syncthreads();
      if (tid == 0) {
        __threadfence();  // the CTA's stores, ordered before the barrier, are visible before its arrival is
        sh.last = atomicAdd(a.ws_cnt + seg_no, 1u) == (unsigned)(parts - 1);
        __threadfence();
      }
      __syncthreads();
      if (sh.last) {
        // `per` warps share a head, each with every per-th partial, four dimensions per lane; their sums meet in o_s
        const int per = max(1, NW / G);
        for (int h0 = 0; h0 < G; h0 += NW / per) {
          const int h = h0 + warp / per, part = warp % per;
          const bool on = h < min(G, h0 + NW / per);
          float Ms = -INFINITY, ms = -INFINITY, L = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          if (on) {
            const size_t base = (size_t)(c_lo + seg_no) * G + h;
            const float4* op = reinterpret_cast<const float4*>(a.ws_o + base * kHeadDim) + lane;
            const float4* mp = a.ws_ml + base;
            const int o_step = G * (kHeadDim / 4);
            constexpr int PRE = 8;
            float4 first_o[PRE];  // this warp's partials part, part + per, ...: asked for together with the maxima
#pragma unroll
            for (int i = 0; i < PRE; ++i) first_o[i] = part + i * per < parts ? __ldcg(op + (size_t)(part + i * per) * o_step) : acc;
            const float4 none = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
            const float4 first_ml = lane < parts ? __ldcg(mp + (size_t)lane * G) : none;
            Ms = first_ml.x;
            ms = first_ml.y;
            for (int p = lane + 32; p < parts; p += 32) {
              const float4 v = __ldcg(mp + (size_t)p * G);
              Ms = fmaxf(Ms, v.x);
              ms = fmaxf(ms, v.y);
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) {
              Ms = fmaxf(Ms, __shfl_xor_sync(0xffffffffu, Ms, off));
              ms = fmaxf(ms, __shfl_xor_sync(0xffffffffu, ms, off));
            }
            const auto add = [&](const float4& v, float f) {
              acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
            };
            int p = part;
            for (int p0 = 0; p0 < parts; p0 += 32) {  // lane p - p0 holds the factor of partial p
              float4 v = first_ml;
              if (p0) v = p0 + lane < parts ? __ldcg(mp + (size_t)(p0 + lane) * G) : none;
              const float f = v.x == Ms ? 1.f : ex2(v.x - Ms);
              if (v.z != 0.f) L = fmaf(v.z, v.y == ms ? 1.f : ex2(v.y - ms), L);
              const int end = min(parts, p0 + 32);
              if (p0 == 0) {
#pragma unroll
                for (int i = 0; i < PRE; ++i) {
                  if (p >= end) continue;
                  add(first_o[i], __shfl_sync(0xffffffffu, f, p));
                  p += per;
                }
              }
#pragma unroll 8
              for (; p < end; p += per) add(__ldcg(op + (size_t)p * o_step), __shfl_sync(0xffffffffu, f, p - p0));
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
            if (per > 1) *reinterpret_cast<float4*>(o_s + warp * OS_PITCH + lane * 4) = acc;
          }
          if (per > 1) __syncthreads();
          if (on && part == 0) {
            for (int w = 1; w < per; ++w) {
              const float4 v = *reinterpret_cast<const float4*>(o_s + (warp + w) * OS_PITCH + lane * 4);
              acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
            }
            write_out(h, acc, Ms, ms, L);
          }
        }
        if (tid == 0) a.ws_cnt[seg_no] = 0u;
      }
    }
    // ---- the next segment ----
    lo = hi;
    if (lo < w1) {
      __syncthreads();  // the merge buffers are free again
      seg_lo = seg_hi;
      seg.tile = seg.nt;
      seg.forward(a, 0);
    }
  }
  cp_async_wait<0>();
}

constexpr int smem_bytes(bool tma, int cols) {
  return kWarps[cols] * STAGES * (tma ? TMA_STAGE : ROWS_STAGE) + 16 * OS_PITCH * 4 + 1024;
}

template <typename T, int FMT, int COLS, bool TMA, bool CLUSTER>
int launch(const A8Args& a, int ctas, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  auto kern = decode_attn_kv8_kernel<T, FMT, COLS, TMA, CLUSTER>;
  if (const int rc = allow_smem(kern, smem_bytes(TMA, COLS), done, CLUSTER)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kWarps[COLS] * 32);
  cfg.dynamicSmemBytes = smem_bytes(TMA, COLS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CLUSTER ? a.cluster : 1;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 2 : 1;
  if (CLUSTER && a.cluster > 8) {  // more than the portable eight: asked once per kernel, size and device
    static std::atomic<unsigned long long> known[17], fits[17];
    int dev = 0, most = 0;
    OMNIKV_CUDA_OK(cudaGetDevice(&dev));
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(known[a.cluster].load(std::memory_order_acquire) & bit)) {
      if (cudaOccupancyMaxActiveClusters(&most, kern, &cfg) != cudaSuccess) (void)cudaGetLastError();
      else if (most > 0) fits[a.cluster].fetch_or(bit, std::memory_order_relaxed);
      known[a.cluster].fetch_or(bit, std::memory_order_release);
    }
    if (!(fits[a.cluster].load(std::memory_order_relaxed) & bit)) {
      A8Args b = a;
      b.cluster = 8;
      return launch<T, FMT, COLS, TMA, CLUSTER>(b, ctas / a.cluster * 8, tm_k, tm_v, st);
    }
  }
  OMNIKV_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a, tm_k, tm_v));
  return OMNIKV_OK;
}

template <typename T, int FMT>
int launch_any(const A8Args& a, int ctas, bool tma, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  const auto go = [&](auto tiles, auto own) -> int {
    constexpr bool TMA = decltype(tiles)::value, CLUSTER = decltype(own)::value;
    return a.G <= 8 ? launch<T, FMT, 1, TMA, CLUSTER>(a, ctas, tm_k, tm_v, st) : launch<T, FMT, 2, TMA, CLUSTER>(a, ctas, tm_k, tm_v, st);
  };
  const std::true_type yes;
  const std::false_type no;
  if (a.cluster) {
    ctas = a.B * a.KVH * a.cluster;
    return tma ? go(yes, yes) : go(no, yes);
  }
  return tma ? go(yes, no) : go(no, no);
}

constexpr int kMaxCtas = 32768;

// CTAs per segment (1: a CTA for each, more: a cluster), or 0: the list cut over all SMs.  The one with the least estimated
// time (ns), the rows being as many as they can be (four fifths of that on average): a start, 1 / warps of a round per tile,
// what a cluster's exchange or the merges through L2 add (15 ns per head and partial of a segment).  kMost: clusters of so many CTAs that run at once on a B200's 148 SMs.  Measured, us, with 8 KV heads:
//   one sequence, list or one CTA, cluster   100 rows 5.5, 5.7   777: 10.3, 5.8   2000: 11.2, 6.6   8781: 11.8, 11.1
//                                            12000: 12.9, 13.2   8781 selected: 13.5, 12.8
//   16 ragged sequences, list, CTA each      700 rows at most: 21.9, 9.9   3000: 30.2, 22.7   12000: 64.0, 70.7
inline int ctas_per_segment(int B, int KVH, int G, int64_t rows, int n_ctas) {
  static constexpr int kMost[17] = {0, 0, 74, 45, 33, 26, 22, 15, 15, 15, 11, 7, 7, 7, 7, 7, 7};
  constexpr int kSms = 148;
  const int segs = B * KVH;
  const double tiles = (double)((rows + TILE - 1) / TILE), per_tile = 2300.0 / kWarps[G <= 8 ? 1 : 2];
  const double all = tiles * segs, ctas = std::min({(double)kSms, all / kWarps[G <= 8 ? 1 : 2], std::sqrt(12.8 * all * segs / G)});
  const double share = all / std::max(ctas, 1.0);
  double best = 5800 + (B == 1 ? per_tile * share + 2000 + 15 * G * ctas / segs : 0.8 * per_tile * share + 8000 + 34 * segs);
  int pick = 0;
  for (int cs = 1; cs <= 16; ++cs) {
    if (cs > 1 && (segs > kMost[cs] || (int64_t)cs * segs > n_ctas || cs * ceil_div(G, cs) > 16)) continue;
    const double ns = ceil_div(segs, cs > 1 ? segs : kSms) * (5300 + per_tile * tiles / cs) + (cs > 1 ? 40 * cs : 0);
    if (ns < best) {
      best = ns;
      pick = cs;
    }
  }
  return pick;
}

inline long long slots_of(int B, int KVH, int ctas) { return (long long)ctas + (long long)B * KVH; }

}  // namespace
}  // namespace omnikv

extern "C" size_t omnikv_kv8_attn_workspace_bytes(int B, int H, int KVH, int n_ctas) {
  using namespace omnikv;
  if (B <= 0 || H <= 0 || KVH <= 0 || H % KVH || n_ctas <= 0) return 0;
  return kAttnCntBytes + (size_t)slots_of(B, KVH, n_ctas) * (H / KVH) * (kHeadDim * sizeof(float) + sizeof(float4));
}

extern "C" int omnikv_kv8_decode_attn(const omnikv_kv8_attn_params* p, void* stream) {
  using namespace omnikv;
  if (!p) return OMNIKV_E_BADARG;
  const omnikv_kv8_cache& c = p->cache;
  if (const int rc = check_kv8_cache(&c)) return rc;
  const auto bad16 = [](const void* q) { return !q || (reinterpret_cast<uintptr_t>(q) & 15); };
  if (bad16(p->q) || bad16(p->out) || !p->len || p->H <= 0 || p->H % c.KVH || p->n_ctas <= 0) return OMNIKV_E_BADARG;
  if (p->q_stride_b % 8 || p->q_stride_h % 8 || p->out_stride_b % 8 || p->out_stride_h % 8) return OMNIKV_E_BADARG;
  if ((c.B > 1 && p->out_stride_b < kHeadDim) || (p->H > 1 && p->out_stride_h < kHeadDim)) return OMNIKV_E_BADARG;
  if (p->idx && (p->idx_cap <= 0 || p->idx_stride < 0)) return OMNIKV_E_BADARG;
  if (p->tail_len && !p->tail_start) return OMNIKV_E_BADARG;
  if (p->score_out && (p->idx || p->tail_len || !p->score_len || p->score_stride <= 0)) return OMNIKV_E_BADARG;
  if (!is_16bit(p->dtype) || p->H / c.KVH > MAX_G) return OMNIKV_E_UNSUPPORTED;
  const int64_t most = (p->idx ? p->idx_cap : (int64_t)c.rows) + (p->tail_len ? c.rows : 0);
  if (most > 0x7fffffff - TILE || (most / TILE + 2) * c.B * c.KVH > 0x7fffffff) return OMNIKV_E_UNSUPPORTED;  // rows and tiles are counted in 32 bits
  if (p->n_ctas > kMaxCtas || (size_t)c.B * c.KVH * 4 > kAttnCntBytes) return OMNIKV_E_UNSUPPORTED;
  if (!p->workspace || p->workspace_bytes < omnikv_kv8_attn_workspace_bytes(c.B, p->H, c.KVH, p->n_ctas)) return OMNIKV_E_WORKSPACE;
  if (bad16(p->workspace)) return OMNIKV_E_BADARG;
  A8Args a;
  a.k = static_cast<const unsigned char*>(c.k); a.v = static_cast<const unsigned char*>(c.v);
  a.sb = c.stride_b; a.sh = c.stride_h; a.sr = c.stride_row;
  a.ks = c.k_scale; a.vs = c.v_scale; a.ssb = c.scale_stride_b; a.ssh = c.scale_stride_h;
  a.shift = __builtin_ctz(c.block); a.rows = c.rows;
  a.q = p->q; a.q_sb = p->q_stride_b; a.q_sh = p->q_stride_h;
  a.out = p->out; a.o_sb = p->out_stride_b; a.o_sh = p->out_stride_h;
  a.idx = p->idx; a.idx_stride = p->idx_stride; a.idx_cap = p->idx_cap;
  a.len = p->len; a.tail_start = p->tail_start; a.tail_len = p->tail_len;
  a.score_out = p->score_out; a.score_stride = p->score_stride; a.score_len = p->score_len;
  a.B = c.B; a.H = p->H; a.KVH = c.KVH; a.G = p->H / c.KVH;
  a.ws_cnt = static_cast<unsigned*>(p->workspace);
  a.ws_ml = reinterpret_cast<float4*>(static_cast<unsigned char*>(p->workspace) + kAttnCntBytes);
  a.ws_o = reinterpret_cast<float*>(a.ws_ml + (size_t)slots_of(c.B, c.KVH, p->n_ctas) * a.G);
  a.status = p->status;
  a.scale = p->scale;
  a.cluster = ctas_per_segment(c.B, c.KVH, a.G, p->idx ? p->idx_cap : c.rows, p->n_ctas);  // a tail is taken to be short
  a.pair = a.v == a.k + kHeadDim;  // V rows right behind their K rows: one copy brings both
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // rows that follow one another come as boxes of a tensor map (where the layout can be described as one)
  CUtensorMap tm_k = {}, tm_v = {};
  const bool tma = !p->idx && !p->tail_len &&
                   make_kv8_tensor_map(&tm_k, c.k, c.rows, c.KVH, c.B, c.stride_row, c.stride_h, c.stride_b, TILE) &&
                   make_kv8_tensor_map(&tm_v, c.v, c.rows, c.KVH, c.B, c.stride_row, c.stride_h, c.stride_b, TILE);
  const bool i8 = c.format == kInt8;
  if (p->dtype == OMNIKV_BF16)
    return i8 ? launch_any<__nv_bfloat16, kInt8>(a, p->n_ctas, tma, tm_k, tm_v, st) : launch_any<__nv_bfloat16, kE4m3>(a, p->n_ctas, tma, tm_k, tm_v, st);
  return i8 ? launch_any<__half, kInt8>(a, p->n_ctas, tma, tm_k, tm_v, st) : launch_any<__half, kE4m3>(a, p->n_ctas, tma, tm_k, tm_v, st);
}
