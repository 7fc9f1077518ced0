// Matrix products in 8-bit integers, one scale per token and per output channel, and the row quantiser in front.
//
//     out[t][c] = (sum_k x[t][k] w[c][k]) * x_scale[t] * w_scale[c] (+ residual[t][c])
//
// The sum is an integer (|sum| <= 128 * 128 * 32768 = 2^29), so it is exact and independent of the order in which slices
// of K are added.  Four kernels: for few tokens a stream of the weights on mma.sync, which starts and ends soonest; for more
// tcgen05 (kind::i8) with the channels on the M side, which leaves the N side to a token count of any size: tiles on single
// SMs that stream a large matrix, tiles shared by a cluster of SMs where there are few of them, tiles on SM pairs for many
// tokens.  linear_plan below chooses by estimates of their times.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "kv8.cuh"
#include "tc05.cuh"
#include "tile_work.cuh"

namespace omnikv {
namespace {

// ---- rows to codes ------------------------------------------------------------------------------------------------
// One CTA per row; the row stays in registers between the maximum and the codes, so it is read once and with one round
// of loads in flight (a single token's row is a latency chain: load, maximum, store).
// VEC: 16-byte pieces per thread at most.
template <typename T, int THREADS, int VEC>
__global__ void __launch_bounds__(THREADS, THREADS > 512 ? 1 : 1024 / THREADS) quant_rows_kernel(const T* x, int64_t x_sr, int K, int8_t* codes, int64_t c_sr,
                                                             float* scale) {
  __shared__ unsigned top[THREADS / 32];
  __shared__ float2 shared;
  pdl_wait();
  pdl_trigger();  // the product behind it may set itself up; it waits for this grid before it reads anything
  const int row = blockIdx.x, tid = threadIdx.x, nvec = K / 8;
  const uint4* src = reinterpret_cast<const uint4*>(x + (size_t)row * x_sr);
  uint4 v[VEC];
#pragma unroll
  for (int u = 0; u < VEC; ++u) {
    v[u] = make_uint4(0, 0, 0, 0);
    if (tid + u * THREADS < nvec) v[u] = src[tid + u * THREADS];
  }
  unsigned m2 = 0;
#pragma unroll
  for (int u = 0; u < VEC; ++u) m2 = max_abs2<T>(m2, v[u]);
  unsigned m = abs_bits_of<T>(m2);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) top[tid >> 5] = m;
  __syncthreads();
  if (tid == 0) {  // the divisions of a rule once per row
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) m = max(m, top[i]);
    const CodeRule rule = code_rule<kInt8>(m);
    shared = shared_rule<kInt8>(rule, m);
    scale[row] = rule.scale;
  }
  __syncthreads();
  const float2 rule = shared;
  uint2* dst = reinterpret_cast<uint2*>(codes + (size_t)row * c_sr);
#pragma unroll
  for (int u = 0; u < VEC; ++u) {
    if (tid + u * THREADS >= nvec) continue;
    dst[tid + u * THREADS] = code8<T, kInt8>(rule, v[u]);
  }
}

// The integer sum with its two scales.  A token of very large values may take sum * x_scale out of fp32's range where the
// result is in it: then the weight's scale, which is of ordinary size, comes first.
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale) {
  const float t = (float)sum * x_scale;
  return fabsf(t) < INFINITY ? t * w_scale : (float)sum * w_scale * x_scale;
}
constexpr float kFarScale = 3.1691265005705735e29f;  // 2^98: below it a sum (at most 2^29) stays in range

struct LinArgs {
  const int8_t* x;
  int64_t x_sr;
  const float* x_scale;
  const int8_t* w;
  int64_t w_sr;
  const float* w_scale;
  const void* res;
  int64_t res_sr;
  void* out;
  int64_t out_sr;
  int n, N, K;
  int* counters;  // tile kernel: [CTAs] arrivals at the tile that a CTA is the first to work on, zero between launches
  int* part;      // tile kernel: [CTAs + tiles][tokens of a tile][128]
  int* status;
  int token_tiles, chunks;  // tiles along the tokens, 128-byte steps of K
  int cluster;              // cluster kernel: CTAs per tile
  int shared, sharers;  // tile kernel: how many tiles, the last ones, are cut into how many pieces (each of a chunk or more)
};

// ---- few tokens: a stream of the weights -------------------------------------------------------------------------------
// A CTA owns 16 channels, its eight warps take 64-byte chunks of K in turn.  The fragments of m16n8k32 come straight from
// global memory with 16-byte loads: inside a chunk of 64 the order of k is free as long as both operands agree, so thread
// (g, t) takes bytes 16 t .. 16 t + 15 of rows g and g + 8 (weights) and of token g, and their words 0..3 are two MMAs.
// DEPTH chunks are asked for while the DEPTH before them are multiplied.  The eight integer sums meet in shared memory.
// More tokens than a CTA takes go to other CTAs, which find the weights in L2.
constexpr int SK_THREADS = 256, SK_WARPS = SK_THREADS / 32, SK_ROWS = 16;

__device__ __forceinline__ void mma_i8(int (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_stream(const int8_t* p) {  // weights: read once
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// NB: blocks of eight tokens of a CTA (four of them spill six registers of 128)
template <typename T, int NB>
__global__ void __launch_bounds__(SK_THREADS, NB == 1 ? 3 : 2) linear_stream_kernel(const LinArgs a) {
  constexpr int SK_DEPTH = NB == 2 ? 3 : 2;
  __shared__ int sums[SK_WARPS][NB * 8][SK_ROWS + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int c0 = blockIdx.x * SK_ROWS, t0 = blockIdx.y * (NB * 8);
  // While the kernel before finishes, this CTA's weights start on their way into L2.  Nothing is read: weights that the
  // kernel before wrote would be wrong in registers, in L2 they are not.
  if (tid < SK_ROWS && c0 + tid < a.N)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(a.w + (size_t)(c0 + tid) * a.w_sr), "r"(a.K) : "memory");
  pdl_wait();
  pdl_trigger();
  const int8_t* w0 = a.w + (size_t)min(c0 + g, a.N - 1) * a.w_sr + 16 * t;  // rows past the end: read again, dropped below
  const int8_t* w1 = a.w + (size_t)min(c0 + g + 8, a.N - 1) * a.w_sr + 16 * t;
  const int8_t* xp[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) xp[b] = a.x + (size_t)min(t0 + b * 8 + g, a.n - 1) * a.x_sr + 16 * t;
  const int chunks = (a.K + 63) >> 6;
  int acc[NB][4];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b][0] = acc[b][1] = acc[b][2] = acc[b][3] = 0;
  uint4 wa[2][SK_DEPTH][2], xb[2][SK_DEPTH][NB];
  const auto fetch = [&](int buf, int first) {
#pragma unroll
    for (int u = 0; u < SK_DEPTH; ++u) {
      const int k = (first + u * SK_WARPS) * 64;
      const bool in = k + 16 * t < a.K;
      wa[buf][u][0] = in ? ld_stream(w0 + k) : make_uint4(0, 0, 0, 0);
      wa[buf][u][1] = in ? ld_stream(w1 + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int b = 0; b < NB; ++b) xb[buf][u][b] = in ? *reinterpret_cast<const uint4*>(xp[b] + k) : make_uint4(0, 0, 0, 0);
    }
  };
  const auto multiply = [&](int buf) {
#pragma unroll
    for (int u = 0; u < SK_DEPTH; ++u) {
      const uint4 p = wa[buf][u][0], q = wa[buf][u][1];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        mma_i8(acc[b], p.x, q.x, p.y, q.y, xb[buf][u][b].x, xb[buf][u][b].y);
        mma_i8(acc[b], p.z, q.z, p.w, q.w, xb[buf][u][b].z, xb[buf][u][b].w);
      }
    }
  };
  constexpr int STEP = SK_DEPTH * SK_WARPS;
  fetch(0, warp);
  for (int c = warp; c < chunks; c += 2 * STEP) {
    fetch(1, c + STEP);
    multiply(0);
    if (c + STEP >= chunks) break;
    fetch(0, c + 2 * STEP);
    multiply(1);
  }
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[warp][b * 8 + 2 * t + (e & 1)][g + 8 * (e >> 1)] = acc[b][e];
  __syncthreads();
  const int c = c0 + tid % SK_ROWS;
  if (c >= a.N) return;
  const float w_scale = a.w_scale[c];
#pragma unroll
  for (int at = tid / SK_ROWS; at < NB * 8; at += SK_THREADS / SK_ROWS) {
    const int tok = t0 + at;
    if (tok >= a.n) return;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < SK_WARPS; ++w) sum += sums[w][at][tid % SK_ROWS];
    float y = scaled(sum, a.x_scale[tok], w_scale);
    if (a.res) y += to_float(static_cast<const T*>(a.res)[(size_t)tok * a.res_sr + c]);
    static_cast<T*>(a.out)[(size_t)tok * a.out_sr + c] = from_float<T>(y);
  }
}

// ---- up to 128 tokens of a large matrix: tiles of 128 channels x BN tokens on tcgen05 ----------------------------------------
// Still a stream of the weights.  Of the tiles every CTA has as many whole ones as all can have.  Where it pays (share_tiles
// below) the chunks (128 bytes of K) of those left over form one list that is cut into equal pieces, at most one per CTA,
// which a CTA works on first: the integer sums of a tile that several CTAs share go to the workspace, the one that arrives
// last adds them up, and all that happens under the stream of the whole tiles.
// Warp 4 fetches 128-byte wide boxes of weights and tokens (TMA, 128-byte swizzle), warp 5 issues the MMAs (K = 32 bytes
// each), int32 accumulators in tensor memory, two of them so that the epilogue of a tile runs under the next tile's MMAs.
// Warps 0-3 read a tile back: thread = channel (TMEM lane), columns = tokens, so a warp's store is 32 neighbouring channels
// of a token whatever the alignment of the output.
constexpr int TK_M = 128, TK_KB = 128, TK_THREADS = 192, TK_CTAS = 148;

template <int BN>
struct TkShape {
  static constexpr int STAGE = (TK_M + BN) * TK_KB;
  static constexpr int STAGES = BN >= 128 ? 6 : 8;
  static constexpr int SMEM = STAGES * STAGE + 1024;
};

__device__ __forceinline__ void tc_mma_i8(unsigned d_tmem, uint64_t a_desc, uint64_t b_desc, unsigned idesc, unsigned accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor (kind::i8): s32 accumulator, signed 8-bit A and B, both K-major.
__host__ __device__ constexpr unsigned i8_instr_desc(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(N >> 3) << 17) | ((unsigned)(M >> 4) << 24);
}
// 16 consecutive 32-bit columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld16i(unsigned taddr, int (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void epilogue_bar() { asm volatile("bar.sync 1, 128;\n" ::: "memory"); }
template <int THREADS>
__device__ __forceinline__ bool epilogue_any(bool pred) {  // OR over the epilogue threads
  unsigned r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, 1, %2, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r)
      : "r"((unsigned)pred), "n"(THREADS)
      : "memory");
  return r != 0;
}

// The results of 16 tokens of one channel: 32 neighbouring channels of a token per warp and store.  What the residual needs
// from memory is asked for one step ahead (`ask`), the full and the ragged step have code of their own.
template <typename T>
struct Channel {
  const T* res;  // this channel's first token, or nullptr
  T* out;        // nullptr: a channel past the end
  int64_t res_sr, out_sr;
  int tokens;
  float w_scale;
  T r[16];
  __device__ __forceinline__ void ask(int j0) {
    if (!res || j0 >= tokens) return;
    const T* p = res + (int64_t)j0 * res_sr;
    if (j0 + 16 <= tokens) {
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = p[j * res_sr];
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = p[min(j, tokens - 1 - j0) * res_sr];
    }
  }
  // far: some token's scale is beyond kFarScale (the check per value slows many tokens by 2 %: 4000 x 4096 x 4096 48.5, 49.6 us)
  __device__ __forceinline__ void put(int j0, const int (&v)[16], const float* x_scale, bool far) {
    if (!out) return;
    float y[16];
    if (far) {
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = scaled(v[j], x_scale[j0 + j], w_scale);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = (float)v[j] * x_scale[j0 + j] * w_scale;
    }
    if (res) {
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] += to_float(r[j]);
      ask(j0 + 16);
    }
    T* p = out + (int64_t)j0 * out_sr;
    if (j0 + 16 <= tokens) {
#pragma unroll
      for (int j = 0; j < 16; ++j) p[j * out_sr] = from_float<T>(y[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j0 + j < tokens) p[j * out_sr] = from_float<T>(y[j]);
    }
  }
};

struct TkShared {
  float x_scale[128];
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2], drained;
  unsigned tmem_base;
  int fail, issued, last, far;
};

template <typename T, int BN>
__global__ void __launch_bounds__(TK_THREADS, 1)
linear_tile_kernel(const LinArgs a, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ TkShared sh;
  constexpr int STAGES = TkShape<BN>::STAGES, STAGE = TkShape<BN>::STAGE;
  constexpr unsigned TMEM_COLS = BN < 16 ? 32 : 2 * BN;
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    sh.fail = 0;
    sh.issued = 0;
    sh.far = 0;
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.acc_full[i], 1);
      mbar_init(&sh.acc_empty[i], 128);
    }
    mbar_init(&sh.drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(&sh.tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = sh.tmem_base;
  const int tiles = ceil_div(a.N, TK_M);
  const TileWork work(tiles, a.shared, a.sharers, a.chunks, gridDim.x, blockIdx.x);  // the host keeps shared * chunks below 2^31
  using Unit = TileWork::Unit;
  // While the kernel before finishes, this CTA's first weights start on their way into L2 (16 x 4096 x 28672: 22.8 -> 21.8 us,
  // 64 x 8192 x 20000: 34.5 -> 33.2); with fewer tiles than SMs it loses (16 x 4096 x 10240: 12.3, 13.1).
  if (tid == 128 && tiles >= TK_CTAS) {
    Unit u;
    int n = 0;
    for (bool more = work.first(u); more && n < STAGES; more = work.next(u))
      for (int k = u.k0; k < u.k1 && n < STAGES; ++k, ++n)
        asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n" ::"l"(reinterpret_cast<uint64_t>(&tm_w)),
                     "r"(k * TK_KB), "r"(u.tile * TK_M)
                     : "memory");
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();

  if (warp == 4) {
    if (lane == 0) {
      int it = 0;
      Unit u;
      for (bool more = work.first(u); more && !sh.fail; more = work.next(u)) {
        for (int k = u.k0; k < u.k1; ++k, ++it) {
          const int st = it % STAGES;
          if (!mbar_wait(&sh.empty[st], ((it / STAGES) & 1) ^ 1, &sh.fail)) {
            if (!sh.fail && a.status) atomicExch(a.status, 7);
            sh.fail = 1;
            break;
          }
          unsigned char* dst = ring + (size_t)st * STAGE;
          mbar_expect_tx(&sh.full[st], STAGE);
          tma_load_2d(dst, &tm_w, k * TK_KB, u.tile * TK_M, &sh.full[st]);
          tma_load_2d(dst + TK_M * TK_KB, &tm_x, k * TK_KB, 0, &sh.full[st]);
          sh.issued = it + 1;
        }
      }
    }
  } else if (warp == 5) {
    if (lane == 0) {
      constexpr unsigned idesc = i8_instr_desc(TK_M, BN);
      bool ok = true;
      int it = 0, n = 0;
      Unit u;
      for (bool more = work.first(u); ok && more; more = work.next(u), ++n) {
        const int buf = n & 1;
        if (!mbar_wait(&sh.acc_empty[buf], ((n >> 1) & 1) ^ 1, &sh.fail)) { ok = false; break; }
        tc_fence_after();
        const unsigned d_tmem = tmem + (unsigned)buf * BN;
        for (int k = u.k0; k < u.k1; ++k, ++it) {
          const int st = it % STAGES;
          if (!mbar_wait(&sh.full[st], (it / STAGES) & 1, &sh.fail)) { ok = false; break; }
          tc_fence_after();
          const unsigned w_base = smem_u32(ring + (size_t)st * STAGE), x_base = w_base + TK_M * TK_KB;
#pragma unroll
          for (int j = 0; j < TK_KB / 32; ++j)
            tc_mma_i8(d_tmem, smem_desc_sw128(w_base + j * 32), smem_desc_sw128(x_base + j * 32), idesc, (k > u.k0 || j) ? 1u : 0u);
          tc_commit(&sh.empty[st]);
        }
        if (ok) tc_commit(&sh.acc_full[buf]);
      }
      if (!ok) {
        if (!sh.fail && a.status) atomicExch(a.status, 7);
        sh.fail = 1;
      }
    }
  } else {
    const int tokens = a.n;
    for (int j = tid; j < tokens; j += 128) {
      const float x = a.x_scale[j];
      sh.x_scale[j] = x;
      if (!(x < kFarScale)) sh.far = 1;
    }
    int n = 0;
    Unit u;
    const auto arrive = [&](const TileWork::Party& p) {  // by one thread; true: the last of them
      __threadfence();  // the stores, ordered before the barrier, are visible before the arrival is
      const bool last = atomicAdd(a.counters + p.first, 1) == p.parts - 1;
      if (last) a.counters[p.first] = 0;  // nobody else touches it any more in this call
      __threadfence();
      return last;
    };
    for (bool more = work.first(u); more; more = work.next(u), ++n) {
      const int buf = n & 1, tile = u.tile, c = tile * TK_M + tid;
      const bool whole = work.whole(u);
      const bool in = c < a.N;
      Channel<T> ch{in && a.res ? static_cast<const T*>(a.res) + c : nullptr, in ? static_cast<T*>(a.out) + c : nullptr,
                    a.res_sr, a.out_sr, tokens, in ? a.w_scale[c] : 0.f};
      if (whole) ch.ask(0);
      const bool got = mbar_wait(&sh.acc_full[buf], (n >> 1) & 1, &sh.fail);
      if (epilogue_any<128>(!got)) {  // the 128 threads leave together
        if (!sh.fail && a.status) atomicExch(a.status, 7);
        sh.fail = 1;
        if (tid == 0) work.give_up(u, arrive);  // the counters end at zero whoever failed: the workspace is used again
        break;
      }
      tc_fence_after();
      const unsigned src = tmem + ((unsigned)(warp * 32) << 16) + (unsigned)buf * BN;
      int* part = a.part + (size_t)(work.cta + tile - work.whole_tiles) * BN * TK_M + tid;  // (CTA, tile) pairs walk a staircase: their sum is unique
#pragma unroll 1
      for (int j0 = 0; j0 < tokens; j0 += 16) {
        int v[16];
        tmem_ld16i(src + j0, v);
        tmem_ld_wait();
        if (whole) {
          ch.put(j0, v, sh.x_scale, sh.far);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) __stcg(part + (j0 + j) * TK_M, v[j]);
        }
      }
      tc_fence_before();
      mbar_arrive(&sh.acc_empty[buf]);
      if (!whole) {
        const TileWork::Party p = work.party(tile);
        const int parts = p.parts;
        epilogue_bar();
        if (tid == 0) sh.last = arrive(p);
        epilogue_bar();
        if (sh.last) {
          const int* all = a.part + (size_t)(p.first + tile - work.whole_tiles) * BN * TK_M + tid;
          const auto fetch = [&](int q, int j0, int (&v)[16]) {  // 16 tokens of partial q (the columns behind the tokens are there too)
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = q < parts && j0 < tokens ? __ldcg(all + ((size_t)q * BN + j0 + j) * TK_M) : 0;
          };
          int v0[16], v1[16], n0[16], n1[16];  // the first two partials are asked for one step ahead
          ch.ask(0);
          fetch(0, 0, v0);
          fetch(1, 0, v1);
#pragma unroll 1
          for (int j0 = 0; j0 < tokens; j0 += 16) {
            fetch(0, j0 + 16, n0);
            fetch(1, j0 + 16, n1);
#pragma unroll
            for (int j = 0; j < 16; ++j) v0[j] += v1[j];
#pragma unroll 1
            for (int q = 2; q < parts; ++q) {
              fetch(q, j0, v1);
#pragma unroll
              for (int j = 0; j < 16; ++j) v0[j] += v1[j];
            }
            ch.put(j0, v0, sh.x_scale, sh.far);
#pragma unroll
            for (int j = 0; j < 16; ++j) v0[j] = n0[j], v1[j] = n1[j];
          }
        }
        epilogue_bar();  // sh.last is used again
      }
    }
  }

  // ---- teardown ----
  tc_fence_before();
  __syncthreads();
  if (sh.fail) {  // wait (bounded) for what is in flight before the memories are given up:
    if (tid == 160) {  // the MMAs, by the thread that issued them,
      tc_commit(&sh.drained);
      mbar_wait(&sh.drained, 0);
    }
    if (tid == 128) {  // and the last requested tile of every stage
      for (int st = 0; st < STAGES; ++st) {
        const int last = sh.issued - 1 - ((sh.issued - 1 - st) % STAGES + STAGES) % STAGES;
        if (sh.issued > st && last >= 0) mbar_wait(&sh.full[st], (last / STAGES) & 1);
      }
    }
    __syncthreads();
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// ---- many tokens: 256 channels x up to 256 tokens on a pair of SMs --------------------------------------------------------
// The same kernel on cta_group::2.  A tile of 128 x 256 on one SM asks for 48 KB of operands per 128 bytes of K, more than
// L2 delivers at the tensor cores' pace; a pair shares the operands of a 256 x 256 tile (each CTA loads half of the
// channels and half of the tokens) and asks for 32 KB per SM.  CTA 0 of the pair issues the MMAs; its barriers count both
// CTAs' bytes, and a commit reports to both.  The token count BN of a tile is a run-time choice (a multiple of 32), made so
// that the last round of tiles is nearly full.  Eight epilogue warps: two per quarter of the TMEM lanes, half of the tokens each.
constexpr int PK_THREADS = 320, PK_STAGES = 6, PK_HALF = 128 * TK_KB, PK_STAGE = 2 * PK_HALF, PK_SMEM = PK_STAGES * PK_STAGE + 1024;

__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, int col, int row, unsigned bar_cluster) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];\n" ::
          "r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(row), "r"(bar_cluster)
      : "memory");
}
__device__ __forceinline__ void pair_mma_i8(unsigned d_tmem, uint64_t a_desc, uint64_t b_desc, unsigned idesc, unsigned accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pair_commit(uint64_t* bar) {  // arrives at this offset in both CTAs
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(smem_u32(bar)),
               "h"((unsigned short)3)
               : "memory");
}
__device__ __forceinline__ void pair_commit_here(uint64_t* bar) {  // ... in this CTA only
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void st_cluster(unsigned addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;\n" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ int ld_cluster(unsigned addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void remote_arrive(unsigned bar_cluster) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar_cluster) : "memory");
}

struct PkShared {
  float x_scale[256];
  uint64_t full[PK_STAGES], empty[PK_STAGES], acc_full[2], acc_empty[2], drained;
  unsigned tmem_base;
  int fail, issued, far;
};

template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PK_THREADS, 1)
linear_pair_kernel(const LinArgs a, const int BN, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ PkShared sh;
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int units = ceil_div(a.N, 2 * TK_M) * a.token_tiles;

  if (tid == 0) {
    sh.fail = 0;
    sh.issued = 0;
    sh.far = 0;
    for (int i = 0; i < PK_STAGES; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.acc_full[i], 1);
      mbar_init(&sh.acc_empty[i], 16);  // the epilogue warps of both CTAs
    }
    mbar_init(&sh.drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&sh.tmem_base)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the barriers of both CTAs are there before either is signalled from the other side
  tc_fence_after();
  const unsigned tmem = sh.tmem_base;
  pdl_wait();
  pdl_trigger();
  const auto give_up = [&]() {  // a wait ran out: both CTAs of the pair stop
    if (!sh.fail && a.status) atomicExch(a.status, 7);
    sh.fail = 1;
    st_cluster(in_cta(smem_u32(&sh.fail), rank ^ 1), 1);
  };

  if (warp == 8) {
    if (lane == 0) {
      int it = 0;
      for (int u = pair; u < units && !sh.fail; u += pairs) {
        const int tt = u % a.token_tiles, ct = u / a.token_tiles;
        for (int k = 0; k < a.chunks; ++k, ++it) {
          const int st = it % PK_STAGES;
          if (!mbar_wait(&sh.empty[st], ((it / PK_STAGES) & 1) ^ 1, &sh.fail)) {
            give_up();
            break;
          }
          unsigned char* dst = ring + (size_t)st * PK_STAGE;
          const unsigned bar = in_cta(smem_u32(&sh.full[st]), 0);
          if (rank == 0) mbar_expect_tx(&sh.full[st], 2 * (TK_M + BN / 2) * TK_KB);
          pair_load(dst, &tm_w, k * TK_KB, (2 * ct + rank) * TK_M, bar);
          pair_load(dst + PK_HALF, &tm_x, k * TK_KB, tt * BN + rank * (BN / 2), bar);
          sh.issued = it + 1;
        }
      }
    }
  } else if (warp == 9) {
    if (lane == 0 && rank == 0) {
      const unsigned idesc = i8_instr_desc(2 * TK_M, BN);
      bool ok = true;
      int it = 0, n = 0;
      for (int u = pair; ok && u < units; u += pairs, ++n) {
        const int buf = n & 1;
        if (!mbar_wait(&sh.acc_empty[buf], ((n >> 1) & 1) ^ 1, &sh.fail)) { ok = false; break; }
        tc_fence_after();
        const unsigned d_tmem = tmem + (unsigned)buf * 256;
        for (int k = 0; k < a.chunks; ++k, ++it) {
          const int st = it % PK_STAGES;
          if (!mbar_wait(&sh.full[st], (it / PK_STAGES) & 1, &sh.fail)) { ok = false; break; }
          tc_fence_after();
          const unsigned w_base = smem_u32(ring + (size_t)st * PK_STAGE), x_base = w_base + PK_HALF;
#pragma unroll
          for (int j = 0; j < TK_KB / 32; ++j)
            pair_mma_i8(d_tmem, smem_desc_sw128(w_base + j * 32), smem_desc_sw128(x_base + j * 32), idesc, (k || j) ? 1u : 0u);
          pair_commit(&sh.empty[st]);
        }
        if (ok) pair_commit(&sh.acc_full[buf]);
      }
      if (!ok) give_up();
    }
  } else {
    const int quarter = warp & 3, half = warp >> 2;
    int n = 0;
    for (int u = pair; u < units; u += pairs, ++n) {
      const int buf = n & 1, t0 = (u % a.token_tiles) * BN, c = (2 * (u / a.token_tiles) + rank) * TK_M + quarter * 32 + lane;
      const int tokens = min(BN, a.n - t0), j_lo = half * (BN / 2), j_hi = min(tokens, j_lo + BN / 2);
      for (int j = tid; j < tokens; j += 256) {  // the unit before ended with a barrier
        const float x = a.x_scale[t0 + j];
        sh.x_scale[j] = x;
        if (!(x < kFarScale)) sh.far = 1;
      }
      const bool in = c < a.N;
      Channel<T> ch{in && a.res ? static_cast<const T*>(a.res) + (int64_t)t0 * a.res_sr + c : nullptr,
                    in ? static_cast<T*>(a.out) + (int64_t)t0 * a.out_sr + c : nullptr, a.res_sr, a.out_sr, j_hi, in ? a.w_scale[c] : 0.f};
      ch.ask(j_lo);
      const bool got = mbar_wait(&sh.acc_full[buf], (n >> 1) & 1, &sh.fail);
      if (epilogue_any<256>(!got)) {  // the 256 threads leave together
        give_up();
        break;
      }
      tc_fence_after();
      const unsigned src = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)buf * 256;
#pragma unroll 1
      for (int j0 = j_lo; j0 < j_hi; j0 += 16) {
        int v[16];
        tmem_ld16i(src + j0, v);
        tmem_ld_wait();
        ch.put(j0, v, sh.x_scale, sh.far);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) remote_arrive(in_cta(smem_u32(&sh.acc_empty[buf]), 0));
      asm volatile("bar.sync 1, 256;\n" ::: "memory");  // sh.x_scale is used again
    }
  }

  // ---- teardown: neither CTA leaves while the other may still signal it ----
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (sh.fail) {  // in both CTAs; wait (bounded) for what is in flight before the memories are given up:
    if (tid == 288 && rank == 0) {  // the MMAs, by the thread that issued them,
      pair_commit_here(&sh.drained);
      mbar_wait(&sh.drained, 0);
    }
    if (tid == 256 && rank == 0) {  // and the last tile of every stage that either CTA has requested its half of
      const int issued = max(sh.issued, ld_cluster(in_cta(smem_u32(&sh.issued), 1)));
      for (int st = 0; st < PK_STAGES; ++st) {
        const int last = issued - 1 - ((issued - 1 - st) % PK_STAGES + PK_STAGES) % PK_STAGES;
        if (issued > st && last >= 0) mbar_wait(&sh.full[st], (last / PK_STAGES) & 1);
      }
    }
    __syncwarp();
    cluster_sync_all();
  }
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
  }
}

// ---- few tiles: a cluster of CTAs per tile ------------------------------------------------------------------------------
// K is cut into as many pieces as the cluster has CTAs.  Behind its MMAs a CTA sends each token's integer sums to the CTA
// that finishes that token (token j: CTA j mod cluster), straight into its shared memory; one cluster barrier later every
// CTA adds up what it was sent.  No workspace, no fences over global memory: partial sums by way of L2 and an arrival counter
// took twice as long (64 x 8192 x 1024: 14.6 us, now 7.1; 128 x 4096 x 4096: 14.8, now 9.5; 256 x 8192 x 1024: 22.6, now 9.4).
// Warps 0-7 read the sums out (two warps per quarter of the TMEM lanes, alternate groups of 16 tokens), 8 fetches, 9 issues.
template <int BN>
struct CkShape {
  static constexpr int STAGE = (TK_M + BN) * TK_KB;
  static constexpr int STAGES = BN >= 128 ? 4 : BN >= 64 ? 6 : 8;
  static constexpr int SUMS = (BN + 8) * TK_M * 4;  // a column more per CTA where the cluster does not divide the columns
  static constexpr int SMEM = STAGES * STAGE + SUMS + 1024;
};
struct CkShared {
  float x_scale[128];
  uint64_t full[8], empty[8], done, drained;
  unsigned tmem_base;
  int fail, issued;
};

constexpr int CK_THREADS = 320;
template <typename T, int BN>
__global__ void __launch_bounds__(CK_THREADS, 1)
linear_cluster_kernel(const LinArgs a, const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ CkShared sh;
  constexpr int STAGES = CkShape<BN>::STAGES, STAGE = CkShape<BN>::STAGE;
  constexpr unsigned TMEM_COLS = BN < 32 ? 32 : BN;
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  int* sums = reinterpret_cast<int*>(ring + STAGES * STAGE);  // [source CTA][this CTA's columns][128]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cs = a.cluster, rank = (int)cluster_rank(), unit = blockIdx.x / cs;
  const int tile = unit / a.token_tiles, t0 = (unit % a.token_tiles) * BN;
  const int k0 = rank * a.chunks / cs, k1 = (rank + 1) * a.chunks / cs;
  const int tokens = min(BN, a.n - t0), cols = (tokens + cs - 1) / cs;

  if (tid == 0) {
    sh.fail = 0;
    sh.issued = 0;
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    mbar_init(&sh.done, 1);
    mbar_init(&sh.drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(&sh.tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = sh.tmem_base;
  cluster_arrive();  // this CTA runs: its shared memory may be written
  pdl_wait();
  pdl_trigger();

  if (warp == 8) {
    if (lane == 0) {
      for (int k = k0, it = 0; k < k1; ++k, ++it) {
        const int st = it % STAGES;
        if (!mbar_wait(&sh.empty[st], ((it / STAGES) & 1) ^ 1, &sh.fail)) {
          if (!sh.fail && a.status) atomicExch(a.status, 7);
          sh.fail = 1;
          break;
        }
        unsigned char* dst = ring + (size_t)st * STAGE;
        mbar_expect_tx(&sh.full[st], STAGE);
        tma_load_2d(dst, &tm_w, k * TK_KB, tile * TK_M, &sh.full[st]);
        tma_load_2d(dst + TK_M * TK_KB, &tm_x, k * TK_KB, t0, &sh.full[st]);
        sh.issued = it + 1;
      }
    }
  } else if (warp == 9) {
    if (lane == 0) {
      constexpr unsigned idesc = i8_instr_desc(TK_M, BN);
      bool ok = true;
      for (int k = k0, it = 0; k < k1; ++k, ++it) {
        const int st = it % STAGES;
        if (!mbar_wait(&sh.full[st], (it / STAGES) & 1, &sh.fail)) { ok = false; break; }
        tc_fence_after();
        const unsigned w_base = smem_u32(ring + (size_t)st * STAGE), x_base = w_base + TK_M * TK_KB;
#pragma unroll
        for (int j = 0; j < TK_KB / 32; ++j)
          tc_mma_i8(tmem, smem_desc_sw128(w_base + j * 32), smem_desc_sw128(x_base + j * 32), idesc, (it || j) ? 1u : 0u);
        tc_commit(&sh.empty[st]);
      }
      if (ok) tc_commit(&sh.done);
      else {
        if (!sh.fail && a.status) atomicExch(a.status, 7);
        sh.fail = 1;
      }
    }
  }
  const int channel = (warp & 3) * 32 + lane, half = (warp >> 2) & 1, c = tile * TK_M + channel;
  float w_scale = 0.f;
  if (warp < 8) {
    if (tid < tokens) sh.x_scale[tid] = a.x_scale[t0 + tid];
    if (c < a.N) w_scale = a.w_scale[c];
  }
  __syncwarp();
  cluster_wait();
  if (warp < 8) {
    const bool got = mbar_wait(&sh.done, 0, &sh.fail);
    if (epilogue_any<256>(!got)) {
      if (!sh.fail && a.status) atomicExch(a.status, 7);
      sh.fail = 1;
    } else {
      tc_fence_after();
      const unsigned mine = smem_u32(sums + (size_t)rank * cols * TK_M + channel);
      int to = (half * 16) % cs, at = (half * 16) / cs;  // token j goes to CTA j % cs as its column j / cs
#pragma unroll 1
      for (int j0 = half * 16; j0 < tokens; j0 += 32) {
        int v[16];
        tmem_ld16i(tmem + ((unsigned)((warp & 3) * 32) << 16) + j0, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (j0 + j < tokens) st_cluster(in_cta(mine + (unsigned)at * (TK_M * 4), to), v[j]);
          if (++to == cs) to = 0, ++at;
        }
        to += 16 % cs, at += 16 / cs;
        if (to >= cs) to -= cs, ++at;
      }
      tc_fence_before();
    }
  }
  __syncwarp();
  cluster_sync_all();  // the sums of every CTA are where they are added up
  if (warp < 8 && c < a.N) {
    const T* res = static_cast<const T*>(a.res) + (int64_t)t0 * a.res_sr + c;
    T* out = static_cast<T*>(a.out) + (int64_t)t0 * a.out_sr + c;
    constexpr int U = 8;
#pragma unroll 1
    for (int i0 = half * U; rank + i0 * cs < tokens; i0 += 2 * U) {
      int sum[U];
      T r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        sum[u] = 0;
        if (a.res) r[u] = res[(int64_t)min(rank + (i0 + u) * cs, tokens - 1) * a.res_sr];
      }
      const int* from = sums + (size_t)i0 * TK_M + channel;
#pragma unroll 2
      for (int q = 0; q < cs; ++q, from += (size_t)cols * TK_M)
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i0 + u < cols) sum[u] += from[u * TK_M];
      float y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = min(rank + (i0 + u) * cs, tokens - 1);
        y[u] = scaled(sum[u], sh.x_scale[j], w_scale);
        if (a.res) y[u] += to_float(r[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = rank + (i0 + u) * cs;
        if (j < tokens) out[(int64_t)j * a.out_sr] = from_float<T>(y[u]);
      }
    }
  }
  __syncthreads();
  if (sh.fail) {  // wait (bounded) for the MMAs and copies in flight
    if (tid == 288) {
      tc_commit(&sh.drained);
      mbar_wait(&sh.drained, 0);
    }
    if (tid == 256)
      for (int st = 0; st < STAGES; ++st) {
        const int last = sh.issued - 1 - ((sh.issued - 1 - st) % STAGES + STAGES) % STAGES;
        if (sh.issued > st && last >= 0) mbar_wait(&sh.full[st], (last / STAGES) & 1);
      }
    __syncthreads();
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// ---- which kernel -----------------------------------------------------------------------------------------------------------
// The one whose estimated time is least.  The estimates are linear fits (in ns) to times measured with weights that are not
// in L2, 1 to 512 tokens, 300 to 28672 channels, K = 512 to 14336, right to 4-6 % on average.  Both sides at some borders, us:
//   stream against a cluster   16 x 4096 x 4096: 5.5, 7.1   64 x 4096 x 2048: 7.2, 6.7   1 x 14336 x 4096: 15.4, 13.1
//   cluster against tiles      64 x 4096 x 6144: 10.1, 13.0   64 x 1024 x 8192: 6.7, 6.1
//   stream against tiles       16 x 4096 x 14336: 17.3, 13.3   1 x 1024 x 8192: 3.6, 5.6
//   cluster against pairs      256 x 8192 x 1024: 9.4, 22.6   512 x 1024 x 2048: 7.9, 6.4
enum LinearKind { kStreamKernel, kTileKernel, kClusterKernel, kPairKernel };
struct LinearPlan {
  LinearKind kind;
  int tokens, token_tiles;  // of a CTA (stream) or a tile, and how many of them
  int tiles, ctas, chunks;  // tiles of both directions; CTAs; 128-byte steps of K
  int cluster;              // CTAs per tile
  int shared, sharers;      // tile kernel: see LinArgs
};
// Tile kernel: into how many pieces the tiles left over behind whole rounds are cut (0: none, they are a round of their own),
// and what that saves (ns).  m pieces per tile save 1 - 1/m of a round and cost m partials' stores and additions; pieces
// that end inside tiles, where there are too many tiles for two each, cost more.  Measured, us without and with: 16 x 4096 x
// 19000 (149 tiles) 23.5, 16.8; 16 x 4096 x 28672 (224) 24.8, 22.8; 128 x 4096 x 28672 27.8, 34.4 (hence whole).
struct Sharing {
  int pieces;
  double saves;
};
inline Sharing share_tiles(int n, long long tiles, long long chunks) {
  const int left = (int)(tiles % TK_CTAS);
  Sharing best = {0, 0.0};
  if (tiles <= TK_CTAS || !left) return best;
  for (int m = 2; m <= 6 && m * left <= TK_CTAS && m <= chunks; ++m) {
    const double saves = 420.0 * chunks * (m - 1) / m - m * (450 + 18 * n);
    if (saves > best.saves) best = Sharing{m * left, saves};
  }
  const double saves = 420.0 * chunks * (TK_CTAS - left) / TK_CTAS - 4000 - 70 * n;
  if (2 * left > TK_CTAS && saves > best.saves) best = Sharing{TK_CTAS, saves};
  return best;
}
inline LinearPlan linear_plan(int n, int N, int K) {
  const long long chunks = ceil_div(K, TK_KB), channel_tiles = ceil_div(N, TK_M);
  const double mega = ((double)N + n) * K * 1e-6;  // operand bytes
  LinearPlan p = {};
  double best = 1e300;
  const auto offer = [&](double ns, LinearKind kind, int tokens, int cluster) {
    if (ns >= best) return;
    best = ns;
    p.kind = kind;
    p.tokens = tokens;
    p.cluster = cluster;
  };
  // Stream, 8, 16 or 32 tokens per CTA: start, the bytes that an SM with the most CTAs fetches, CTAs, bytes of weights.
  static constexpr double kStream[3][4] = {{1450, 12.6, 272, 53}, {1430, 10.4, 584, 42}, {1880, 11.1, 738, 13}};
  for (int i = 0; i < 3 && n <= 128; ++i) {
    const int tokens = 8 << i;
    if (i && n <= tokens / 2) break;
    const double ctas = (double)ceil_div(N, SK_ROWS) * ceil_div(n, tokens);
    offer(kStream[i][0] + kStream[i][1] * std::ceil(ctas / TK_CTAS) * K * 1e-3 * (SK_ROWS + tokens) + kStream[i][2] * ctas / TK_CTAS +
              kStream[i][3] * N * 1e-6 * K, kStreamKernel, tokens, 1);
  }
  // Tiles: start, tokens read out, rounds (by a CTA's operands from L2, or by all weights from HBM).
  if (n <= 128) {
    const int BN = n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : 128;
    const double whole = channel_tiles / TK_CTAS, rest = channel_tiles % TK_CTAS ? 1 : 0;
    offer(3400 + 11.3 * n + chunks * (whole * std::max(1.25 * (TK_M + BN), 370.0) + rest * std::max(1.25 * (TK_M + BN), 270.0)) -
              share_tiles(n, channel_tiles, chunks).saves, kTileKernel, BN, 1);
  }
  // Clusters, as many as can run at once: start, tokens read out and added up, the operands of a CTA, of all, the sums sent.
  static constexpr int kCluster[5][2] = {{2, 74}, {3, 45}, {4, 33}, {6, 22}, {8, 15}};  // CTAs, clusters
  for (int BN = 16; BN <= 128 && (BN == 16 || n > BN / 2); BN *= 2) {
    const long long units = channel_tiles * ceil_div(n, BN);
    for (const auto& c : kCluster) {
      if (units > c[1] || c[0] > chunks) break;
      const int tokens = min(n, BN);
      offer(3180 + 8.6 * tokens + 16.9 * tokens / c[0] + 1.255 * ((chunks + c[0] - 1) / c[0]) * (TK_M + BN) + 82.6 * mega +
                0.0586 * units * c[0] * tokens, kClusterKernel, BN, c[0]);
    }
  }
  // Pairs: the token count whose rounds of tiles over the SM pairs take least.  A round goes by the operands' way from L2
  // rather than by its MMAs: measured 10.3, 11.3, 13.0 us for 128, 192, 256 tokens at K = 4096.
  for (int BN = 256; BN >= 32 && n > 16; BN -= 32) {
    const double units = std::ceil(channel_tiles / 2.0) * ceil_div(n, BN);
    const double round = chunks * (BN >= 128 ? 0.586 * BN + 211 : 0.16 * BN + 266);
    offer(3380 + std::max(std::ceil(units / (TK_CTAS / 2)) * round, 170 * mega) + 5.6 * BN + 22 * mega, kPairKernel, BN, 2);
  }
  p.chunks = (int)chunks;
  p.token_tiles = ceil_div(n, p.tokens);
  const long long tiles = p.kind == kPairKernel ? (channel_tiles + 1) / 2 * p.token_tiles : channel_tiles * p.token_tiles;
  p.tiles = (int)std::min<long long>(tiles, 0x7fffffff);
  switch (p.kind) {
    case kStreamKernel: break;  // a grid of its own
    case kClusterKernel: p.ctas = p.tiles * p.cluster; break;
    case kPairKernel: p.ctas = 2 * min(TK_CTAS / 2, p.tiles); break;
    case kTileKernel:
      p.ctas = min(TK_CTAS, p.tiles);
      p.sharers = share_tiles(n, p.tiles, chunks).pieces;
      if (p.sharers) p.shared = p.tiles % TK_CTAS;
  }
  return p;
}
constexpr int kMostRows = 0x7fffffff - 256;  // tokens or channels: rounded up to a tile they still fit 32 bits
inline size_t linear_workspace(const LinearPlan& p) {
  return p.shared ? 1024 + (size_t)(p.sharers + p.shared) * p.tokens * TK_M * sizeof(int) : 0;
}

inline bool bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15); }

template <typename T, int BN>
int launch_tile(const LinArgs& a, const LinearPlan& pl, const CUtensorMap& tm_w, const CUtensorMap& tm_x, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  auto kern = linear_tile_kernel<T, BN>;
  if (const int rc = allow_smem(kern, TkShape<BN>::SMEM, done)) return rc;
  OMNIKV_CUDA_OK(launch_pdl_smem_args(kern, dim3(pl.ctas), dim3(TK_THREADS), TkShape<BN>::SMEM, st, a, tm_w, tm_x));
  return OMNIKV_OK;
}

template <typename T, int BN>
int launch_cluster(const LinArgs& a, const LinearPlan& pl, const CUtensorMap& tm_w, const CUtensorMap& tm_x, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  auto kern = linear_cluster_kernel<T, BN>;
  if (const int rc = allow_smem(kern, CkShape<BN>::SMEM, done)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.ctas);
  cfg.blockDim = dim3(CK_THREADS);
  cfg.dynamicSmemBytes = CkShape<BN>::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = pl.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  OMNIKV_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, a, tm_w, tm_x));
  return OMNIKV_OK;
}

template <typename T, int BN>
int launch_single(const LinArgs& a, const LinearPlan& pl, const CUtensorMap& tm_w, const CUtensorMap& tm_x, cudaStream_t st) {
  return pl.kind == kClusterKernel ? launch_cluster<T, BN>(a, pl, tm_w, tm_x, st) : launch_tile<T, BN>(a, pl, tm_w, tm_x, st);
}

template <typename T>
int launch_pair(const LinArgs& a, const LinearPlan& pl, const CUtensorMap& tm_w, const CUtensorMap& tm_x, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  auto kern = linear_pair_kernel<T>;
  if (const int rc = allow_smem(kern, PK_SMEM, done)) return rc;
  OMNIKV_CUDA_OK(launch_pdl_smem_args(kern, dim3(pl.ctas), dim3(PK_THREADS), PK_SMEM, st, a, pl.tokens, tm_w, tm_x));
  return OMNIKV_OK;
}

template <typename T>
int launch_linear(const LinArgs& a, const LinearPlan& pl, cudaStream_t st) {
  if (pl.kind == kStreamKernel) {
    auto kern = pl.tokens == 8 ? linear_stream_kernel<T, 1> : pl.tokens == 16 ? linear_stream_kernel<T, 2> : linear_stream_kernel<T, 4>;
    OMNIKV_CUDA_OK(launch_pdl(kern, dim3(ceil_div(a.N, SK_ROWS), pl.token_tiles), dim3(SK_THREADS), 0, st, a));
    return OMNIKV_OK;
  }
  CUtensorMap tm_w, tm_x;
  if (!make_bytes_tensor_map(&tm_w, a.w, a.N, a.K, a.w_sr, TK_M) ||
      !make_bytes_tensor_map(&tm_x, a.x, a.n, a.K, a.x_sr, pl.kind == kPairKernel ? pl.tokens / 2 : pl.tokens))
    return OMNIKV_E_UNSUPPORTED;
  if (pl.kind == kPairKernel) return launch_pair<T>(a, pl, tm_w, tm_x, st);
  switch (pl.tokens) {
    case 16: return launch_single<T, 16>(a, pl, tm_w, tm_x, st);
    case 32: return launch_single<T, 32>(a, pl, tm_w, tm_x, st);
    case 64: return launch_single<T, 64>(a, pl, tm_w, tm_x, st);
    default: return launch_single<T, 128>(a, pl, tm_w, tm_x, st);
  }
}

}  // namespace
}  // namespace omnikv

extern "C" int omnikv_quant_rows(int dtype, const void* x, int64_t x_stride_row, int n, int K, int8_t* codes,
                                 int64_t code_stride_row, float* scale, void* stream) {
  using namespace omnikv;
  if (bad16(x) || bad16(codes) || !scale || n <= 0 || K <= 0 || K % 16 || x_stride_row % 8 || code_stride_row % 16 ||
      code_stride_row < K)
    return OMNIKV_E_BADARG;
  if (!is_16bit(dtype) || K > 32768) return OMNIKV_E_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto kern, int threads, auto tag) -> int {
    OMNIKV_CUDA_OK(launch_pdl_args(kern, dim3(n), dim3(threads), st, static_cast<const decltype(tag)*>(x), x_stride_row, K, codes,
                                   code_stride_row, scale));
    return OMNIKV_OK;
  };
  const auto pick = [&](auto tag) -> int {  // few pieces per thread: a row is one round of loads, and several rows share an SM
    using T = decltype(tag);
    if (K <= 256 * 8 * 2) return go(quant_rows_kernel<T, 256, 2>, 256, tag);
    if (K <= 512 * 8 * 2) return go(quant_rows_kernel<T, 512, 2>, 512, tag);
    if (K <= 512 * 8 * 4) return go(quant_rows_kernel<T, 512, 4>, 512, tag);
    return go(quant_rows_kernel<T, 1024, 4>, 1024, tag);
  };
  return dtype == OMNIKV_BF16 ? pick(__nv_bfloat16()) : pick(__half());
}

extern "C" size_t omnikv_linear_w8a8_workspace_bytes(int n_tokens, int channels, int K) {
  using namespace omnikv;
  if (n_tokens <= 0 || channels <= 0 || K <= 0 || n_tokens > kMostRows || channels > kMostRows) return 0;
  return linear_workspace(linear_plan(n_tokens, channels, K));
}

extern "C" int omnikv_linear_w8a8(const omnikv_linear_w8a8_params* p, void* stream) {
  using namespace omnikv;
  if (!p || bad16(p->x) || bad16(p->w) || !p->x_scale || !p->w_scale || !p->out) return OMNIKV_E_BADARG;
  if (p->n_tokens <= 0 || p->channels <= 0 || p->K <= 0 || p->K % 16) return OMNIKV_E_BADARG;
  if (p->x_stride_row % 16 || p->w_stride_row % 16 || p->x_stride_row < p->K || p->w_stride_row < p->K) return OMNIKV_E_BADARG;
  if (p->out_stride_row < p->channels || (p->residual && p->residual_stride_row && p->residual_stride_row < p->channels)) return OMNIKV_E_BADARG;
  if (p->n_tokens > kMostRows || p->channels > kMostRows) return OMNIKV_E_UNSUPPORTED;
  if (p->K > 32768 || (p->out_dtype != OMNIKV_F32 && !is_16bit(p->out_dtype))) return OMNIKV_E_UNSUPPORTED;
  LinArgs a{p->x, p->x_stride_row, p->x_scale, p->w, p->w_stride_row, p->w_scale, p->residual, p->residual_stride_row,
            p->out, p->out_stride_row, p->n_tokens, p->channels, p->K};
  const LinearPlan pl = linear_plan(a.n, a.N, a.K);
  if (pl.tiles == 0x7fffffff) return OMNIKV_E_UNSUPPORTED;  // tiles are counted in 32 bits
  const size_t need = linear_workspace(pl);
  if (need && (!p->workspace || p->workspace_bytes < need)) return OMNIKV_E_WORKSPACE;
  if (need && bad16(p->workspace)) return OMNIKV_E_BADARG;
  a.counters = static_cast<int*>(p->workspace);
  a.part = a.counters + 256;
  a.status = p->status;
  a.token_tiles = pl.token_tiles;
  a.shared = pl.shared;
  a.sharers = pl.sharers;
  a.chunks = pl.chunks;
  a.cluster = pl.cluster;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (p->out_dtype) {
    case OMNIKV_F32: return launch_linear<float>(a, pl, st);
    case OMNIKV_BF16: return launch_linear<__nv_bfloat16>(a, pl, st);
    default: return launch_linear<__half>(a, pl, st);
  }
}
