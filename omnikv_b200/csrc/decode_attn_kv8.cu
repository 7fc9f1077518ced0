// Decode attention over a KV cache held in 8 bits.
//
// Grid (n_splits, KVH, B): a CTA owns a contiguous share of its sequence's row list, writes one un-normalised partial
// (o, m, l) per query head, and the CTA that finishes last for a (sequence, KV head) merges them, so a call is one launch.
#include "kv8.cuh"

namespace omnikv {
namespace {

constexpr int MAX_G = 16;
constexpr int NW = 4, NT = NW * 32;

struct A8Args {
  const unsigned char *k, *v;
  int64_t sb, sh, sr;
  const float *ks, *vs;
  int64_t ssb, ssh;
  int shift, rows;
  const void* q;
  int64_t q_sb, q_sh;
  void* out;
  const int* idx;
  int64_t idx_stride;
  int idx_cap;
  const int *len, *tail_start, *tail_len;
  float* score_out;
  int64_t score_stride;
  const int* score_len;
  float *ws_o, *ws_ml;
  unsigned* ws_cnt;
  int B, H, KVH, G, S;
  float scale;
};

// The rows of a sequence: nA listed ones, then the tail [t0, t0 + nB).
struct RowList {
  int nA, nB, t0;
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

template <typename T, int FMT>
__global__ void __launch_bounds__(NT) decode_attn_kv8_kernel(const A8Args a) {
  __shared__ float o_s[NW][MAX_G][kHeadDim];
  __shared__ float ml_s[NW][MAX_G][2];
  __shared__ int last_flag;
  pdl_wait();
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.G;
  const RowList list = row_list(a, b);
  const int n = list.nA + list.nB;
  const int chunk = ceil_div(n, a.S), r0 = min(n, split * chunk), r1 = min(n, r0 + chunk);
  const unsigned char* k = a.k + (size_t)b * a.sb + (size_t)kvh * a.sh;
  const unsigned char* v = a.v + (size_t)b * a.sb + (size_t)kvh * a.sh;
  const float* ks = a.ks + (size_t)b * a.ssb + (size_t)kvh * a.ssh;
  const float* vs = a.vs + (size_t)b * a.ssb + (size_t)kvh * a.ssh;
  const int score_lim = a.score_out ? min(a.score_len[b], list.nA) : 0;
  float* score_row = a.score_out ? a.score_out + ((size_t)kvh * a.B + b) * a.score_stride : nullptr;
  const T* q = static_cast<const T*>(a.q) + (size_t)b * a.q_sb + (size_t)kvh * G * a.q_sh;
  for (int g = 0; g < G; ++g) {
    float qv[4];
    for (int e = 0; e < 4; ++e) qv[e] = to_float(q[(size_t)g * a.q_sh + lane * 4 + e]) * a.scale;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r = r0 + warp; r < r1; r += NW) {
      const int64_t row = r < list.nA ? (a.idx ? a.idx[(size_t)b * a.idx_stride + r] : r) : list.t0 + (r - list.nA);
      if (row < 0 || row >= a.rows) continue;
      const unsigned kw = *reinterpret_cast<const unsigned*>(k + row * a.sr + lane * 4);
      const unsigned vw = *reinterpret_cast<const unsigned*>(v + row * a.sr + lane * 4);
      float s = 0.f;
      for (int e = 0; e < 4; ++e) s = fmaf(qv[e], code_value<FMT>((kw >> (8 * e)) & 0xffu), s);
      for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
      s *= ks[row >> a.shift];
      if (lane == 0 && r < score_lim) score_row[r] = g == 0 ? s : fmaxf(score_row[r], s);
      const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : expf(m - mn), p = expf(s - mn);
      const float pv = p * vs[row >> a.shift];
      l = l * c + p;
      for (int e = 0; e < 4; ++e) o[e] = o[e] * c + pv * code_value<FMT>((vw >> (8 * e)) & 0xffu);
      m = mn;
    }
    for (int e = 0; e < 4; ++e) o_s[warp][g][lane * 4 + e] = o[e];
    if (lane == 0) {
      ml_s[warp][g][0] = m;
      ml_s[warp][g][1] = l;
    }
  }
  __syncthreads();
  for (int g = 0; g < G; ++g) {
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml_s[w][g][0]);
    for (int w = 0; w < NW; ++w) {
      const float c = ml_s[w][g][0] == -INFINITY ? 0.f : expf(ml_s[w][g][0] - M);
      L += ml_s[w][g][1] * c;
      acc += o_s[w][g][tid] * c;
    }
    const size_t base = (size_t)(b * a.H + kvh * G + g) * a.S + split;
    a.ws_o[base * kHeadDim + tid] = acc;
    if (tid == 0) {
      a.ws_ml[base * 2] = M;
      a.ws_ml[base * 2 + 1] = L;
    }
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) last_flag = atomicAdd(a.ws_cnt + b * a.KVH + kvh, 1u) == (unsigned)(a.S - 1);
  __syncthreads();
  if (!last_flag) return;
  __threadfence();
  for (int g = 0; g < G; ++g) {
    const size_t base = (size_t)(b * a.H + kvh * G + g) * a.S;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int s = 0; s < a.S; ++s) M = fmaxf(M, __ldcg(a.ws_ml + (base + s) * 2));
    for (int s = 0; s < a.S; ++s) {
      const float ms = __ldcg(a.ws_ml + (base + s) * 2), c = ms == -INFINITY ? 0.f : expf(ms - M);
      L += __ldcg(a.ws_ml + (base + s) * 2 + 1) * c;
      acc += __ldcg(a.ws_o + (base + s) * kHeadDim + tid) * c;
    }
    static_cast<T*>(a.out)[(size_t)b * a.q_sb + (size_t)(kvh * G + g) * a.q_sh + tid] = from_float<T>(L == 0.f ? 0.f : acc / L);
  }
  if (tid == 0) a.ws_cnt[b * a.KVH + kvh] = 0u;
}

}  // namespace
}  // namespace omnikv

extern "C" size_t omnikv_kv8_attn_workspace_bytes(int B, int H, int n_splits) {
  if (B <= 0 || H <= 0 || n_splits <= 0) return 0;
  return omnikv::kAttnCntBytes +
         (omnikv::attn_ws_o_floats(B, H, n_splits) + omnikv::attn_ws_ml_floats(B, H, n_splits)) * sizeof(float);
}

extern "C" int omnikv_kv8_decode_attn(const omnikv_kv8_attn_params* p, void* stream) {
  using namespace omnikv;
  if (!p) return OMNIKV_E_BADARG;
  const omnikv_kv8_cache& c = p->cache;
  if (const int rc = check_kv8_cache(&c)) return rc;
  const auto bad16 = [](const void* q) { return !q || (reinterpret_cast<uintptr_t>(q) & 15); };
  if (bad16(p->q) || bad16(p->out) || !p->len || p->H <= 0 || p->H % c.KVH || p->n_splits <= 0) return OMNIKV_E_BADARG;
  if (p->q_stride_b % 8 || p->q_stride_h % 8) return OMNIKV_E_BADARG;
  if (p->idx && (p->idx_cap <= 0 || p->idx_stride < 0)) return OMNIKV_E_BADARG;
  if (p->tail_len && !p->tail_start) return OMNIKV_E_BADARG;
  if (p->score_out && (p->idx || p->tail_len || !p->score_len || p->score_stride <= 0)) return OMNIKV_E_BADARG;
  if (!is_16bit(p->dtype) || p->H / c.KVH > MAX_G) return OMNIKV_E_UNSUPPORTED;
  if (p->n_splits > 512 || (size_t)c.B * c.KVH * 4 > kAttnCntBytes) return OMNIKV_E_UNSUPPORTED;
  if (!p->workspace || p->workspace_bytes < omnikv_kv8_attn_workspace_bytes(c.B, p->H, p->n_splits)) return OMNIKV_E_WORKSPACE;
  if (bad16(p->workspace)) return OMNIKV_E_BADARG;
  A8Args a;
  a.k = static_cast<const unsigned char*>(c.k); a.v = static_cast<const unsigned char*>(c.v);
  a.sb = c.stride_b; a.sh = c.stride_h; a.sr = c.stride_row;
  a.ks = c.k_scale; a.vs = c.v_scale; a.ssb = c.scale_stride_b; a.ssh = c.scale_stride_h;
  a.shift = __builtin_ctz(c.block); a.rows = c.rows;
  a.q = p->q; a.q_sb = p->q_stride_b; a.q_sh = p->q_stride_h; a.out = p->out;
  a.idx = p->idx; a.idx_stride = p->idx_stride; a.idx_cap = p->idx_cap;
  a.len = p->len; a.tail_start = p->tail_start; a.tail_len = p->tail_len;
  a.score_out = p->score_out; a.score_stride = p->score_stride; a.score_len = p->score_len;
  a.ws_cnt = static_cast<unsigned*>(p->workspace);
  a.ws_o = reinterpret_cast<float*>(static_cast<unsigned char*>(p->workspace) + kAttnCntBytes);
  a.ws_ml = a.ws_o + attn_ws_o_floats(c.B, p->H, p->n_splits);
  a.B = c.B; a.H = p->H; a.KVH = c.KVH; a.G = p->H / c.KVH; a.S = p->n_splits;
  a.scale = p->scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(a.S, a.KVH, a.B);
  const bool i8 = c.format == kInt8;
  auto kern = p->dtype == OMNIKV_BF16
                  ? (i8 ? decode_attn_kv8_kernel<__nv_bfloat16, kInt8> : decode_attn_kv8_kernel<__nv_bfloat16, kE4m3>)
                  : (i8 ? decode_attn_kv8_kernel<__half, kInt8> : decode_attn_kv8_kernel<__half, kE4m3>);
  OMNIKV_CUDA_OK(launch_pdl(kern, grid, dim3(NT), 0, st, a));
  return OMNIKV_OK;
}
