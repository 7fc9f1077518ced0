// Matrix products in 8-bit integers, one scale per token and per output channel, and the row quantiser in front.
#include "kv8.cuh"

namespace omnikv {
namespace {

// ---- rows to codes ------------------------------------------------------------------------------------------------
// One CTA per row; the row stays in registers between the maximum and the codes, so it is read once and with one round
// of loads in flight (a single token's row is a latency chain: load, maximum, store).
constexpr int QR_VEC = 8;  // 16-byte pieces per thread at most

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) quant_rows_kernel(const T* x, int64_t x_sr, int K, int8_t* codes, int64_t c_sr,
                                                             float* scale) {
  __shared__ unsigned top[THREADS / 32];
  pdl_wait();
  const int row = blockIdx.x, tid = threadIdx.x, nvec = K / 8;
  const uint4* src = reinterpret_cast<const uint4*>(x + (size_t)row * x_sr);
  uint4 v[QR_VEC];
#pragma unroll
  for (int u = 0; u < QR_VEC; ++u) {
    v[u] = make_uint4(0, 0, 0, 0);
    if (tid + u * THREADS < nvec) v[u] = src[tid + u * THREADS];
  }
  unsigned m = 0;
#pragma unroll
  for (int u = 0; u < QR_VEC; ++u) {
    const unsigned* w = reinterpret_cast<const unsigned*>(&v[u]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack16<T>(w[i]);
      m = max(m, max(abs_bits(f.x), abs_bits(f.y)));
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((tid & 31) == 0) top[tid >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) m = max(m, top[i]);
  const CodeRule rule = code_rule<kInt8>(m);
  if (tid == 0) scale[row] = rule.scale;
  uint2* dst = reinterpret_cast<uint2*>(codes + (size_t)row * c_sr);
#pragma unroll
  for (int u = 0; u < QR_VEC; ++u) {
    if (tid + u * THREADS >= nvec) continue;
    const unsigned* w = reinterpret_cast<const unsigned*>(&v[u]);
    unsigned o[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack16<T>(w[i]);
      o[i >> 1] |= (code_with<kInt8>(rule, f.x) | code_with<kInt8>(rule, f.y) << 8) << (16 * (i & 1));
    }
    dst[tid + u * THREADS] = make_uint2(o[0], o[1]);
  }
}

// ---- the product: one thread per output -----------------------------------------------------------------------------
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
};

template <typename T>
__global__ void __launch_bounds__(256) linear_w8a8_kernel(const LinArgs a) {
  pdl_wait();
  const int c = blockIdx.x * 32 + (threadIdx.x >> 3), t = blockIdx.y * 8 + (threadIdx.x & 7);
  if (c >= a.N || t >= a.n) return;
  const int4* w = reinterpret_cast<const int4*>(a.w + (size_t)c * a.w_sr);
  const int4* x = reinterpret_cast<const int4*>(a.x + (size_t)t * a.x_sr);
  int acc = 0;
  for (int i = 0; i < a.K / 16; ++i) {
    const int4 p = w[i], q = x[i];
    acc = __dp4a(p.x, q.x, __dp4a(p.y, q.y, __dp4a(p.z, q.z, __dp4a(p.w, q.w, acc))));
  }
  float y = (float)acc * a.x_scale[t] * a.w_scale[c];
  if (a.res) y += to_float(static_cast<const T*>(a.res)[(size_t)t * a.res_sr + c]);
  static_cast<T*>(a.out)[(size_t)t * a.out_sr + c] = from_float<T>(y);
}

inline bool bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15); }

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
  const auto go = [&](auto tag, auto threads) -> int {
    using T = decltype(tag);
    constexpr int TH = decltype(threads)::value;
    OMNIKV_CUDA_OK(launch_pdl_args(quant_rows_kernel<T, TH>, dim3(n), dim3(TH), st, static_cast<const T*>(x), x_stride_row, K,
                                   codes, code_stride_row, scale));
    return OMNIKV_OK;
  };
  using Small = std::integral_constant<int, 128>;
  using Large = std::integral_constant<int, 512>;
  const bool small = K <= 128 * 8 * QR_VEC;
  if (dtype == OMNIKV_BF16) return small ? go(__nv_bfloat16(), Small()) : go(__nv_bfloat16(), Large());
  return small ? go(__half(), Small()) : go(__half(), Large());
}

extern "C" size_t omnikv_linear_w8a8_workspace_bytes(int, int, int) { return 0; }

extern "C" int omnikv_linear_w8a8(const omnikv_linear_w8a8_params* p, void* stream) {
  using namespace omnikv;
  if (!p || bad16(p->x) || bad16(p->w) || !p->x_scale || !p->w_scale || !p->out) return OMNIKV_E_BADARG;
  if (p->n_tokens <= 0 || p->channels <= 0 || p->K <= 0 || p->K % 16) return OMNIKV_E_BADARG;
  if (p->x_stride_row % 16 || p->w_stride_row % 16 || p->x_stride_row < p->K || p->w_stride_row < p->K) return OMNIKV_E_BADARG;
  if (p->out_stride_row < p->channels || (p->residual && p->residual_stride_row < p->channels)) return OMNIKV_E_BADARG;
  if (p->K > 32768 || (p->out_dtype != OMNIKV_F32 && !is_16bit(p->out_dtype))) return OMNIKV_E_UNSUPPORTED;
  LinArgs a{p->x, p->x_stride_row, p->x_scale, p->w, p->w_stride_row, p->w_scale, p->residual, p->residual_stride_row,
            p->out, p->out_stride_row, p->n_tokens, p->channels, p->K};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(ceil_div(a.N, 32), ceil_div(a.n, 8));
  auto kern = p->out_dtype == OMNIKV_F32 ? linear_w8a8_kernel<float>
              : p->out_dtype == OMNIKV_BF16 ? linear_w8a8_kernel<__nv_bfloat16> : linear_w8a8_kernel<__half>;
  OMNIKV_CUDA_OK(launch_pdl(kern, grid, dim3(256), 0, st, a));
  return OMNIKV_OK;
}
