// Filling and reading a KV cache held in 8 bits: a prompt's rows, one row per sequence, rows back in 16 bits.
//
// All three are streams: 2 bytes in and 1 out per element (store), 1 in and 2 out (load), and a row per head (append),
// so HBM (or, for one row, latency) bounds them.
#include "kv8.cuh"

namespace omnikv {
namespace {

struct Kv8View {
  unsigned char *k, *v;
  int64_t sb, sh, sr;
  float *ks, *vs;
  int64_t ssb, ssh;
  int block, rows;
};

inline Kv8View view_of(const omnikv_kv8_cache* c) {
  return Kv8View{static_cast<unsigned char*>(c->k), static_cast<unsigned char*>(c->v), c->stride_b, c->stride_h,
                 c->stride_row, c->k_scale, c->v_scale, c->scale_stride_b, c->scale_stride_h, c->block, c->rows};
}

// ---- store ------------------------------------------------------------------------------------------------------
// A CTA takes 128 rows (256, and twice the threads, where a scale block is that long: 179 -> 140 us for 131072 rows of 8 heads
// against twice the rows per thread) of one (sequence, head) of K or V: sixteen lanes hold a row, eight elements each, in
// registers between the two steps (maximum of the block, codes), so every element is read once.  One thread per scale block
// turns its maximum into the rule for its codes: the divisions that takes were a third of the instructions when every thread
// did it (131072 rows of 8 heads, one tensor as K and V: 149 -> 123 us; two tensors: 128 us, 123 at the copy rate).

struct StoreArgs {
  Kv8View c;
  const void *k, *v;
  int64_t k_sb, k_sh, k_sr, v_sb, v_sh, v_sr;
  int start, n, KVH;
  const int* lens;
};

// PPB: passes of THREADS / 16 rows per scale block; 0: blocks shorter than a pass (one row: 165 us with a reduction per pass,
// 144 with one for all passes).
constexpr int kStorePasses = 8;
template <typename T, int FMT, int ST_THREADS, int PPB>
__global__ void __launch_bounds__(ST_THREADS) kv8_store_kernel(const StoreArgs a) {
  constexpr int PASSES = kStorePasses, ST_ROWS = ST_THREADS / 16, R = PASSES * ST_ROWS, WARPS = ST_THREADS / 32, BLOCKS = PPB ? PASSES / PPB : R;
  __shared__ unsigned top[BLOCKS][PPB ? WARPS : 1];  // largest magnitude of each scale block, by warp
  __shared__ float2 rules[BLOCKS];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane16 = tid & 15, row16 = tid >> 4;
  const int h = blockIdx.y >> 1, b = blockIdx.z;
  const bool is_v = blockIdx.y & 1;
  const int n = a.lens ? min(a.n, a.lens[b]) : a.n;
  const int r0 = blockIdx.x * R;
  if (r0 >= n) return;
  const int shift = 31 - __clz(a.c.block);
  const int64_t s_sr = is_v ? a.v_sr : a.k_sr;
  const T* src = static_cast<const T*>(is_v ? a.v : a.k) + (size_t)b * (is_v ? a.v_sb : a.k_sb) + (size_t)h * (is_v ? a.v_sh : a.k_sh) +
                 (int64_t)(r0 + row16) * s_sr + lane16 * 8;
  uint4 x[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    x[p] = make_uint4(0, 0, 0, 0);
    if (r0 + p * ST_ROWS + row16 < n) x[p] = *reinterpret_cast<const uint4*>(src + p * ST_ROWS * s_sr);
  }
  if constexpr (PPB > 0) {
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i) {
      unsigned m2 = 0;
#pragma unroll
      for (int p = i * PPB; p < (i + 1) * PPB; ++p) m2 = max_abs2<T>(m2, x[p]);
      const unsigned m = __reduce_max_sync(0xffffffffu, abs_bits_of<T>(m2));
      if ((tid & 31) == 0) top[i][tid >> 5] = m;
    }
  } else {
    if (shift)
      for (int i = tid; i < R; i += ST_THREADS) top[i][0] = 0;
    // the rows' maxima over sixteen lanes: at each step a lane hands half of its passes over and keeps the other half
    unsigned m[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) m[p] = abs_bits_of<T>(max_abs2<T>(0u, x[p]));
#pragma unroll
    for (int n = PASSES / 2, off = 8; n > 0; n >>= 1, off >>= 1)
#pragma unroll
      for (int p = 0; p < n; ++p) {
        const unsigned keep = lane16 & off ? m[p + n] : m[p], give = lane16 & off ? m[p] : m[p + n];
        m[p] = max(keep, __shfl_xor_sync(0xffffffffu, give, off));
      }
    m[0] = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], 1));
    const int row = (lane16 >> 1) * ST_ROWS + row16;  // bits 3, 2, 1 of the lane: the pass it has been left with
    if (shift) {
      __syncthreads();
      if (!(lane16 & 1) && m[0]) atomicMax(&top[row >> shift][0], m[0]);
    } else if (!(lane16 & 1)) {
      top[row][0] = m[0];
    }
  }
  __syncthreads();
  if (tid < (PPB ? BLOCKS : R >> shift)) {
    unsigned m = top[tid][0];
    if constexpr (PPB > 0)
#pragma unroll
      for (int w = 1; w < WARPS; ++w) m = max(m, top[tid][w]);
    const CodeRule rule = code_rule<FMT>(m);
    rules[tid] = shared_rule<FMT>(rule, m);
    float* scale = (is_v ? a.c.vs : a.c.ks) + (size_t)b * a.c.ssb + (size_t)h * a.c.ssh + ((a.start + r0) >> shift);
    if (r0 + (tid << shift) < n) scale[tid] = rule.scale;
  }
  __syncthreads();
  unsigned char* dst = (is_v ? a.c.v : a.c.k) + (size_t)b * a.c.sb + (size_t)h * a.c.sh + ((int64_t)a.start + r0 + row16) * a.c.sr + lane16 * 8;
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int lr = p * ST_ROWS + row16;
    if (r0 + lr < n) *reinterpret_cast<uint2*>(dst + p * ST_ROWS * a.c.sr) = code8<T, FMT>(rules[PPB ? p / (PPB ? PPB : 1) : lr >> shift], x[p]);
  }
}

// ---- append -----------------------------------------------------------------------------------------------------
// One CTA per (sequence, head) of K or V.  Every warp finds the row's maximum for itself (four elements per lane), so
// only the old scale has to be read by all before one thread replaces it.  Rows that follow a grown scale are re-coded
// by all threads, 16 codes each.
constexpr int AP_THREADS = 128;

template <typename T, int FMT>
__global__ void __launch_bounds__(AP_THREADS) kv8_append_kernel(const Kv8View c, const T* k_new, const T* v_new,
                                                                int64_t n_sb, int64_t n_sh, const int* pos_dev) {
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31;
  const int h = blockIdx.x >> 1, b = blockIdx.y;
  const bool is_v = blockIdx.x & 1;
  const int pos = pos_dev[b];
  if (pos < 0 || pos >= c.rows) return;
  const int shift = 31 - __clz(c.block), in_block = pos & (c.block - 1);
  unsigned char* code = (is_v ? c.v : c.k) + (size_t)b * c.sb + (size_t)h * c.sh;
  float* scale = (is_v ? c.vs : c.ks) + (size_t)b * c.ssb + (size_t)h * c.ssh + (pos >> shift);
  const uint2 raw = *reinterpret_cast<const uint2*>((is_v ? v_new : k_new) + (size_t)b * n_sb + (size_t)h * n_sh + lane * 4);
  const float s0 = in_block ? *scale : 0.f;
  const float2 f0 = unpack16<T>(raw.x), f1 = unpack16<T>(raw.y);
  unsigned m = max(max(abs_bits(f0.x), abs_bits(f0.y)), max(abs_bits(f1.x), abs_bits(f1.y)));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
  CodeRule rule = code_rule<FMT>(m);
  const bool fits = s0 > rule.scale || s0 != s0;  // the old scale stands (a block that reads as NaN stays so)
  float s1 = rule.scale;
  if (fits) {
    s1 = s0;
    rule.mul = 1.f;
    rule.den = s0;
    rule.live = __float_as_uint(s0) < 0x7f800000u;
  }
  __syncthreads();  // every warp has read the old scale
  if (tid < 32) {
    const unsigned w = code_with<FMT>(rule, f0.x) | code_with<FMT>(rule, f0.y) << 8 | code_with<FMT>(rule, f1.x) << 16 |
                       code_with<FMT>(rule, f1.y) << 24;
    *reinterpret_cast<unsigned*>(code + (int64_t)pos * c.sr + lane * 4) = w;
    if (lane == 0) *scale = s1;
  }
  if (fits || s1 == s0) return;
  const float ratio = s0 / s1;
  const bool finite = abs_bits(s1) < 0x7f800000u;  // else the block reads as NaN: codes 0
  unsigned char* first = code + (int64_t)(pos - in_block) * c.sr;
  for (int i = tid; i < in_block * 8; i += AP_THREADS) {
    uint4* p = reinterpret_cast<uint4*>(first + (int64_t)(i >> 3) * c.sr) + (i & 7);
    uint4 q = *p;
    unsigned* w = reinterpret_cast<unsigned*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned o = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (finite) o |= code_of<FMT>(code_value<FMT>((w[j] >> (8 * e)) & 0xffu) * ratio) << (8 * e);
      w[j] = o;
    }
    *p = q;
  }
}

// ---- load -------------------------------------------------------------------------------------------------------
// Eight threads per row of 128 codes, sixteen codes each; a CTA takes K and V of 16 * STEPS rows of a head.  The heads of
// the same rows are neighbours in the grid: where a token's heads lie together (the layout of layers that read selected
// tokens), the scattered reads of a token then come close in time.
constexpr int LD_THREADS = 256;
constexpr int kLoadIdxSteps = 4;  // rows per thread of scattered reads (2048 of 20000 rows, 16 sequences: 39.4, 35.5, 34.7 us for 1, 2, 4)

template <typename T, int FMT, int STEPS>
__global__ void __launch_bounds__(LD_THREADS) kv8_load_kernel(const Kv8View c, int KVH, int start, int n, const int* idx,
                                                              int64_t idx_stride, T* k_out, T* v_out, int64_t o_sb,
                                                              int64_t o_sh, int64_t o_sr) {
  pdl_wait();
  pdl_trigger();
  const int h = blockIdx.x % KVH, i0 = (blockIdx.x / KVH) * (16 * STEPS) + (threadIdx.x >> 4), b = blockIdx.y;
  const bool is_v = (threadIdx.x >> 3) & 1;
  const int piece = threadIdx.x & 7, shift = 31 - __clz(c.block);
  const unsigned char* code = (is_v ? c.v : c.k) + (size_t)b * c.sb + (size_t)h * c.sh + piece * 16;
  const float* scale = (is_v ? c.vs : c.ks) + (size_t)b * c.ssb + (size_t)h * c.ssh;
  T* out = (is_v ? v_out : k_out) + (size_t)b * o_sb + (size_t)h * o_sh + piece * 16;
  int64_t row[STEPS];
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    const int i = i0 + 16 * u;
    row[u] = i >= n ? -1 : idx ? (int64_t)idx[(size_t)b * idx_stride + i] : (int64_t)start + i;
    if (row[u] >= c.rows) row[u] = -1;
  }
  uint4 q[STEPS];
  float s[STEPS];
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    q[u] = make_uint4(0, 0, 0, 0);
    s[u] = 0.f;
    if (row[u] >= 0) {
      q[u] = *reinterpret_cast<const uint4*>(code + row[u] * c.sr);
      s[u] = scale[row[u] >> shift];
    }
  }
#pragma unroll
  for (int u = 0; u < STEPS; ++u) {
    const int i = i0 + 16 * u;
    if (i >= n) continue;
    const unsigned* w = reinterpret_cast<const unsigned*>(&q[u]);
    unsigned o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned two = w[j >> 1] >> (16 * (j & 1));
      o[j] = pack2<T>(code_value<FMT>(two & 0xffu) * s[u], code_value<FMT>((two >> 8) & 0xffu) * s[u]);
    }
    uint4* dst = reinterpret_cast<uint4*>(out + (int64_t)i * o_sr);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

template <typename T, int FMT>
int launch_store(const StoreArgs& a, int B, cudaStream_t st) {
  const auto go = [&](auto kern, int threads) -> int {
    OMNIKV_CUDA_OK(launch_pdl(kern, dim3(ceil_div(a.n, kStorePasses * threads / 16), 2 * a.KVH, B), dim3(threads), 0, st, a));
    return OMNIKV_OK;
  };
  switch (a.c.block) {
    case 16: return go(kv8_store_kernel<T, FMT, 256, 1>, 256);
    case 32: return go(kv8_store_kernel<T, FMT, 256, 2>, 256);
    case 64: return go(kv8_store_kernel<T, FMT, 256, 4>, 256);
    case 128: return go(kv8_store_kernel<T, FMT, 256, 8>, 256);
    case 256: return go(kv8_store_kernel<T, FMT, 512, 8>, 512);
    default: return go(kv8_store_kernel<T, FMT, 256, 0>, 256);
  }
}

// kernel<element type, format> for the two 16-bit types and the two formats
#define OMNIKV_KV8_DISPATCH(dtype, format, CALL)                          \
  (dtype == OMNIKV_BF16 ? (format == kInt8 ? CALL(__nv_bfloat16, kInt8) : CALL(__nv_bfloat16, kE4m3)) \
                        : (format == kInt8 ? CALL(__half, kInt8) : CALL(__half, kE4m3)))

inline bool bad16(const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15); }

}  // namespace
}  // namespace omnikv

extern "C" int omnikv_kv8_store(const omnikv_kv8_cache* c, int dtype, const void* k, int64_t k_stride_b,
                                int64_t k_stride_h, int64_t k_stride_row, const void* v, int64_t v_stride_b,
                                int64_t v_stride_h, int64_t v_stride_row, int start, int n, const int32_t* lens,
                                void* stream) {
  using namespace omnikv;
  if (const int rc = check_kv8_written(c)) return rc;
  if (bad16(k) || bad16(v) || n <= 0 || start < 0 || start % c->block || n > c->rows - start) return OMNIKV_E_BADARG;
  if (!is_16bit(dtype)) return OMNIKV_E_UNSUPPORTED;
  if (k_stride_b % 8 || k_stride_h % 8 || k_stride_row % 8 || v_stride_b % 8 || v_stride_h % 8 || v_stride_row % 8)
    return OMNIKV_E_BADARG;
  StoreArgs a{view_of(c), k, v, k_stride_b, k_stride_h, k_stride_row, v_stride_b, v_stride_h, v_stride_row,
              start, n, c->KVH, lens};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define OMNIKV_CALL(T, F) launch_store<T, F>(a, c->B, st)
  return OMNIKV_KV8_DISPATCH(dtype, c->format, OMNIKV_CALL);
#undef OMNIKV_CALL
}

extern "C" int omnikv_kv8_append(const omnikv_kv8_cache* c, int dtype, const void* k_new, const void* v_new,
                                 int64_t new_stride_b, int64_t new_stride_h, const int32_t* pos, void* stream) {
  using namespace omnikv;
  if (const int rc = check_kv8_written(c)) return rc;
  if (bad16(k_new) || bad16(v_new) || !pos || new_stride_b % 8 || new_stride_h % 8) return OMNIKV_E_BADARG;
  if (!is_16bit(dtype)) return OMNIKV_E_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(2 * c->KVH, c->B);
#define OMNIKV_CALL(T, F)                                                                                             \
  launch_pdl_args(kv8_append_kernel<T, F>, grid, dim3(AP_THREADS), st, view_of(c), static_cast<const T*>(k_new),     \
                  static_cast<const T*>(v_new), new_stride_b, new_stride_h, pos)
  OMNIKV_CUDA_OK(OMNIKV_KV8_DISPATCH(dtype, c->format, OMNIKV_CALL));
#undef OMNIKV_CALL
  return OMNIKV_OK;
}

extern "C" int omnikv_kv8_load(const omnikv_kv8_cache* c, int dtype, int start, int n, const int32_t* idx,
                               int64_t idx_stride, void* k_out, void* v_out, int64_t out_stride_b, int64_t out_stride_h,
                               int64_t out_stride_row, void* stream) {
  using namespace omnikv;
  if (const int rc = check_kv8_cache(c)) return rc;
  if (bad16(k_out) || bad16(v_out) || n <= 0 || start < 0 || (idx && (start || idx_stride < 0)))
    return OMNIKV_E_BADARG;
  if (out_stride_b % 8 || out_stride_h % 8 || out_stride_row % 8 || out_stride_row < kHeadDim) return OMNIKV_E_BADARG;
  if (!is_16bit(dtype)) return OMNIKV_E_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int steps = idx ? kLoadIdxSteps : 1;
  const int64_t blocks = ((int64_t)n + 16 * steps - 1) / (16 * steps) * c->KVH;
  if (blocks > 0x7fffffff) return OMNIKV_E_UNSUPPORTED;
  const auto go = [&](auto kern, auto tag) -> int {
    using T = decltype(tag);
    OMNIKV_CUDA_OK(launch_pdl_args(kern, dim3((unsigned)blocks, c->B), dim3(LD_THREADS), st, view_of(c), c->KVH, start, n, idx, idx_stride,
                                   static_cast<T*>(k_out), static_cast<T*>(v_out), out_stride_b, out_stride_h, out_stride_row));
    return OMNIKV_OK;
  };
#define OMNIKV_CALL(T, F) (idx ? go(kv8_load_kernel<T, F, kLoadIdxSteps>, T()) : go(kv8_load_kernel<T, F, 1>, T()))
  return OMNIKV_KV8_DISPATCH(dtype, c->format, OMNIKV_CALL);
#undef OMNIKV_CALL
}

extern "C" unsigned long long omnikv_capture_id(void* stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &id) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

extern "C" int omnikv_capture_retain(void* stream, void (*release)(void*), void* arg) {
  using namespace omnikv;
  if (!release) return OMNIKV_E_BADARG;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  cudaGraph_t graph = nullptr;
  OMNIKV_CUDA_OK(cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, nullptr, &graph));
  if (status != cudaStreamCaptureStatusActive || !graph) return OMNIKV_E_BADARG;
  cudaUserObject_t object = nullptr;
  OMNIKV_CUDA_OK(cudaUserObjectCreate(&object, arg, release, 1, cudaUserObjectNoDestructorSync));
  OMNIKV_CUDA_OK(cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove));
  return OMNIKV_OK;
}
