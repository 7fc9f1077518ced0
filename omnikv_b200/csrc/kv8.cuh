// 8-bit codes of keys, values, activations and weights: how a value becomes a code and back.
#pragma once

#include <cuda_fp8.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace omnikv {

enum : int { kInt8 = OMNIKV_KV8_INT8, kE4m3 = OMNIKV_KV8_E4M3 };

template <int FMT>
__host__ __device__ constexpr float code_top() {
  return FMT == kInt8 ? 127.f : 448.f;
}

// |x| as an unsigned integer: its order is the order of the magnitudes, infinities above all numbers and NaN above
// infinities, so an integer maximum finds a block's largest magnitude and carries NaN along.
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int FMT>
__device__ __forceinline__ unsigned code_of(float v) {
  if constexpr (FMT == kInt8) return (unsigned)__float2int_rn(v) & 0xffu;
  else return (unsigned)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
template <int FMT>
__device__ __forceinline__ float code_value(unsigned byte) {
  if constexpr (FMT == kInt8) return (float)(int)(signed char)byte;
  else return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

// How the values of a block with largest magnitude a (bits) are coded: code = round(top x / a), scale = a / top.
//
// One value (code_with): IEEE division.  For 16-bit x the quotient is a ratio of integers, and one that is not exactly in
// the middle between two codes is at least 2^-19 of itself away from it (int8: |254 X - (2k+1) A 2^m| >= 1 against 254 X
// with X < 2^11; e4m3: 2^-16), so the rounded fp32 quotient lies on the true side and the code is that of exact arithmetic.
// (top x could overflow for a >= 2^64: both sides are scaled down by a power of two there.)
//
// Four values (code4), a third of a division's instructions (a store of 131072 rows of 8 heads, one tensor as K and V:
// 269 -> 123 us).  A product with the rounded factor top / a is within 2^-23 of the quotient, which is the true side for
// every quotient but an exact middle; and exact middles do occur.
//   int8: (2k+1) A 2^m = 254 X has, unless 127 divides A, the one solution 2k+1 = 127, x = a / 2, which rounds to the even 64,
//   away from zero: so the factor is rounded up.  Where 127 divides A the factor is a power of two and nothing is rounded, or
//   (fp16 only) the values are divided.  The sum with 1.5 * 2^23 rounds the exact product to an integer, ties to even.
//   e4m3: middles fall to both sides.  Rounding the product to 21 bits puts those, which have at most 8 bits, back in their
//   place and moves no other quotient by more than 2^-20.6.
struct CodeRule {
  float mul, den, scale, factor;
  bool live;  // false: all codes are zero (nothing but zeros, or something that is not finite)
  bool divide;  // code4 divides: top / a could overflow, or see above
};
template <int FMT>
__device__ __forceinline__ CodeRule code_rule(unsigned a_bits) {
  const float a = __uint_as_float(a_bits);
  CodeRule r;
  r.scale = __fdiv_rn(a, code_top<FMT>());
  r.live = a_bits > 0 && a_bits < 0x7f800000u;
  const float f = a >= 18446744073709551616.f ? 5.421010862427522e-20f : 1.f;  // 2^64, 2^-64
  r.mul = code_top<FMT>() * f;
  r.den = r.live ? a * f : 1.f;
  r.divide = a < 7.888609052210118e-31f;  // 2^-100
  r.factor = 0.f;
  if (r.live && !r.divide) {
    r.factor = FMT == kInt8 ? __fdiv_ru(127.f, a) : __fdiv_rn(code_top<FMT>(), a);
    if (FMT == kInt8 && fmaf(r.scale, 127.f, -a) == 0.f && fmaf(r.factor, a, -127.f) != 0.f) r.divide = true;
  }
  return r;
}
template <int FMT>
__device__ __forceinline__ unsigned code_with(const CodeRule& r, float x) {
  return r.live ? code_of<FMT>(__fdiv_rn(x * r.mul, r.den)) : 0u;
}
// What the threads of a CTA share of a rule: {factor, a}; factor 0: all codes zero, negative: divide.
template <int FMT>
__device__ __forceinline__ float2 shared_rule(const CodeRule& r, unsigned a_bits) {
  return make_float2(!r.live ? 0.f : r.divide ? -1.f : r.factor, __uint_as_float(a_bits));
}
__device__ __forceinline__ float to_21_bits(float x) { return __uint_as_float((__float_as_uint(x) + 4u) & ~7u); }
// Two 16-bit elements of a 32-bit word as floats.
template <typename T>
__device__ __forceinline__ float2 unpack16(unsigned u);
template <>
__device__ __forceinline__ float2 unpack16<__nv_bfloat16>(unsigned u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack16<__half>(unsigned u) {
  return __half22float2(*reinterpret_cast<__half2*>(&u));
}

// The codes of four values, packed.
template <int FMT>
__device__ __forceinline__ unsigned code4(const float2& rule, float2 x, float2 y) {
  const float f = rule.x;
  if (f <= 0.f) {
    if (f == 0.f) return 0u;
    const CodeRule r = code_rule<FMT>(__float_as_uint(rule.y));
    return code_with<FMT>(r, x.x) | code_with<FMT>(r, x.y) << 8 | code_with<FMT>(r, y.x) << 16 | code_with<FMT>(r, y.y) << 24;
  }
  if constexpr (FMT == kInt8) {
    constexpr float kBig = 12582912.f;
    const unsigned q0 = __float_as_uint(fmaf(x.x, f, kBig)), q1 = __float_as_uint(fmaf(x.y, f, kBig));
    const unsigned q2 = __float_as_uint(fmaf(y.x, f, kBig)), q3 = __float_as_uint(fmaf(y.y, f, kBig));
    return __byte_perm(__byte_perm(q0, q1, 0x0040), __byte_perm(q2, q3, 0x0040), 0x5410);
  } else {
    return (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(to_21_bits(x.x * f), to_21_bits(x.y * f)), __NV_SATFINITE, __NV_E4M3) |
           (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(to_21_bits(y.x * f), to_21_bits(y.y * f)), __NV_SATFINITE, __NV_E4M3) << 16;
  }
}
// ... of the eight 16-bit elements of a 16-byte piece
template <typename T, int FMT>
__device__ __forceinline__ uint2 code8(const float2& rule, const uint4& v) {
  return make_uint2(code4<FMT>(rule, unpack16<T>(v.x), unpack16<T>(v.y)), code4<FMT>(rule, unpack16<T>(v.z), unpack16<T>(v.w)));
}

// Running largest magnitudes of the two 16-bit elements of a word, side by side (a NaN stays), and the larger of both as
// the bits of a float.
template <typename T>
__device__ __forceinline__ unsigned max_abs2(unsigned m, unsigned w) {
  unsigned r;
  if constexpr (std::is_same<T, __half>::value)
    asm("max.NaN.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(m), "r"(w & 0x7fff7fffu));
  else
    asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(m), "r"(w & 0x7fff7fffu));
  return r;
}
template <typename T>
__device__ __forceinline__ unsigned max_abs2(unsigned m, const uint4& v) {
  return max_abs2<T>(max_abs2<T>(max_abs2<T>(max_abs2<T>(m, v.x), v.y), v.z), v.w);
}
template <typename T>
__device__ __forceinline__ unsigned abs_bits_of(unsigned m2) {
  const unsigned m = max(m2 & 0x7fffu, (m2 >> 16) & 0x7fffu);  // the order of the patterns is the order of the magnitudes
  if constexpr (std::is_same<T, __half>::value) return abs_bits(__half2float(__ushort_as_half((unsigned short)m)));
  else return m << 16;
}

// Thread-block clusters: this CTA's rank, a shared-memory address in CTA `rank`, and the barrier of all threads in two halves.
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned in_cta(unsigned addr, unsigned rank) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_sync_all() {
  cluster_arrive();
  cluster_wait();
}

// Host: an omnikv_kv8_cache that the kernels can read.
inline int check_kv8_cache(const omnikv_kv8_cache* c) {
  const auto bad16 = [](const void* p) { return !p || (reinterpret_cast<uintptr_t>(p) & 15); };
  if (!c || bad16(c->k) || bad16(c->v) || !c->k_scale || !c->v_scale) return OMNIKV_E_BADARG;
  if (c->B <= 0 || c->KVH <= 0 || c->rows <= 0) return OMNIKV_E_BADARG;
  if (c->head_dim != kHeadDim) return OMNIKV_E_UNSUPPORTED;
  if (c->format != kInt8 && c->format != kE4m3) return OMNIKV_E_UNSUPPORTED;
  if (c->block <= 0 || c->block > 256 || (c->block & (c->block - 1))) return OMNIKV_E_UNSUPPORTED;
  if (c->stride_b % 16 || c->stride_h % 16 || c->stride_row % 16 || c->stride_row < kHeadDim) return OMNIKV_E_BADARG;
  if (c->B > 65535 || c->KVH > 32767) return OMNIKV_E_UNSUPPORTED;  // grid dimensions
  return OMNIKV_OK;
}
// ... and write: no two sequences or heads in the same memory.
inline int check_kv8_written(const omnikv_kv8_cache* c) {
  if (const int rc = check_kv8_cache(c)) return rc;
  const auto shared = [](int n, int64_t codes, int64_t scales) { return n > 1 && (!codes || !scales); };
  return shared(c->B, c->stride_b, c->scale_stride_b) || shared(c->KVH, c->stride_h, c->scale_stride_h) ? OMNIKV_E_BADARG : OMNIKV_OK;
}
// Tensor map over the codes of an 8-bit cache (false: the layout cannot be described as one).
bool make_kv8_tensor_map(CUtensorMap* map, const void* base, int64_t rows, int KVH, int B, int64_t sr, int64_t sh,
                         int64_t sb, int box_rows);

// Tensor map over a row-major matrix of bytes: box 128 bytes x box_rows rows, 128-byte swizzle, zeros past its edges.
bool make_bytes_tensor_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows);

// cudaFuncSetAttribute once per kernel and device (large_cluster: more than eight CTAs to a cluster, too).
template <typename Kern>
int allow_smem(Kern kern, int bytes, std::atomic<unsigned long long>& done, bool large_cluster = false) {
  int dev = 0;
  OMNIKV_CUDA_OK(cudaGetDevice(&dev));
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return OMNIKV_OK;
  OMNIKV_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (large_cluster) OMNIKV_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  done.fetch_or(bit, std::memory_order_release);
  return OMNIKV_OK;
}

inline bool is_16bit(int dtype) { return dtype == OMNIKV_BF16 || dtype == OMNIKV_F16; }

}  // namespace omnikv
