// 8-bit codes of keys, values, activations and weights: how a value becomes a code and back.
#pragma once

#include <cuda_fp8.h>

#include <atomic>

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

// num / den with den > 0 to the nearest code.  IEEE division: for 16-bit x the quotient top * x / a is a ratio of
// integers of at most 18 and 11 bits, so an fp32 quotient never crosses the middle between two codes and the code is
// the one exact arithmetic gives.
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

// How the values of a block with largest magnitude a (bits) are coded: code = round(x * mul / den), scale = a / top.
// Both sides of the quotient are scaled down by a power of two where top * x could overflow.
struct CodeRule {
  float mul, den, scale;
  bool live;  // false: all codes are zero (nothing but zeros, or something that is not finite)
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
  return r;
}
template <int FMT>
__device__ __forceinline__ unsigned code_with(const CodeRule& r, float x) {
  return r.live ? code_of<FMT>(__fdiv_rn(x * r.mul, r.den)) : 0u;
}

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
// Tensor map over the codes of an 8-bit cache (false: the layout cannot be described as one).
bool make_kv8_tensor_map(CUtensorMap* map, const void* base, int64_t rows, int KVH, int B, int64_t sr, int64_t sh,
                         int64_t sb, int box_rows);

// Tensor map over a row-major matrix of bytes: box 128 bytes x box_rows rows, 128-byte swizzle, zeros past its edges.
bool make_bytes_tensor_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows);

// cudaFuncSetAttribute once per kernel and device.
template <typename Kern>
int allow_smem(Kern kern, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  OMNIKV_CUDA_OK(cudaGetDevice(&dev));
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return OMNIKV_OK;
  OMNIKV_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_release);
  return OMNIKV_OK;
}

inline bool is_16bit(int dtype) { return dtype == OMNIKV_BF16 || dtype == OMNIKV_F16; }

}  // namespace omnikv
