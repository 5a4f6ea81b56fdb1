// What the kernels along the vocabulary axis share: the soft cap in its roundings, keys that order logits as integers, and
// block-wide reductions whose result does not depend on anything but the inputs.
#pragma once

#include "common.cuh"

namespace xl {

constexpr int VOCAB_MAX = 1 << 19;   // longest row: sums of weights in 2^-44 stay below 2^63
constexpr int TOPK_MAX = 1024;       // teacher entries of a row

// cap * tanh(x / cap) with quotient, tanh and product rounded to T each, as the reference's eager soft_cap does.
template <typename T> __device__ __forceinline__ float capped_rounded(T x, float cap) {
  const T q = from_float<T>(to_float(x) / cap);
  const T t = from_float<T>(tanhf(to_float(q)));
  return to_float(from_float<T>(cap * to_float(t)));
}

// ---------------------------------------------------------------------------------------------
// keys: a < b  <=>  key(a) < key(b), -0 and +0 alike, every NaN below -inf.  bf16 keys have 16 bits, fp32 keys 32.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t key_of_float(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);   // (-0 + 0 is +0)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float float_of_key(uint32_t k) {
  if (k == 0u) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
template <typename T> struct VocabKey;
template <> struct VocabKey<float> {
  static constexpr int BITS = 32;
  static __device__ __forceinline__ uint32_t of(float x) { return key_of_float(x); }
  static __device__ __forceinline__ float value(uint32_t k) { return float_of_key(k); }
};
template <> struct VocabKey<__nv_bfloat16> {   // the fp32 key's lower half says nothing: 0 or, below zero, all ones
  static constexpr int BITS = 16;
  static __device__ __forceinline__ uint32_t of(__nv_bfloat16 x) { return key_of_float(__bfloat162float(x)) >> 16; }
  static __device__ __forceinline__ float value(uint32_t k) { return float_of_key(k & 0x8000u ? k << 16 : k ? (k << 16) | 0xffffu : 0u); }
};

// ---------------------------------------------------------------------------------------------
// reductions over a block of WARPS full warps; `s` is shared memory of WARPS elements.  Every thread gets the result.
// ---------------------------------------------------------------------------------------------
template <int WARPS, typename V, typename F> __device__ __forceinline__ V block_reduce(V v, F f, V* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();   // (the last use of `s` is over)
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) v = f(v, s[w]);
  return v;
}
struct OpMax {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; }
};
struct OpSum {
  template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};

// what row-wise entries over logits check in common
static inline int vocab_validate(int rows, int V, int64_t row_stride, float cap, int dtype) {
  if (dtype != XL_F32 && dtype != XL_BF16) return XL_ERR_BAD_DTYPE;
  if (rows <= 0 || V <= 0 || !(cap >= 0.f) || cap > 3.0e38f) return XL_ERR_BAD_SHAPE;
  if (rows > 1 && row_stride < V) return XL_ERR_BAD_STRIDE;
  if (V > VOCAB_MAX) return XL_ERR_TOO_LARGE;
  return XL_OK;
}

}  // namespace xl
