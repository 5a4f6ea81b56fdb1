// What the kernels along the vocabulary axis share: the soft cap in its roundings, keys that order logits as integers, and
// block-wide reductions whose result does not depend on anything but the inputs.
#pragma once

#include "common.cuh"

namespace xl {

constexpr int VOCAB_MAX = 1 << 18;   // longest row: sums of weights in 2^-44 stay below 2^63
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
  __syncwarp();   // shuffles of a warp whose lanes have not met again take some 200 cycles each, of one whose have 30
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

// ---------------------------------------------------------------------------------------------
// 64-bit arithmetic with short chains: the result of a 64-bit instruction takes some forty cycles
// ---------------------------------------------------------------------------------------------
// Conversions between 64-bit numbers and integers or fp32 go through the slowest unit of the SM; here they are bit moves and
// additions of powers of two.
__device__ __forceinline__ double double_of(float v) {   // (what is below 2^-126 counts as 0)
  const uint32_t b = __float_as_uint(v), m = b & 0x7fffffffu;
  return m < 0x00800000u ? 0.0 : __hiloint2double((int)((b & 0x80000000u) | ((m >> 3) + 0x38000000u)), (int)(m << 29));
}
// e^x for x <= 0 (below -700: e^-700): 2^n times the Taylor series of 2^f, |f| <= 1/2, to degree 10: relative error 3e-13
__device__ __forceinline__ double exp64(double x) {
  constexpr double LOG2E_64 = 1.4426950408889634, ROUND = 6755399441055744.0;   // 1.5 * 2^52: adding it rounds to whole numbers
  x = x > -700.0 ? x : -700.0;
  const double r = fma(x, LOG2E_64, ROUND), f = fma(x, LOG2E_64, ROUND - r);
  const double f2 = f * f, f4 = f2 * f2;   // (in halves of halves: a chain of five instead of ten)
  const double p0 = fma(fma(0.05550410866482158, f, 0.24022650695910072), f2, fma(0.6931471805599453, f, 1.0));
  const double p1 = fma(fma(1.5252733804059841e-05, f, 0.0001540353039338161), f2, fma(0.0013333558146428443, f, 0.009618129107628477));
  const double p2 = fma(7.054911620801123e-09, f2, fma(1.01780860092397e-07, f, 1.321548679014431e-06));
  const double p = fma(fma(p2, f4, p1), f4, p0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(r) << 20), __double2loint(p));   // (exponent >= -1010: no subnormal)
}
// 1 / d, 1 <= d <= 2: a Newton step from the fp32 reciprocal (2^-22 squared)
__device__ __forceinline__ double inverse64(double d) {
  const uint32_t hi = (uint32_t)__double2hiint(d), lo = (uint32_t)__double2loint(d);
  const float f = hi >= 0x40000000u ? 2.f : __uint_as_float(0x3f800000u | (hi & 0x000fffffu) << 3 | lo >> 29);
  const double r = double_of(__fdividef(1.f, f));
  return fma(r, fma(-d, r, 1.0), r);
}
// log2(x) of x >= 0: the fp32 logarithm of the mantissa, and what e^x says is missing from it (error 1e-13)
__device__ __forceinline__ double log2_64(double x) {
  if (!(x > 0.0) || x > 1.7e308) return x == 0.0 ? -(double)INFINITY : x;   // (NaN, infinity; not of negative numbers)
  const int hi = __double2hiint(x), e = (hi >> 20) - 1023;
  const double m = __hiloint2double((hi & 0x000fffff) | 0x3ff00000, __double2loint(x));
  const float l = log2f((float)m);
  const double missing = fma(m, exp64((double)l * -0.69314718055994530942), -1.0);
  return fma(missing, 1.4426950408889634, (double)l) + (double)e;
}

// ---------------------------------------------------------------------------------------------
// fp32 arithmetic of the capped logits, two elements to an instruction
//
// Packed fma/mul/add take two cycles of the fp32 pipe but one issue slot for two elements (measured: 65 packed against 125
// plain instructions per cycle and SM), and a row's passes are as much bound by issue slots as by the pipe.
// ---------------------------------------------------------------------------------------------
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 f2_pack(float a, float b) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ f32x2 f2_bits(uint32_t a, uint32_t b) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b)); return r; }
__device__ __forceinline__ f32x2 f2_dup(float a) { return f2_pack(a, a); }
__device__ __forceinline__ void f2_unpack(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 f2_mul(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 f2_fma(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ float exp2_approx(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

constexpr float LOG2E = 1.4426950408889634f;

// tanh(z) = z P(z^2) for |z| <= 0.75, relative error within 3 * 2^-24 (least-squares weights driven to the minimax, degree 5).
// Rows whose logits all stay below three quarters of the cap are fast; what larger ones cost stands at the kernels.
// Beyond it 1 - 2 / (1 + e^2|z|), whose quotient is below 0.37 there.
constexpr float TANH_SMALL = 0.75f;
__device__ __forceinline__ float tanh_large(float z) {
  const float q = 1.f - __fdividef(2.f, 1.f + exp2_approx(fminf(fabsf(z), 20.f) * (2.f * LOG2E)));
  return z != z ? z : copysignf(q, z);
}

// A vector of 16 bytes of logits as packed fp32 pairs.
template <typename T> struct Vec16;
template <> struct Vec16<__nv_bfloat16> {
  static constexpr int N = 8;
  f32x2 p[4];
  uint4 raw;
  __device__ __forceinline__ void set(const uint4& u) {
    raw = u;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = f2_bits(w[i] << 16, w[i] & 0xffff0000u);
  }
  // running largest magnitude (NaN does not count)
  typedef __nv_bfloat162 Mag;
  static __device__ __forceinline__ Mag no_mag() { return __float2bfloat162_rn(0.f); }
  __device__ __forceinline__ Mag track(Mag m) const {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __hmax2(m, __habs2(h[i]));
    return m;
  }
  static __device__ __forceinline__ float largest(Mag m) { return __bfloat162float(__hmax(__low2bfloat16(m), __high2bfloat16(m))); }
  static __device__ __forceinline__ uint4 round(const f32x2 (&v)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      f2_unpack(v[i], a, b);
      w[i] = pack_bf16x2(a, b);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec16<float> {
  static constexpr int N = 4;
  f32x2 p[2];
  __device__ __forceinline__ void set(const uint4& u) { p[0] = f2_bits(u.x, u.y); p[1] = f2_bits(u.z, u.w); }
  typedef float Mag;
  static __device__ __forceinline__ Mag no_mag() { return 0.f; }
  __device__ __forceinline__ Mag track(Mag m) const {
    float a, b, c, d;
    f2_unpack(p[0], a, b);
    f2_unpack(p[1], c, d);
    return fmaxf(m, fmaxf(fmaxf(fabsf(a), fabsf(b)), fmaxf(fabsf(c), fabsf(d))));
  }
  static __device__ __forceinline__ float largest(Mag m) { return m; }
  static __device__ __forceinline__ uint4 round(const f32x2 (&v)[2]) {
    uint4 u;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(u.x), "=r"(u.y) : "l"(v[0]));
    asm("mov.b64 {%0, %1}, %2;" : "=r"(u.z), "=r"(u.w) : "l"(v[1]));
    return u;
  }
};

// z = a * tanh(x / cap) with a = cap log2(e) / T, or (x - ref) * log2(e) / T without a cap: exponents of two.  `ref` is a number
// near the row's largest logit, so that rows near the type's lowest value (masks) do not overflow.
template <bool CAP> struct CappedZ {
  float a, icap, ref, flat;   // flat = 1 / a^2: the cap's slope is 1 - flat z^2
  // z = x Q(x^2) for magnitudes up to `limit`: the polynomial's coefficients with a and the powers of the cap inside, which
  // saves the product x / cap; for caps outside 1/8 .. 1024, whose powers leave fp32, nothing counts as small
  float q0, q1, q2, q3, q4, q5, limit;
  CappedZ(float cap, float temperature) {   // (on the host: the constants are kernel parameters)
    const double scale = 1.4426950408889634 / (double)temperature, wide = CAP ? scale * (double)cap : scale;
    a = (float)wide;
    ref = 0.f;
    icap = CAP ? (float)(1.0 / (double)cap) : 0.f;
    flat = CAP ? (float)(1.0 / (wide * wide)) : 0.f;
    const bool fits = CAP && cap >= 0.125f && cap <= 1024.f;
    const double i1 = fits ? 1.0 / (double)cap : 0.0, i2 = i1 * i1;
    q0 = (float)(wide * i1);
    q1 = (float)(wide * C1 * i1 * i2);
    q2 = (float)(wide * C2 * i1 * i2 * i2);
    q3 = (float)(wide * C3 * i1 * i2 * i2 * i2);
    q4 = (float)(wide * C4 * i1 * i2 * i2 * i2 * i2);
    q5 = (float)(wide * C5 * i1 * i2 * i2 * i2 * i2 * i2);
    limit = fits ? TANH_SMALL * cap : -1.f;
  }
  static constexpr float C1 = -0.33332958817481995f, C2 = 0.1332540661096573f, C3 = -0.05334443226456642f, C4 = 0.01958290860056877f, C5 = -0.004716257099062204f;
  __device__ __forceinline__ float operator()(float x) const {
    if (!CAP) return (x - ref) * a;
    const float z = x * icap, s = z * z;
    if (fabsf(z) > TANH_SMALL) return a * tanh_large(z);
    return z * fmaf(s, fmaf(s, fmaf(s, fmaf(s, fmaf(s, a * C5, a * C4), a * C3), a * C2), a * C1), a);
  }
  __device__ __forceinline__ void set_ref(float largest) { ref = fabsf(largest) <= 3.4028234e38f ? largest : 0.f; }   // (not of infinities)
  // tanh(x / cap)
  __device__ __forceinline__ float tanh_of(float x) const {
    const float z = x * icap, s = z * z;
    if (fabsf(z) > TANH_SMALL) return tanh_large(z);
    return z * fmaf(s, fmaf(s, fmaf(s, fmaf(s, fmaf(s, C5, C4), C3), C2), C1), 1.f);
  }
  __device__ __forceinline__ bool small(float magnitude) const { return !CAP || magnitude <= limit; }
  // of a vector's elements; SMALL: the caller has seen that all magnitudes are small
  template <bool SMALL, typename T> __device__ __forceinline__ void of(const Vec16<T>& v, f32x2 (&out)[Vec16<T>::N / 2]) const {
    if (!CAP) {
#pragma unroll
      for (int i = 0; i < Vec16<T>::N / 2; ++i) out[i] = f2_mul(f2_add(v.p[i], f2_dup(-ref)), f2_dup(a));
      return;
    }
    if (SMALL) {
#pragma unroll
      for (int i = 0; i < Vec16<T>::N / 2; ++i) {
        const f32x2 x = v.p[i], s = f2_mul(x, x);
        f32x2 q = f2_fma(s, f2_dup(q5), f2_dup(q4));
        q = f2_fma(s, q, f2_dup(q3));
        q = f2_fma(s, q, f2_dup(q2));
        q = f2_fma(s, q, f2_dup(q1));
        out[i] = f2_mul(x, f2_fma(s, q, f2_dup(q0)));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < Vec16<T>::N / 2; ++i) {
      float x0, x1;
      f2_unpack(v.p[i], x0, x1);
      out[i] = f2_pack((*this)(x0), (*this)(x1));
    }
  }
};

// How a row that may start anywhere lies in 16-byte vectors, and which of them are this block's: `head` elements in front of
// the first boundary (block 0 of the row), vectors [v0, v1), and the rest behind the last vector (the last block).
// place(j) numbers the elements so that vector v holds N (v + 1) .. N (v + 1) + N - 1.
template <typename T> struct RowSlice {
  static constexpr int N = Vec16<T>::N;
  int head, vectors, v0, v1, first, end;   // places [first, end) are this block's
  int V;
  __device__ __forceinline__ RowSlice(const T* x, int V_, int rank, int blocks) : V(V_) {
    const int mis = (int)((reinterpret_cast<uintptr_t>(x) / sizeof(T)) % N);
    head = min(V, mis ? N - mis : 0);
    vectors = (V - head) / N;
    const int per = (vectors + blocks - 1) / blocks;
    v0 = min(vectors, rank * per);
    v1 = min(vectors, v0 + per);
    first = rank == 0 ? 0 : N * (v0 + 1);
    end = rank == blocks - 1 ? place(V) : N * (v1 + 1);
  }
  __device__ __forceinline__ int place(int j) const { return j - head + N; }
  __device__ __forceinline__ int element(int v) const { return head + v * N; }
  // places of the block's single elements: n_single of them, the i-th is element single(i)
  __device__ __forceinline__ int n_single(int rank, int blocks) const {
    return (rank == 0 ? head : 0) + (rank == blocks - 1 ? V - head - vectors * N : 0);
  }
  __device__ __forceinline__ int single(int i, int rank) const {
    const int h = rank == 0 ? head : 0;
    return i < h ? i : head + vectors * N + i - h;
  }
};

// With a cap |z| <= a = cap log2(e) / T: up to 100, sums of 2^z need no maximum in front (2^a * 2^18 and 2^-a are normal numbers).
static inline bool vocab_bounded(float cap, float temperature) { return cap > 0.f && 1.45 * (double)cap <= 100.0 * (double)temperature; }
// temperatures of the entries that compute in fp32
static inline bool vocab_temperature(float t) { return t >= 1e-4f && t <= 1e6f; }
// what row-wise entries over logits check in common
static inline bool vocab_aligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == XL_F32 ? 3u : 1u)) == 0; }
static inline int vocab_validate(const void* logits, int rows, int V, int64_t row_stride, float cap, int dtype) {
  if (dtype != XL_F32 && dtype != XL_BF16) return XL_ERR_BAD_DTYPE;
  if (rows <= 0 || V <= 0 || !(cap == 0.f || (cap >= 1e-6f && cap <= 1e6f))) return XL_ERR_BAD_SHAPE;
  if (rows > 1 && row_stride < V) return XL_ERR_BAD_STRIDE;
  if (V > VOCAB_MAX) return XL_ERR_TOO_LARGE;
  if (!vocab_aligned(logits, dtype)) return XL_ERR_BAD_ALIGNMENT;   // (whole elements; 16 bytes are not asked for)
  return XL_OK;
}

}  // namespace xl
