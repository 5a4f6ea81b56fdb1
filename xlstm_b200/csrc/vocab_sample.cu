// Sampling head: one token per row of logits from temperature, top-k, top-p, min-p and a given uniform number.
//
// Mathematics.  With y = cap tanh(x / cap) and w = exp((y - y_max) / T) the tokens stand in the order of descending logit,
// lower index first among equals.  Every filter keeps a prefix of that order, so all that is asked of a row are prefix
// questions -- the mass of the first k tokens, the first token where the running mass reaches top_p of it, and the first
// where it exceeds u times the mass kept -- and none of them needs the row sorted.  Three ways to the answers:
//   list       top_k up to 256, or min_p alone: only the few tokens that can be kept are collected (vocab_select.cuh) and sorted;
//   counts     bf16 logits take few values: a histogram of the 16-bit patterns in shared memory (32 768 pairs of 16-bit counters),
//              its non-empty bins in order of value (some 2 500 of a row of 50 304), one weight each, and one scan of the masses;
//   digits     everything else: count and mass of the leading 11 bits of the keys, then of the next bits inside the bin where a
//              running sum crosses its goal, down to one key, inside which the rank follows by division.
// All three sum the same whole numbers, so a token does not depend on the way taken.
//
// Precision.  The result is a whole number: a running sum that is off by d in relative terms picks another token with a
// probability of up to d times the number of tokens.  Weights are therefore formed in 64 bits and summed as integers in
// units of 2^-44 (rows are at most 2^18 long), which is exact and independent of the order of the atomics.
//
// What bounds it.  Not memory (8 rows of 50 304 in bf16 are 0.1 us, 256 rows 4 us) but the chain of one block, since what a row
// needs next always depends on all of it.  Counts: 16 - 18 us a row, of which 128 KB of counters to clear 1.3, a shared-memory atomic
// per logit 3.4 (random addresses: about 12 lanes a cycle), listing the values 2.7, their weights 2.6, scan and questions 2.5, the
// index of the token 2.1; 256 rows take two rounds on 148 SMs, 29 us.  List: 11 us for 64 rows, k = 50, cut over clusters of four
// blocks whose slices stay in registers.  Digits: a weight in 64 bits per logit and four to six passes, 0.14 ms for rows of 50 304
// in fp32, up to one an SM.  Temperature 0: 21 us for 8 rows, 43 for 256 (the argmax head alone: 6 and 35).
#include "vocab_select.cuh"

namespace xl {

constexpr int VS_LIST_K = 256, VS_WIDE = 1024, VS_NARROW = 256;
constexpr int VS_BINS = 2048;
constexpr int VS_VALUES = 4096;   // distinct bf16 values of a row that the counts way takes
constexpr double VS_ONE = 17592186044416.0;   // 2^44
typedef unsigned long long u64;

// (64-bit conversions go through the slowest unit of the SM: see vocab_row.cuh)
__device__ __forceinline__ u64 vs_whole(double w) {   // rint(w 2^44), 0 <= w <= 1
  return (u64)__double_as_longlong(fma(w, VS_ONE, 4503599627370496.0)) & 0x000fffffffffffffull;
}
__device__ __forceinline__ double vs_number(u64 m) {   // m < 2^63
  return fma((double)(int)(m >> 32), 4294967296.0, (double)(uint32_t)m);
}

// what a row's tokens weigh
struct VsWeights {
  double cap, icap, ymax, invT;
  float largest;
  __device__ __forceinline__ double capped(float v) const {
    if (!(cap > 0.0)) return (double)v;
    const double e = exp64(-2.0 * double_of(fabsf(v)) * icap);
    const double y = cap * (1.0 - e) * inverse64(1.0 + e);
    return v < 0.f ? -y : y;
  }
  __device__ __forceinline__ void set(double cap_, double icap_, double invT_, float largest_) {
    cap = cap_;
    icap = icap_;
    invT = invT_;
    largest = largest_;
  }
  __device__ __forceinline__ void set_max() { ymax = capped(largest); }
  __device__ __forceinline__ double of(float v, double y) const {
    const double w = exp64((y - ymax) * invT);
    return v == largest ? 1.0 : !(v > -INFINITY) || (largest == INFINITY && !(cap > 0.0)) ? 0.0 : w;   // 0: NaN and -inf; next to +inf without a cap
  }
  __device__ __forceinline__ double of(float v) const { return of(v, capped(v)); }
  // several at a time, the largest's cap among them: a 64-bit instruction's result takes some forty cycles
  template <int M> __device__ __forceinline__ void of(const float (&v)[M], double (&out)[M]) {
    double y[M];
    set_max();
#pragma unroll
    for (int i = 0; i < M; ++i) y[i] = capped(v[i]);
#pragma unroll
    for (int i = 0; i < M; ++i) out[i] = of(v[i], y[i]);
  }
  static __device__ __forceinline__ u64 whole(double w) { return vs_whole(w); }
};

// ceil(sum / each), at most 2^18: the fp32 quotient is off by one at most.  (A place that a mass ends in weighs something; the loop
// ends without that, too.)
__device__ __forceinline__ unsigned int vs_steps(u64 sum, u64 each) {
  if (each == 0ull) return 1u;
  unsigned int q = (unsigned int)((float)sum / (float)each);
  while ((u64)q * each < sum) ++q;
  while (q > 0u && (u64)(q - 1u) * each >= sum) --q;
  return q;
}

struct VsPlace {
  uint32_t key;        // key of the token found
  unsigned int rank;   // how many tokens of the same key stand in front of it
  u64 upto;            // running mass, the token included
};

// ---------------------------------------------------------------------------------------------- the settings of a row
struct VsSettings {
  float temperature, top_p, min_p, u;
  int top_k;
  __device__ __forceinline__ VsSettings(const xl_sample_params& p, long long row) {
    temperature = p.temperature_rows ? p.temperature_rows[row] : p.temperature;
    top_k = p.top_k_rows ? p.top_k_rows[row] : p.top_k;
    if (top_k <= 0 || top_k > p.V) top_k = p.V;
    top_p = p.top_p_rows ? p.top_p_rows[row] : p.top_p;
    min_p = p.min_p_rows ? p.min_p_rows[row] : p.min_p;
    u = p.u[row];
  }
  // the running mass that top_p asks for; at most 1 (in units): the first token alone
  __device__ __forceinline__ double top_p_goal(u64 kept) const { return ceil((double)top_p * vs_number(kept)); }
  // and the one that u asks for
  __device__ __forceinline__ u64 goal(u64 kept) const {
    const double at = (double)(u > 0.f ? fminf(u, 1.f) : 0.f) * vs_number(kept);   // (NaN: the first)
    return min(kept, (u64)at + 1ull);
  }
};

// exclusive running sums over a block, and the total
template <int THREADS> struct VsScan {
  unsigned int c[THREADS / 32];
  u64 m[THREADS / 32];
};
template <int THREADS> __device__ void vs_scan(VsScan<THREADS>& s, unsigned int& c, u64& m, unsigned int* total_c, u64* total_m) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned int ic = c;
  u64 im = m;
  __syncwarp();   // (see block_reduce)
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned int oc = __shfl_up_sync(0xffffffffu, ic, o);
    const u64 om = __shfl_up_sync(0xffffffffu, im, o);
    if (lane >= o) { ic += oc; im += om; }
  }
  __syncthreads();
  if (lane == 31) { s.c[warp] = ic; s.m[warp] = im; }
  __syncthreads();
  if (warp == 0) {
    constexpr int W = THREADS / 32;
    const unsigned int c0 = lane < W ? s.c[lane] : 0u;
    const u64 m0 = lane < W ? s.m[lane] : 0ull;
    unsigned int ac = c0;
    u64 am = m0;
#pragma unroll
    for (int o = 1; o < W; o <<= 1) {
      const unsigned int oc = __shfl_up_sync(0xffffffffu, ac, o);
      const u64 om = __shfl_up_sync(0xffffffffu, am, o);
      if (lane >= o) { ac += oc; am += om; }
    }
    if (lane < W) { s.c[lane] = ac; s.m[lane] = am; }   // inclusive over warps
  }
  __syncthreads();
  *total_c = s.c[THREADS / 32 - 1];
  *total_m = s.m[THREADS / 32 - 1];
  c = ic - c + (warp ? s.c[warp - 1] : 0u);
  m = im - m + (warp ? s.m[warp - 1] : 0ull);
}

// ---------------------------------------------------------------------------------------------- digits
struct VsHist {   // masses in two words: 64-bit additions to shared memory would be loops of compare-and-swap
  unsigned int count[VS_BINS], low[VS_BINS], high[VS_BINS];
  __device__ __forceinline__ void clear(int b) { count[b] = low[b] = high[b] = 0u; }
  __device__ __forceinline__ u64 mass(int b) const { return (u64)high[b] << 32 | low[b]; }
  __device__ __forceinline__ void add(int b, u64 m, bool counts) {
    if (counts) atomicAdd(&count[b], 1u);
    const unsigned int lo = (unsigned int)m;
    unsigned int hi = (unsigned int)(m >> 32);
    if (lo && atomicAdd(&low[b], lo) > 0xffffffffu - lo) ++hi;   // (the carry, whatever the order)
    if (hi) atomicAdd(&high[b], hi);
  }
};
template <int THREADS> struct VsDigits {
  VsHist top, sub;   // leading 11 bits; the bits of the descent at work
  unsigned int bin, base_cnt;
  u64 base_mass;
};

template <typename T, int THREADS> struct VsRow {
  VsDigits<THREADS>& s;
  VsScan<THREADS>& scan;
  const T* x;
  int V;
  VsWeights w;
  bool counts;   // whether somebody asks for counts

  // f of every logit of the row
  template <typename F> __device__ __forceinline__ void each(F f) const {
    const RowSlice<T> slice(x, V, 0, 1);
    for_vectors<THREADS, 4>(reinterpret_cast<const uint4*>(x + slice.head), threadIdx.x, slice.vectors, [&](const uint4& u, int) {
#pragma unroll 1
      for (int i = 0; i < Vec16<T>::N; ++i) f(vec_element<T>(u, i));
    });
    for (int i = threadIdx.x; i < slice.n_single(0, 1); i += THREADS) f(x[slice.single(i, 0)]);
  }

  // one prefix question over a histogram: the bin, from the top, in which the running count (or mass) reaches `goal`
  __device__ void find(const VsHist& h, int bins, bool by_mass, u64 goal, unsigned int base_cnt, u64 base_mass) {
    constexpr int PER = VS_BINS / THREADS;
    const int b0 = bins - 1 - PER * (int)threadIdx.x;
    unsigned int c = 0u, tc;
    u64 m = 0ull, tm;
    for (int i = 0; i < PER; ++i)
      if (b0 - i >= 0) { c += h.count[b0 - i]; m += h.mass(b0 - i); }
    vs_scan<THREADS>(scan, c, m, &tc, &tm);
    c += base_cnt;
    m += base_mass;
    for (int i = 0; i < PER && b0 - i >= 0; ++i) {
      const unsigned int bc = h.count[b0 - i];
      const u64 bm = h.mass(b0 - i), before = by_mass ? m : c, end = before + (by_mass ? bm : bc);
      if (before < goal && goal <= end) { s.bin = (unsigned int)(b0 - i); s.base_cnt = c; s.base_mass = m; }
      c += bc;
      m += bm;
    }
    __syncthreads();
  }

  __device__ __noinline__ void histogram(VsHist& h, int left, int step, uint32_t prefix) {
    const int bins = 1 << step;
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += THREADS) h.clear(b);
    __syncthreads();
    each([&](T e) {
      const uint32_t key = VocabKey<T>::of(e);
      if (left < VocabKey<T>::BITS && key >> left != prefix) return;
      const uint32_t b = (key >> (left - step)) & (uint32_t)(bins - 1);
      h.add((int)b, VsWeights::whole(w.of(to_float(e))), counts);
    });
    __syncthreads();
  }

  // first token, in sampling order, whose running count (or mass) reaches `goal`, which the whole row does
  __device__ VsPlace descend(bool by_mass, u64 goal) {
    constexpr int BITS = VocabKey<T>::BITS;
    find(s.top, VS_BINS, by_mass, goal, 0u, 0ull);
    uint32_t prefix = s.bin;
    for (int left = BITS - 11; left > 0;) {
      const int step = left > 11 ? 11 : left;
      const unsigned int base_cnt = s.base_cnt;
      const u64 base_mass = s.base_mass;
      histogram(s.sub, left, step, prefix);
      find(s.sub, 1 << step, by_mass, goal, base_cnt, base_mass);
      prefix = (prefix << step) | s.bin;
      left -= step;
    }
    const u64 each = VsWeights::whole(w.of(VocabKey<T>::value(prefix)));   // of every token of this key
    VsPlace r;
    r.key = prefix;
    r.rank = by_mass ? vs_steps(goal - s.base_mass, each) - 1u : (unsigned int)(goal - s.base_cnt) - 1u;
    r.upto = s.base_mass + (u64)(r.rank + 1u) * each;
    __syncthreads();
    return r;
  }

  __device__ VsPlace sample(const VsSettings& set) {
    constexpr int BITS = VocabKey<T>::BITS;
    histogram(s.top, BITS, 11, 0u);
    // the whole row's mass, and what min_p leaves of it
    u64 all = 0ull, over = 0ull, t;
    unsigned int none = 0u, tc;
    for (int b = threadIdx.x; b < VS_BINS; b += THREADS) all += s.top.mass(b);
    if (set.min_p > 0.f)
      each([&](T e) {
        const double v = w.of(to_float(e));
        if (v >= (double)set.min_p) over += VsWeights::whole(v);
      });
    vs_scan<THREADS>(scan, none, all, &tc, &t);
    u64 kept = t;
    if (set.top_k < V) kept = descend(false, (u64)set.top_k).upto;
    const u64 one = (u64)VS_ONE;
    if (set.top_p < 1.f) {
      const double goal = set.top_p_goal(kept);
      kept = goal > 1.0 ? descend(true, min((u64)goal, kept)).upto : one;
    }
    if (!(set.min_p <= 0.f)) {   // (NaN: nothing but the first token)
      vs_scan<THREADS>(scan, none, over, &tc, &t);
      kept = min(kept, t);
    }
    kept = max(one, kept);
    return descend(true, set.goal(kept));
  }
};

// ---------------------------------------------------------------------------------------------- counts (bf16)
struct VsCounts {
  union {
    unsigned int pair[32768];        // counters of the patterns 2 i and 2 i + 1
    u64 each[VS_VALUES];             // when the values have been listed: the weight of a token of each
  };
  unsigned int value[VS_VALUES];     // pattern << 16 | count, in order of descending value
  unsigned int group[256];           // non-empty bins of 256 patterns each, in that order; then those in front
  unsigned int values, counted;
  int last;                          // values of weight min_p and more
  u64 over;                          // their mass
  VsPlace place;
};

// The row's values in order.  Units of eight patterns (16 bytes) come in the order of descending value: the positive ones
// from the top, then the negative ones; 32 units are a group, and the groups go round the warps, since most of a row's
// values sit side by side.  false: too many values, or a counter ran over 65 535 (then they do not sum up to V).
template <int THREADS> __device__ bool vs_counts(VsCounts& s, const __nv_bfloat16* x, int V) {
  constexpr int WARPS = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // (eight loads a thread are under way while the counters are cleared: the whole of a row of up to 65 536)
  constexpr int BATCH = 8;
  const RowSlice<__nv_bfloat16> slice(x, V, 0, 1);
  const uint4* xv = reinterpret_cast<const uint4*>(x + slice.head);
  uint4 u[BATCH];
  auto load = [&](int v) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (v + i * THREADS < slice.vectors) u[i] = __ldg(xv + v + i * THREADS);
  };
  load(tid);
  for (int i = tid; i < 8192; i += THREADS) reinterpret_cast<uint4*>(s.pair)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) { s.counted = 0u; s.last = 0; }
  __syncthreads();
  auto count = [&](uint32_t bits) { atomicAdd(&s.pair[bits >> 1], bits & 1u ? 0x10000u : 1u); };
#pragma unroll 1
  for (int v = tid; v < slice.vectors;) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (v + i * THREADS < slice.vectors) {
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
        for (int h = 0; h < 4; ++h) { count(w[h] & 0xffffu); count(w[h] >> 16); }
      }
    v += BATCH * THREADS;
    load(v);
  }
  for (int i = tid; i < slice.n_single(0, 1); i += THREADS) count(__bfloat16_as_ushort(x[slice.single(i, 0)]));
  __syncthreads();
  if (tid == 0) {   // -0 goes with +0
    const unsigned int minus = s.pair[0x4000] & 0xffffu;
    s.pair[0x4000] -= minus;
    s.pair[0] += minus;
  }
  __syncthreads();
  const uint4* units = reinterpret_cast<const uint4*>(s.pair);
  auto unit_of = [&](int g) { return g < 128 ? 4095 - (g * 32 + lane) : g * 32 + lane; };
  // a unit's non-empty bins as bits, NaN (patterns above infinity, which starts the units 0xff0 and 0x1ff0) aside
  auto filled = [](const uint4& u, int unit) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    unsigned int m = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= (w[i] & 0xffffu ? 1u : 0u) << (2 * i) | (w[i] >> 16 ? 2u : 0u) << (2 * i);
    const int in_sign = unit & 0xfff;
    return in_sign < 0xff0 ? m : in_sign == 0xff0 ? m & 1u : 0u;
  };
  constexpr int ROUNDS = 256 / WARPS;
  uint4 mine[ROUNDS];   // (a thread's units stay in registers for the second look)
  unsigned int sum = 0u;
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) mine[i] = units[unit_of(i * WARPS + warp)];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const uint4 u = mine[i];
    unsigned int n = 0u;
    __syncwarp();
    if (__any_sync(0xffffffffu, (u.x | u.y | u.z | u.w) != 0u)) {
      n = __reduce_add_sync(0xffffffffu, __popc(filled(u, unit_of(i * WARPS + warp))));
      sum += (u.x & 0xffffu) + (u.x >> 16) + (u.y & 0xffffu) + (u.y >> 16) + (u.z & 0xffffu) + (u.z >> 16) + (u.w & 0xffffu) + (u.w >> 16);
    }
    if (lane == 0) s.group[i * WARPS + warp] = n;
  }
  if (V > 65535) {
    __syncwarp();
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) atomicAdd(&s.counted, sum);
  }
  __syncthreads();
  if (warp == 0) {
    unsigned int c[8], n = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) n += c[i] = s.group[8 * lane + i];
    unsigned int upto = n;
    __syncwarp();
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) s.values = upto;
    upto -= n;
#pragma unroll
    for (int i = 0; i < 8; ++i) { s.group[8 * lane + i] = upto; upto += c[i]; }
  }
  __syncthreads();
  if ((V > 65535 && s.counted != (unsigned int)V) || s.values > VS_VALUES) return false;
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int g = i * WARPS + warp, unit = unit_of(g);
    const uint4 u = mine[i];
    __syncwarp();
    if (!__any_sync(0xffffffffu, (u.x | u.y | u.z | u.w) != 0u)) continue;
    const unsigned int m = filled(u, unit), n = __popc(m);
    unsigned int upto = n;
    __syncwarp();
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    unsigned int* out = s.value + s.group[g] + upto - n;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int b = 0; b < 8; ++b)
      if (m >> b & 1u) {
        const unsigned int front = g < 128 ? __popc(m >> b) - 1u : __popc(m & ((1u << b) - 1u));
        out[front] = (uint32_t)(8 * unit + b) << 16 | (w[b >> 1] >> (16 * (b & 1)) & 0xffffu);
      }
  }
  __syncthreads();
  return true;
}

// The weights by all threads; the scan and the questions by the first 256 only: shuffles and barriers of 32 warps take longer than
// a few more additions a thread (8 rows: 17.4 us with 256, 18.0 with 512, 20.5 with 1024).
constexpr int VS_FIRST = 256;
__device__ __forceinline__ void vs_first_barrier() {
  __syncwarp();   // (whole warps arrive)
  asm volatile("bar.sync 1, %0;" ::"n"(VS_FIRST) : "memory");
}

template <int THREADS>
__device__ VsPlace vs_counted_sample(VsCounts& s, VsScan<THREADS>& scan, VsWeights& w, const VsSettings& set, int V) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, values = (int)s.values;
  int last = 0;   // values of weight min_p and more
#pragma unroll 1
  for (int i = tid; i < values; i += 3 * THREADS) {
    uint32_t e[3];
    float x[3];
    double v[3];
#pragma unroll
    for (int h = 0; h < 3; ++h) { e[h] = s.value[min(i + h * THREADS, values - 1)]; x[h] = __uint_as_float(e[h] & 0xffff0000u); }
    w.of(x, v);
#pragma unroll
    for (int h = 0; h < 3; ++h)
      if (i + h * THREADS < values) {
        s.each[i + h * THREADS] = VsWeights::whole(v[h]);
        if (v[h] >= (double)set.min_p) last = i + h * THREADS + 1;
      }
  }
  if (set.min_p > 0.f) {
    __syncwarp();
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0 && last) atomicMax(&s.last, last);
  }
  __syncthreads();
  if (tid < VS_FIRST) {
    const int per = (values + VS_FIRST - 1) / VS_FIRST, i0 = min(values, tid * per), i1 = min(values, i0 + per);
    u64 mass = 0ull, over = 0ull;
    unsigned int count = 0u;
#pragma unroll 4
    for (int i = i0; i < i1; ++i) {
      const unsigned int c = s.value[i] & 0xffffu;
      mass += s.each[i] * c;
      count += c;
      if (i < s.last) over = mass;
    }
    // masses and counts in front of this thread's values, and their sums
    u64 before_m = mass;
    unsigned int before_c = count;
    __syncwarp();
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 om = __shfl_up_sync(0xffffffffu, before_m, o);
      const unsigned int oc = __shfl_up_sync(0xffffffffu, before_c, o);
      if (lane >= o) { before_m += om; before_c += oc; }
    }
    if (lane == 31) { scan.m[warp] = before_m; scan.c[warp] = before_c; }
    vs_first_barrier();
    u64 all = 0ull;
    unsigned int tc = 0u;
    before_m -= mass;
    before_c -= count;
#pragma unroll
    for (int i = 0; i < VS_FIRST / 32; ++i) {
      if (i < warp) { before_m += scan.m[i]; before_c += scan.c[i]; }
      all += scan.m[i];
      tc += scan.c[i];
    }
    if (set.min_p > 0.f && i0 < s.last && s.last <= i1) s.over = before_m + over;
    // one prefix question; the thread that has the place works it out
    auto find = [&](bool by_mass, u64 goal) {
      const u64 lo = by_mass ? before_m : before_c, hi = lo + (by_mass ? mass : count);
      if (lo < goal && goal <= hi) {
        u64 m = before_m;
        unsigned int c = before_c;
#pragma unroll 2
        for (int i = i0;; ++i) {
          const unsigned int bc = s.value[i] & 0xffffu;
          const u64 each = s.each[i], bm = each * bc;
          if (goal <= (by_mass ? m + bm : (u64)(c + bc))) {
            s.place.key = VocabKey<__nv_bfloat16>::of(__ushort_as_bfloat16((unsigned short)(s.value[i] >> 16)));
            s.place.rank = by_mass ? vs_steps(goal - m, each) - 1u : (unsigned int)(goal - c) - 1u;
            s.place.upto = m + (u64)(s.place.rank + 1u) * each;
            break;
          }
          m += bm;
          c += bc;
        }
      }
      vs_first_barrier();
      const u64 upto = s.place.upto;
      vs_first_barrier();
      return upto;
    };
    u64 kept = all;
    if (set.top_k < V && set.top_k < (int)tc) kept = find(false, (u64)set.top_k);   // (NaN is not counted here: fewer tokens than top_k are all kept)
    const u64 one = (u64)VS_ONE;
    if (set.top_p < 1.f) {
      const double goal = set.top_p_goal(kept);
      kept = goal > 1.0 ? find(true, min((u64)goal, kept)) : one;
    }
    if (set.min_p > 0.f) {
      vs_first_barrier();   // (s.over)
      kept = min(kept, s.last ? s.over : 0ull);
    } else if (!(set.min_p <= 0.f)) {
      kept = 0ull;   // (NaN: nothing but the first token)
    }
    find(true, set.goal(max(one, kept)));
  }
  __syncthreads();
  return s.place;
}

// places of a vector's elements that equal v, as bits (-0 equals +0)
template <typename T> __device__ __forceinline__ unsigned int vs_equal(const uint4& u, T v);
template <> __device__ __forceinline__ unsigned int vs_equal<__nv_bfloat16>(const uint4& u, __nv_bfloat16 v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 two = __halves2bfloat162(v, v);
  unsigned int m = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) m |= (__heq2_mask(h[i], two) & 0x00020001u) << (2 * i);   // bits 2 i and 2 i + 17
  return (m | m >> 16) & 0xffu;
}
template <> __device__ __forceinline__ unsigned int vs_equal<float>(const uint4& u, float v) {
  return (__uint_as_float(u.x) == v ? 1u : 0u) | (__uint_as_float(u.y) == v ? 2u : 0u) | (__uint_as_float(u.z) == v ? 4u : 0u) | (__uint_as_float(u.w) == v ? 8u : 0u);
}

// index of the token of key `key` (a number's) that has `rank` others in front of it; every warp takes a stretch of the row
template <typename T, int THREADS> __device__ void vs_locate(unsigned int* wc, const T* x, int V, uint32_t key, unsigned int rank, int64_t* out) {
  constexpr int WARPS = THREADS / 32, KEEP = 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T value = from_float<T>(VocabKey<T>::value(key));
  const float number = to_float(value);
  const RowSlice<T> slice(x, V, 0, 1);
  const uint4* xv = reinterpret_cast<const uint4*>(x + slice.head);
  // stretches of whole vectors; the first warp has the elements in front of the vectors, too, the last those behind
  const int per = (slice.vectors + WARPS - 1) / WARPS, v0 = min(slice.vectors, warp * per), v1 = min(slice.vectors, v0 + per);
  const int tail = slice.element(slice.vectors);
  unsigned int n = 0u, kept[KEEP];   // the first eight rounds' places stay in registers (rows up to 65 536 bf16)
  if (warp == 0 && lane < slice.head) n += to_float(x[lane]) == number;
  if (warp == WARPS - 1 && tail + lane < V) n += to_float(x[tail + lane]) == number;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int v = v0 + 32 * i + lane;
    kept[i] = v < v1 ? vs_equal<T>(__ldg(xv + v), value) : 0u;
    n += __popc(kept[i]);
  }
  for (int v = v0 + 32 * KEEP + lane; v < v1; v += 32) n += __popc(vs_equal<T>(__ldg(xv + v), value));
  __syncwarp();
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if (lane == 0) wc[warp] = n;
  __syncthreads();
  unsigned int before = __reduce_add_sync(0xffffffffu, lane < warp ? wc[lane] : 0u);
  if (rank < before || rank >= before + n) return;
  auto single = [&](int j0, int j1) {
    const bool hit = j0 + lane < j1 && to_float(x[j0 + lane]) == number;
    const unsigned int mask = __ballot_sync(0xffffffffu, hit);
    if (hit && before + __popc(mask & ((1u << lane) - 1u)) == rank) *out = j0 + lane;
    before += __popc(mask);
  };
  // the round of 32 vectors that has the token, from the counts of all at once
  auto inside = [&](unsigned int m, int v) {
    unsigned int upto = __popc(m);
    __syncwarp();
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int c = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += c;
    }
    unsigned int at = before + upto - __popc(m);
    for (unsigned int b = m; b; b &= b - 1u, ++at)
      if (at == rank) *out = slice.element(v + lane) + __ffs(b) - 1;
  };
  if (warp == 0) single(0, slice.head);
  if (rank < before) return;
  unsigned int sums[KEEP];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < KEEP; ++i) sums[i] = __reduce_add_sync(0xffffffffu, __popc(kept[i]));
  unsigned int m = 0u;
  int at = -1;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    if (at < 0 && rank < before + sums[i]) { at = i; m = kept[i]; }
    if (at < 0) before += sums[i];
  }
  if (at >= 0) { inside(m, v0 + 32 * at); return; }
  for (int v = v0 + 32 * KEEP; v < v1; v += 32) {
    m = v + lane < v1 ? vs_equal<T>(__ldg(xv + v + lane), value) : 0u;
    const unsigned int sum = __reduce_add_sync(0xffffffffu, __popc(m));
    if (rank < before + sum) { inside(m, v); return; }
    before += sum;
  }
  if (warp == WARPS - 1) single(tail, V);
}

// ---------------------------------------------------------------------------------------------- list
// From the n entries in order (those that can be kept, all of them if fewer than top_k)
template <typename T, int THREADS>
__device__ void vs_listed_sample(VsScan<THREADS>& scan, const u64* list, const VsWeights& w, const VsSettings& set, int n, int64_t* out) {
  constexpr int PER = SEL_CAP / THREADS;
  const int tid = threadIdx.x;
  n = min(n, set.top_k);
  const int per = (n + THREADS - 1) / THREADS, i0 = min(n, tid * per);
  u64 each[PER], mass = 0ull, over = 0ull, kept, t;
  unsigned int none = 0u, tc;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    each[i] = 0ull;
    if (i < per && i0 + i < n) {
      const double v = w.of(list_value<T>(list[i0 + i]));
      each[i] = VsWeights::whole(v);
      if (v >= (double)set.min_p) over += each[i];
      mass += each[i];
    }
  }
  u64 before = mass;
  vs_scan<THREADS>(scan, none, before, &tc, &kept);
  const u64 one = (u64)VS_ONE;
  __shared__ u64 reached;
  // the first entry whose running mass reaches `goal`; `then` takes its place and running mass
  auto find = [&](u64 goal, auto then) {
    if (before < goal && goal <= before + mass) {
      u64 m = before;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (m < goal && goal <= m + each[i]) then(i0 + i, m + each[i]);
        m += each[i];
      }
    }
  };
  if (set.top_p < 1.f) {
    const double goal = set.top_p_goal(kept);
    if (goal > 1.0) {
      find(min((u64)goal, kept), [&](int, u64 upto) { reached = upto; });
      __syncthreads();
      kept = reached;
    } else {
      kept = one;
    }
  }
  if (!(set.min_p <= 0.f)) {
    vs_scan<THREADS>(scan, none, over, &tc, &t);
    kept = min(kept, t);
  }
  kept = max(one, kept);
  find(set.goal(kept), [&](int i, u64) { *out = (int64_t)(uint32_t)~(uint32_t)list[i]; });
}

// ---------------------------------------------------------------------------------------------- greedy rows
// the token of xl_softcap_argmax
template <typename T, int THREADS> __device__ void vs_greedy(const T* x, int V, float cap, int64_t* out) {
  __shared__ float fv[THREADS / 32];
  __shared__ int iv[THREADS / 32];
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  for (int j = threadIdx.x; j < V; j += THREADS) {
    const float y = cap > 0.f ? capped_rounded<T>(x[j], cap) : to_float(x[j]);
    if (y > bv || (y == bv && j < bi)) { bv = y; bi = j; }
  }
  __syncwarp();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
  }
  if ((threadIdx.x & 31) == 0) { fv[threadIdx.x >> 5] = bv; iv[threadIdx.x >> 5] = bi; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < THREADS / 32; ++w)
      if (fv[w] > bv || (fv[w] == bv && iv[w] < bi)) { bv = fv[w]; bi = iv[w]; }
    *out = bi == 0x7fffffff ? 0 : bi;
  }
}

// ---------------------------------------------------------------------------------------------- the kernel
template <typename T, int THREADS> __host__ __device__ constexpr bool vs_counting() { return THREADS == VS_WIDE && VocabKey<T>::BITS == 16; }
template <typename T, int THREADS> constexpr size_t vs_smem() {
  return vs_counting<T, THREADS>() && sizeof(VsCounts) > sizeof(VsDigits<THREADS>) ? sizeof(VsCounts) : sizeof(VsDigits<THREADS>);
}

template <typename T, int THREADS, int KEEP> __global__ void __launch_bounds__(THREADS) sample_kernel(const xl_sample_params p, const double icap, const int blocks) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ SelShared<THREADS> ss;
  __shared__ VsScan<THREADS> scan;
  __shared__ double invT;   // a 64-bit division: by one thread, and out of the way early
  const int rank = blocks > 1 ? (int)cluster_ctarank() : 0;
  const long long row = blockIdx.x / blocks;
  const VsSettings set(p, row);
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  if (threadIdx.x == 0) invT = 1.0 / (double)set.temperature;   // (read behind the first barrier)
  if (!(set.temperature > 0.f)) {
    if (rank == 0) vs_greedy<T, THREADS>(x, p.V, p.cap, p.tokens + row);
    return;
  }
  const bool few = set.top_k <= VS_LIST_K || p.V <= SEL_CAP, alone = !few && set.top_k == p.V && set.top_p >= 1.f && set.min_p > 0.f;
  VsWeights w;
  auto weigh = [&](float largest) {
    w.set(p.cap, icap, invT, largest);
    w.set_max();
  };
  VsPlace place;
  bool found = false;
  if (few || alone || !vs_counting<T, THREADS>()) {
    Selector<T, THREADS, KEEP> sel(ss, x, p.V, rank, blocks);
    sel.bound(few ? set.top_k : 1);
    const float largest = float_of_key(ss.top);
    if (!(largest > -INFINITY)) {
      if (rank == 0 && threadIdx.x == 0) p.tokens[row] = 0;
      return;
    }
    weigh(largest);
    if (few || alone) {
      float least = sel.least();
      bool whole = ss.bound == 0u;   // the list has every token that can be chosen
      if (!(least > -INFINITY)) {    // (fewer than top_k are not masked: those)
        whole = true;
        least = VocabKey<T>::BITS == 16 ? -3.3895314e38f : -3.4028235e38f;
      }
      if (alone) {   // the smallest key of weight min_p, five bits at a time: every lane asks for one of 32
        uint32_t key = 0u;
        const uint32_t kmax = VocabKey<T>::of(from_float<T>(largest));
        for (int shift = VocabKey<T>::BITS; shift > 0;) {
          const int step = shift < 5 ? shift : 5, lane = threadIdx.x & 31;
          shift -= step;
          const uint32_t mine = key | (uint32_t)lane << shift | ((1u << shift) - 1u);   // the largest key of the lane's stretch
          __syncwarp();
          const bool in = lane >> step == 0 && (mine >= kmax || w.of(VocabKey<T>::value(mine)) >= (double)set.min_p);
          const unsigned int some = __ballot_sync(0xffffffffu, in);
          key |= (uint32_t)(some ? __ffs(some) - 1 : 0) << shift;
        }
        least = fminf(VocabKey<T>::value(key), largest);
      }
      sel.collect(least, [](const uint4&, int) {}, [](T) {});
      const unsigned int n = sel.gather();
      if (rank != 0) return;
      if (n <= SEL_CAP && (alone || whole || n >= (unsigned int)set.top_k)) {
        sort_list<THREADS>(ss.list, (int)n);
        vs_listed_sample<T, THREADS>(scan, ss.list, w, set, (int)n, p.tokens + row);
        return;
      }
    }
  }
  if constexpr (vs_counting<T, THREADS>()) {
    VsCounts& s = *reinterpret_cast<VsCounts*>(smem);
    if (vs_counts<THREADS>(s, x, p.V)) {
      const float largest = s.values ? __bfloat162float(__ushort_as_bfloat16((unsigned short)(s.value[0] >> 16))) : -INFINITY;
      if (!(largest > -INFINITY)) {
        if (threadIdx.x == 0) p.tokens[row] = 0;
        return;
      }
      w.set(p.cap, icap, invT, largest);
      place = vs_counted_sample<THREADS>(s, scan, w, set, p.V);
      found = true;
    } else if (!few && !alone) {   // (the digits need the largest logit)
      Selector<T, THREADS, 0> sel(ss, x, p.V, 0, 1);
      sel.bound(1);
      const float largest = float_of_key(ss.top);
      if (!(largest > -INFINITY)) {
        if (threadIdx.x == 0) p.tokens[row] = 0;
        return;
      }
      weigh(largest);
    }
    __syncthreads();
  }
  if (!found) {
    VsRow<T, THREADS> r = {*reinterpret_cast<VsDigits<THREADS>*>(smem), scan, x, p.V, w, set.top_k < p.V};
    place = r.sample(set);
  }
  vs_locate<T, THREADS>(scan.c, x, p.V, place.key, place.rank, p.tokens + row);
}

// Rows whose tokens are surely few take narrow blocks, several of them an SM, and where there are idle SMs a cluster of them;
// all others one wide block each, whose shared memory holds the counts.
template <typename T, int THREADS, int KEEP> static int vs_go(const xl_sample_params* p, int blocks, cudaStream_t st) {
  auto kern = sample_kernel<T, THREADS, KEEP>;
  const size_t smem = vs_smem<T, THREADS>();
  XL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p->rows * blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  XL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, *p, p->cap > 0.f ? 1.0 / (double)p->cap : 0.0, blocks));
  return check_launch("xl_softcap_sample");
}

template <typename T> static int vs_launch(const xl_sample_params* p, cudaStream_t st) {
  const bool few = p->V <= SEL_CAP || (!p->top_k_rows && p->top_k > 0 && p->top_k <= VS_LIST_K);
  if (!few) return vs_go<T, VS_WIDE, 0>(p, 1, st);
  int blocks = 1;
  while (blocks < SEL_BLOCKS && p->rows * (blocks * 2) <= 2 * 148 && p->V >= 2048 * (blocks * 2) && p->top_k * 3 <= SEL_CAP) blocks *= 2;
  const int vectors = p->V / Vec16<T>::N;
  if ((vectors + blocks - 1) / blocks <= 8 * VS_NARROW) return vs_go<T, VS_NARROW, 8>(p, blocks, st);
  return vs_go<T, VS_NARROW, 0>(p, blocks, st);
}

}  // namespace xl

extern "C" int xl_softcap_sample(const xl_sample_params* p, void* cuda_stream) {
  using namespace xl;
  if (!p || !p->logits || !p->tokens || !p->u) return XL_ERR_NULL_POINTER;
  const int rc = vocab_validate(p->logits, p->rows, p->V, p->row_stride, p->cap, p->dtype);
  if (rc != XL_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  return p->dtype == XL_F32 ? vs_launch<float>(p, st) : vs_launch<__nv_bfloat16>(p, st);
}
