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
#include "vocab_select.cuh"

namespace xl {

constexpr int VS_LIST_K = 256, VS_WIDE = 1024, VS_NARROW = 256;
constexpr int VS_BINS = 2048;
constexpr int VS_VALUES = 4096;   // distinct bf16 values of a row that the counts way takes
constexpr double VS_ONE = 17592186044416.0;   // 2^44
typedef unsigned long long u64;

// e^x for x <= 0: 2^n times the Taylor series of 2^f, |f| <= 1/2, to degree 13 (relative error 3e-16)
__device__ __forceinline__ double vs_exp(double x) {
  const double t = fmax(x, -700.0) * 1.4426950408889634, n = rint(t);
  const double f = fma(fmax(x, -700.0), 1.4426950408889634, -n);
  double p = 1.3691488853904128e-12;
  p = fma(p, f, 2.5678435993488206e-11);
  p = fma(p, f, 4.4455382718708116e-10);
  p = fma(p, f, 7.054911620801123e-09);
  p = fma(p, f, 1.01780860092397e-07);
  p = fma(p, f, 1.321548679014431e-06);
  p = fma(p, f, 1.5252733804059841e-05);
  p = fma(p, f, 0.0001540353039338161);
  p = fma(p, f, 0.0013333558146428443);
  p = fma(p, f, 0.009618129107628477);
  p = fma(p, f, 0.05550410866482158);
  p = fma(p, f, 0.24022650695910072);
  p = fma(p, f, 0.6931471805599453);
  p = fma(p, f, 1.0);
  return __hiloint2double(__double2hiint(p) + ((int)n << 20), __double2loint(p));   // (n >= -1010: no subnormal)
}
// 1 / d, 1 <= d <= 2: two Newton steps from the fp32 reciprocal
__device__ __forceinline__ double vs_inverse(double d) {
  double r = (double)__frcp_rn((float)d);
  r = fma(r, fma(-d, r, 1.0), r);
  return fma(r, fma(-d, r, 1.0), r);
}

// what a row's tokens weigh
template <typename T> struct VsWeights {
  double cap, icap, ymax, invT;
  uint32_t kmax;
  __device__ __forceinline__ void set(float cap_, float temperature, float largest) {
    cap = cap_;
    icap = cap_ > 0.f ? 1.0 / (double)cap_ : 0.0;
    invT = 1.0 / (double)temperature;
    kmax = VocabKey<T>::of(from_float<T>(largest));
    ymax = capped(largest);
  }
  __device__ __forceinline__ double capped(float v) const {
    if (!(cap > 0.0)) return v;
    const double e = vs_exp(-2.0 * fabs((double)v) * icap);
    return copysign(cap * (1.0 - e) * vs_inverse(1.0 + e), (double)v);
  }
  __device__ __forceinline__ double of(uint32_t key) const {
    if (key == kmax) return 1.0;
    const float v = VocabKey<T>::value(key);
    if (!(v > -INFINITY) || ymax == INFINITY) return 0.0;   // NaN and -inf; next to +inf
    return vs_exp(fmin((capped(v) - ymax) * invT, 0.0));
  }
  static __device__ __forceinline__ u64 whole(double w) { return __double2ull_rn(w * VS_ONE); }
};

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
  __device__ __forceinline__ double top_p_goal(u64 kept) const { return ceil((double)top_p * (double)kept); }
  // and the one that u asks for
  __device__ __forceinline__ u64 goal(u64 kept) const {
    const double at = (double)u * (double)kept;
    return min(kept, at > 0.0 ? (u64)at + 1ull : 1ull);   // (NaN: the first)
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
struct VsHist {
  unsigned int count[VS_BINS];
  u64 mass[VS_BINS];
};
template <int THREADS> struct VsDigits {
  VsHist top, sub;   // leading 11 bits; the bits of the descent at work
  unsigned int bin, cnt, base_cnt;
  u64 base_mass, bin_mass;
};

template <typename T, int THREADS> struct VsRow {
  VsDigits<THREADS>& s;
  VsScan<THREADS>& scan;
  const T* x;
  int V;
  VsWeights<T> w;

  // one prefix question over a histogram: the bin, from the top, in which the running count (or mass) reaches `goal`
  __device__ void find(const VsHist& h, int bins, bool by_mass, u64 goal, unsigned int base_cnt, u64 base_mass) {
    constexpr int PER = VS_BINS / THREADS;
    const int b0 = bins - 1 - PER * (int)threadIdx.x;
    unsigned int c = 0u, tc;
    u64 m = 0ull, tm;
    for (int i = 0; i < PER; ++i)
      if (b0 - i >= 0) { c += h.count[b0 - i]; m += h.mass[b0 - i]; }
    vs_scan<THREADS>(scan, c, m, &tc, &tm);
    c += base_cnt;
    m += base_mass;
    for (int i = 0; i < PER && b0 - i >= 0; ++i) {
      const unsigned int bc = h.count[b0 - i];
      const u64 bm = h.mass[b0 - i], before = by_mass ? m : c, end = before + (by_mass ? bm : bc);
      if (before < goal && goal <= end) { s.bin = (unsigned int)(b0 - i); s.cnt = bc; s.bin_mass = bm; s.base_cnt = c; s.base_mass = m; }
      c += bc;
      m += bm;
    }
    __syncthreads();
  }

  __device__ __noinline__ void histogram(VsHist& h, int left, int step, uint32_t prefix) {
    const int bins = 1 << step;
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += THREADS) { h.count[b] = 0u; h.mass[b] = 0ull; }
    __syncthreads();
    for (int j = threadIdx.x; j < V; j += THREADS) {
      const uint32_t key = VocabKey<T>::of(x[j]);
      if (left < VocabKey<T>::BITS && key >> left != prefix) continue;
      const uint32_t b = (key >> (left - step)) & (uint32_t)(bins - 1);
      atomicAdd(&h.count[b], 1u);
      const u64 m = VsWeights<T>::whole(w.of(key));
      if (m) atomicAdd(&h.mass[b], m);
    }
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
    const u64 each = s.bin_mass / s.cnt;   // of every token of this key
    VsPlace r;
    r.key = prefix;
    r.rank = by_mass ? (unsigned int)((goal - s.base_mass + each - 1) / each) - 1u : (unsigned int)(goal - s.base_cnt) - 1u;
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
    for (int b = threadIdx.x; b < VS_BINS; b += THREADS) all += s.top.mass[b];
    if (set.min_p > 0.f)
      for (int j = threadIdx.x; j < V; j += THREADS) {
        const double v = w.of(VocabKey<T>::of(x[j]));
        if (v >= (double)set.min_p) over += VsWeights<T>::whole(v);
      }
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
  unsigned int pair[32768];          // counters of the patterns 2 i and 2 i + 1
  unsigned int value[VS_VALUES];     // pattern << 16 | count, in order of descending value
  unsigned int bits, cnt, base_cnt;
  u64 base_mass, each;
};

// The pattern of rank-th value of a block of 64: blocks 511 .. 0 of positive patterns from the top, then 512 .. 1023 of negative ones.
// false: too many values, or a counter ran over (then they do not sum up to V).
template <int THREADS> __device__ bool vs_counts(VsCounts& s, VsScan<THREADS>& scan, const __nv_bfloat16* x, int V, int* values) {
  static_assert(THREADS == 1024, "a block of 64 patterns per thread");
  const int tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < 8192; i += THREADS) reinterpret_cast<uint4*>(s.pair)[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  auto count = [&](uint32_t bits) { atomicAdd(&s.pair[bits >> 1], bits & 1u ? 0x10000u : 1u); };
  const RowSlice<__nv_bfloat16> slice(x, V, 0, 1);
  for_vectors<THREADS>(reinterpret_cast<const uint4*>(x + slice.head), tid, slice.vectors, [&](const uint4& u, int) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { count(w[i] & 0xffffu); count(w[i] >> 16); }
  });
  for (int i = tid; i < slice.n_single(0, 1); i += THREADS) count(__bfloat16_as_ushort(x[slice.single(i, 0)]));
  __syncthreads();
  if (tid == 0) {   // -0 goes with +0
    const unsigned int minus = s.pair[0x4000] & 0xffffu;
    s.pair[0x4000] -= minus;
    s.pair[0] += minus;
  }
  __syncthreads();
  const bool positive = tid < 512;
  const int block = positive ? 511 - tid : tid;   // of 64 patterns
  const unsigned int* words = s.pair + 32 * block;
  const int first_nan = block == 510 || block == 1022 ? 1 : block == 511 || block == 1023 ? 0 : 64;   // (inf is pattern 0 of block 510)
  u64 mask = 0ull;
  unsigned int sum = 0u;
  for (int i = 0; i < 32; ++i) {   // (each lane starts at another word: another bank)
    const int at = (i + lane) & 31;
    const unsigned int w = words[at], lo = w & 0xffffu, hi = w >> 16;
    sum += lo + hi;
    if (2 * at < first_nan && lo) mask |= 1ull << (2 * at);
    if (2 * at + 1 < first_nan && hi) mask |= 2ull << (2 * at);
  }
  unsigned int n = (unsigned int)__popcll(mask), total;
  u64 counted = sum, all;
  vs_scan<THREADS>(scan, n, counted, &total, &all);
  *values = (int)total;
  if (all != (u64)V || total > VS_VALUES) return false;
  for (int i = 0; i < 32; ++i) {
    const int at = (i + lane) & 31;
    const unsigned int w = words[at];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int b = 2 * at + h;
      if (!(mask >> b & 1ull)) continue;
      const unsigned int front = positive ? (unsigned int)__popcll(mask >> b) - 1u : (unsigned int)__popcll(mask & ((1ull << b) - 1ull));
      s.value[n + front] = (uint32_t)(64 * block + b) << 16 | (h ? w >> 16 : w & 0xffffu);
    }
  }
  __syncthreads();
  return true;
}

template <int THREADS>
__device__ VsPlace vs_counted_sample(VsCounts& s, VsScan<THREADS>& scan, const VsWeights<__nv_bfloat16>& w, const VsSettings& set, int values, int V) {
  constexpr int PER = VS_VALUES / THREADS;
  const int tid = threadIdx.x, per = (values + THREADS - 1) / THREADS, i0 = min(values, tid * per);
  auto key_of = [](uint32_t e) { return VocabKey<__nv_bfloat16>::of(__ushort_as_bfloat16((unsigned short)(e >> 16))); };
  u64 each[PER], mass = 0ull, over = 0ull, all, t;
  unsigned int cnt[PER], count = 0u, tc;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    each[i] = 0ull;
    cnt[i] = 0u;
    if (i < per && i0 + i < values) {
      const uint32_t e = s.value[i0 + i];
      const double v = w.of(key_of(e));
      each[i] = VsWeights<__nv_bfloat16>::whole(v);
      cnt[i] = e & 0xffffu;
      mass += each[i] * cnt[i];
      count += cnt[i];
      if (v >= (double)set.min_p) over += each[i] * cnt[i];
    }
  }
  u64 before_m = mass;
  unsigned int before_c = count;
  vs_scan<THREADS>(scan, before_c, before_m, &tc, &all);
  auto find = [&](bool by_mass, u64 goal) {
    u64 m = before_m;
    unsigned int c = before_c;
    const u64 lo = by_mass ? m : c, hi = lo + (by_mass ? mass : count);
    if (lo < goal && goal <= hi) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const u64 bm = each[i] * cnt[i], b = by_mass ? m : c, e = b + (by_mass ? bm : cnt[i]);
        if (b < goal && goal <= e) { s.bits = s.value[i0 + i] >> 16; s.cnt = cnt[i]; s.base_cnt = c; s.base_mass = m; s.each = each[i]; }
        m += bm;
        c += cnt[i];
      }
    }
    __syncthreads();
    VsPlace r;
    r.key = key_of(s.bits << 16);
    r.rank = by_mass ? (unsigned int)((goal - s.base_mass + s.each - 1) / s.each) - 1u : (unsigned int)(goal - s.base_cnt) - 1u;
    r.upto = s.base_mass + (u64)(r.rank + 1u) * s.each;
    __syncthreads();
    return r;
  };
  u64 kept = all;
  if (set.top_k < (int)tc) kept = find(false, (u64)set.top_k).upto;   // (NaN is not counted here: fewer tokens than top_k are all kept)
  const u64 one = (u64)VS_ONE;
  if (set.top_p < 1.f) {
    const double goal = set.top_p_goal(kept);
    kept = goal > 1.0 ? find(true, min((u64)goal, kept)).upto : one;
  }
  if (!(set.min_p <= 0.f)) {
    unsigned int none = 0u;
    vs_scan<THREADS>(scan, none, over, &tc, &t);
    kept = min(kept, t);
  }
  kept = max(one, kept);
  return find(true, set.goal(kept));
}

// index of the token of key `key` that has `rank` others in front of it; every warp takes a stretch of the row
template <typename T, int THREADS> __device__ void vs_locate(unsigned int* wc, const T* x, int V, uint32_t key, unsigned int rank, int64_t* out) {
  constexpr int WARPS = THREADS / 32, N = Vec16<T>::N;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const RowSlice<T> slice(x, V, 0, 1);
  const uint4* xv = reinterpret_cast<const uint4*>(x + slice.head);
  // stretches of whole vectors; the first warp has the elements in front of the vectors, too, the last those behind
  const int per = (slice.vectors + WARPS - 1) / WARPS, v0 = min(slice.vectors, warp * per), v1 = min(slice.vectors, v0 + per);
  const int tail = slice.head + slice.vectors * N;
  auto equals = [&](const uint4& u) {
    const T* e = reinterpret_cast<const T*>(&u);
    unsigned int m = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) m |= (VocabKey<T>::of(e[i]) == key ? 1u : 0u) << i;
    return m;
  };
  unsigned int n = 0u;
  if (warp == 0 && lane < slice.head) n += VocabKey<T>::of(x[lane]) == key;
  if (warp == WARPS - 1 && tail + lane < V) n += VocabKey<T>::of(x[tail + lane]) == key;
  for (int v = v0 + lane; v < v1; v += 32) n += __popc(equals(__ldg(xv + v)));
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if (lane == 0) wc[warp] = n;
  __syncthreads();
  unsigned int before = 0u;
  for (int w = 0; w < warp; ++w) before += wc[w];
  if (rank < before || rank >= before + n) return;
  auto single = [&](int j0, int j1) {
    const bool hit = j0 + lane < j1 && VocabKey<T>::of(x[j0 + lane]) == key;
    const unsigned int mask = __ballot_sync(0xffffffffu, hit);
    if (hit && before + __popc(mask & ((1u << lane) - 1u)) == rank) *out = j0 + lane;
    before += __popc(mask);
  };
  if (warp == 0) single(0, slice.head);
  for (int v = v0; v < v1; v += 32) {
    const unsigned int m = v + lane < v1 ? equals(__ldg(xv + v + lane)) : 0u;
    unsigned int upto = __popc(m);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int c = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += c;
    }
    unsigned int at = before + upto - __popc(m);
    for (unsigned int b = m; b; b &= b - 1u, ++at)
      if (at == rank) *out = slice.element(v + lane) + __ffs(b) - 1;
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (warp == WARPS - 1) single(tail, V);
}

// ---------------------------------------------------------------------------------------------- list
// From the n entries in order (those that can be kept, all of them if fewer than top_k)
template <typename T, int THREADS>
__device__ void vs_listed_sample(VsScan<THREADS>& scan, const u64* list, const VsWeights<T>& w, const VsSettings& set, int n, int64_t* out) {
  constexpr int PER = SEL_CAP / THREADS, SHIFT = 32 - VocabKey<T>::BITS;
  const int tid = threadIdx.x;
  n = min(n, set.top_k);
  const int per = (n + THREADS - 1) / THREADS, i0 = min(n, tid * per);
  u64 each[PER], mass = 0ull, over = 0ull, kept, t;
  unsigned int none = 0u, tc;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    each[i] = 0ull;
    if (i < per && i0 + i < n) {
      const double v = w.of((uint32_t)(list[i0 + i] >> 32) >> SHIFT);
      each[i] = VsWeights<T>::whole(v);
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

template <typename T, int THREADS> __global__ void __launch_bounds__(THREADS) sample_kernel(const xl_sample_params p, const int blocks) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ SelShared<THREADS> ss;
  __shared__ VsScan<THREADS> scan;
  const int rank = blocks > 1 ? (int)cluster_ctarank() : 0;
  const long long row = blockIdx.x / blocks;
  const VsSettings set(p, row);
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  if (!(set.temperature > 0.f)) {
    if (rank == 0) vs_greedy<T, THREADS>(x, p.V, p.cap, p.tokens + row);
    return;
  }
  const bool few = set.top_k <= VS_LIST_K || p.V <= SEL_CAP, alone = !few && set.top_k == p.V && set.top_p >= 1.f && set.min_p > 0.f;
  Selector<T, THREADS> sel(ss, x, p.V, rank, blocks);
  sel.bound(few ? set.top_k : 1);
  const float largest = float_of_key(ss.top);
  if (!(largest > -INFINITY)) {
    if (rank == 0 && threadIdx.x == 0) p.tokens[row] = 0;
    return;
  }
  VsWeights<T> w;
  w.set(p.cap, set.temperature, largest);
  if (few || alone) {
    float least = sel.least();
    if (alone) {   // the smallest key of weight min_p, five bits at a time: every lane asks for one of 32
      uint32_t key = 0u;
      for (int shift = VocabKey<T>::BITS; shift > 0;) {
        const int step = shift < 5 ? shift : 5, lane = threadIdx.x & 31;
        shift -= step;
        const uint32_t mine = key | (uint32_t)lane << shift | ((1u << shift) - 1u);   // the largest key of the lane's stretch
        const bool in = lane >> step == 0 && (mine >= w.kmax || w.of(mine) >= (double)set.min_p);
        const unsigned int some = __ballot_sync(0xffffffffu, in);
        key |= (uint32_t)(some ? __ffs(some) - 1 : 0) << shift;
      }
      least = fminf(VocabKey<T>::value(key), largest);
    }
    sel.collect(least, [](const uint4&, int) {}, [](T) {});
    __syncthreads();
    const unsigned int n = sel.gather();
    if (rank != 0) return;
    if (n <= SEL_CAP && (alone || n >= (unsigned int)set.top_k || ss.bound == 0u)) {
      sort_list<THREADS>(ss.list, (int)n);
      vs_listed_sample<T, THREADS>(scan, ss.list, w, set, (int)n, p.tokens + row);
      return;
    }
  }
  if (rank != 0) return;
  VsPlace place;
  bool found = false;
  if constexpr (vs_counting<T, THREADS>()) {
    VsCounts& s = *reinterpret_cast<VsCounts*>(smem);
    int values;
    if (vs_counts<THREADS>(s, scan, x, p.V, &values)) {
      place = vs_counted_sample<THREADS>(s, scan, w, set, values, p.V);
      found = true;
    }
    __syncthreads();
  }
  if (!found) {
    VsRow<T, THREADS> r = {*reinterpret_cast<VsDigits<THREADS>*>(smem), scan, x, p.V, w};
    place = r.sample(set);
  }
  vs_locate<T, THREADS>(scan.c, x, p.V, place.key, place.rank, p.tokens + row);
}

// Rows whose tokens are surely few take narrow blocks, several of them an SM, and where there are idle SMs a cluster of them;
// all others one wide block each, whose shared memory holds the counts.
template <typename T, int THREADS> static int vs_go(const xl_sample_params* p, int blocks, cudaStream_t st) {
  auto kern = sample_kernel<T, THREADS>;
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
  XL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, *p, blocks));
  return check_launch("xl_softcap_sample");
}

template <typename T> static int vs_launch(const xl_sample_params* p, cudaStream_t st) {
  const bool few = p->V <= SEL_CAP || (!p->top_k_rows && p->top_k > 0 && p->top_k <= VS_LIST_K);
  if (!few) return vs_go<T, VS_WIDE>(p, 1, st);
  int blocks = 1;
  while (blocks < SEL_BLOCKS && p->rows * (blocks * 2) <= 2 * 148 && p->V >= 4096 * (blocks * 2) && p->top_k * blocks * 4 <= SEL_CAP) blocks *= 2;
  return vs_go<T, VS_NARROW>(p, blocks, st);
}

}  // namespace xl

extern "C" int xl_softcap_sample(const xl_sample_params* p, void* cuda_stream) {
  using namespace xl;
  if (!p || !p->logits || !p->tokens || !p->u) return XL_ERR_NULL_POINTER;
  const int rc = vocab_validate(p->rows, p->V, p->row_stride, p->cap, p->dtype);
  if (rc != XL_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  return p->dtype == XL_F32 ? vs_launch<float>(p, st) : vs_launch<__nv_bfloat16>(p, st);
}
