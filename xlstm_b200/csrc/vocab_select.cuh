// The largest logits of a row, sorted, without sorting the row.
//
// Mathematics.  The row falls into G groups of places (a thread's vectors, or the even and the odd places of them apart).  If the
// k-th largest of the group maxima is t, at least k logits are >= t: t bounds the k-th largest logit from below, and only about
// -G ln(1 - k/G) logits reach it (74 for k = 64, G = 256).  So a first pass takes maxima, one warp finds t by bisection over the
// leading 16 bits of the keys -- the whole block waits for its rounds, hence no more groups than k needs --, a second pass
// collects what reaches t into a list, and only the list is sorted, by (key, lower index).  Rows where too many logits reach t (crowds of equal ones, or all large logits in few
// groups) are told by the length of the list, and left to the caller's exact selection.
//
// A row may be cut over a cluster of b blocks: where every slice has k / b group maxima >= t the row has k, so the smallest of the
// slices' (k / b)-th largest holds; all blocks write to the list of block 0 through the cluster's shared memory.
#pragma once

#include "vocab_row.cuh"

namespace xl {

constexpr int SEL_CAP = 1024;      // entries of the list
constexpr int SEL_BLOCKS = 8;
constexpr int SEL_GROUPS = 512;    // at most; as few of 64, 128, 256, 512 as 3/8 of them are k

__device__ __forceinline__ uint32_t add_cluster_u32(uint32_t addr, uint32_t v) {
  uint32_t old;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
  return old;
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

template <int THREADS> struct SelShared {
  static constexpr int GROUPS = 2 * THREADS < SEL_GROUPS ? 2 * THREADS : SEL_GROUPS;
  unsigned long long list[SEL_CAP];     // key (32 bits) and ~index
  unsigned short group[GROUPS];         // leading 16 bits of the groups' largest keys
  unsigned int from[2][SEL_BLOCKS];     // of the row's blocks: bound, largest key; written once a launch
  unsigned int largest[THREADS / 32];
  unsigned int n, mine;                 // entries that reached the bound, also those beyond the list: of the row (block 0's), of the slice
  unsigned int bound, top;              // leading 16 bits of the bound's key; key of the largest logit
};

template <typename T> __device__ __forceinline__ uint32_t list_key(T x) { return VocabKey<T>::of(x) << (32 - VocabKey<T>::BITS); }
template <typename T> __device__ __forceinline__ float list_value(unsigned long long e) { return VocabKey<T>::value((uint32_t)(e >> 32) >> (32 - VocabKey<T>::BITS)); }

// running maxima of the even and odd places of a thread's vectors; NaN does not count
template <typename T> struct GroupMax;
template <> struct GroupMax<__nv_bfloat16> {
  __nv_bfloat162 m;
  __device__ __forceinline__ GroupMax() : m(__float2bfloat162_rn(-INFINITY)) {}
  __device__ __forceinline__ void add(const uint4& u) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    m = __hmax2(m, __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  }
  __device__ __forceinline__ void add_one(__nv_bfloat16 x) { m = __hmax2(m, __halves2bfloat162(x, __float2bfloat16(-INFINITY))); }
  __device__ __forceinline__ float even() const { return __low2float(m); }
  __device__ __forceinline__ float odd() const { return __high2float(m); }
};
template <> struct GroupMax<float> {
  float a, b;
  __device__ __forceinline__ GroupMax() : a(-INFINITY), b(-INFINITY) {}
  __device__ __forceinline__ void add(const uint4& u) {
    a = fmaxf(a, fmaxf(__uint_as_float(u.x), __uint_as_float(u.z)));
    b = fmaxf(b, fmaxf(__uint_as_float(u.y), __uint_as_float(u.w)));
  }
  __device__ __forceinline__ void add_one(float x) { a = fmaxf(a, x); }
  __device__ __forceinline__ float even() const { return a; }
  __device__ __forceinline__ float odd() const { return b; }
};

// places of a vector's elements that are >= v, as bits
template <typename T> __device__ __forceinline__ unsigned int vec_reach(const uint4& u, float v);
template <> __device__ __forceinline__ unsigned int vec_reach<__nv_bfloat16>(const uint4& u, float v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 two = __float2bfloat162_rn(v);   // (a bf16 number, or -inf)
  unsigned int m = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) m |= (__hge2_mask(h[i], two) & 0x00020001u) << (2 * i);   // bits 2 i and 2 i + 17
  return (m | m >> 16) & 0xffu;
}
template <> __device__ __forceinline__ unsigned int vec_reach<float>(const uint4& u, float v) {
  return (__uint_as_float(u.x) >= v ? 1u : 0u) | (__uint_as_float(u.y) >= v ? 2u : 0u) | (__uint_as_float(u.z) >= v ? 4u : 0u) | (__uint_as_float(u.w) >= v ? 8u : 0u);
}
// whether one is (or is NaN)
template <typename T> __device__ __forceinline__ bool vec_any(const uint4& u, float v);
template <> __device__ __forceinline__ bool vec_any<__nv_bfloat16>(const uint4& u, float v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  return !__hblt2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])), __float2bfloat162_rn(v));
}
template <> __device__ __forceinline__ bool vec_any<float>(const uint4& u, float v) {
  return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w))) >= v;
}
template <typename T> __device__ __forceinline__ T vec_element(const uint4& u, int i);   // (selects: the vector stays in registers)
template <> __device__ __forceinline__ __nv_bfloat16 vec_element<__nv_bfloat16>(const uint4& u, int i) {
  const uint32_t w = i < 4 ? (i < 2 ? u.x : u.y) : (i < 6 ? u.z : u.w);
  return __ushort_as_bfloat16((unsigned short)(i & 1 ? w >> 16 : w & 0xffffu));
}
template <> __device__ __forceinline__ float vec_element<float>(const uint4& u, int i) {
  return __uint_as_float(i < 2 ? (i == 0 ? u.x : u.y) : (i == 2 ? u.z : u.w));
}

// f(vector, its number) for v, v + STEP, .. below end, BATCH loads under way at a time
template <int STEP, int BATCH, typename F> __device__ __forceinline__ void for_vectors(const uint4* xv, int v, int end, F f) {
  const int over = 31 - (int)(threadIdx.x & 31) + (BATCH - 1) * STEP;   // of the warp's last lane in the batch's last round
#pragma unroll 1
  for (; v + over < end; v += BATCH * STEP) {   // (all lanes together: f may part them)
    uint4 u[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) u[i] = __ldg(xv + v + i * STEP);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      f(u[i], v + i * STEP);
      __syncwarp();
    }
  }
#pragma unroll 1
  for (; v < end; v += STEP) f(__ldg(xv + v), v);
}

// a warp's 32 values in descending order over its lanes
template <typename V> __device__ __forceinline__ V run_sorted(V e) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int len = 2; len <= 32; len <<= 1)
#pragma unroll
    for (int step = len >> 1; step > 0; step >>= 1) {
      const V o = __shfl_xor_sync(0xffffffffu, e, step);
      const bool larger = ((lane & len) == 0) == ((lane & step) == 0);   // whether this lane keeps the larger one
      e = (e > o) == larger ? e : o;
    }
  return e;
}
// how many values of the sorted runs but run `own` are larger than e
template <typename V> __device__ __forceinline__ int above_in_runs(const V* list, int runs, int own, V e) {
  int above = 0;
#pragma unroll 4
  for (int q = 0; q < runs; ++q) {
    const V* run = list + 32 * q;
    int c = 0;
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) c += run[c + step - 1] > e ? step : 0;
    c += run[c] > e ? 1 : 0;   // (32 if all are larger)
    above += q == own ? 0 : c;
  }
  return above;
}

// KEEP: the slice has at most KEEP vectors a thread, which stay in registers between the passes; 0: it is read twice
template <typename T, int THREADS, int KEEP> struct Selector {
  static constexpr int N = Vec16<T>::N, GROUPS = SelShared<THREADS>::GROUPS;
  SelShared<THREADS>& s;
  const T* x;
  RowSlice<T> slice;
  int rank, blocks, singles;
  const uint4* xv;
  uint4 kept[KEEP ? KEEP : 1];

  __device__ __forceinline__ Selector(SelShared<THREADS>& s_, const T* x_, int V, int rank_, int blocks_)
      : s(s_), x(x_), slice(x_, V, rank_, blocks_), rank(rank_), blocks(blocks_) {
    xv = reinterpret_cast<const uint4*>(x + slice.head);
    singles = slice.n_single(rank, blocks);
  }

  // First pass: s.bound (a lower bound of the k-th largest) and s.top (the largest, NaN aside), both of the whole row.  Ends behind a
  // barrier.
  __device__ void bound(int k) {
    const int tid = threadIdx.x, lane = tid & 31;
    __syncwarp();
    if (blocks > 1) cluster_arrive();
    GroupMax<T> g;
    if (KEEP) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (slice.v0 + tid + i * THREADS < slice.v1) kept[i] = __ldg(xv + slice.v0 + tid + i * THREADS);
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (slice.v0 + tid + i * THREADS < slice.v1) g.add(kept[i]);
    } else {
      for_vectors<THREADS, 8>(xv, slice.v0 + tid, slice.v1, [&](const uint4& u, int) { g.add(u); });
    }
    for (int i = tid; i < singles; i += THREADS) g.add_one(x[slice.single(i, rank)]);
    // the groups' largest keys: of a thread's even and odd places, of both, of two or more threads together
    k = (k + blocks - 1) / blocks;
    int groups = 64;
    while (groups < GROUPS && 8 * k > 3 * groups) groups *= 2;
    uint32_t ge = key_of_float(g.even()) >> 16, go = key_of_float(g.odd()) >> 16;
    const bool both = groups < 2 * THREADS;
    if (both) ge = max(ge, go);
    const int share = both ? THREADS / groups : 1;   // threads of a group
    __syncwarp();
    for (int o = 1; o < share; o <<= 1) ge = max(ge, __shfl_xor_sync(0xffffffffu, ge, o));
    if (k > 1 && tid % share == 0) {
      s.group[tid / share] = (unsigned short)ge;
      if (!both) s.group[THREADS + tid] = (unsigned short)go;
    }
    __syncwarp();
    const uint32_t mine = __reduce_max_sync(0xffffffffu, key_of_float(fmaxf(g.even(), g.odd())));
    if (lane == 0) s.largest[tid >> 5] = mine;
    if (tid == 0) s.n = s.mine = 0u;
    __syncthreads();
    if (tid < 32) {
      const uint32_t* two = reinterpret_cast<const uint32_t*>(s.group);
      const uint32_t top = __reduce_max_sync(0xffffffffu, lane < THREADS / 32 ? s.largest[lane] : 0u);
      uint32_t t = top >> 16;
      if (k > groups) t = 0u;
      else if (k > 1) t = groups == 64 ? bisect<1>(two, k) : groups == 128 ? bisect<2>(two, k) : groups == 256 ? bisect<4>(two, k) : bisect<GROUPS / 64>(two, k);
      if (blocks > 1) {
        __syncwarp();
        cluster_wait();
        if (lane < blocks) {
          st_cluster_u32(mapa_u32(smem_u32(&s.from[0][rank]), lane), t);
          st_cluster_u32(mapa_u32(smem_u32(&s.from[1][rank]), lane), top);
        }
      } else if (lane == 0) {
        s.bound = t;
        s.top = top;
      }
    }
    if (blocks > 1) {
      if (tid >= 32) cluster_wait();
      __syncwarp();
      cluster_sync_all();
      if (tid == 0) {
        uint32_t t = 0xffffu, top = 0u;
        for (int r = 0; r < blocks; ++r) { t = min(t, s.from[0][r]); top = max(top, s.from[1][r]); }
        s.bound = t;
        s.top = top;
      }
    }
    __syncthreads();
  }

  // the k-th largest of 64 PAIRS >= k keys, by one warp: bit by bit below the bits that all share
  template <int PAIRS> static __device__ __forceinline__ uint32_t bisect(const uint32_t* two, int k) {
    const int lane = threadIdx.x & 31;
    uint32_t key[2 * PAIRS], lo = 0xffffu, hi = 0u;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const uint32_t w = two[i * 32 + lane];
      key[2 * i] = w >> 16;
      key[2 * i + 1] = w & 0xffffu;
      lo = min(lo, min(key[2 * i], key[2 * i + 1]));
      hi = max(hi, max(key[2 * i], key[2 * i + 1]));
    }
    __syncwarp();
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    uint32_t bit = lo == hi ? 0u : 0x80000000u >> __clz(lo ^ hi), t = bit ? hi & ~(2u * bit - 1u) : hi;
#pragma unroll 1
    for (; bit; bit >>= 1) {
      const uint32_t c = t | bit;
      int n = 0;
#pragma unroll
      for (int i = 0; i < 2 * PAIRS; ++i) n += key[i] >= c;
      if (__reduce_add_sync(0xffffffffu, n) >= k) t = c;
    }
    return t;
  }

  // the bound as a number; -inf where there are too few groups for one
  __device__ __forceinline__ float least() const {
    return s.bound == 0u ? -INFINITY : VocabKey<T>::value(s.bound << (VocabKey<T>::BITS - 16));
  }

  // Second pass over the slice: what reaches `least` into block 0's list; `also(vector, number)` and `also_one(element)` see
  // everything.
  template <typename F, typename G> __device__ void collect(float least, F also, G also_one) {
    const int tid = threadIdx.x;
    const uint32_t n0 = mapa_u32(smem_u32(&s.n), 0), list0 = mapa_u32(smem_u32(s.list), 0);
    bool full = false;   // (a crowd need not be counted)
    auto take = [&](T e, int j) {
      if (full) return;
      const unsigned long long entry = (unsigned long long)list_key(e) << 32 | (uint32_t)~j;
      const unsigned int mine = atomicAdd(&s.mine, 1u);
      full = mine >= SEL_CAP;
      if (blocks == 1) {
        if (mine < SEL_CAP) s.list[mine] = entry;
      } else {
        const unsigned int at = add_cluster_u32(n0, 1u);
        if (at < SEL_CAP) st_cluster_u64(list0 + 8 * at, entry);
      }
    };
    auto look = [&](const uint4& u, int v) {
      also(u, v);
      if (!vec_any<T>(u, least)) return;
      for (unsigned int m = vec_reach<T>(u, least); m; m &= m - 1u) {
        const int i = __ffs(m) - 1;
        take(vec_element<T>(u, i), slice.element(v) + i);
      }
    };
    if (KEEP) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (slice.v0 + tid + i * THREADS < slice.v1) look(kept[i], slice.v0 + tid + i * THREADS);
    } else {
      for_vectors<THREADS, 4>(xv, slice.v0 + tid, slice.v1, look);
    }
    for (int i = tid; i < singles; i += THREADS) {
      const int j = slice.single(i, rank);
      also_one(x[j]);
      if (to_float(x[j]) >= least) take(x[j], j);
    }
  }

  // Behind collect(), by all blocks; the others than block 0 are done then and may end.  Returns the number of entries in block 0's
  // list (above SEL_CAP: too many).  A barrier for block 0.
  __device__ unsigned int gather() {
    if (blocks == 1) {
      __syncthreads();
      return s.mine;
    }
    __syncwarp();
    cluster_arrive();
    if (rank != 0) return 0u;
    cluster_wait();
    return s.n;
  }
};

// The exact selection, for rows that the bound does not thin out: the k <= SEL_CAP largest of the row into `list`, in any order,
// by a histogram of the leading 11 bits of the keys, one of the next bits inside the bin of the k-th, and so on.  NaN counts as
// the smallest.  One block; ends behind a barrier.
constexpr int SEL_BINS = 2048;
template <int THREADS> struct SelExact {
  unsigned int count[SEL_BINS];
  unsigned int wc[THREADS / 32], bin, above, n;
};
template <typename T, int THREADS> __device__ __noinline__ void select_exact(SelExact<THREADS>& s, unsigned long long* list, const T* x, int V, int k) {
  constexpr int BITS = VocabKey<T>::BITS, WARPS = THREADS / 32, PER = SEL_BINS / THREADS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t prefix = 0u;
  unsigned int want = (unsigned int)k;   // of those that share the prefix
  for (int left = BITS; left > 0;) {
    const int step = left > 11 ? 11 : left, bins = 1 << step;
    __syncthreads();
    for (int b = tid; b < bins; b += THREADS) s.count[b] = 0u;
    __syncthreads();
    for (int j = tid; j < V; j += THREADS) {
      const uint32_t key = VocabKey<T>::of(x[j]);
      if (left < BITS && key >> left != prefix) continue;
      atomicAdd(&s.count[(key >> (left - step)) & (uint32_t)(bins - 1)], 1u);
    }
    __syncthreads();
    const int b0 = bins - 1 - PER * tid;   // PER bins a thread, from the top
    unsigned int sum = 0u;
    for (int i = 0; i < PER; ++i) sum += b0 - i >= 0 ? s.count[b0 - i] : 0u;
    unsigned int upto = sum;
    __syncwarp();
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) s.wc[warp] = upto;
    __syncthreads();
    unsigned int before = upto - sum;
    for (int w = 0; w < warp; ++w) before += s.wc[w];
    for (int i = 0; i < PER; ++i) {
      const unsigned int c = b0 - i >= 0 ? s.count[b0 - i] : 0u;
      if (before < want && want <= before + c) { s.bin = (unsigned int)(b0 - i); s.above = before; }
      before += c;
    }
    __syncthreads();
    prefix = (prefix << step) | s.bin;
    want -= s.above;
    left -= step;
  }
  // the tokens above it, in any order, then the first `want` of its equals in index order (every warp takes a stretch)
  if (tid == 0) s.n = 0u;
  const int per = (V + WARPS - 1) / WARPS, j0 = min(V, warp * per), j1 = min(V, j0 + per);
  __syncthreads();
  auto entry = [](uint32_t key, int j) { return (unsigned long long)(key << (32 - BITS)) << 32 | (uint32_t)~j; };
  unsigned int n = 0u;
  for (int j = j0 + lane; j < j1; j += 32) {
    const uint32_t key = VocabKey<T>::of(x[j]);
    if (key > prefix) list[atomicAdd(&s.n, 1u)] = entry(key, j);
    n += key == prefix;
  }
  __syncwarp();
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) s.wc[warp] = n;
  __syncthreads();
  unsigned int before = 0u;
  for (int w = 0; w < warp; ++w) before += s.wc[w];
  if (n > 0u && before < want)
    for (int j = j0; j < j1 && before < want; j += 32) {
      const bool hit = j + lane < j1 && VocabKey<T>::of(x[j + lane]) == prefix;
      const unsigned int mask = __ballot_sync(0xffffffffu, hit), mine = before + __popc(mask & ((1u << lane) - 1u));
      if (hit && mine < want) list[k - want + mine] = entry(prefix, j + lane);
      before += __popc(mask);
    }
  __syncthreads();
}

// Descending sort of the n <= SEL_CAP entries (all different, none zero); ends behind a barrier.  Every warp sorts runs of 32 in
// registers; an entry's place then is its place in its run plus, from a binary search of each other run, how many are larger.
// (223 entries: 4 900 cycles by comparing all with all, 352: 11 500 by a bitonic sort in shared memory.)
template <int THREADS> __device__ void sort_list(unsigned long long* list, int n) {
  constexpr int WARPS = THREADS / 32, PER = SEL_CAP / THREADS > 0 ? SEL_CAP / THREADS : 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, runs = (n + 31) / 32;
  unsigned long long mine[PER];
  int place[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = warp + i * WARPS, at = 32 * r + lane;
    if (r >= runs) break;
    mine[i] = run_sorted(at < n ? list[at] : 0ull);
    list[at] = mine[i];   // (at < SEL_CAP: whole runs)
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = warp + i * WARPS;
    if (r >= runs) break;
    place[i] = lane + above_in_runs<unsigned long long>(list, runs, r, mine[i]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (warp + i * WARPS >= runs) break;
    if (mine[i]) list[place[i]] = mine[i];
  }
  __syncthreads();
}

}  // namespace xl
