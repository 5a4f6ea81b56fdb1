// Sampling head: one token per row of logits from temperature, top-k, top-p, min-p and a given uniform number.
//
// Mathematics.  With y = cap tanh(x / cap) and w = exp((y - y_max) / T) the tokens stand in the order of descending logit,
// lower index first among equals.  Every filter keeps a prefix of that order, so all that is asked of a row are three
// prefix questions -- the mass of the first k tokens, the first token where the running mass reaches top_p of it, and the
// first where it exceeds u times the mass kept -- and none of them needs the row sorted: a histogram (count and mass) of
// the leading key bits answers each up to a bin, one over the next bits inside that bin up to a finer one, and so on down
// to a single key, inside which all weights are the same and the rank follows by division.
//
// Precision.  The result is a whole number: a running sum that is off by d in relative terms picks another token with a
// probability of up to d times the number of tokens.  Weights are therefore formed in 64 bits and summed as integers in
// units of 2^-44 (rows are at most 2^18 long), which is exact and independent of the order of the atomics.
#include "vocab_row.cuh"

namespace xl {

constexpr int VS_THREADS = 1024, VS_WARPS = VS_THREADS / 32, VS_BINS = 2048;
constexpr double VS_ONE = 17592186044416.0;   // 2^44

struct VsHist {
  unsigned int count[VS_BINS];
  unsigned long long mass[VS_BINS];
};
struct VsShared {
  VsHist top, sub;                    // leading 11 bits; the bits of the descent at work
  unsigned int wc[VS_WARPS];
  unsigned long long wm[VS_WARPS];
  float fv[VS_WARPS];
  int iv[VS_WARPS];
  // answer of a descent step
  unsigned int bin, cnt, base_cnt;
  unsigned long long base_mass, bin_mass;
};

// One prefix question over a histogram: the bin, from the top, in which the running count (or mass) reaches `goal`.
__device__ void vs_find(VsShared& s, const VsHist& h, int bins, bool by_mass, unsigned long long goal, unsigned int base_cnt, unsigned long long base_mass) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b0 = bins - 1 - 2 * tid, b1 = b0 - 1;
  const unsigned int c0 = b0 >= 0 ? h.count[b0] : 0u, c1 = b1 >= 0 ? h.count[b1] : 0u;
  const unsigned long long m0 = b0 >= 0 ? h.mass[b0] : 0ull, m1 = b1 >= 0 ? h.mass[b1] : 0ull;
  unsigned int c = c0 + c1;
  unsigned long long m = m0 + m1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned int oc = __shfl_up_sync(0xffffffffu, c, o);
    const unsigned long long om = __shfl_up_sync(0xffffffffu, m, o);
    if (lane >= o) { c += oc; m += om; }
  }
  __syncthreads();
  if (lane == 31) { s.wc[warp] = c; s.wm[warp] = m; }
  __syncthreads();
  unsigned int ec = base_cnt + c - c0 - c1;   // in front of this thread's bins
  unsigned long long em = base_mass + m - m0 - m1;
  for (int w = 0; w < warp; ++w) { ec += s.wc[w]; em += s.wm[w]; }
  const unsigned long long before = by_mass ? em : ec, mid = before + (by_mass ? m0 : c0), end = mid + (by_mass ? m1 : c1);
  if (before < goal && goal <= end) {
    const bool first = goal <= mid;
    s.bin = first ? b0 : b1;
    s.cnt = first ? c0 : c1;
    s.bin_mass = first ? m0 : m1;
    s.base_cnt = first ? ec : ec + c0;
    s.base_mass = first ? em : em + m0;
  }
  __syncthreads();
}

struct VsPlace {
  uint32_t key;             // key of the token found
  unsigned int rank;        // how many tokens of the same key stand in front of it
  unsigned long long upto;  // running mass, the token included
};

template <typename T> struct VsRow {
  const T* x;
  int V;
  double cap, ymax, invT;
  uint32_t kmax;

  __device__ __forceinline__ double capped(float v) const { return cap > 0.0 ? cap * tanh((double)v / cap) : (double)v; }
  __device__ __forceinline__ double weight(uint32_t key) const {
    if (key == kmax) return 1.0;
    const float v = VocabKey<T>::value(key);
    if (!(v > -INFINITY) || ymax == INFINITY) return 0.0;   // NaN and -inf; next to +inf
    return exp((capped(v) - ymax) * invT);
  }

  // first token, in sampling order, whose running count (or mass) reaches `goal`, which the whole row does
  __device__ VsPlace descend(VsShared& s, bool by_mass, unsigned long long goal) const {
    constexpr int BITS = VocabKey<T>::BITS;
    vs_find(s, s.top, VS_BINS, by_mass, goal, 0u, 0ull);
    uint32_t prefix = s.bin;
    for (int left = BITS - 11; left > 0;) {
      const int step = left > 11 ? 11 : left;
      const int bins = 1 << step;
      const unsigned int base_cnt = s.base_cnt;
      const unsigned long long base_mass = s.base_mass;
      __syncthreads();
      for (int b = threadIdx.x; b < bins; b += VS_THREADS) { s.sub.count[b] = 0u; s.sub.mass[b] = 0ull; }
      __syncthreads();
      for (int j = threadIdx.x; j < V; j += VS_THREADS) {
        const uint32_t key = VocabKey<T>::of(x[j]);
        if (key >> left != prefix) continue;
        const uint32_t b = (key >> (left - step)) & (uint32_t)(bins - 1);
        atomicAdd(&s.sub.count[b], 1u);
        atomicAdd(&s.sub.mass[b], __double2ull_rn(weight(key) * VS_ONE));
      }
      __syncthreads();
      vs_find(s, s.sub, bins, by_mass, goal, base_cnt, base_mass);
      prefix = (prefix << step) | s.bin;
      left -= step;
    }
    const unsigned long long w = s.bin_mass / s.cnt;   // of every token of this key
    VsPlace r;
    r.key = prefix;
    r.rank = by_mass ? (unsigned int)((goal - s.base_mass + w - 1) / w) - 1u : (unsigned int)(goal - s.base_cnt) - 1u;
    r.upto = s.base_mass + (unsigned long long)(r.rank + 1u) * w;
    __syncthreads();
    return r;
  }

  // index of the token of key `key` that has `rank` others in front of it; every warp takes a stretch of the row
  __device__ void locate(VsShared& s, uint32_t key, unsigned int rank, int64_t* out) const {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (V + VS_WARPS - 1) / VS_WARPS, j0 = min(V, warp * per), j1 = min(V, j0 + per);
    unsigned int n = 0;
    for (int j = j0 + lane; j < j1; j += 32) n += VocabKey<T>::of(x[j]) == key;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s.wc[warp] = n;
    __syncthreads();
    unsigned int before = 0;
    for (int w = 0; w < warp; ++w) before += s.wc[w];
    if (rank < before || rank >= before + n) return;
    for (int j = j0; j < j1; j += 32) {
      const bool hit = j + lane < j1 && VocabKey<T>::of(x[j + lane]) == key;
      const unsigned int mask = __ballot_sync(0xffffffffu, hit);
      const unsigned int mine = before + __popc(mask & ((1u << lane) - 1u));
      if (hit && mine == rank) *out = j + lane;
      before += __popc(mask);
    }
  }
};

// the token of xl_softcap_argmax
template <typename T> __device__ void vs_greedy(VsShared& s, const T* x, int V, float cap, int64_t* out) {
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  for (int j = threadIdx.x; j < V; j += VS_THREADS) {
    const float y = cap > 0.f ? capped_rounded<T>(x[j], cap) : to_float(x[j]);
    if (y > bv || (y == bv && j < bi)) { bv = y; bi = j; }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
  }
  if ((threadIdx.x & 31) == 0) { s.fv[threadIdx.x >> 5] = bv; s.iv[threadIdx.x >> 5] = bi; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < VS_WARPS; ++w)
      if (s.fv[w] > bv || (s.fv[w] == bv && s.iv[w] < bi)) { bv = s.fv[w]; bi = s.iv[w]; }
    *out = bi == 0x7fffffff ? 0 : bi;
  }
}

template <typename T> __global__ void __launch_bounds__(VS_THREADS) sample_kernel(const xl_sample_params p) {
  extern __shared__ __align__(16) unsigned char smem[];
  VsShared& s = *reinterpret_cast<VsShared*>(smem);
  const int row = blockIdx.x, tid = threadIdx.x;
  const float temp = p.temperature_rows ? p.temperature_rows[row] : p.temperature;
  const int top_k = p.top_k_rows ? p.top_k_rows[row] : p.top_k;
  const float top_p = p.top_p_rows ? p.top_p_rows[row] : p.top_p, min_p = p.min_p_rows ? p.min_p_rows[row] : p.min_p;
  VsRow<T> r;
  r.x = static_cast<const T*>(p.logits) + (long long)row * p.row_stride;
  r.V = p.V;
  if (!(temp > 0.f)) { vs_greedy<T>(s, r.x, p.V, p.cap, p.tokens + row); return; }
  // the largest logit
  uint32_t km = 0u;
  for (int j = tid; j < p.V; j += VS_THREADS) km = max(km, VocabKey<T>::of(r.x[j]));
  r.kmax = block_reduce<VS_WARPS>(km, OpMax(), s.wc);
  r.cap = p.cap;
  const float xmax = VocabKey<T>::value(r.kmax);
  if (!(xmax > -INFINITY)) { if (tid == 0) p.tokens[row] = 0; return; }
  r.ymax = r.capped(xmax);
  r.invT = 1.0 / (double)temp;
  // histogram of the leading bits, and the mass that min_p leaves
  for (int b = tid; b < VS_BINS; b += VS_THREADS) { s.top.count[b] = 0u; s.top.mass[b] = 0ull; }
  __syncthreads();
  unsigned long long all = 0ull, over = 0ull;
  for (int j = tid; j < p.V; j += VS_THREADS) {
    const uint32_t key = VocabKey<T>::of(r.x[j]), b = key >> (VocabKey<T>::BITS - 11);
    const double w = r.weight(key);
    const unsigned long long m = __double2ull_rn(w * VS_ONE);
    atomicAdd(&s.top.count[b], 1u);
    atomicAdd(&s.top.mass[b], m);
    all += m;
    if (w >= (double)min_p) over += m;
  }
  all = block_reduce<VS_WARPS>(all, OpSum(), s.wm);
  over = block_reduce<VS_WARPS>(over, OpSum(), s.wm);
  __syncthreads();
  const unsigned long long one = (unsigned long long)VS_ONE;
  unsigned long long kept = all;
  if (top_k > 0 && top_k < p.V) kept = r.descend(s, false, (unsigned long long)top_k).upto;
  if (top_p < 1.f) {
    const double goal = ceil((double)top_p * (double)kept);
    kept = goal > 1.0 ? r.descend(s, true, min((unsigned long long)goal, kept)).upto : one;   // (one: the first token alone)
  }
  kept = max(one, min(kept, over));
  const double at = (double)p.u[row] * (double)kept;
  unsigned long long goal = at > 0.0 ? (unsigned long long)at + 1ull : 1ull;   // (NaN: the first)
  const VsPlace place = r.descend(s, true, min(goal, kept));
  r.locate(s, place.key, place.rank, p.tokens + row);
}

}  // namespace xl

extern "C" int xl_softcap_sample(const xl_sample_params* p, void* cuda_stream) {
  using namespace xl;
  if (!p || !p->logits || !p->tokens || !p->u) return XL_ERR_NULL_POINTER;
  const int rc = vocab_validate(p->rows, p->V, p->row_stride, p->cap, p->dtype);
  if (rc != XL_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  const size_t smem = sizeof(VsShared);
  if (p->dtype == XL_F32) {
    XL_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    sample_kernel<float><<<p->rows, VS_THREADS, smem, st>>>(*p);
  } else {
    XL_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    sample_kernel<__nv_bfloat16><<<p->rows, VS_THREADS, smem, st>>>(*p);
  }
  return check_launch("xl_softcap_sample");
}
