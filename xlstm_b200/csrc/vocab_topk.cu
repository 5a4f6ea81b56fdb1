// Top logits: the k largest soft-capped logits of every row, their ids and the row's log-sum-exp.
//
// Mathematics.  The cap is strictly increasing, so the order is that of the logits as they come, compared as integer keys.
// The key of the k-th largest is found by a histogram of the leading key bits, then of the next ones inside the bin that the
// k-th falls into, and so on; what lies above it is fewer than k tokens, and as many of its equals as are missing join
// them in index order.  Sorting the k survivors by (key, index) in shared memory gives the output order.
#include "vocab_row.cuh"

namespace xl {

constexpr int TK_THREADS = 512, TK_WARPS = TK_THREADS / 32, TK_BINS = 2048;

struct TkShared {
  unsigned int count[TK_BINS];
  unsigned long long list[TOPK_MAX];   // key << 32 | ~index
  unsigned int wc[TK_WARPS];
  float wf[TK_WARPS];
  unsigned int bin, above, n;
};

__device__ __forceinline__ float capped_f32(float x, float cap) { return cap > 0.f ? cap * tanhf(x / cap) : x; }

template <typename T> __global__ void __launch_bounds__(TK_THREADS) topk_kernel(const xl_topk_params p) {
  __shared__ TkShared s;
  constexpr int BITS = VocabKey<T>::BITS;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.V, k = p.k;
  const T* x = static_cast<const T*>(p.logits) + (long long)row * p.row_stride;
  // key of the k-th largest
  uint32_t prefix = 0u;
  unsigned int want = (unsigned int)k;   // ... of those that share the prefix
  for (int left = BITS; left > 0;) {
    const int step = left > 11 ? 11 : left, bins = 1 << step;
    for (int b = tid; b < bins; b += TK_THREADS) s.count[b] = 0u;
    __syncthreads();
    for (int j = tid; j < V; j += TK_THREADS) {
      const uint32_t key = VocabKey<T>::of(x[j]);
      if (left < BITS && key >> left != prefix) continue;
      atomicAdd(&s.count[(key >> (left - step)) & (uint32_t)(bins - 1)], 1u);
    }
    __syncthreads();
    // four bins a thread, from the top
    const int b0 = bins - 1 - 4 * tid;
    unsigned int c[4], sum = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += c[i] = b0 - i >= 0 ? s.count[b0 - i] : 0u;
    unsigned int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) s.wc[warp] = upto;
    __syncthreads();
    unsigned int before = upto - sum;
    for (int w = 0; w < warp; ++w) before += s.wc[w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < want && want <= before + c[i]) { s.bin = (unsigned int)(b0 - i); s.above = before; }
      before += c[i];
    }
    __syncthreads();
    prefix = (prefix << step) | s.bin;
    want -= s.above;
    left -= step;
    __syncthreads();
  }
  // the tokens above it, in any order, then the first `want` of its equals in index order (every warp takes a stretch)
  if (tid == 0) s.n = 0u;
  for (int i = tid; i < TOPK_MAX; i += TK_THREADS) s.list[i] = 0ull;
  const int per = (V + TK_WARPS - 1) / TK_WARPS, j0 = min(V, warp * per), j1 = min(V, j0 + per);
  __syncthreads();
  unsigned int n = 0u;
  for (int j = j0 + lane; j < j1; j += 32) {
    const uint32_t key = VocabKey<T>::of(x[j]);
    if (key > prefix) s.list[atomicAdd(&s.n, 1u)] = (unsigned long long)key << 32 | (uint32_t)~j;
    n += key == prefix;
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) s.wc[warp] = n;
  __syncthreads();
  unsigned int before = 0u;
  for (int w = 0; w < warp; ++w) before += s.wc[w];
  if (n > 0u && before < want)
    for (int j = j0; j < j1 && before < want; j += 32) {
      const bool hit = j + lane < j1 && VocabKey<T>::of(x[j + lane]) == prefix;
      const unsigned int mask = __ballot_sync(0xffffffffu, hit), mine = before + __popc(mask & ((1u << lane) - 1u));
      if (hit && mine < want) s.list[k - want + mine] = (unsigned long long)prefix << 32 | (uint32_t)~(j + lane);
      before += __popc(mask);
    }
  __syncthreads();
  // descending bitonic sort of the list, padded with zeros to a power of two
  int size = 1;
  while (size < k) size <<= 1;
  for (int len = 2; len <= size; len <<= 1)
    for (int step = len >> 1; step > 0; step >>= 1) {
      for (int i = tid; i < size / 2; i += TK_THREADS) {
        const int a = 2 * i - (i & (step - 1)), b = a + step;
        const unsigned long long u = s.list[a], v = s.list[b];
        if ((u < v) == ((a & len) == 0)) { s.list[a] = v; s.list[b] = u; }
      }
      __syncthreads();
    }
  for (int i = tid; i < k; i += TK_THREADS) {
    const unsigned long long e = s.list[i];
    p.values[(long long)row * k + i] = capped_f32(VocabKey<T>::value((uint32_t)(e >> 32)), p.cap);
    p.ids[(long long)row * k + i] = (int32_t)~(uint32_t)e;
  }
  if (!p.lse) return;
  const float ymax = capped_f32(VocabKey<T>::value((uint32_t)(s.list[0] >> 32)), p.cap);
  float sum = 0.f;
  for (int j = tid; j < V; j += TK_THREADS) {
    const float y = capped_f32(to_float(x[j]), p.cap);
    sum += expf((y - ymax) / p.temperature);
  }
  sum = block_reduce<TK_WARPS>(sum, OpSum(), s.wf);
  if (tid == 0) p.lse[row] = isinf(ymax) ? ymax : ymax / p.temperature + logf(sum);
}

}  // namespace xl

extern "C" int xl_softcap_topk(const xl_topk_params* p, void* cuda_stream) {
  using namespace xl;
  if (!p || !p->logits || !p->values || !p->ids) return XL_ERR_NULL_POINTER;
  int rc = vocab_validate(p->rows, p->V, p->row_stride, p->cap, p->dtype);
  if (rc != XL_OK) return rc;
  if (p->k <= 0 || p->k > p->V || !vocab_temperature(p->temperature)) return XL_ERR_BAD_SHAPE;
  if (p->k > TOPK_MAX) return XL_ERR_TOO_LARGE;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  if (p->dtype == XL_F32) topk_kernel<float><<<p->rows, TK_THREADS, 0, st>>>(*p);
  else topk_kernel<__nv_bfloat16><<<p->rows, TK_THREADS, 0, st>>>(*p);
  return check_launch("xl_softcap_topk");
}
