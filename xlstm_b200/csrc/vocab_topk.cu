// Top logits: the k largest soft-capped logits of every row, their ids and the row's log-sum-exp.
//
// Mathematics.  The cap is strictly increasing, so the order is that of the logits as they come.  Two passes over the row: maxima
// of groups for a bound of the k-th largest (vocab_select.cuh), then the list of what reaches it together with the sum of
// 2^(z - z_max) in fp32.  The second pass finds the row in L2, so memory is read once.
//
// What bounds it.  Many rows: waiting; no unit is full.  15 instructions a logit in both passes (of which the cap's polynomial,
// exponential and sum are 7.5) at 2.1 a cycle and SM of 4; per instruction a warp waits 3.3 cycles for loads and 2.4 at barriers, the fp32
// units are busy 37 % of the time, those of the special functions 34 %.  4096 rows of 50 304 in bf16, k = 64, take 144 us, where their
// 412 MB are 63 us of memory (k = 256: 217 us; from k of some 440 on the list overflows and the exact selection does all: k = 512, 1.5 ms).
// A logit beyond three quarters of the cap sends its thread over its vectors again: one a row 211 us, 64 a row 266.
// Few rows: the chain of maxima, bisection, list and sort, 8.2 - 8.9 us for 16 rows, cut over clusters of eight blocks.
#include "vocab_select.cuh"

namespace xl {

template <int THREADS> struct TkShared {
  SelShared<THREADS> sel;
  SelExact<THREADS> exact;
  float wf[THREADS / 32], from[SEL_BLOCKS];
};

template <typename T, bool CAP, bool BOUNDED, int THREADS, int KEEP> __global__ void __launch_bounds__(THREADS, KEEP ? 2 : 1024 / THREADS) topk_kernel(const xl_topk_params p, const CappedZ<CAP> Z0, const double invT, const int blocks) {
  __shared__ TkShared<THREADS> s;
  constexpr int N = Vec16<T>::N;
  const int tid = threadIdx.x, k = p.k, rank = blocks > 1 ? (int)cluster_ctarank() : 0;
  const long long row = blockIdx.x / blocks;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  Selector<T, THREADS, KEEP> sel(s.sel, x, p.V, rank, blocks);
  sel.bound(k);
  const float least = sel.least(), largest = float_of_key(s.sel.top);
  CappedZ<CAP> Z = Z0;
  Z.set_ref(largest);
  const float zmax = CAP && !BOUNDED ? Z(largest) : 0.f;   // what z is taken relative to
  float sum = 0.f;
  f32x2 acc[2] = {0ull, 0ull};
  const f32x2 shift = f2_dup(-zmax);
  typename Vec16<T>::Mag mag = Vec16<T>::no_mag();
  auto add = [&](const f32x2 (&z)[N / 2]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      float z0, z1;
      f2_unpack(CAP && !BOUNDED ? f2_add(z[i], shift) : z[i], z0, z1);
      acc[i & 1] = f2_add(acc[i & 1], f2_pack(exp2_approx(z0), exp2_approx(z1)));
    }
  };
  sel.collect(least, [&](const uint4& u, int) {
    Vec16<T> a;
    a.set(u);
    if (CAP) mag = a.track(mag);
    f32x2 z[N / 2];
    Z.template of<true, T>(a, z);
    add(z);
  }, [&](T e) { sum += exp2_approx(Z(to_float(e)) - zmax); });
  if (!Z.small(Vec16<T>::largest(mag))) {   // a logit near the cap: this thread's vectors again
    acc[0] = acc[1] = 0ull;
#pragma unroll 1
    for (int v = sel.slice.v0 + tid; v < sel.slice.v1; v += THREADS) {
      Vec16<T> a;
      a.set(__ldg(sel.xv + v));
      f32x2 z[N / 2];
      Z.template of<false, T>(a, z);
      add(z);
    }
  }
  {
    float a0, a1;
    f2_unpack(f2_add(acc[0], acc[1]), a0, a1);
    sum = block_reduce<THREADS / 32>(sum + (a0 + a1), OpSum(), s.wf);   // (a barrier: the list is there, too)
  }
  if (blocks > 1 && tid == 0) st_cluster_f32(mapa_u32(smem_u32(&s.from[rank]), 0), sum);
  __syncwarp();
  const unsigned int n = sel.gather();
  if (rank != 0) return;
  if (tid == 0 && p.lse) {
    if (blocks > 1) {
      sum = s.from[0];
      for (int r = 1; r < blocks; ++r) sum += s.from[r];
    }
    p.lse[row] = (float)((log2_64((double)sum) + (double)zmax) * 0.69314718055994530942 + (CAP ? 0.0 : (double)Z.ref * invT));
  }
  if (n > SEL_CAP || n < (unsigned int)k) {
    select_exact<T, THREADS>(s.exact, s.sel.list, x, p.V, k);
    sort_list<THREADS>(s.sel.list, k);
  } else {
    sort_list<THREADS>(s.sel.list, (int)n);
  }
  for (int i = tid; i < k; i += THREADS) {
    const unsigned long long e = s.sel.list[i];
    const float v = list_value<T>(e);
    p.values[row * k + i] = CAP ? p.cap * Z.tanh_of(v) : v;
    p.ids[row * k + i] = (int32_t)~(uint32_t)e;
  }
}

// Blocks of a row: one, and up to eight where there are idle SMs; the bound over slices is a little weaker, and the list should hold
// what reaches it.
static int tk_blocks(int rows, int V, int k) {
  int blocks = 1;
  while (blocks < SEL_BLOCKS && rows * (blocks * 2) <= 4 * 148 && V >= 2048 * (blocks * 2) && k * 3 <= SEL_CAP) blocks *= 2;
  return blocks;
}

template <typename T, bool CAP, bool BOUNDED, int THREADS, int KEEP> static int tk_go(const xl_topk_params* p, int blocks, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p->rows * blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  XL_CUDA_TRY(cudaLaunchKernelEx(&cfg, topk_kernel<T, CAP, BOUNDED, THREADS, KEEP>, *p, CappedZ<CAP>(p->cap, p->temperature), 1.0 / (double)p->temperature, blocks));
  return check_launch("xl_softcap_topk");
}

// Slices of up to eight vectors a thread stay in registers; longer ones are read twice, by blocks of 256 threads, four an SM: with
// eight of 128 so many rows are under way that L2 loses half of them before the second pass (4096 rows of 50 304: 173 us, 158).
template <typename T, bool CAP, bool BOUNDED> static int tk_launch(const xl_topk_params* p, cudaStream_t st) {
  const int blocks = tk_blocks(p->rows, p->V, p->k), vectors = p->V / Vec16<T>::N;
  if ((vectors + blocks - 1) / blocks <= 8 * 256) return tk_go<T, CAP, BOUNDED, 256, 8>(p, blocks, st);
  return tk_go<T, CAP, BOUNDED, 256, 0>(p, blocks, st);
}
template <typename T> static int tk_choose(const xl_topk_params* p, cudaStream_t st) {
  if (!(p->cap > 0.f)) return tk_launch<T, false, false>(p, st);
  return vocab_bounded(p->cap, p->temperature) ? tk_launch<T, true, true>(p, st) : tk_launch<T, true, false>(p, st);
}

}  // namespace xl

extern "C" int xl_softcap_topk(const xl_topk_params* p, void* cuda_stream) {
  using namespace xl;
  if (!p || !p->logits || !p->values || !p->ids) return XL_ERR_NULL_POINTER;
  int rc = vocab_validate(p->logits, p->rows, p->V, p->row_stride, p->cap, p->dtype);
  if (rc != XL_OK) return rc;
  if (p->k <= 0 || p->k > p->V || !vocab_temperature(p->temperature)) return XL_ERR_BAD_SHAPE;
  if (p->k > TOPK_MAX) return XL_ERR_TOO_LARGE;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  return p->dtype == XL_F32 ? tk_choose<float>(p, st) : tk_choose<__nv_bfloat16>(p, st);
}
