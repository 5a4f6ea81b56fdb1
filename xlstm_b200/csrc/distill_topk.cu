// Distillation from a teacher's top logits: loss and gradient along the vocabulary axis.
//
// Mathematics.  z = soft_cap(x) / T, q = softmax(z), S = the tokens that a row's teacher entries name, R = all others ("tail").
// With l_R = log sum_R e^z, l_S = log sum_S e^z and l = log(e^{l_R} + e^{l_S}):
//   loss / T^2 = sum_k p_k (log p_k - z[id_k] + l) + p_t (log p_t - l_R + l)
//   dloss/dz_j / T^2 = W e^{z_j - l} - sum_{k: id_k = j} p_k            for j in S
//                    = e^{z_j - l_R} (W e^{l_R - l} - p_t)              for j in R
// Both sums over the row are taken apart from the start (a bit per token says which one it belongs to), so neither a tail of
// 1e-9 behind a confident student nor the named tokens behind a flat one come out of a difference of large numbers, and
// the tail's factor W e^{l_R - l} - p_t is one number a row.  The K teacher entries are few: their terms are in 64 bits.
#include "vocab_row.cuh"

namespace xl {

constexpr int DT_THREADS = 256, DT_WARPS = DT_THREADS / 32;
// what a row leaves for its gradient
enum { ST_LR = 0, ST_L = 1, ST_B = 2, ST_W = 3, ST_TEACHER = 4, ST_LIVE = 5 };

struct DtShared {
  int id[TOPK_MAX];          // -1: unused
  float p[TOPK_MAX], z[TOPK_MAX];
  double wd[DT_WARPS];
  float wf[DT_WARPS];
  int wi[DT_WARPS];
};

struct DtTeacher {
  double L;        // subtracted from t / T
  double psum;
  bool live;       // the row counts: an entry is used and, without the teacher's own sum, has mass
};

__device__ __forceinline__ float dt_tanh(float x, float cap) { return tanhf(x / cap); }

// ids and probabilities of the teacher entries of a row into shared memory
__device__ DtTeacher dt_teacher(DtShared& s, const xl_distill_params& p, long long row) {
  const double invT = 1.0 / (double)p.temperature;
  const float* val = p.values + row * p.K;
  const bool given = p.teacher_lse != nullptr;
  double m = -INFINITY;
  int any = 0;
  for (int k = threadIdx.x; k < p.K; k += DT_THREADS) {
    const long long id = p.ids64 ? static_cast<const int64_t*>(p.ids)[row * p.K + k] : (long long)static_cast<const int32_t*>(p.ids)[row * p.K + k];
    const bool used = id >= 0 && id < p.V;
    if (id >= p.V && p.status) atomicExch(p.status, 4);
    s.id[k] = used ? (int)id : -1;
    any |= used;
    if (used) m = fmax(m, (double)val[k] * invT);
    if (used && val[k] != val[k]) m = val[k];
  }
  // (NaN has to survive the maximum)
  m = block_reduce<DT_WARPS>(m, [](double a, double b) { return a != a ? a : b != b ? b : fmax(a, b); }, s.wd);
  DtTeacher t;
  any = block_reduce<DT_WARPS>(any, OpMax(), s.wi);
  t.live = any && (given || m != -INFINITY);
  t.L = 0.0;
  if (t.live && !given) {
    double sum = 0.0;
    for (int k = threadIdx.x; k < p.K; k += DT_THREADS)
      if (s.id[k] >= 0) sum += exp((double)val[k] * invT - m);
    sum = block_reduce<DT_WARPS>(sum, OpSum(), s.wd);
    t.L = m + log(sum);
  } else if (given) {
    t.L = (double)p.teacher_lse[row];
  }
  double psum = 0.0;
  for (int k = threadIdx.x; k < p.K; k += DT_THREADS) {
    const double pk = s.id[k] >= 0 && t.live ? exp((double)val[k] * invT - t.L) : 0.0;
    s.p[k] = (float)pk;
    psum += pk;
  }
  t.psum = block_reduce<DT_WARPS>(psum, OpSum(), s.wd);
  return t;
}

template <typename T, bool LOSS, bool GRAD> __global__ void __launch_bounds__(DT_THREADS) distill_kernel(const xl_distill_params p) {
  extern __shared__ __align__(16) unsigned int named[];   // a bit per token
  __shared__ DtShared s;
  const int tid = threadIdx.x, V = p.V, K = p.K;
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const float invT = 1.f / p.temperature, cap = p.cap;
  float* st = p.stats ? p.stats + row * 8 : nullptr;
  auto z_of = [&](float v) { return (cap > 0.f ? cap * dt_tanh(v, cap) : v) * invT; };
  auto in_top = [&](int j) { return (named[j >> 5] >> (j & 31)) & 1u; };

  const DtTeacher t = dt_teacher(s, p, row);
  for (int w = tid; w < (V + 31) / 32; w += DT_THREADS) named[w] = 0u;
  __syncthreads();
  int count = 0;   // of tokens named
  for (int k = tid; k < K; k += DT_THREADS)
    if (s.id[k] >= 0) count += !((atomicOr(&named[s.id[k] >> 5], 1u << (s.id[k] & 31)) >> (s.id[k] & 31)) & 1u);
  count = block_reduce<DT_WARPS>(count, OpSum(), s.wi);   // (and the bits are there)

  float lR, l, B, W;
  if (LOSS) {
    float mR = -INFINITY, mS = -INFINITY;
    for (int j = tid; j < V; j += DT_THREADS) {
      const float z = z_of(to_float(x[j]));
      if (in_top(j)) mS = fmaxf(mS, z);
      else mR = fmaxf(mR, z);
    }
    mR = block_reduce<DT_WARPS>(mR, OpMax(), s.wf);
    mS = block_reduce<DT_WARPS>(mS, OpMax(), s.wf);
    const float m = fmaxf(mR, mS);
    float sR = 0.f, sS = 0.f;
    const float aR = mR == -INFINITY ? 0.f : mR, aS = mS == -INFINITY ? 0.f : mS;
    for (int j = tid; j < V; j += DT_THREADS) {
      const float z = z_of(to_float(x[j]));
      if (in_top(j)) sS += expf(z - aS);
      else sR += expf(z - aR);
    }
    sR = block_reduce<DT_WARPS>(sR, OpSum(), s.wf);
    sS = block_reduce<DT_WARPS>(sS, OpSum(), s.wf);
    lR = aR + logf(sR);
    const float lS = aS + logf(sS);
    l = m == -INFINITY ? m : m + logf(expf(lR - m) + expf(lS - m));
    const double pt = p.teacher_lse && t.live && count < V ? fmax(0.0, 1.0 - t.psum) : 0.0;
    const double T2 = (double)p.temperature * (double)p.temperature;
    double loss = 0.0;
    for (int k = tid; k < K; k += DT_THREADS) {
      const float pk = s.p[k];
      if (!(pk == 0.f)) loss += (double)pk * ((double)p.values[row * K + k] / (double)p.temperature - t.L - (double)z_of(to_float(x[s.id[k]])) + (double)l);
    }
    loss = block_reduce<DT_WARPS>(loss, OpSum(), s.wd);
    if (!(pt == 0.0)) loss += pt * (log(pt) - (double)lR + (double)l);
    W = (float)(t.psum + pt);
    B = lR == -INFINITY ? 0.f : (float)((double)W * exp((double)lR - (double)l) - pt);
    if (tid == 0) {
      p.loss[row] = (float)(T2 * loss);
      if (st) { st[ST_LR] = lR; st[ST_L] = l; st[ST_B] = B; st[ST_W] = W; }
    }
  } else {
    lR = st[ST_LR]; l = st[ST_L]; B = st[ST_B]; W = st[ST_W];
  }
  if (!GRAD) return;
  const float g = (p.weight ? p.weight[row * p.weight_stride] : 1.f) * p.temperature;
  T* dx = static_cast<T*>(p.dlogits) + row * p.dlogits_stride;
  for (int j = tid; j < V; j += DT_THREADS) {
    const float v = to_float(x[j]);
    const float th = cap > 0.f ? dt_tanh(v, cap) : 0.f, z = (cap > 0.f ? cap * th : v) * invT;
    if (!in_top(j)) dx[j] = from_float<T>(t.live ? g * B * expf(z - lR) * (1.f - th * th) : 0.f);
  }
  for (int k = tid; k < K; k += DT_THREADS) {
    const int id = s.id[k];
    if (id < 0) continue;
    const float v = to_float(x[id]);
    const float th = cap > 0.f ? dt_tanh(v, cap) : 0.f, z = (cap > 0.f ? cap * th : v) * invT;
    float pk = 0.f;
    for (int i = 0; i < K; ++i) pk += s.id[i] == id ? s.p[i] : 0.f;   // (every entry of a token named twice writes the same value)
    dx[id] = from_float<T>(t.live ? g * (W * expf(z - l) - pk) * (1.f - th * th) : 0.f);
  }
}

static int dt_validate(const xl_distill_params* p) {
  if (!p || !p->logits || !p->values || !p->ids) return XL_ERR_NULL_POINTER;
  const int rc = vocab_validate(p->rows, p->V, p->row_stride, p->cap, p->dtype);
  if (rc != XL_OK) return rc;
  if (p->K <= 0 || !(p->temperature > 0.f) || p->temperature > 3.0e38f) return XL_ERR_BAD_SHAPE;
  if (p->K > TOPK_MAX) return XL_ERR_TOO_LARGE;
  if (p->dlogits && p->rows > 1 && p->dlogits_stride < p->V) return XL_ERR_BAD_STRIDE;
  if (p->dlogits) {
    const uintptr_t size = p->dtype == XL_F32 ? 4 : 2, n = (uintptr_t)p->V * size, last = (uintptr_t)(p->rows - 1) * size;
    const uintptr_t a = reinterpret_cast<uintptr_t>(p->logits), b = reinterpret_cast<uintptr_t>(p->dlogits);
    if (a < b + last * (uintptr_t)p->dlogits_stride + n && b < a + last * (uintptr_t)p->row_stride + n) return XL_ERR_ALIASING;
  }
  return XL_OK;
}

template <typename T> static int dt_launch(const xl_distill_params* p, bool loss, cudaStream_t st) {
  const size_t smem = (size_t)((p->V + 31) / 32) * 4;
  auto go = [&](auto kern) -> int {
    XL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, VOCAB_MAX / 8));
    kern<<<p->rows, DT_THREADS, smem, st>>>(*p);
    return check_launch("xl_distill_topk");
  };
  if (!loss) return go(distill_kernel<T, false, true>);
  return p->dlogits ? go(distill_kernel<T, true, true>) : go(distill_kernel<T, true, false>);
}

}  // namespace xl

extern "C" int xl_distill_topk(const xl_distill_params* p, void* cuda_stream) {
  using namespace xl;
  const int rc = dt_validate(p);
  if (rc != XL_OK) return rc;
  if (!p->loss) return XL_ERR_NULL_POINTER;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  return p->dtype == XL_F32 ? dt_launch<float>(p, true, st) : dt_launch<__nv_bfloat16>(p, true, st);
}

extern "C" int xl_distill_topk_backward(const xl_distill_params* p, void* cuda_stream) {
  using namespace xl;
  const int rc = dt_validate(p);
  if (rc != XL_OK) return rc;
  if (!p->dlogits || !p->stats) return XL_ERR_NULL_POINTER;
  cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
  return p->dtype == XL_F32 ? dt_launch<float>(p, false, st) : dt_launch<__nv_bfloat16>(p, false, st);
}
