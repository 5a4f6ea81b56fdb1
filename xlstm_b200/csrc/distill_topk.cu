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
//
// What bounds it.  Waiting, with the fp32 units half and those of the special functions two fifths busy and 2.1 instructions a cycle and
// SM of 4: per instruction a warp waits 3 cycles for loads in the loss (11 instructions a logit; 2048 rows of 50 304 in bf16: 58 us, their
// 206 MB are 31 us of memory), 10 in the gradient alone (10 instructions; 77 us, 413 MB, 63 us), 5 and 2.4 at barriers with both in
// one launch (22 instructions; 4096 rows: 236 us; the logits come from memory once, 826 MB in all, 126 us).  Few rows: the chain ids ->
// logits there -> 64-bit exponentials -> sums -> logarithms -> gradient, 12 us for 64 rows cut over clusters of eight blocks.
// These are rows whose logits stay below three quarters of the cap.  One beyond it sends its thread over its vectors again, with a
// branch and a division an element, and in the backward launch the whole row: one such logit a row 111 us for the loss, 230 for
// loss and gradient through autograd (135 without), 368 for 4096 rows in one launch (64 of them a row: 139, 259, 427).
#include "vocab_row.cuh"

namespace xl {

constexpr int DT_WARPS = 8, DT_BLOCKS = 8;   // warps: at most
// threads of a block: small ones hide each other's serial parts best (2048 rows of 50 304: loss 59 us with 128, 63 with 256), but
// with both directions in one launch the second pass finds more of its row in L1 where fewer rows are under way (265, 247 for 4096 rows)
__host__ __device__ constexpr int dt_threads(bool both) { return both ? 256 : 128; }
constexpr double DT_LN2 = 0.69314718055994530942;
// what a row leaves for its gradient; ST_FLAGS: 1 if its logits stay below three quarters of the cap, and 2 if a token is named
// twice; the last two places hold a double.  Without a cap ST_LR is what the tail's exponents are relative to, ST_REF what those of
// the tokens named are, and ST_B has the tail's sum in it.
enum { ST_LR = 0, ST_L = 1, ST_B = 2, ST_W = 3, ST_FLAGS = 4, ST_REF = 5, ST_TEACHER = 6 };

struct DtShared {
  double wd[3][DT_WARPS];
  float wf[2][DT_WARPS], from[4][DT_BLOCKS];   // from: of the row's blocks; a place is written once a launch
  int wi[2][DT_WARPS];
  float lR, l, B, W, pscale;
  int again;   // a token of the slice is named twice (here, not in a register through the passes)
};
// Dynamic shared memory: K entries -- t / T, id (-1: unused), z of the student there, e^(t / T - shift) -- and a bit per token of
// the slice.
struct DtEntries {
  double* t;
  int* id;
  float *z, *e;
  unsigned int* bits;
  __device__ __forceinline__ DtEntries(unsigned char* m, int K) {
    t = reinterpret_cast<double*>(m);
    id = reinterpret_cast<int*>(t + K);
    z = reinterpret_cast<float*>(id + K);
    e = z + K;
    bits = reinterpret_cast<unsigned int*>(e + K);
  }
};
static size_t dt_smem(int K, int V, int N, int blocks) {
  const size_t vectors = (size_t)V / N, per = (vectors + blocks - 1) / blocks;
  return (size_t)K * 20 + ((per + 3) * N + 31) / 32 * 4 + 4;
}

// one value of every block of the row's cluster, in rank order, combined by `f`
template <typename F> __device__ __forceinline__ float dt_exchange(float v, float* from, int rank, int blocks, F f) {
  if (threadIdx.x < blocks) st_cluster_f32(mapa_u32(smem_u32(from + rank), threadIdx.x), v);
  __syncwarp();
  cluster_sync_all();
  v = from[0];
  for (int r = 1; r < blocks; ++r) v = f(v, from[r]);
  return v;
}

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

// f(vector, its number) for v, v + STEP, .. below end, four loads under way at a time
template <int STEP, typename F> __device__ __forceinline__ void dt_vectors(const uint4* xv, int v, int end, F f) {
  const int over = 31 - (int)(threadIdx.x & 31) + 3 * STEP;
#pragma unroll 1
  for (; v + over < end; v += 4 * STEP) {   // (all lanes together: f may part them)
    uint4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __ldg(xv + v + i * STEP);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f(u[i], v + i * STEP);
      __syncwarp();
    }
  }
#pragma unroll 1
  for (; v < end; v += STEP) f(__ldg(xv + v), v);
}

__device__ __forceinline__ double dt_nanmax(double a, double b) { return a != a || b != b ? a + b : fmax(a, b); }   // (NaN survives)

template <typename T, bool CAP, bool BOUNDED, bool LOSS, bool GRAD>
__global__ void __launch_bounds__(dt_threads(LOSS && GRAD), LOSS && GRAD ? 4 : 8) distill_kernel(const xl_distill_params p, const CappedZ<CAP> Z0, const double invT, const int blocks) {
  CappedZ<CAP> Z = Z0;
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ DtShared s;
  constexpr int N = Vec16<T>::N, THREADS = dt_threads(LOSS && GRAD), WARPS = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.V, K = p.K;
  const int rank = blocks > 1 ? (int)cluster_ctarank() : 0;
  const long long row = blockIdx.x / blocks;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  const RowSlice<T> slice(x, V, rank, blocks);
  const uint4* xv = reinterpret_cast<const uint4*>(x + slice.head);
  const int singles = slice.n_single(rank, blocks);
  // (shared memory of another block may be written once that block runs: the other half of this barrier is in front of the first exchange)
  if (LOSS && blocks > 1) cluster_arrive();
  const DtEntries en(dynamic, K);
  const bool given = p.teacher_lse != nullptr;
  float* st = p.stats ? p.stats + row * 8 : nullptr;
  const unsigned char* bytes = reinterpret_cast<const unsigned char*>(en.bits) + (N == 8 ? 1 - slice.first / 8 : 0);
  auto flags = [&](int v) -> unsigned int {   // bits of the vector's elements
    if (N == 8) return bytes[v];
    const int o = N * (v + 1) - slice.first;
    return (unsigned int)(bytes[o >> 3] >> (o & 4)) & 15u;
  };
  auto flag = [&](int j) -> bool {
    const int o = slice.place(j) - slice.first;
    return (en.bits[o >> 5] >> (o & 31)) & 1u;
  };

  if (!LOSS && !CAP) Z.ref = st[ST_REF];
  // the teacher's entries, the student's logits there, and the bits of the tokens named
  if (LOSS) {
    for (int w = tid; w < (slice.end - slice.first + 31) / 32; w += THREADS) en.bits[w] = 0u;
    __syncthreads();
  }
  const int with = min(WARPS, (K + 31) / 32);   // warps that have entries
  double m = -INFINITY;   // of t / T
  float xS = -INFINITY;   // largest logit of the tokens named
  int any = 0, twice = 0, count = 0;
  if (warp < with) {
    for (int k = tid; k < K; k += THREADS) {
      const long long at = row * K + k, id = p.ids64 ? static_cast<const int64_t*>(p.ids)[at] : (long long)static_cast<const int32_t*>(p.ids)[at];
      const double t = (double)p.values[at] * invT;
      const bool used = id >= 0 && id < V;
      if (id >= V && p.status) atomicExch(p.status, 4);
      en.id[k] = used ? (int)id : -1;
      en.z[k] = 0.f;
      if (!used) continue;
      en.t[k] = t;
      any = 1;
      m = dt_nanmax(m, t);
      const float xk = to_float(x[id]);
      en.z[k] = LOSS && !CAP ? xk : Z(xk);   // (without a cap z waits for the row's largest)
      xS = fmaxf(xS, xk);
      const int o = slice.place((int)id) - slice.first;
      if (LOSS && o >= 0 && o < slice.end - slice.first) {
        const int old = (atomicOr(&en.bits[o >> 5], 1u << (o & 31)) >> (o & 31)) & 1u;
        twice |= old;
        count += 1 - old;
      }
    }
    __syncwarp();   // (see block_reduce)
    if (LOSS) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        m = dt_nanmax(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (!BOUNDED) xS = fmaxf(xS, __shfl_xor_sync(0xffffffffu, xS, o));
      }
      if (K >= V) count = __reduce_add_sync(0xffffffffu, count);
    }
    any = (__any_sync(0xffffffffu, any) ? 1 : 0) | (__any_sync(0xffffffffu, twice) ? 2 : 0);
    if (lane == 0) { s.wd[2][warp] = m; s.wf[0][warp] = xS; s.wi[0][warp] = any; s.wi[1][warp] = count; }
  }
  __syncthreads();   // (the bits are there, too)
  any = 0;
  count = 0;
  for (int w = 0; w < with; ++w) {
    if (LOSS) {
      m = dt_nanmax(m, s.wd[2][w]);
      if (!BOUNDED) xS = fmaxf(xS, s.wf[0][w]);
      count += s.wi[1][w];
    }
    any |= s.wi[0][w];
  }
  const bool everything = K >= V && count == V;   // no token is left for the tail
  bool again = any & 2, live = any & 1;
  if (LOSS && tid == 0) s.again = any & 2;
  double L = 0.0;   // shift of the teacher's exponents; with its own sum, or in the backward pass, the right one from the start
  if (LOSS) {
    live = live && (given || m != -INFINITY);
    if (live) L = given ? (double)p.teacher_lse[row] : m;
  } else {
    live = live && st[ST_W] != 0.f;
    again = (int)st[ST_FLAGS] & 2;
    L = *reinterpret_cast<const double*>(st + ST_TEACHER);
  }
  // Shifts of the two sums.  Bounded z: none.  Under a cap their largest z.  Without one z may lie anywhere down to the type's
  // lowest value, where a step of fp32 is 2e31: each sum takes its logits relative to its own largest, refR or refS, from the start,
  // and the two come together in 64 bits.
  float mR = 0.f, mS = 0.f, refR = 0.f, refS = 0.f;
  if (LOSS) {
    __syncwarp();
    if (blocks > 1) cluster_wait();
    if (!BOUNDED) {
      float xm = -INFINITY;
      dt_vectors<THREADS>(xv, slice.v0 + tid, slice.v1, [&](const uint4& u, int v) {
        Vec16<T> a;
        a.set(u);
        const unsigned int f = flags(v);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          float x0, x1;
          f2_unpack(a.p[i], x0, x1);
          if (!(f >> (2 * i) & 1u)) xm = fmaxf(xm, x0);
          if (!(f >> (2 * i + 1) & 1u)) xm = fmaxf(xm, x1);
        }
      });
      for (int i = tid; i < singles; i += THREADS) {
        const int j = slice.single(i, rank);
        if (!flag(j)) xm = fmaxf(xm, to_float(x[j]));
      }
      xm = block_reduce<WARPS>(xm, OpMax(), s.wf[0]);
      if (blocks > 1) xm = dt_exchange(xm, s.from[2], rank, blocks, OpMax());
      if (CAP) {   // (-inf is a value like any other)
        mR = Z(xm);
        mS = Z(xS);
      } else {
        Z.set_ref(xm);
        refR = Z.ref;
        Z.set_ref(xS);
        refS = Z.ref;
        Z.set_ref(fmaxf(xm, xS));
      }
    }
  }
  float sS = 0.f;   // of the slice's tokens named
  if (warp < with) {
    double E = 0.0, F = 0.0;   // sum of e_k, and of e_k (t_k - z_k)
    for (int k = tid; k < K; k += THREADS) {
      double zk = 0.0;   // z of the student there, without a cap from the logit itself: near the type's lowest value en.z is -inf
      float zS = en.z[k] - mS;
      if (LOSS && CAP) zk = (double)en.z[k] * DT_LN2;
      if (LOSS && !CAP) {
        zk = ((double)en.z[k] - (double)Z.ref) * invT;
        zS = (en.z[k] - refS) * Z.a;
        en.z[k] = Z(en.z[k]);
      }
      double e = 0.0;
      if (en.id[k] >= 0 && live) {
        const double d = en.t[k] - L;
        e = d < -690.0 ? 0.0 : d <= 0.0 ? exp64(d) : exp(d);   // (above 0: a teacher's sum that is not the sum)
        if (LOSS && !(e == 0.0)) F += e * (en.t[k] - zk);
      }
      en.e[k] = (float)e;
      E += e;
      if (LOSS && en.id[k] >= 0) {
        const int o = slice.place(en.id[k]);
        bool first = o >= slice.first && o < slice.end;
        if (again)   // a token named twice is summed once
          for (int i = 0; i < k; ++i) first = first && en.id[i] != en.id[k];
        if (first) sS += exp2_approx(zS);
      }
    }
    __syncwarp();
    if (LOSS) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        E += __shfl_xor_sync(0xffffffffu, E, o);
        F += __shfl_xor_sync(0xffffffffu, F, o);
        sS += __shfl_xor_sync(0xffffffffu, sS, o);
      }
      if (lane == 0) { s.wd[0][warp] = E; s.wd[1][warp] = F; s.wf[1][warp] = sS; }
    }
  }

  const float ref = Z.ref;   // of the tokens named
  if (LOSS && !CAP) Z.ref = refR;
  bool small = true;   // (this thread's, in the second pass: this warp's) logits stay below three quarters of the cap
  if (LOSS) {
    // both sums over the slice.  The first try takes every magnitude for a small one and looks at the largest behind it;
    // a thread that met a large one sums its vectors again.
    float sR = 0.f;
    f32x2 acc[2] = {0ull, 0ull};
    const f32x2 shift = f2_dup(-mR);
    typename Vec16<T>::Mag mag = Vec16<T>::no_mag();
    auto sum = [&](auto is_small, const uint4& u, int v) {
      Vec16<T> a;
      a.set(u);
      if (CAP && decltype(is_small)::value) mag = a.track(mag);
      f32x2 z[N / 2];
      Z.template of<decltype(is_small)::value, T>(a, z);
      const unsigned int f = flags(v);
      if (f != 0u) {   // (K of V tokens; their part is summed with the entries)
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          float z0, z1;
          f2_unpack(z[i], z0, z1);
          z[i] = f2_pack(f >> (2 * i) & 1u ? -INFINITY : z0, f >> (2 * i + 1) & 1u ? -INFINITY : z1);
        }
      }
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        float z0, z1;
        f2_unpack(BOUNDED || !CAP ? z[i] : f2_add(z[i], shift), z0, z1);
        acc[i & 1] = f2_add(acc[i & 1], f2_pack(exp2_approx(z0), exp2_approx(z1)));
      }
    };
    dt_vectors<THREADS>(xv, slice.v0 + tid, slice.v1, [&](const uint4& u, int v) { sum(Yes(), u, v); });
    small = Z.small(Vec16<T>::largest(mag));
    if (!small) {
      sR = 0.f;
      acc[0] = acc[1] = 0ull;
#pragma unroll 1
      for (int v = slice.v0 + tid; v < slice.v1; v += THREADS) sum(No(), __ldg(xv + v), v);
    }
    for (int i = tid; i < singles; i += THREADS) {
      const int j = slice.single(i, rank);
      const float z = Z(to_float(x[j]));
      if (!flag(j)) sR += exp2_approx(z - mR);
    }
    {
      float a0, a1;
      f2_unpack(f2_add(acc[0], acc[1]), a0, a1);
      sR += a0 + a1;
    }
    __syncwarp();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sR += __shfl_xor_sync(0xffffffffu, sR, o);
    if (GRAD) small = __all_sync(0xffffffffu, small);   // the second pass's loops meet in whole warps: one way for all lanes
    __syncwarp();
    int all_small = __syncthreads_and(small);   // (and the maximum in s.wf[0] has been read)
    if (lane == 0) s.wf[0][warp] = sR;
    __syncthreads();
    if (warp == 0) {
      sR = sS = 0.f;
      for (int w = 0; w < WARPS; ++w) sR += s.wf[0][w];
      for (int w = 0; w < with; ++w) sS += s.wf[1][w];
    }
    if (blocks > 1) {
      if (tid < blocks) {
        st_cluster_f32(mapa_u32(smem_u32(s.from[1] + rank), tid), sS);
        st_cluster_f32(mapa_u32(smem_u32(s.from[3] + rank), tid), (all_small ? 1.f : 0.f) + (float)s.again);
      }
      sR = dt_exchange(sR, s.from[0], rank, blocks, OpSum());
    }
    if (warp == 0) {
      __syncwarp();
      int named_twice = s.again;   // in any of the slices
      if (blocks > 1) {
        sS = 0.f;
        for (int r = 0; r < blocks; ++r) {
          const int flags_r = (int)s.from[3][r];
          sS += s.from[1][r];
          all_small = all_small && (flags_r & 1);
          named_twice |= flags_r & 2;
        }
      }
      double E = 0.0, F = 0.0;
      for (int w = 0; w < with; ++w) { E += s.wd[0][w]; F += s.wd[1][w]; }
      const double left = given && live && !everything ? fmax(0.0, 1.0 - E) : 0.0;   // p_tail
      // sums in one scale, and the four logarithms in four lanes
      double oR = (double)mR, oS = (double)mS;   // (without a cap the larger one is 0)
      if (!CAP) {
        const double scale = invT * 1.4426950408889634;
        oR = ((double)refR - (double)ref) * scale;
        oS = ((double)refS - (double)ref) * scale;
        mR = (float)oR;
        mS = (float)oS;
      }
      const float top = BOUNDED || !CAP ? 0.f : sR > 0.f ? (sS > 0.f ? fmaxf(mR, mS) : mR) : mS;
      const double tR = BOUNDED || sR == 0.f ? sR : sR * exp2_approx(mR - top), tS = BOUNDED || sS == 0.f ? sS : sS * exp2_approx(mS - top);
      const double lg = log2_64(lane == 0 ? (double)sR : lane == 1 ? tR + tS : lane == 2 ? E : left);
      const double lR = __shfl_sync(0xffffffffu, lg, 0) + oR, l = __shfl_sync(0xffffffffu, lg, 1) + (double)top;   // log2(0) = -inf
      const double lE = __shfl_sync(0xffffffffu, lg, 2), lleft = __shfl_sync(0xffffffffu, lg, 3);
      if (lane == 0) {
        double loss = 0.0, W = 0.0;
        const double r = (double)(1.f / (float)E), iE = fma(r, fma(-E, r, 1.0), r);   // 1 / E
        if (live) {
          W = given ? E + left : 1.0;
          loss = given ? F + E * (l * DT_LN2 - L) : F * iE + (l - lE) * DT_LN2 - L;
          if (!(left == 0.0)) loss += left * (lleft - lR + l) * DT_LN2;
        }
        s.lR = !CAP ? refR : sR == 0.f ? 0.f : (float)lR;
        s.l = (float)l;
        s.B = sR == 0.f ? 0.f : (float)(W * (double)((float)tR / (float)(tR + tS)) - left);
        if (!CAP && sR != 0.f) s.B /= sR;
        s.W = (float)W;
        s.pscale = given ? 1.f : (float)iE;
        if (rank == 0) {
          p.loss[row] = (float)((double)p.temperature * (double)p.temperature * loss);
          if (st) {
            st[ST_LR] = s.lR; st[ST_L] = s.l; st[ST_B] = s.B; st[ST_W] = s.W; st[ST_FLAGS] = (all_small ? 1.f : 0.f) + (float)named_twice; st[ST_REF] = ref;
            *reinterpret_cast<double*>(st + ST_TEACHER) = given ? L : L + lE * DT_LN2;
          }
        }
      }
    }
  } else {
    if (tid == 0) { s.lR = st[ST_LR]; s.l = st[ST_L]; s.B = st[ST_B]; s.W = st[ST_W]; s.pscale = 1.f; }
    small = (int)st[ST_FLAGS] & 1;
  }
  if (!GRAD) return;
  __syncthreads();

  T* dx = static_cast<T*>(p.dlogits) + row * p.dlogits_stride;
  const bool wide = (reinterpret_cast<uintptr_t>(dx + slice.head) & 15u) == 0;   // the gradient's vectors lie like the logits'
  const float g = live ? (p.weight ? p.weight[row * p.weight_stride] : 1.f) * p.temperature : 0.f, gB = g * s.B, lR = CAP ? s.lR : 0.f;
  if (!CAP) Z.ref = s.lR;
  const float bend = CAP ? gB * Z.flat : 0.f;   // slope 1 - tanh^2 = 1 - (z / a)^2
  const f32x2 gB2 = f2_dup(gB), bend2 = f2_dup(-bend), shift = f2_dup(-lR);
  auto store = [&](const uint4& out, int v) {
    if (wide) {
      __stcs(reinterpret_cast<uint4*>(dx + slice.head) + v, out);
    } else {
      const T* o = reinterpret_cast<const T*>(&out);
#pragma unroll
      for (int i = 0; i < N; ++i) dx[slice.element(v) + i] = o[i];
    }
  };
  auto grad = [&](const f32x2 (&z)[N / 2], int v) {
    f32x2 d[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      float e0, e1;
      f2_unpack(CAP ? f2_add(z[i], shift) : z[i], e0, e1);
      const f32x2 e = f2_pack(exp2_approx(e0), exp2_approx(e1));
      d[i] = f2_mul(e, CAP ? f2_fma(f2_mul(z[i], z[i]), bend2, gB2) : gB2);
    }
    store(Vec16<T>::round(d), v);
  };
  if (!live) {   // (`live` is one for the block, `small` for the warp or, from `stats`, for the row: dt_vectors wants whole warps)
    for (int v = slice.v0 + tid; v < slice.v1; v += THREADS) store(make_uint4(0u, 0u, 0u, 0u), v);
  } else if (small) {
    dt_vectors<THREADS>(xv, slice.v0 + tid, slice.v1, [&](const uint4& u, int v) {
      Vec16<T> a;
      a.set(u);
      f32x2 z[N / 2];
      Z.template of<true, T>(a, z);
      grad(z, v);
    });
  } else {
#pragma unroll 1
    for (int v = slice.v0 + tid; v < slice.v1; v += THREADS) {
      Vec16<T> a;
      a.set(__ldg(xv + v));
      f32x2 z[N / 2];
      Z.template of<false, T>(a, z);
      grad(z, v);
    }
  }
  for (int i = tid; i < singles; i += THREADS) {
    const int j = slice.single(i, rank);
    const float z = Z(to_float(x[j]));
    dx[j] = from_float<T>(live ? exp2_approx(z - lR) * (CAP ? fmaf(-bend * z, z, gB) : gB) : 0.f);
  }
  __syncthreads();   // the named tokens got the tail's gradient, too: theirs follows
  const float l = s.l, W = s.W;
  for (int k = tid; k < K; k += THREADS) {
    const int id = en.id[k];
    if (id < 0 || !live) continue;
    const int o = slice.place(id);
    if (o < slice.first || o >= slice.end) continue;
    float pk = en.e[k];
    if (LOSS ? s.again != 0 : again) {   // a token named twice: all its entries write the same value
      pk = 0.f;
      for (int i = 0; i < K; ++i) pk += en.id[i] == id ? en.e[i] : 0.f;
    }
    const float z = en.z[k];
    dx[id] = from_float<T>(g * (W * exp2_approx(z - l) - pk * s.pscale) * (CAP ? 1.f - Z.flat * z * z : 1.f));
  }
}

static int dt_validate(const xl_distill_params* p) {
  if (!p || !p->logits || !p->values || !p->ids) return XL_ERR_NULL_POINTER;
  const int rc = vocab_validate(p->logits, p->rows, p->V, p->row_stride, p->cap, p->dtype);
  if (rc != XL_OK) return rc;
  if (p->K <= 0 || !vocab_temperature(p->temperature)) return XL_ERR_BAD_SHAPE;
  if (p->K > TOPK_MAX) return XL_ERR_TOO_LARGE;
  if ((p->stats && (reinterpret_cast<uintptr_t>(p->stats) & 7u)) || (p->dlogits && !vocab_aligned(p->dlogits, p->dtype))) return XL_ERR_BAD_ALIGNMENT;
  if (p->dlogits && p->rows > 1 && p->dlogits_stride < p->V) return XL_ERR_BAD_STRIDE;
  if (p->dlogits) {
    const uintptr_t size = p->dtype == XL_F32 ? 4 : 2, n = (uintptr_t)p->V * size, last = (uintptr_t)(p->rows - 1) * size;
    const uintptr_t a = reinterpret_cast<uintptr_t>(p->logits), b = reinterpret_cast<uintptr_t>(p->dlogits);
    if (a < b + last * (uintptr_t)p->dlogits_stride + n && b < a + last * (uintptr_t)p->row_stride + n) return XL_ERR_ALIASING;
  }
  return XL_OK;
}

// Blocks of a row: one, and with fewer than 592 rows up to eight slices of at least 2048 tokens, which exchange their sums through
// the cluster's shared memory (515 rows of 10 007 in fp32: 10 us whole, 13 in halves).
static int dt_blocks(int rows, int V) {
  int blocks = 1;
  while (blocks < DT_BLOCKS && rows * (blocks * 2) <= 4 * 148 && V >= 2048 * (blocks * 2)) blocks *= 2;
  return blocks;
}

template <typename T, bool CAP, bool BOUNDED, bool LOSS, bool GRAD> static int dt_go(const xl_distill_params* p, cudaStream_t st) {
  const int blocks = dt_blocks(p->rows, p->V);
  auto kern = distill_kernel<T, CAP, BOUNDED, LOSS, GRAD>;
  const size_t smem = dt_smem(p->K, p->V, Vec16<T>::N, blocks);
  // (one limit for all calls: the attribute is the kernel's, and another host thread may set it between here and the launch)
  if (smem > 40 * 1024) XL_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dt_smem(TOPK_MAX, VOCAB_MAX, Vec16<T>::N, 1)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p->rows * blocks);
  cfg.blockDim = dim3(dt_threads(LOSS && GRAD));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  XL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, *p, CappedZ<CAP>(p->cap, p->temperature), 1.0 / (double)p->temperature, blocks));
  return check_launch("xl_distill_topk");
}

template <typename T> static int dt_launch(const xl_distill_params* p, bool loss, cudaStream_t st) {
  const bool cap = p->cap > 0.f, bounded = vocab_bounded(p->cap, p->temperature);
  if (!loss) return cap ? dt_go<T, true, true, false, true>(p, st) : dt_go<T, false, false, false, true>(p, st);
  if (p->dlogits) {
    if (bounded) return dt_go<T, true, true, true, true>(p, st);
    return cap ? dt_go<T, true, false, true, true>(p, st) : dt_go<T, false, false, true, true>(p, st);
  }
  if (bounded) return dt_go<T, true, true, true, false>(p, st);
  return cap ? dt_go<T, true, false, true, false>(p, st) : dt_go<T, false, false, true, false>(p, st);
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
