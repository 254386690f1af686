// Distillation from a teacher's top logits: loss and gradient of a student's logits in one pass (sm_100a).
//
// Row r has student logits x [V], the teacher's logits t_k at K token ids j_k (the set J), optionally the log-sum-exp R
// of the teacher's other logits over tau, and a label y. With q = softmax(x / tau), q_0 the sum of q outside J and
// p the softmax of (t_1 / tau, ..., t_K / tau, R):
//
//   loss_r = (1 - h) tau^2 [ sum_k p_k (log p_k - log q_jk) + p_0 (log p_0 - log q_0) ] + h (lse(x) - x_y)
//   dx_v   = s [ (1 - h) tau (q_v - p_k) + h (softmax(x)_v - [v = y]) ]              v = j_k
//   dx_v   = s [ (1 - h) tau q_v (1 - p_0 / q_0) + h (softmax(x)_v - [v = y]) ]      v outside J
//
// and the loss is the mean over the rows that count; s is the gradient of the loss over their number.
//
// The sums run over the tokens outside J and over J apart: q_0 as 1 - sum q_jk would lose what a good student leaves to
// the others. The tokens of J are marked in shared memory and read as -inf in the pass over the row, which leaves their
// base gradient at zero; one thread for each entry then writes its gradient over it.
//
// A row is read once, into registers: a CTA of 512 threads holds up to 64 KB of it (NV vectors of 16 bytes a thread),
// a longer row is shared by a cluster of CTAs that exchange their maxima and sums through distributed shared memory.
#include <cooperative_groups.h>

#include "launch.cuh"
#include "logits.cuh"

namespace astrai {

namespace cg = cooperative_groups;

constexpr int DST_THREADS = 512;
constexpr int DST_WARPS = DST_THREADS / 32;
constexpr int DST_MAX_K = 1024;
constexpr int DST_KI = DST_MAX_K / DST_THREADS;  // entries of a thread
constexpr int DST_MAX_CLUSTER = 16;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct DistillArgs {
  const void* x;
  long long ldx;
  void* dx;
  long long lddx;
  const void* ids;     // [rows, K], int32 or int64
  int ids64;
  const void* values;  // [rows, K]
  int values_type;     // 0 bf16, 1 fp16, 2 fp32
  const float* rest;   // [rows] or null
  const long long* target;  // [rows] or null
  long long ignore;
  int rows, V, K, cluster;
  float inv_tau, kl_loss, kl_grad, hard;  // 1 / tau, (1 - h) tau^2, (1 - h) tau, h
  const float* count;     // rows that count, null: all
  const float* grad;      // gradient of the loss, null: `expected`
  float expected;
  int unless_expected;    // nothing is done if *grad == expected
  float* row_loss;        // null: not wanted
};

__device__ __forceinline__ bool row_counts(const long long* target, long long ignore, int row, int V, long long& y) {
  y = -1;
  if (!target) return true;
  y = target[row];
  return y != ignore && y >= 0 && y < V;
}

// Several values of every thread reduced over the CTA, the same result in all threads: MAX of them as maxima, the others as
// sums in a fixed order. `part` holds N floats per warp; a barrier separates two uses of it.
template <int N, bool MAX>
__device__ __forceinline__ void block_reduce(float (&v)[N], float* part) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = MAX ? warp_max(v[i]) : warp_sum(v[i]);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) part[i * DST_WARPS + w] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = part[i * DST_WARPS + (lane & (DST_WARPS - 1))];
#pragma unroll
    for (int o = DST_WARPS / 2; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffff, v[i], o);
      v[i] = MAX ? fmaxf(v[i], u) : v[i] + u;
    }
  }
}

__device__ __forceinline__ float teacher_value(const DistillArgs& a, long long i) {
  if (a.values_type == 0) return __bfloat162float(static_cast<const __nv_bfloat16*>(a.values)[i]);
  if (a.values_type == 1) return __half2float(static_cast<const __half*>(a.values)[i]);
  return static_cast<const float*>(a.values)[i];
}

// a finite reference for a maximum
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }

// The student's mass at one temperature: outside J and on J as sums of 2^((x - ref) c), joined. With d = (J's reference -
// that outside) c and m = max(d, 0), `sum` is all of it relative to 2^m at the reference outside: neither part overflows.
struct Mass {
  float outside, d, m, sum;
  __device__ Mass(float outside_, float on, float d_) : outside(outside_), d(d_), m(fmaxf(d_, 0.f)) {
    sum = outside * exp2_fast(-m) + on * exp2_fast(d - m);
  }
  __device__ float log2_all_over_outside() const { return m + log2f(sum) - log2f(outside); }  // -log2 q_0
  __device__ float log2_rel_outside() const { return m + log2f(sum); }  // of all of it, relative to each reference
  __device__ float log2_rel_on() const { return m - d + log2f(sum); }
  __device__ float inv_rel_outside() const { return exp2_fast(-m) / sum; }  // 1 / all of it, relative to each reference
  __device__ float inv_rel_on() const { return exp2_fast(d - m) / sum; }
};

template <typename T, int NV, bool TRAIN, bool TWO>
__global__ void __launch_bounds__(DST_THREADS, 2) distill_kernel(const DistillArgs a) {
  constexpr int E = LogitType<T>::E;
  __shared__ __align__(4) uint8_t mask[DST_THREADS * NV];
  __shared__ float part_max[3 * DST_WARPS], part_sum[6 * DST_WARPS];
  __shared__ float mine[6];
  __shared__ int twice;
  const int t = threadIdx.x;
  const int cs = a.cluster, rank = cs > 1 ? (int)cg::this_cluster().block_rank() : 0;
  const int row = blockIdx.x / cs;
  begin_early();
  float g = a.expected;
  if (a.grad) {
    g = *a.grad;
    if (a.unless_expected && g == a.expected) return;
  }
  const T* x = static_cast<const T*>(a.x) + (long long)row * a.ldx;
  T* dx = TRAIN ? static_cast<T*>(a.dx) + (long long)row * a.lddx : nullptr;
  const RowVecs<T> vecs(x, a.V);
  const int per = (vecs.n + cs - 1) / cs, v0 = rank * per, v1 = min(v0 + per, vecs.n);
  long long y;
  if (!row_counts(a.target, a.ignore, row, a.V, y)) {  // the same for the whole cluster
    if constexpr (TRAIN)
      for (int v = v0 + t; v < v1; v += DST_THREADS) vecs.store(dx, v, make_uint4(0, 0, 0, 0));
    if (a.row_loss && rank == 0 && t == 0) a.row_loss[row] = 0.f;
    return;
  }

  uint4 u[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = v0 + t + i * DST_THREADS;
    u[i] = v < v1 ? vecs.load(v) : vec_neg_inf<T>();
  }
  const auto id_at = [&](int k) -> long long {
    const long long at = (long long)row * a.K + k;
    return a.ids64 ? static_cast<const long long*>(a.ids)[at] : static_cast<const int*>(a.ids)[at];
  };
  int id[DST_KI];
  float tv[DST_KI], xj[DST_KI];
#pragma unroll
  for (int i = 0; i < DST_KI; ++i) {
    const int k = t + i * DST_THREADS;
    id[i] = -1;
    tv[i] = xj[i] = -INFINITY;
    if (k < a.K) {
      const long long j = id_at(k);
      if (j >= 0 && j < a.V) {
        id[i] = (int)j;
        tv[i] = teacher_value(a, (long long)row * a.K + k) * a.inv_tau;
        xj[i] = LogitType<T>::one(x[j]);
      }
    }
  }
  const float rest = a.rest ? a.rest[row] : -INFINITY;
  const float xy = y >= 0 ? LogitType<T>::one(x[y]) : 0.f;
  for (int i = t; i < DST_THREADS * NV / 4; i += DST_THREADS) reinterpret_cast<uint32_t*>(mask)[i] = 0;
  if (t == 0) twice = 0;
  __syncthreads();
  // marks of the entries in this CTA's part of the row
  bool here[DST_KI], first[DST_KI];
#pragma unroll
  for (int i = 0; i < DST_KI; ++i) {
    const int v = (id[i] + vecs.head) / E;
    first[i] = here[i] = id[i] >= 0 && v >= v0 && v < v1;
    if (here[i]) {
      const uint32_t b = 1u << (8 * ((v - v0) & 3) + (id[i] + vecs.head) % E);
      if (atomicOr(reinterpret_cast<uint32_t*>(mask) + (v - v0) / 4, b) & b) twice = 1;
    }
  }
  __syncthreads();
  if (twice) {  // an id that comes again: the student's mass there counts once, with the first of them
#pragma unroll 1
    for (int i = 0; i < DST_KI; ++i)
      for (int l = 0; first[i] && l < t + i * DST_THREADS; ++l)
        if (id_at(l) == id[i]) first[i] = false;
  }

  const float c = a.inv_tau * LOG2E;
  float mx[3] = {rest, -INFINITY, -INFINITY};  // teacher; student on J, outside J
#pragma unroll
  for (int i = 0; i < DST_KI; ++i) {
    mx[0] = fmaxf(mx[0], tv[i]);
    mx[1] = fmaxf(mx[1], xj[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t bits = mask[t + i * DST_THREADS];
    if (bits) vec_mask<T>(u[i], bits);
    float f[E];
    vec_floats<T>(u[i], f);
#pragma unroll
    for (int e = 0; e < E; ++e) mx[2] = fmaxf(mx[2], f[e]);
  }
  block_reduce<3, true>(mx, part_max);
  const float mt = ref_of(mx[0]), mj = ref_of(mx[1]), mr = ref_of(mx[2]);

  // teacher's mass on J; sum of its mass * (log p - log q) up to constants; student's sums on J and outside, over tau and
  // at 1
  float sum[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float pe[DST_KI];
#pragma unroll
  for (int i = 0; i < DST_KI; ++i) {
    const float th = tv[i] - mt, zh = (xj[i] - mj) * a.inv_tau;
    pe[i] = id[i] >= 0 ? exp2_fast(th * LOG2E) : 0.f;
    sum[0] += pe[i];
    if (pe[i] != 0.f) sum[1] += pe[i] * (th - zh);
    if (first[i]) {
      sum[2] += exp2_fast(zh * LOG2E);
      if constexpr (TWO) sum[3] += exp2_fast((xj[i] - mj) * LOG2E);
    }
  }
  float mo = mr;  // the logit that the sums outside J are relative to
  const Pair c2(c, c), log2e2(LOG2E, LOG2E);
  {
    const Pair ref2(-mo, -mo);
    Pair s2(0.f, 0.f), s1(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pair p[E / 2];
      vec_pairs<T>(u[i], p);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const Pair d = p[e] + ref2;
        s2 = s2 + exp2_fast(d * c2);
        if constexpr (TWO) s1 = s1 + exp2_fast(d * log2e2);
      }
    }
    sum[4] = s2.sum();
    if constexpr (TWO) sum[5] = s1.sum();
  }
  block_reduce<6, false>(sum, part_sum);

  float on = sum[2], on1 = sum[3], out = sum[4], out1 = sum[5];
  if (cs > 1) {  // the sums of all CTAs, those outside J relative to this one's reference
    cg::cluster_group cl = cg::this_cluster();
    if (t == 0) {
      mine[0] = mx[2];
      mine[1] = out;
      mine[2] = out1;
      mine[3] = on;
      mine[4] = on1;
    }
    cl.sync();
    const int lane = t & 31;
    const float* theirs = cl.map_shared_rank(mine, lane < cs ? lane : 0);
    const float m = lane < cs ? theirs[0] : -INFINITY;
    if (mx[2] == -INFINITY) mo = ref_of(warp_max(m));  // none of its own: one that others have
    const bool some = m != -INFINITY;
    out = warp_sum(some ? theirs[1] * exp2_fast((m - mo) * c) : 0.f);
    if constexpr (TWO) out1 = warp_sum(some ? theirs[2] * exp2_fast((m - mo) * LOG2E) : 0.f);
    on = warp_sum(lane < cs ? theirs[3] : 0.f);
    if constexpr (TWO) on1 = warp_sum(lane < cs ? theirs[4] : 0.f);
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  if (out == 0.f) mo = mj;  // nothing outside J
  const Mass z(out, on, on == 0.f ? -INFINITY : (mj - mo) * c);
  const Mass z1(TWO ? out1 : out, TWO ? on1 : on, on == 0.f ? -INFINITY : (mj - mo) * (TWO ? LOG2E : c));
  // the teacher's share outside J
  const float pr = rest == -INFINITY ? 0.f : exp2_fast((rest - mt) * LOG2E);
  const float mass = sum[0] + pr, inv = mass != 0.f ? 1.f / mass : 0.f;
  const float p0 = pr * inv;

  if (a.row_loss && rank == 0 && t == 0) {
    // sum_k p_k (log p_k - log q_jk) = (sum e_k (th - zh)) / mass + (sum of p_k) (log of q's sum - log mass)
    float loss = 0.f;
    if (mass != 0.f) {
      const float logm = logf(mass);
      if (sum[0] != 0.f) loss = sum[1] * inv + sum[0] * inv * (z.log2_rel_on() * LN2 - logm);
      if (p0 != 0.f) loss += p0 * ((rest - mt) - logm + z.log2_all_over_outside() * LN2);
      loss *= a.kl_loss;
    }
    if (a.hard > 0.f) loss += a.hard * ((mo - xy) + z1.log2_rel_outside() * LN2);
    a.row_loss[row] = loss;
  }
  if constexpr (TRAIN) {
    const float s = g / (a.count ? fmaxf(*a.count, 1.f) : (float)max(a.rows, 1));
    const float all = mass != 0.f ? 1.f : 0.f;
    const float kl = s * a.kl_grad, ce = s * a.hard;
    const float share = out != 0.f ? p0 / out : 0.f;
    const float base = kl * (all * z.inv_rel_outside() - share) + (TWO ? 0.f : ce * z.inv_rel_outside());
    const float base1 = TWO ? ce * z1.inv_rel_outside() : 0.f;
    const Pair ref2(-mo, -mo), base2(base, base), base12(base1, base1);
    const auto outside = [&](Pair p) {
      p = p + ref2;
      const Pair d = base2 * exp2_fast(p * c2);
      if constexpr (TWO) return fma2(base12, exp2_fast(p * log2e2), d);
      return d;
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = v0 + t + i * DST_THREADS;
      if (v >= v1) break;
      Pair p[E / 2];
      vec_pairs<T>(u[i], p);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) p[e] = outside(p[e]);
      vecs.store(dx, v, pairs_round<T>(p));
    }
    __syncthreads();  // the base gradient lies before the entries' gradients
#pragma unroll 1
    for (int i = 0; i < DST_KI; ++i) {
      if (!here[i]) continue;
      float p = pe[i] * inv;
      if (twice) {  // the teacher's mass of all entries with this id, the same whichever of them writes it
        p = 0.f;
        for (int l = 0; l < a.K; ++l)
          if (id_at(l) == id[i])
            p += exp2_fast((teacher_value(a, (long long)row * a.K + l) * a.inv_tau - mt) * LOG2E) * inv;
      }
      const float q = exp2_fast((xj[i] - mj) * c) * z.inv_rel_on();
      const float q1 = TWO ? exp2_fast((xj[i] - mj) * LOG2E) * z1.inv_rel_on() : q;
      dx[id[i]] = LogitType<T>::round(kl * (q * all - p) + ce * (q1 - (id[i] == y ? 1.f : 0.f)));
    }
    if (t == 0 && y >= 0 && ce != 0.f) {
      const int v = ((int)y + vecs.head) / E, bit = ((int)y + vecs.head) % E;
      if (v >= v0 && v < v1 && !(mask[v - v0] >> bit & 1)) dx[y] = LogitType<T>::round(outside(Pair(xy, xy)).get().x - ce);
    }
  }
  if (cs > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // others may still read `mine`
}

// count[0] = rows that count
__global__ void __launch_bounds__(1024) distill_count_kernel(const long long* target, long long ignore, int rows, int V,
                                                             float* count) {
  __shared__ int part[32];
  begin_early();
  int n = 0;
  long long y;
  for (int r = threadIdx.x; r < rows; r += 1024) n += row_counts(target, ignore, r, V, y);
  n = __reduce_add_sync(0xffffffff, n);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x < 32) {
    n = __reduce_add_sync(0xffffffff, part[threadIdx.x]);
    if (threadIdx.x == 0) *count = (float)n;
  }
}

// loss = sum of the rows' losses / count, in a fixed order
__global__ void __launch_bounds__(1024) distill_mean_kernel(const float* row_loss, int rows, const float* count,
                                                            float* loss) {
  __shared__ double part[32];
  begin_early();
  double s = 0.;
  for (int r = threadIdx.x; r < rows; r += 1024) s += row_loss[r];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffff, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = part[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffff, s, o);
    if (threadIdx.x == 0) *loss = (float)(s / (count ? fmaxf(*count, 1.f) : (float)max(rows, 1)));
  }
}

template <typename T, int NV, bool TRAIN, bool TWO>
void distill_launch(const DistillArgs& a, cudaStream_t s) {
  auto* kernel = distill_kernel<T, NV, TRAIN, TWO>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a.rows * a.cluster);
  cfg.blockDim = dim3(DST_THREADS);
  cfg.stream = s;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = a.cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.cluster > 1 ? 2 : 1;
  if (a.cluster > 8) cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  note_launch();
  cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, bool TRAIN, bool TWO>
void distill_sized(DistillArgs a, cudaStream_t s) {
  constexpr int E = LogitType<T>::E;
  const int vecs = (a.V + E - 1) / E + 1;  // one more where a row starts off the grid
  int cs = 1;
  while ((vecs + cs - 1) / cs > DST_THREADS * 8) cs *= 2;
  a.cluster = cs;
  const int per = (vecs + cs - 1) / cs;
  if (per <= DST_THREADS) return distill_launch<T, 1, TRAIN, TWO>(a, s);
  if (per <= DST_THREADS * 2) return distill_launch<T, 2, TRAIN, TWO>(a, s);
  if (per <= DST_THREADS * 4) return distill_launch<T, 4, TRAIN, TWO>(a, s);
  distill_launch<T, 8, TRAIN, TWO>(a, s);
}

template <typename T>
void distill_typed(const DistillArgs& a, cudaStream_t s) {
  const bool two = a.hard > 0.f && a.inv_tau != 1.f;
  if (a.dx)
    two ? distill_sized<T, true, true>(a, s) : distill_sized<T, true, false>(a, s);
  else
    two ? distill_sized<T, false, true>(a, s) : distill_sized<T, false, false>(a, s);
}

}  // namespace astrai

namespace astrai_host {
using namespace astrai;

int distill_max_k() { return DST_MAX_K; }
// longest row for elements of this size
int distill_max_vocab(int elem) { return DST_MAX_CLUSTER * DST_THREADS * 8 * (16 / elem) - 16 / elem; }

void distill(const void* x, long long ldx, void* dx, long long lddx, const void* ids, bool ids64, const void* values,
             int values_type, const float* rest, const long long* target, long long ignore, int rows, int V, int K,
             float tau, float hard, const float* grad, float expected, bool unless_expected, float* row_loss,
             float* count, bool have_count, float* loss, int dtype, cudaStream_t s) {
  if (target && !have_count)
    launch_early(distill_count_kernel, dim3(1), dim3(1024), 0, s, target, ignore, rows, V, count);
  DistillArgs a{x, ldx, dx, lddx, ids, ids64, values, values_type, rest, target, ignore, rows, V, K, 1, 1.f / tau,
                (1.f - hard) * tau * tau, (1.f - hard) * tau, hard, target ? count : nullptr, grad, expected,
                unless_expected, row_loss};
  if (rows > 0) {
    if (dtype == 0) distill_typed<__nv_bfloat16>(a, s);
    else if (dtype == 1) distill_typed<__half>(a, s);
    else distill_typed<float>(a, s);
  }
  if (loss)
    launch_early(distill_mean_kernel, dim3(1), dim3(1024), 0, s, (const float*)row_loss, rows,
                 (const float*)(target ? count : nullptr), loss);
}

}  // namespace astrai_host
