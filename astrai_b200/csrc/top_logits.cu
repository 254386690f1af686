// The k largest logits of each row in order, and the log-sum-exp of all others (sm_100a).
//
// Equal logits rank by id, the lowest first; a NaN ranks above every number. `rest` is log sum exp(x_v / tau) over the
// tokens that are not among the k.
//
// A row is read once, into registers: a CTA of 512 threads holds up to 64 KB of it, a longer row is shared by a cluster.
// Nothing is sorted but a few candidates. Every warp finds the j-th largest of its 32 threads' maxima, and the smallest of
// those over the G warps of the row is a bound that at least G j >= k logits reach: for k = 64 of 32000 about 150 do. Those
// become candidates in shared memory, ranked by comparing each with all, and read as -inf in the sum over the rest of the
// row. Where more than TOP_CAP logits reach the bound (ties), the exact k-th largest and the id that cuts its ties are found
// by bisection, and the row is read again.
#include <cooperative_groups.h>

#include "launch.cuh"
#include "logits.cuh"

namespace astrai {

namespace cg = cooperative_groups;

constexpr int TOP_THREADS = 512;
constexpr int TOP_WARPS = TOP_THREADS / 32;
constexpr int TOP_MAX_K = 256;
constexpr int TOP_CAP = 1024;
constexpr int TOP_MAX_CLUSTER = 16;

struct TopArgs {
  const void* x;
  long long ldx;
  int rows, V, k, cluster;
  float inv_tau;
  int* ids;      // [rows, k]
  void* values;  // [rows, k]
  float* rest;   // [rows]
};

struct TopShared {
  unsigned long long list[TOP_CAP];  // key, then the id's complement: greater ranks first
  float left[TOP_CAP];                     // logits of candidates that are not among the k
  uint32_t bound[TOP_WARPS], most[TOP_WARPS];
  float part[TOP_WARPS];
  int counts[TOP_WARPS];
  uint32_t cluster_bound;
  int cluster_count;
  int n;                                   // the leader's: candidates of the row
  float max_of[TOP_MAX_CLUSTER], sum_of[TOP_MAX_CLUSTER];  // the leader's: each CTA's part of the rest
};

// Sum over the row's threads, the same in all of them.
__device__ __forceinline__ int row_count(TopShared& sh, int n, int cs) {
  n = __reduce_add_sync(0xffffffff, n);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.counts[threadIdx.x >> 5] = n;
  __syncthreads();
  n = __reduce_add_sync(0xffffffff, (threadIdx.x & 31) < TOP_WARPS ? sh.counts[threadIdx.x & 31] : 0);
  if (cs == 1) return n;
  cg::cluster_group cl = cg::this_cluster();
  if (threadIdx.x == 0) sh.cluster_count = n;
  cl.sync();
  n = 0;
  for (int i = 0; i < cs; ++i) n += *cl.map_shared_rank(&sh.cluster_count, i);
  cl.sync();
  return n;
}

template <typename T, int NV>
__global__ void __launch_bounds__(TOP_THREADS, 2) top_logits_kernel(const TopArgs a) {
  constexpr int E = LogitType<T>::E;
  __shared__ TopShared sh;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int cs = a.cluster, rank = cs > 1 ? (int)cg::this_cluster().block_rank() : 0;
  const int row = blockIdx.x / cs;
  begin_early();
  const RowVecs<T> vecs(static_cast<const T*>(a.x) + (long long)row * a.ldx, a.V);
  const int per = (vecs.n + cs - 1) / cs, v0 = rank * per, v1 = min(v0 + per, vecs.n);
  uint4 u[NV];
  float most[NV];
  const auto load = [&] {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = v0 + t + i * TOP_THREADS;
      u[i] = v < v1 ? vecs.load(v) : vec_neg_inf<T>();
    }
  };
  load();
  if (t == 0) sh.n = 0;
  TopShared* lead = &sh;
  if (cs > 1) lead = cg::this_cluster().map_shared_rank(&sh, 0);

  // The bound: warps whose lanes all hold logits, the last CTA's may be fewer.
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    most[i] = vec_max<T>(u[i]);
    top = max_nan(top, most[i]);
  }
  const int tail = vecs.n - (cs - 1) * per;  // vectors of the last CTA
  const auto full = [&](int n) { return min(max(n, 0) / 32, TOP_WARPS); };
  const int warps = (cs - 1) * full(per) + full(tail);
  const int j = warps > 0 ? (a.k + warps - 1) / warps : 33;
  uint32_t key = key_of(top), bound = 0xFFFFFFFFu;
  if (j > 32) {
    bound = 0;
  } else if (w < full(v1 - v0)) {
    for (int i = 0;; ++i) {
      bound = __reduce_max_sync(0xffffffff, key);
      if (i == j - 1) break;
      if (lane == __ffs(__ballot_sync(0xffffffff, key == bound)) - 1) key = 0;
    }
  }
  if (lane == 0) sh.bound[w] = bound;
  __syncthreads();
  bound = __reduce_min_sync(0xffffffff, sh.bound[lane & (TOP_WARPS - 1)]);
  if (cs > 1) {
    cg::cluster_group cl = cg::this_cluster();
    if (t == 0) sh.cluster_bound = bound;
    cl.sync();
    bound = __reduce_min_sync(0xffffffff, *cl.map_shared_rank(&sh.cluster_bound, lane < cs ? lane : 0));
  }

  int cut = a.V;  // of the logits equal to the bound, those with smaller ids
  for (int attempt = 0;; ++attempt) {
    // Candidates out of the row; the largest logit that stays, and its sum.
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (key_of(most[i]) >= bound) {
        const int v = v0 + t + i * TOP_THREADS, at = vecs.first(v);
        float f[E];
        vec_floats<T>(u[i], f);
        uint32_t out = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t ke = key_of(f[e]);
          const int id = at + e;
          if (ke < bound || (ke == bound && id >= cut) || id < 0 || id >= a.V || v >= v1) continue;
          out |= 1u << e;
          const int slot = atomicAdd(&lead->n, 1);
          if (slot < TOP_CAP) lead->list[slot] = (unsigned long long)ke << 32 | (uint32_t)~id;
        }
        vec_mask<T>(u[i], out);
        mx = max_nan(mx, vec_max<T>(u[i]));
      } else {
        mx = fmaxf(mx, most[i]);
      }
    }
    uint32_t km = __reduce_max_sync(0xffffffff, key_of(mx));
    if (lane == 0) sh.most[w] = km;
    __syncthreads();
    km = __reduce_max_sync(0xffffffff, sh.most[lane & (TOP_WARPS - 1)]);
    mx = of_key(km);
    const float c = a.inv_tau * 1.4426950408889634f, ref = mx == -INFINITY ? 0.f : mx;
    const Pair c2(c, c), ref2(-ref, -ref);
    Pair s2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pair p[E / 2];
      vec_pairs<T>(u[i], p);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) s2 = s2 + exp2_fast((p[e] + ref2) * c2);
    }
    float s = warp_sum(s2.sum());
    if (lane == 0) sh.part[w] = s;
    __syncthreads();
    if (t == 0) {
      s = 0.f;
      for (int i = 0; i < TOP_WARPS; ++i) s += sh.part[i];
      lead->max_of[rank] = mx;
      lead->sum_of[rank] = s;
    }
    if (cs > 1) cg::this_cluster().sync();
    else __syncthreads();
    const int n = lead->n;
    if (n <= TOP_CAP) break;
    // Too many. The exact k-th largest key, and the id up to which the logits equal to it are taken.
    const auto count = [&](uint32_t more_than, uint32_t equal, int below) {  // keys above, and equal ones with ids below
      int got = 0;
#pragma unroll 1
      for (int v = v0 + t; v < v1; v += TOP_THREADS) {
        const int at = vecs.first(v);
        float f[E];
        vec_floats<T>(vecs.load(v), f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t ke = key_of(f[e]);
          const int id = at + e;
          got += id >= 0 && id < a.V && (ke > more_than || (ke == equal && id < below));
        }
      }
      return row_count(sh, got, cs);
    };
    uint32_t kth = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
      const uint32_t next = kth | 1u << b;
      if (count(next, next, a.V) >= a.k) kth = next;
    }
    int low = 0;  // fewer than k are above, or equal with an id below `low`
#pragma unroll 1
    for (int b = 31 - __clz(a.V); b >= 0; --b)
      if (low + (1 << b) <= a.V && count(kth, kth, low + (1 << b)) < a.k) low += 1 << b;
    bound = kth;
    cut = low + 1;
    load();
#pragma unroll
    for (int i = 0; i < NV; ++i) most[i] = of_key(0xFFFFFFFFu);  // every vector may hold a candidate
    if (rank == 0 && t == 0) sh.n = 0;
    if (cs > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  if (rank > 0) {  // the leader stays until its memory has been read
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    return;
  }
  if (cs > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

  // Ranks: four threads for each candidate compare it with a quarter of the others.
  const int n = sh.n, quarter = t & 3;
  float mx = -INFINITY, s = 0.f;
  for (int i = 0; i < cs; ++i) {
    if (sh.max_of[i] == -INFINITY) continue;
    const float m = max_nan(mx, sh.max_of[i]);
    s = s * exp2_fast((mx - m) * a.inv_tau * 1.4426950408889634f) +
        sh.sum_of[i] * exp2_fast((sh.max_of[i] - m) * a.inv_tau * 1.4426950408889634f);
    mx = m;
  }
  float left_max = -INFINITY;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += TOP_THREADS / 4) {
    const int i = i0 + t / 4;
    const unsigned long long mine = i < n ? sh.list[i] : 0;
    int r = 0;
    for (int l = quarter; l < n; l += 4) r += sh.list[l] > mine;
    r += __shfl_xor_sync(0xffffffff, r, 1);
    r += __shfl_xor_sync(0xffffffff, r, 2);
    if (i >= n || quarter != 0) continue;
    const float value = of_key((uint32_t)(mine >> 32));
    if (r < a.k) {
      const long long at = (long long)row * a.k + r;
      a.ids[at] = (int)~(uint32_t)mine;
      static_cast<T*>(a.values)[at] = LogitType<T>::round(value);
    } else {
      sh.left[r - a.k] = value;  // by rank: the order in which candidates came must not reach the sum
      left_max = max_nan(left_max, value);
    }
  }
  // the candidates that are not among the k
  uint32_t kl = __reduce_max_sync(0xffffffff, key_of(left_max));
  if (lane == 0) sh.bound[w] = kl;
  __syncthreads();
  left_max = of_key(__reduce_max_sync(0xffffffff, sh.bound[lane & (TOP_WARPS - 1)]));
  const float m = max_nan(mx, left_max), ref = m == -INFINITY ? 0.f : m;
  const float c = a.inv_tau * 1.4426950408889634f;
  float sl = 0.f;
  for (int i = t; i < n - a.k; i += TOP_THREADS) sl += exp2_fast((sh.left[i] - ref) * c);
  sl = warp_sum(sl);
  if (lane == 0) sh.part[w] = sl;
  __syncthreads();
  if (t == 0) {
    s *= exp2_fast((mx - ref) * c);
    for (int i = 0; i < TOP_WARPS; ++i) s += sh.part[i];
    a.rest[row] = isinf(m) ? m : fmaf(ref, a.inv_tau, logf(s));
  }
  if (cs > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int NV>
void top_launch(const TopArgs& a, cudaStream_t s) {
  auto* kernel = top_logits_kernel<T, NV>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a.rows * a.cluster);
  cfg.blockDim = dim3(TOP_THREADS);
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

template <typename T>
void top_sized(TopArgs a, cudaStream_t s) {
  constexpr int E = LogitType<T>::E;
  const int vecs = (a.V + E - 1) / E + 1;  // one more where a row starts off the grid
  int cs = 1;
  while ((vecs + cs - 1) / cs > TOP_THREADS * 8) cs *= 2;
  a.cluster = cs;
  const int per = (vecs + cs - 1) / cs;
  if (per <= TOP_THREADS) return top_launch<T, 1>(a, s);
  if (per <= TOP_THREADS * 2) return top_launch<T, 2>(a, s);
  if (per <= TOP_THREADS * 4) return top_launch<T, 4>(a, s);
  top_launch<T, 8>(a, s);
}

}  // namespace astrai

namespace astrai_host {
using namespace astrai;

int top_logits_max_k() { return TOP_MAX_K; }
// longest row for elements of this size
int top_logits_max_vocab(int elem) { return TOP_MAX_CLUSTER * TOP_THREADS * 8 * (16 / elem) - 16 / elem; }

void top_logits(const void* x, long long ldx, int rows, int V, int k, float tau, int* ids, void* values, float* rest,
                int dtype, cudaStream_t s) {
  const TopArgs a{x, ldx, rows, V, k, 1, 1.f / tau, ids, values, rest};
  if (dtype == 0) top_sized<__nv_bfloat16>(a, s);
  else if (dtype == 1) top_sized<__half>(a, s);
  else top_sized<float>(a, s);
}

}  // namespace astrai_host
