// The k largest logits of each row in order, and the log-sum-exp of all others (sm_100a).
//
// Equal logits rank by id, the lowest first; a NaN ranks above every number. `rest` is log sum exp(x_v / tau) over the
// tokens that are not among the k.
//
// A CTA takes a row and reads it twice, from memory and then from L2. Nothing is sorted but a few candidates: in the first
// reading the largest logits of both halves of every thread's part make 64 numbers a warp, and the smallest, over the W warps,
// of each warp's j-th largest is a bound that at least W j >= k logits reach (for k = 64 of 32000 about 100 do). The second
// reading finds those and sums the others, relative to the bound, for `rest`; the candidates that do not make it are added.
// Where more than TOP_CAP logits reach the bound, the exact k-th largest and the id that cuts its ties are found by bisection,
// in some fifty passes over the row. That is so with ties; and with 128 threads a row, whose 4 warps have 256 numbers for the
// bound, where k comes near 256: 8192 rows of 32000 bf16 take 338 us at k = 200, 439 at 224, 1890 at 240, 5800 at 248 and 12500
// at 256 (8192 rows of 16000 fp32: 296, 385, 1200, 2860, 6550), 999 rows of 50021 fp32 with 512 threads 104 and 112 at 200 and
// 256.
//
// What bounds it is a row's chain of steps with a barrier behind each, so small CTAs of 64 registers a thread, 32 warps of them
// on an SM, hide most of it: 8192 rows of 32000 bf16, k = 64, take 195 us (2.7 TB/s of what has to be read; the
// exponentials alone, 16 a clock and SM, 58 us) with 128 threads a row, 225 with 256 and 346 with 512. Rows kept in shared memory
// between the readings left room for 24 warps and took 261 us. More threads take a row where there are too few rows to fill
// the GPU, or where the rows of all CTAs at a time would not stay in L2 (2048 rows of 50021 bf16: 128 threads 119 us, 256 threads
// 107 us; 999 rows of 50021 fp32: 125 us, and 107 with 512).
#include <algorithm>

#include "launch.cuh"
#include "logits.cuh"

namespace astrai {

constexpr int TOP_MAX_K = 256;
constexpr int TOP_CAP = 1024;
constexpr long long TOP_L2 = 96ll << 20;  // bytes of rows that stay in L2 between a row's two readings

struct TopArgs {
  const void* x;
  long long ldx;
  int rows, V, k;
  float inv_tau;
  int* ids;      // [rows, k]
  void* values;  // [rows, k]
  float* rest;   // [rows]
};

struct TopShared {
  unsigned long long list[TOP_CAP];  // key, then the id's complement: greater ranks first
  float left[TOP_CAP];                   // logits of candidates that are not among the k
  uint32_t vecs[TOP_CAP];                // vectors that hold candidates
  uint32_t part[2][32];
  float sum[32];
  int n;
};

template <typename T, int NT>
struct TopRow {
  static constexpr int E = LogitType<T>::E, W = NT / 32;
  TopShared& sh;
  RowVecs<T> vecs;
  int chunk, w0, mine;  // a warp's vectors, this thread's: w0 + i * 32 + lane
  int turn = 0;
  float below = 0.f;  // this thread's sum of 2^((x - bound) c) over the logits below gather()'s bound

  __device__ __forceinline__ void load(int i, uint4 (&u)[4]) const { vecs.load(w0 + i * 32, chunk / 32 - i, mine - i, u); }
  __device__ int first(int i) const { return vecs.first(w0 + i * 32 + (threadIdx.x & 31)); }
  // f(vector, its number), four in flight; some behind the last read as -inf
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int i = 0; i < mine; i += 4) {
      uint4 u[4];
      load(i, u);
#pragma unroll
      for (int j = 0; j < 4; ++j) f(u[j], i + j);
    }
  }
  // over the CTA, the same in all threads
  template <typename F>
  __device__ __forceinline__ uint32_t reduce(uint32_t v, F f) {
    v = f(v);
    if ((threadIdx.x & 31) == 0) sh.part[turn][threadIdx.x >> 5] = v;
    __syncthreads();
    v = f(sh.part[turn][threadIdx.x & (W - 1)]);
    turn ^= 1;
    return v;
  }
  __device__ uint32_t max_of(uint32_t v) {
    return reduce(v, [](uint32_t x) { return __reduce_max_sync(0xffffffff, x); });
  }
  __device__ uint32_t min_of(uint32_t v) {
    return reduce(v, [](uint32_t x) { return __reduce_min_sync(0xffffffff, x); });
  }
  __device__ int count_of(int n) {
    return (int)reduce((uint32_t)n, [](uint32_t x) { return __reduce_add_sync(0xffffffff, x); }) / (32 / W);
  }
  // The place in a list of this thread's `mine` entries, by thread; `n`, what the list has, counts on.
  __device__ __forceinline__ int place(int& n, int mine) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int before = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(0xffffffff, before, d);
      if (lane >= d) before += other;
    }
    if (lane == 31) sh.part[turn][w] = before;
    __syncthreads();
    const int of_warp = lane < W ? (int)sh.part[turn][lane] : 0;
    turn ^= 1;
    const int at = n + before - mine + __reduce_add_sync(0xffffffff, lane < w ? of_warp : 0);
    n += __reduce_add_sync(0xffffffff, of_warp);
    return at;
  }
  __device__ float sum_of(float s) {
    s = warp_sum(s);
    if ((threadIdx.x & 31) == 0) sh.sum[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += sh.sum[i];
    __syncthreads();
    return s;
  }
  // Keys above `more_than`, and those equal to it with ids below `below`.
  __device__ __noinline__ int count(uint32_t more_than, int below) {
    int n = 0;
    each([&](const uint4& u, int i) {
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t key = key_of(x[e]);
        const int id = first(i) + e;
        n += i < mine && id >= 0 && id < vecs.V && (key > more_than || (key == more_than && id < below));
      }
    });
    return count_of(n);
  }
  // Candidates: keys from `bound` on; their number, or more than TOP_CAP. First the vectors that hold any, then those vectors'
  // elements: a warp in which a few lanes look at eight elements each takes as long as if all did. A thread marks its vectors
  // in a word first, and the CTA takes its places in the list at once: at 64 of 32000 nearly every warp has some in every turn.
  // Both steps sum what is below the bound. The lists are in the threads' order, so that the sum's order is always the same.
  __device__ __noinline__ int gather(uint32_t bound, float c) {
    const int t = threadIdx.x;
    const float edge = of_key(bound);
    const Pair edge2(-edge, -edge), c2(c, c);
    Pair sum(0.f, 0.f);
    int n_vecs = 0, n = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < chunk / 32; i0 += 32) {
      uint32_t marks = 0;
#pragma unroll 1
      for (int i = i0; i < min(i0 + 32, chunk / 32); i += 4) {
        uint4 u[4];
        load(i, u);
        uint32_t some4 = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool some = !(vec_max<T>(u[j]) < edge);  // a NaN too
          some4 |= (uint32_t)some << j;
          Pair x[E / 2];
          vec_pairs<T>(u[j], x);
          Pair s = exp2_fast((x[0] + edge2) * c2);
#pragma unroll
          for (int e = 1; e < E / 2; ++e) s = s + exp2_fast((x[e] + edge2) * c2);
          if (!some) sum = sum + s;
        }
        marks |= some4 << (i - i0);
      }
      if (mine - i0 < 32) marks &= (1u << max(mine - i0, 0)) - 1;
      int to = place(n_vecs, __popc(marks));
#pragma unroll 1
      for (; marks && to < TOP_CAP; marks &= marks - 1) sh.vecs[to++] = (i0 + __ffs(marks) - 1) * NT + t;
    }
    if (n_vecs > TOP_CAP) return TOP_CAP + 1;
    __syncthreads();
#pragma unroll 1
    for (int q0 = 0; q0 < n_vecs; q0 += NT) {
      const int q = q0 + t;
      uint32_t marks = 0;
      int at = 0;
      if (q < n_vecs) {
        const int v = sh.vecs[q], of = v % NT, number = of / 32 * chunk + v / NT * 32 + of % 32;
        at = vecs.first(number);
        float x[E];
        vec_floats<T>(vecs.load(number), x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool some = key_of(x[e]) >= bound;
          marks |= (uint32_t)(some && at + e >= 0 && at + e < vecs.V) << e;
          if (some) x[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < E; e += 2) sum = sum + exp2_fast((Pair(x[e], x[e + 1]) + edge2) * c2);
      }
      int to = place(n, __popc(marks));
#pragma unroll 1
      for (; marks && to < TOP_CAP; marks &= marks - 1) {
        const int e = __ffs(marks) - 1;
        sh.list[to++] = (unsigned long long)key_of(LogitType<T>::one(vecs.row[at + e])) << 32 | (uint32_t)~(at + e);
      }
    }
    below = sum.sum();
    return n;
  }
  // Candidates: keys above `bound`, and those equal to it with ids below `cut`; their number.
  __device__ __noinline__ int gather_cut(uint32_t bound, int cut) {
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    each([&](const uint4& u, int i) {
      if (key_of(vec_max<T>(u)) < bound || i >= mine) return;
      float x[E];
      vec_floats<T>(u, x);
      const int at = first(i);
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t key = key_of(x[e]);
        const int id = at + e;
        bits |= (uint32_t)(id >= 0 && id < vecs.V && (key > bound || (key == bound && id < cut))) << e;
      }
      if (!bits) return;
      int to = atomicAdd(&sh.n, __popc(bits));
#pragma unroll 1
      for (; bits; bits &= bits - 1, ++to) {
        const int e = __ffs(bits) - 1;
        float one = x[0];
#pragma unroll
        for (int j = 1; j < E; ++j) one = e == j ? x[j] : one;
        if (to < TOP_CAP) sh.list[to] = (unsigned long long)key_of(one) << 32 | (uint32_t)~(at + e);
      }
    });
    __syncthreads();
    return sh.n;
  }
  // This thread's sum of 2^((x - ref) c) over the logits below the bound, and those equal to it with ids from `cut` on.
  __device__ __noinline__ float mass_below(uint32_t bound, int cut, float ref, float c) {
    float s = 0.f;
    each([&](const uint4& u, int i) {
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t key = key_of(x[e]);
        s += exp2_fast(((key > bound || (key == bound && first(i) + e < cut) ? -INFINITY : x[e]) - ref) * c);
      }
    });
    return s;
  }
  // The largest of them.
  __device__ __noinline__ float max_below(uint32_t bound, int cut) {
    uint32_t most = 0;
    each([&](const uint4& u, int i) {
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t key = key_of(x[e]);
        const int id = first(i) + e;
        if (i < mine && id >= 0 && id < vecs.V && (key < bound || (key == bound && id >= cut))) most = max(most, key);
      }
    });
    most = max_of(most);
    return most ? of_key(most) : -INFINITY;
  }
};

template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) top_logits_kernel(const TopArgs a) {
  constexpr int W = NT / 32;
  __shared__ __align__(16) TopShared sh;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5, row = blockIdx.x;
  begin_early();
  TopRow<T, NT> r{sh, RowVecs<T>(static_cast<const T*>(a.x) + (long long)row * a.ldx, a.V)};
  r.chunk = (r.vecs.n + NT - 1) / NT * 32;
  r.w0 = w * r.chunk;
  r.mine = max(0, min(r.chunk / 32, (min(r.w0 + r.chunk, r.vecs.n) - r.w0 - lane + 31) / 32));

  // the largest of the thread's first and second half
  float top[2] = {-INFINITY, -INFINITY};
  const int half = (r.mine + 1) / 2;
#pragma unroll 1
  for (int i0 = 0; i0 < r.mine; i0 += 4) {
    uint4 u[4];
    r.load(i0, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float most = vec_max<T>(u[i]);
      if (i0 + i < half) top[0] = max_nan(top[0], most);
      else top[1] = max_nan(top[1], most);
    }
  }
  // The bound, from the warps whose lanes all hold logits.
  const int warps = r.vecs.n < 32 ? 0 : min((r.vecs.n - 32) / r.chunk + 1, W);
  const int j = warps > 0 ? (a.k + warps - 1) / warps : 65;
  uint32_t key = key_of(top[0]), second = r.mine > 1 ? key_of(top[1]) : 0, bound = 0xFFFFFFFFu;
  if (second > key) {
    const uint32_t swap = key;
    key = second;
    second = swap;
  }
  if (j > 64 || a.V <= a.k) {
    bound = 0;
  } else if (w < warps) {
#pragma unroll 1
    for (int i = 0;; ++i) {
      bound = __reduce_max_sync(0xffffffff, key);
      if (i == j - 1) break;
      if (lane == __ffs(__ballot_sync(0xffffffff, key == bound)) - 1) key = second, second = 0;
    }
  }
  bound = r.min_of(bound);
  int cut = a.V;  // of the logits equal to the bound, those with smaller ids
  const float c = a.inv_tau * 1.4426950408889634f;
  int n = r.gather(bound, c);
  bool usual = n <= TOP_CAP && bound > key_of(-INFINITY);
  if (n > TOP_CAP) {
    // The exact k-th largest key, and the id up to which the logits equal to it are taken.
    uint32_t kth = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
      const uint32_t next = kth | 1u << b;
      if (r.count(next, a.V) >= a.k) kth = next;
    }
    int low = 0;  // fewer than k are above, or equal with an id below `low`
#pragma unroll 1
    for (int b = 31 - __clz(a.V); b >= 0; --b)
      if (low + (1 << b) <= a.V && r.count(kth, low + (1 << b)) < a.k) low += 1 << b;
    bound = kth;
    cut = low + 1;
    n = r.gather_cut(bound, cut);
  }

  // Ranks: each warp sorts 32 candidates at a time; one's rank is its place there and, by bisection, how many of each other 32
  // are greater.
  float left_max = -INFINITY;
  const int runs = (n + 31) / 32;
  __syncthreads();
#pragma unroll 1
  for (int i = t; i < runs * 32; i += NT) {
    unsigned long long v = i < n ? sh.list[i] : 0;
#pragma unroll
    for (int of = 2; of <= 32; of *= 2)
#pragma unroll
      for (int d = of / 2; d; d /= 2) {
        const unsigned long long other = __shfl_xor_sync(0xffffffff, v, d);
        if ((other > v) == (((lane & d) == 0) == ((lane & of) == 0))) v = other;
      }
    sh.list[i] = v;
  }
  __syncthreads();
#pragma unroll 1
  for (int i = t; i < n; i += NT) {
    const unsigned long long mine = sh.list[i];
    int rank = lane;
#pragma unroll 2
    for (int run = 0; run < runs; ++run) {
      const unsigned long long* const sorted = sh.list + run * 32;
      int greater = 0;
#pragma unroll
      for (int step = 16; step; step /= 2) greater += sorted[greater + step - 1] > mine ? step : 0;
      greater += sorted[greater] > mine;
      rank += run == i / 32 ? 0 : greater;
    }
    const float value = of_key((uint32_t)(mine >> 32));
    if (rank < a.k) {
      const long long at = (long long)row * a.k + rank;
      a.ids[at] = (int)~(uint32_t)mine;
      static_cast<T*>(a.values)[at] = LogitType<T>::round(value);
    } else {
      sh.left[rank - a.k] = value;  // by rank: the order in which candidates came must not reach the sum
      left_max = max_nan(left_max, value);
    }
  }
  // The rest relative to the bound or to the largest candidate in it; where that is too far above the others or is not a
  // number, to its largest.
  left_max = of_key(r.max_of(key_of(left_max)));  // and its barrier for `left`
  float ref = n < a.V ? max_nan(of_key(bound), left_max) : left_max, s = 0.f;
  const auto left = [&] {
    float sl = 0.f;
    for (int i = t; i < n - a.k; i += NT) sl += exp2_fast((sh.left[i] - ref) * c);
    return sl;
  };
  if (n == a.V) {
    if (fabsf(ref) < INFINITY) s = r.sum_of(left());
  } else if (usual && fabsf(ref) < INFINITY) {
    s = r.sum_of(r.below * exp2_fast((of_key(bound) - ref) * c) + left());
  }
  if (n < a.V && !(s >= 1e-24f)) {
    ref = max_nan(r.max_below(bound, cut), left_max);
    if (fabsf(ref) < INFINITY) s = r.sum_of(r.mass_below(bound, cut, ref, c) + left());
  }
  if (t == 0) a.rest[row] = !(fabsf(ref) < INFINITY) ? ref : s == 0.f ? -INFINITY : fmaf(ref, a.inv_tau, logf(s));
}

template <typename T>
void top_typed(const TopArgs& a, cudaStream_t s) {
  const auto launch = [&](auto* kernel, int threads) { launch_early(kernel, dim3((unsigned)a.rows), dim3(threads), 0, s, a); };
  constexpr int SMS = 148;
  const long long vecs = (a.V + LogitType<T>::E - 1) / LogitType<T>::E;
  int threads = 128;
  const auto rows = [&](int n) { return std::min<long long>(a.rows, SMS * (1024 / n)); };  // at a time
  while (threads < 1024 && ((rows(threads) == rows(2 * threads) && vecs >= 16 * threads) || rows(threads) * vecs * 16 > TOP_L2))
    threads *= 2;
  if (threads == 128) launch(top_logits_kernel<T, 128>, 128);
  else if (threads == 256) launch(top_logits_kernel<T, 256>, 256);
  else if (threads == 512) launch(top_logits_kernel<T, 512>, 512);
  else launch(top_logits_kernel<T, 1024>, 1024);
}

}  // namespace astrai

namespace astrai_host {
using namespace astrai;

int top_logits_max_k() { return TOP_MAX_K; }

void top_logits(const void* x, long long ldx, int rows, int V, int k, float tau, int* ids, void* values, float* rest,
                int dtype, cudaStream_t s) {
  const TopArgs a{x, ldx, rows, V, k, 1.f / tau, ids, values, rest};
  if (dtype == 0) top_typed<__nv_bfloat16>(a, s);
  else if (dtype == 1) top_typed<__half>(a, s);
  else top_typed<float>(a, s);
}

}  // namespace astrai_host
