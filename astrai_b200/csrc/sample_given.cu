// One token per row from a given uniform number, under temperature, top-k, top-p and min-p (sm_100a).
//
// With w_v = exp((x_v - max x) / T) the tokens that are kept are those
//   not below the k-th largest logit,
//   whose strictly larger logits (of what top-k kept) hold at most p of its mass, and
//   with w_v >= min_p,
// and the token is the first kept one, in the order of ids, at which the running sum of w exceeds u times the whole. T = 0
// takes the largest logit. All three rules are bounds on the logit, so tokens of equal logits are kept or dropped together.
//
// The result is that of 64-bit arithmetic: an error of 1e-7 in a sum would move the token's border past u in one of a few
// hundred rows. Where top-k, min-p or top-p leave few tokens, these are gathered and everything about them is computed in
// 64 bits. Sums over a whole row are taken in 32 bits first, with a bound on their error; a row whose answer lies within it
// is summed again in 64 bits.
//
// A row is read once, into shared memory: a CTA of 512 threads holds up to 64 KB of it, a longer row is shared by a cluster. The
// bound that gathers the candidates is the one of the top logits: the smallest, over the row's warps, of each warp's j-th
// largest thread maximum.
#include <cooperative_groups.h>

#include "launch.cuh"
#include "logits.cuh"

namespace astrai {

namespace cg = cooperative_groups;

constexpr int SG_THREADS = 512;
constexpr int SG_WARPS = SG_THREADS / 32;
constexpr int SG_VECS = 8;  // 16-byte vectors of a thread
constexpr int SG_LIST_K = 256;  // top-k up to here, and the largest logits looked at for top-p, go by the list
constexpr int SG_CAP = 1024;
constexpr int SG_MAX_CLUSTER = 16;

struct SampleGivenArgs {
  const void* x;
  long long ldx;
  int rows, V, cluster;
  const void* uniform;  // [rows] fp32 or fp64
  int uniform64;
  const float* temperature;  // [rows]
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* token;  // [rows]
  float* logprob;    // [rows] or null
};

enum Verdict { kDone = 0, kAmbiguous = 1, kIncomplete = 2 };

struct SampleShared {
  unsigned long long list[SG_CAP];    // candidates: key, then the id's complement
  unsigned long long sorted[SG_CAP];  // greatest first
  double weight[SG_CAP];              // of the sorted ones
  double before[SG_CAP];              // mass of those before it
  double warp_sum[2][SG_WARPS];
  double sums[2];                     // of this CTA
  uint32_t warp_key[SG_WARPS];
  int warp_count[SG_WARPS];
  uint32_t key;  // of this CTA
  int count;     // of this CTA
  int n;         // the leader's: candidates of the row
  int verdict;   // the leader's
};

// What the rows' settings say, and the sums over threads, CTAs and the cluster.
struct SampleRow {
  SampleShared& sh;
  int cs, rank, t, lane, w;
  float max_x;
  double T64, p, m, draw;
  bool use_k, use_p, use_m;
  int k;

  __device__ void sync() const {
    if (cs > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  // The results of these are the same in all threads of the row.
  __device__ uint32_t max_key(uint32_t key) const {
    key = __reduce_max_sync(0xffffffff, key);
    __syncthreads();
    if (lane == 0) sh.warp_key[w] = key;
    __syncthreads();
    key = __reduce_max_sync(0xffffffff, sh.warp_key[lane & (SG_WARPS - 1)]);
    if (cs > 1) {
      if (t == 0) sh.key = key;
      cg::this_cluster().sync();
      key = __reduce_max_sync(0xffffffff, *cg::this_cluster().map_shared_rank(&sh.key, lane < cs ? lane : 0));
      cg::this_cluster().sync();
    }
    return key;
  }
  __device__ int count(int n) const {
    n = __reduce_add_sync(0xffffffff, n);
    __syncthreads();
    if (lane == 0) sh.warp_count[w] = n;
    __syncthreads();
    n = __reduce_add_sync(0xffffffff, lane < SG_WARPS ? sh.warp_count[lane] : 0);
    if (cs > 1) {
      if (t == 0) sh.count = n;
      cg::this_cluster().sync();
      n = __reduce_add_sync(0xffffffff, lane < cs ? *cg::this_cluster().map_shared_rank(&sh.count, lane) : 0);
      cg::this_cluster().sync();
    }
    return n;
  }
  __device__ static double warp_add(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
    return v;
  }
  // Two sums. The first one's parts: before this CTA, in it, and whether CTAs after it have any; its warps' parts stay in
  // sh.warp_sum[0].
  struct Part {
    double before, here;
    bool last;
  };
  __device__ Part sum(double& s0, double& s1) const {
    s0 = warp_add(s0);
    s1 = warp_add(s1);
    __syncthreads();
    if (lane == 0) sh.warp_sum[0][w] = s0, sh.warp_sum[1][w] = s1;
    __syncthreads();
    s0 = s1 = 0.;
    for (int i = 0; i < SG_WARPS; ++i) s0 += sh.warp_sum[0][i], s1 += sh.warp_sum[1][i];
    Part part{0., s0, true};
    if (cs > 1) {
      if (t == 0) sh.sums[0] = s0, sh.sums[1] = s1;
      cg::this_cluster().sync();
      s0 = s1 = 0.;
      for (int i = 0; i < cs; ++i) {
        const double* theirs = cg::this_cluster().map_shared_rank(sh.sums, i);
        if (i == rank) part.before = s0;
        if (i > rank && theirs[0] > 0.) part.last = false;
        s0 += theirs[0];
        s1 += theirs[1];
      }
      cg::this_cluster().sync();
    }
    return part;
  }
  __device__ double weight(float x) const { return x == -INFINITY ? 0. : exp(((double)x - (double)max_x) / T64); }
};

__device__ __forceinline__ uint32_t key_part(unsigned long long e) { return (uint32_t)(e >> 32); }
__device__ __forceinline__ int id_part(unsigned long long e) { return (int)~(uint32_t)e; }

// The leader's candidates in order, their weights and running mass.
__device__ void order_list(const SampleRow& r, int n) {
  SampleShared& sh = r.sh;
  const int quarter = r.t & 3;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += SG_THREADS / 4) {
    const int i = i0 + r.t / 4;
    const unsigned long long mine = i < n ? sh.list[i] : 0;
    int above = 0;
    for (int l = quarter; l < n; l += 4) above += sh.list[l] > mine;
    above += __shfl_xor_sync(0xffffffff, above, 1);
    above += __shfl_xor_sync(0xffffffff, above, 2);
    if (i < n && quarter == 0) {
      sh.sorted[above] = mine;
      sh.weight[above] = r.weight(of_key(key_part(mine)));
    }
  }
  __syncthreads();
  if (r.w == 0) {
    const int each = (n + 31) / 32, a = min(n, r.lane * each), b = min(n, a + each);
    double s = 0.;
    for (int i = a; i < b; ++i) s += sh.weight[i];
    double run = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffff, run, o);
      if (r.lane >= o) run += up;
    }
    run -= s;
    for (int i = a; i < b; ++i) {
      sh.before[i] = run;
      run += sh.weight[i];
    }
  }
  __syncthreads();
}

// The leader's answer from its candidates. `total` +- `error` is the mass of the row that top-p takes a share of, where top-k
// is off; `complete`: no token below the candidates can be kept.
__device__ void answer_from_list(const SampleRow& r, int n, bool complete, double total, double error, long long* token,
                                 float* logprob) {
  SampleShared& sh = r.sh;
  const uint32_t kth = r.use_k && r.k <= n ? key_part(sh.sorted[r.k - 1]) : 0;
  int nk = n;
  if (r.use_k) {
    nk = 0;
    for (int i0 = 0; i0 < n; i0 += SG_THREADS) nk += __syncthreads_count(i0 + r.t < n && key_part(sh.sorted[i0 + r.t]) >= kth);
    total = nk > 0 ? sh.before[nk - 1] + sh.weight[nk - 1] : 0.;
    error = 0.;
  }
  const double share = r.p * total, blur = r.p * error;
  bool unsure = false;
  int kept = 0;
  for (int i0 = 0; i0 < n; i0 += SG_THREADS) {
    const int i = i0 + r.t;
    bool keep = i < nk;
    if (keep && r.use_p) {
      int first = 0, last = i;  // where its value begins
      const uint32_t key = key_part(sh.sorted[i]);
      while (first < last) {
        const int mid = (first + last) / 2;
        if (key_part(sh.sorted[mid]) == key) last = mid;
        else first = mid + 1;
      }
      keep = !(sh.before[first] > share);
      unsure |= first > 0 && blur > 0. && fabs(sh.before[first] - share) <= blur;
    }
    if (keep && r.use_m) keep = sh.weight[i] >= r.m;
    kept += __syncthreads_count(keep);
  }
  int verdict = kDone;
  if (!complete && r.use_p) {  // is the bound of top-p among the candidates?
    const double all = sh.before[n - 1] + sh.weight[n - 1];
    unsure |= blur > 0. && fabs(all - share) <= blur;
    if (!(all > share)) verdict = kIncomplete;
  }
  if (__syncthreads_or(unsure)) verdict = kAmbiguous;
  if (verdict == kDone) {
    const double mass = sh.before[kept - 1] + sh.weight[kept - 1], target = r.draw * mass;
    const int quarter = r.t & 3;
    uint32_t best = 0;   // complement of the id: the first at which the running sum in the order of ids is above the target
    int last = -1;       // and the last with any mass
#pragma unroll 1
    for (int i0 = 0; i0 < kept; i0 += SG_THREADS / 4) {
      const int i = i0 + r.t / 4;
      const int id = i < kept ? id_part(sh.sorted[i]) : -1;
      double s = 0.;
      for (int l = quarter; l < kept; l += 4)
        if (id_part(sh.sorted[l]) <= id) s += sh.weight[l];
      s += __shfl_xor_sync(0xffffffff, s, 1);
      s += __shfl_xor_sync(0xffffffff, s, 2);
      if (i < kept) {
        if (s > target) best = max(best, ~(uint32_t)id);
        if (sh.weight[i] > 0.) last = max(last, id);
      }
    }
    best = __reduce_max_sync(0xffffffff, best);
    last = __reduce_max_sync(0xffffffff, last);
    __syncthreads();
    if (r.lane == 0) sh.warp_key[r.w] = best, sh.warp_count[r.w] = last;
    __syncthreads();
    best = __reduce_max_sync(0xffffffff, sh.warp_key[r.lane & (SG_WARPS - 1)]);
    last = __reduce_max_sync(0xffffffff, sh.warp_count[r.lane & (SG_WARPS - 1)]);
    const int id = best ? (int)~best : last;
    for (int i = r.t; i < kept; i += SG_THREADS)
      if (id_part(sh.sorted[i]) == id) {
        *token = id;
        if (logprob) *logprob = (float)log(sh.weight[i] / mass);
      }
  }
  if (r.t == 0) sh.verdict = verdict;
}

template <typename T>
__global__ void __launch_bounds__(SG_THREADS, 2) sample_given_kernel(const SampleGivenArgs a) {
  constexpr int E = LogitType<T>::E;
  extern __shared__ uint4 held[];  // vector i of thread t at i * 512 + t
  __shared__ SampleShared sh;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int cs = a.cluster, rank = cs > 1 ? (int)cg::this_cluster().block_rank() : 0;
  const int row = blockIdx.x / cs;
  begin_early();
  const RowVecs<T> vecs(static_cast<const T*>(a.x) + (long long)row * a.ldx, a.V);
  const int per = (vecs.n + cs - 1) / cs, v0 = rank * per, v1 = min(v0 + per, vecs.n);
  // every warp holds vectors one after another, so that sums over warps are sums over ids
  const int chunk = (per + SG_THREADS - 1) / SG_THREADS * 32, w0 = v0 + w * chunk, w1 = min(w0 + chunk, v1);
  const int mine = max(0, min(chunk / 32, (w1 - w0 - lane + 31) / 32));  // vectors of this thread
  float top = -INFINITY;
  bool nan = false;
  {
    uint4 u[SG_VECS];
#pragma unroll
    for (int i = 0; i < SG_VECS; ++i) u[i] = i < mine ? vecs.load(w0 + i * 32 + lane) : vec_neg_inf<T>();
#pragma unroll
    for (int i = 0; i < SG_VECS; ++i) {
      if (i < mine) held[i * SG_THREADS + t] = u[i];
      const float most = vec_max<T>(u[i]);
      nan |= most != most;
      top = fmaxf(top, most);
    }
  }
  SampleRow r{sh, cs, rank, t, lane, w};
  const float temperature = a.temperature[row];
  const bool greedy = !(temperature > 0.f);
  r.T64 = (double)(greedy ? 1.f : fminf(fmaxf(temperature, 1e-8f), 3.4e38f));
  r.k = a.top_k[row];
  r.use_k = !greedy && r.k > 0 && r.k < a.V;
  const float p = a.top_p[row], m = a.min_p[row];
  r.use_p = !greedy && p < 1.f;
  r.use_m = !greedy && m > 0.f;
  r.p = r.use_p ? fmax((double)p, 0.) : 1.;
  r.m = r.use_m ? fmin((double)m, 1.) : 0.;
  r.draw = a.uniform64 ? static_cast<const double*>(a.uniform)[row] : (double)static_cast<const float*>(a.uniform)[row];
  r.draw = fmin(fmax(r.draw, 0.), 1.);  // a NaN becomes 0
  SampleShared* lead = &sh;
  if (cs > 1) lead = cg::this_cluster().map_shared_rank(&sh, 0);
  if (t == 0) sh.n = 0;

  const float c = (float)(1.4426950408889634 / r.T64);
  r.max_x = of_key(r.max_key(key_of(nan ? of_key(0xFFFFFFFFu) : top)));

  // f(element, id) over this thread's elements
  const auto each = [&](auto f) {
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      const int at = vecs.first(w0 + i * 32 + lane);
      float x[E];
      vec_floats<T>(held[i * SG_THREADS + t], x);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at + e >= 0 && at + e < a.V) f(x[e], at + e);
    }
  };
  const bool none = !(fabsf(r.max_x) < INFINITY);
  if (none) {  // a NaN, an infinity or nothing allowed: no distribution; the largest logit that is a number
    uint32_t key = 0;
    each([&](float x, int) { if (x == x) key = max(key, key_of(x)); });
    key = r.max_key(key);
    uint32_t first = 0;
    each([&](float x, int id) { if (x == x && key_of(x) == key) first = max(first, ~(uint32_t)id); });
    first = r.max_key(first);
    if (rank == 0 && t == 0) {
      a.token[row] = key ? (int)~first : 0;
      if (a.logprob) a.logprob[row] = __int_as_float(0x7FC00000);
    }
    return;
  }

  // Mass of what `keep` leaves of a vector, and its sum of w |t|. In 32 bits each exponential is within 2^-22 of itself and
  // 3 |t| 2^-24 ln 2 for the roundings of t = (x - max) c, and eight of them are added in a tree.
  const auto vec_mass = [&](int i, bool precise, auto keep, float& spread) {
    float x[E];
    vec_floats<T>(held[i * SG_THREADS + t], x);
    if (precise) {
      double s = 0.;
#pragma unroll 1
      for (int e = 0; e < E; ++e)
        if (x[e] > -INFINITY && keep(x[e])) s += r.weight(x[e]);
      return s;
    }
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float arg = (x[e] - r.max_x) * c;
      s[e] = x[e] > -INFINITY && keep(x[e]) ? exp2_fast(arg) : 0.f;
      if (s[e] > 0.f) spread -= s[e] * arg;
    }
#pragma unroll
    for (int o = E / 2; o > 0; o >>= 1)
#pragma unroll
      for (int e = 0; e < o; ++e) s[e] += s[e + o];
    return (double)s[0];
  };
  SampleRow::Part part;
  const auto masses = [&](bool precise, auto keep, double& total, double& error) {
    double spread = 0.;
    total = 0.;
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      float d = 0.f;
      total += vec_mass(i, precise, keep, d);
      spread += d;
    }
    part = r.sum(total, spread);
    error = precise ? 0. : 4.5e-7 * total + 1.3e-7 * spread;
  };
  // Draws among what `keep` leaves.
  const auto draw = [&](auto keep) {
#pragma unroll 1
    for (int precise = 0; precise < 2; ++precise) {
      if (rank == 0 && t == 0) sh.verdict = kDone;
      double total, error;
      masses(precise, keep, total, error);
      // The CTA in whose part the target lies, and there, counted from its start, the warp. Should rounding leave the
      // target at the very end, the last one with any mass takes it.
      double target = r.draw * total;
      const bool here = part.here > 0. && part.before <= target && (target < part.before + part.here || part.last);
      target -= part.before;
      double before = 0.;
      for (int i = 0; i < w; ++i) before += sh.warp_sum[0][i];
      bool last = true;
      for (int i = w + 1; i < SG_WARPS; ++i) last &= !(sh.warp_sum[0][i] > 0.);
      const double hi = before + sh.warp_sum[0][w];
      if (here && before < hi && before <= target && (target < hi || last)) {
        int at_i = 0, last_i = 0;
        double at_before = -1., last_before = before, s;
#pragma unroll 1
        for (int i = 0; i < chunk / 32; ++i) {
          float d = 0.f;
          s = SampleRow::warp_add(i < mine ? vec_mass(i, precise, keep, d) : 0.);
          if (s > 0.) last_i = i, last_before = before;
          if (at_before < 0. && before + s > target) at_i = i, at_before = before;
          before += s;
        }
        if (at_before < 0.) at_i = last_i, at_before = last_before;
        float d = 0.f;
        s = at_i < mine ? vec_mass(at_i, precise, keep, d) : 0.;
        double scan = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffff, scan, o);
          if (lane >= o) scan += up;
        }
        const uint32_t above = __ballot_sync(0xffffffff, s > 0. && at_before + scan > target);
        const uint32_t some = __ballot_sync(0xffffffff, s > 0.);
        const int who = above ? __ffs(above) - 1 : 31 - __clz(some);
        if (lane == who) {
          double run = at_before + (scan - s), c0 = run, c1 = run;
          int id = -1;
          float chosen = 0.f, x[E];
          vec_floats<T>(held[at_i * SG_THREADS + t], x);
          const int at = vecs.first(w0 + at_i * 32 + lane);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            if (!(x[e] > -INFINITY) || !keep(x[e])) continue;
            const double one = precise ? r.weight(x[e]) : (double)exp2_fast((x[e] - r.max_x) * c);
            if (one > 0. && (id < 0 || !(c1 > target))) {  // the first above the target, or the last with any mass
              id = at + e;
              chosen = x[e];
              c0 = run;
              c1 = run + one;
            }
            run += one;
          }
          if (!precise && (target - c0 <= 2. * error || c1 - target <= 2. * error)) {
            lead->verdict = kAmbiguous;
          } else {
            a.token[row] = id;
            if (a.logprob) a.logprob[row] = (float)log(r.weight(chosen) / total);
          }
        }
      }
      r.sync();
      const int verdict = lead->verdict;
      r.sync();
      if (verdict == kDone) return;
    }
  };

  double total = 0., error = 0.;
  if (greedy) {
    uint32_t first = 0;
    each([&](float x, int id) { if (x == r.max_x) first = max(first, ~(uint32_t)id); });
    first = r.max_key(first);
    masses(false, [](float) { return true; }, total, error);
    if (rank == 0 && t == 0) {
      a.token[row] = (int)~first;
      if (a.logprob) a.logprob[row] = (float)-log(total);
    }
    return;
  }

  const auto all = [](float) { return true; };
  const bool by_k = r.use_k && r.k <= SG_LIST_K;
  if (by_k || (!r.use_k && (r.use_p || r.use_m))) {
    // A bound that all candidates reach.
    uint32_t bound = 0;
    if (r.use_m && !(by_k && r.use_p)) {
      const double x = r.max_x + r.T64 * log(r.m);
      bound = key_of((float)(x - 1e-6 * (fabs(x) + fabs(r.max_x) + r.T64)));
    }
    bool complete = by_k || r.use_m;
    if (by_k || r.use_p) {
      const auto full = [&](int n) { return n < 32 ? 0 : min((n - 32) / chunk + 1, SG_WARPS); };
      const int warps = (cs - 1) * full(per) + full(vecs.n - (cs - 1) * per);
      const int j = warps > 0 ? ((by_k ? r.k : SG_LIST_K) + warps - 1) / warps : 33;
      uint32_t key = key_of(top), low = 0xFFFFFFFFu;
      if (j > 32) {
        low = 0;
      } else if (w < full(v1 - v0)) {
        for (int i = 0;; ++i) {
          low = __reduce_max_sync(0xffffffff, key);
          if (i == j - 1) break;
          if (lane == __ffs(__ballot_sync(0xffffffff, key == low)) - 1) key = 0;
        }
      }
      low = ~r.max_key(~low);
      if (low > bound) {
        complete = by_k || low == 0;
        bound = low;
      }
      complete |= low == 0;
    }
    if (r.use_p && !by_k) masses(false, all, total, error);
    each([&](float x, int id) {
      const uint32_t key = key_of(x);
      if (key < bound) return;
      const int slot = atomicAdd(&lead->n, 1);
      if (slot < SG_CAP) lead->list[slot] = (unsigned long long)key << 32 | (uint32_t)~id;
    });
    r.sync();
    const int n = lead->n;
    if (n <= SG_CAP) {
      if (rank == 0) order_list(r, n);
      for (int precise = 0;; ++precise) {
        if (rank == 0) answer_from_list(r, n, complete, total, error, a.token + row, a.logprob ? a.logprob + row : nullptr);
        r.sync();
        const int verdict = lead->verdict;
        r.sync();
        if (verdict == kDone) return;
        if (verdict == kIncomplete) break;
        masses(true, all, total, error);
      }
    } else {
      r.sync();  // the leader's count has been read
    }
  }

  // Many tokens stay: the bounds of top-k and top-p by bisection of the key.
  uint32_t kth = 0;
  if (r.use_k) {
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
      const uint32_t next = kth | 1u << b;
      int n = 0;
      each([&](float x, int) { n += key_of(x) >= next; });
      if (r.count(n) >= r.k) kth = next;
    }
  }
  uint32_t low = kth;
  if (r.use_p) {
#pragma unroll 1
    for (int precise = 0; precise < 2; ++precise) {
      bool unsure = false;
      masses(precise, [&](float x) { return key_of(x) >= kth; }, total, error);
      const double share = r.p * total, blur = r.p * error;
      uint32_t cut = 0;  // the largest key such that it and those above hold more than the share
#pragma unroll 1
      for (int b = 31; b >= 0; --b) {
        const uint32_t next = cut | 1u << b;
        double s, e;
        masses(precise, [&](float x) { return key_of(x) >= kth && key_of(x) >= next; }, s, e);
        unsure |= fabs(s - share) <= e + blur;
        if (s > share) cut = next;
      }
      low = max(kth, cut);
      if (!unsure) break;
    }
  }
  const float near = r.use_m ? r.max_x + (float)r.T64 * logf((float)r.m) : -INFINITY;
  const float slack = 1e-4f * (fabsf(r.max_x) + fabsf(near) + (float)r.T64);
  draw([&](float x) {
    if (key_of(x) < low) return false;
    if (!r.use_m || x > near + slack) return true;
    return x >= near - slack && r.weight(x) >= r.m;
  });
}

template <typename T>
void sample_given_launch(const SampleGivenArgs& a, int smem, cudaStream_t s) {
  auto* kernel = sample_given_kernel<T>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a.rows * a.cluster);
  cfg.blockDim = dim3(SG_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SG_VECS * SG_THREADS * 16);
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
void sample_given_sized(SampleGivenArgs a, cudaStream_t s) {
  constexpr int E = LogitType<T>::E;
  const int vecs = (a.V + E - 1) / E + 1;  // one more where a row starts off the grid
  int cs = 1;
  while ((vecs + cs - 1) / cs > SG_THREADS * SG_VECS) cs *= 2;
  a.cluster = cs;
  const int per = (vecs + cs - 1) / cs;
  sample_given_launch<T>(a, (per + SG_THREADS - 1) / SG_THREADS * SG_THREADS * 16, s);
}

}  // namespace astrai

namespace astrai_host {
using namespace astrai;

// longest row for elements of this size
int sample_given_max_vocab(int elem) { return SG_MAX_CLUSTER * SG_THREADS * SG_VECS * (16 / elem) - 16 / elem; }

void sample_given(const void* x, long long ldx, int rows, int V, const void* uniform, bool uniform64,
                  const float* temperature, const int* top_k, const float* top_p, const float* min_p, long long* token,
                  float* logprob, int dtype, cudaStream_t s) {
  const SampleGivenArgs a{x, ldx, rows, V, 1, uniform, uniform64, temperature, top_k, top_p, min_p, token, logprob};
  if (dtype == 0) sample_given_sized<__nv_bfloat16>(a, s);
  else if (dtype == 1) sample_given_sized<__half>(a, s);
  else sample_given_sized<float>(a, s);
}

}  // namespace astrai_host
