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
// A CTA of 512 threads takes a row, or where the rows are too few for the SMs a cluster of CTAs does. Up to 64 KB of logits
// stay in the CTA's shared memory between the passes over them, more than that come from L2 again.
// The bound that gathers the candidates is the one of the top logits: the smallest, over the row's warps, of each warp's j-th
// largest thread maximum. Where top-p reaches below them (flat rows) or k is large, a histogram of the logits over 4096 equal
// steps shows in which steps the bound must lie, and the few logits there are ordered and decided exactly.
#include <cooperative_groups.h>

#include <cstdlib>

#include "launch.cuh"
#include "logits.cuh"

namespace astrai {

namespace cg = cooperative_groups;

constexpr int SG_THREADS = 512;
constexpr int SG_WARPS = SG_THREADS / 32;
constexpr int SG_VECS = 8;  // 16-byte vectors of a thread
constexpr int SG_LIST_K = 256;  // top-k up to here, and the largest logits looked at for top-p, go by the list
constexpr int SG_CAP = 1024;
constexpr int SG_BINS = 4096;
constexpr int SG_MAX_CLUSTER = 8;

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

// 2^t for t <= 0 in 64 bits, within 2^-46 of itself (below 2^-1000: zero): e^z = sum z^n / n! at |z| <= ln 2 / 2, whose 13th
// term is below 2^-53, times a power of two.
__device__ __forceinline__ double exp2_64(double t) {
  constexpr double kRound = 6755399441055744.;  // 1.5 * 2^52: adding it rounds to a whole number
  const double n = t + kRound, z = (t - (n - kRound)) * 0.6931471805599453;
  double e = 1. / 479001600.;
  e = fma(e, z, 1. / 39916800.);
  e = fma(e, z, 1. / 3628800.);
  e = fma(e, z, 1. / 362880.);
  e = fma(e, z, 1. / 40320.);
  e = fma(e, z, 1. / 5040.);
  e = fma(e, z, 1. / 720.);
  e = fma(e, z, 1. / 120.);
  e = fma(e, z, 1. / 24.);
  e = fma(e, z, 1. / 6.);
  e = fma(e, z, 0.5);
  e = fma(e, z, 1.);
  e = fma(e, z, 1.);
  return t > -1000. ? __hiloint2double(__double2hiint(e) + (__double2loint(n) << 20), __double2loint(e)) : 0.;
}

enum Verdict { kDone = 0, kAmbiguous = 1, kIncomplete = 2 };

struct SampleShared {
  unsigned long long list[SG_CAP];    // candidates: key, then the id's complement
  unsigned long long sorted[SG_CAP];  // greatest first
  uint16_t by_id[SG_CAP];             // places among the sorted ones, in the order of ids
  union {
    struct {
      double weight[SG_CAP];  // of the sorted ones
      double before[SG_CAP];  // mass of those before it
    };
    uint32_t bins[SG_BINS];
  };
  double warp_sum[2][SG_WARPS];  // two of each: a reduction writes one while the last one's may still be read
  double sums[2];                // of this CTA
  uint32_t warp_key[2][SG_WARPS], key[2];
  int n;         // the leader's: candidates of the row
  int verdict;   // the leader's
  uint32_t low;  // the least key that min-p keeps; the leader's: the least key that the row keeps
  uint32_t scan[SG_WARPS];
  double scan64[SG_WARPS];
  int found;
  uint32_t found_above;
};

// What the row's settings say, and the reductions over warps, CTAs and the cluster: their results are the same in all
// threads of the row.
struct SampleRow {
  SampleShared& sh;
  int cs, rank, t, lane, w;
  float max_x;
  double T64, c64, p, m, draw;  // c64: log2(e) / T
  bool use_k, use_p, use_m;
  int k;
  int turn = 0;

  __device__ void sync() const {
    if (cs > 1) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename F>
  __device__ uint32_t reduce(uint32_t v, F f) {
    const int at = turn ^= 1;
    v = f(v);
    if (lane == 0) sh.warp_key[at][w] = v;
    __syncthreads();
    v = f(sh.warp_key[at][lane & (SG_WARPS - 1)]);
    if (cs > 1) {
      if (t == 0) sh.key[at] = v;
      cg::this_cluster().sync();
      v = f(*cg::this_cluster().map_shared_rank(&sh.key[at], lane < cs ? lane : 0));
    }
    return v;
  }
  __device__ uint32_t max_key(uint32_t v) {
    return reduce(v, [](uint32_t x) { return __reduce_max_sync(0xffffffff, x); });
  }
  __device__ uint32_t min_key(uint32_t v) {
    return reduce(v, [](uint32_t x) { return __reduce_min_sync(0xffffffff, x); });
  }
  __device__ int count(int n) {
    const int at = turn ^= 1;
    n = __reduce_add_sync(0xffffffff, n);
    if (lane == 0) sh.warp_key[at][w] = n;
    __syncthreads();
    n = __reduce_add_sync(0xffffffff, lane < SG_WARPS ? (int)sh.warp_key[at][lane] : 0);
    if (cs > 1) {
      if (t == 0) sh.key[at] = n;
      cg::this_cluster().sync();
      n = __reduce_add_sync(0xffffffff, lane < cs ? (int)*cg::this_cluster().map_shared_rank(&sh.key[at], lane) : 0);
    }
    return n;
  }
  __device__ static double warp_add(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
    return v;
  }
  // A sum and its parts: before this CTA, in it, and whether no CTA after it has any; in this warp and the warps before it in
  // the CTA, and whether no warp after it has any.
  struct Part {
    double total, before, here, warp_before, warp;
    bool last, warp_last;
  };
  __device__ Part sum(double s) {
    const int at = turn ^= 1;
    Part part;
    part.warp = s = warp_add(s);
    if (lane == 0) sh.warp_sum[at][w] = s;
    __syncthreads();
    const double theirs = sh.warp_sum[at][lane & (SG_WARPS - 1)];
    double scan = theirs;
#pragma unroll
    for (int o = 1; o < SG_WARPS; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffff, scan, o, SG_WARPS);
      if ((lane & (SG_WARPS - 1)) >= o) scan += up;
    }
    part.total = part.here = __shfl_sync(0xffffffff, scan, SG_WARPS - 1);
    part.warp_before = __shfl_sync(0xffffffff, scan, max(w - 1, 0));
    if (w == 0) part.warp_before = 0.;
    part.warp_last = (__ballot_sync(0xffffffff, theirs > 0.) & ((1u << SG_WARPS) - 1)) >> (w + 1) == 0;
    part.before = 0.;
    part.last = true;
    if (cs > 1) {
      if (t == 0) sh.sums[at] = part.here;
      cg::this_cluster().sync();
      const double others = lane < cs ? *cg::this_cluster().map_shared_rank(&sh.sums[at], lane) : 0.;
      scan = others;
#pragma unroll
      for (int o = 1; o < SG_MAX_CLUSTER; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffff, scan, o);
        if (lane >= o) scan += up;
      }
      part.total = __shfl_sync(0xffffffff, scan, SG_MAX_CLUSTER - 1);
      part.before = __shfl_sync(0xffffffff, scan, max(rank - 1, 0));
      if (rank == 0) part.before = 0.;
      part.last = __ballot_sync(0xffffffff, others > 0.) >> (rank + 1) == 0;
    }
    return part;
  }
  __device__ double weight(float x) const { return exp2_64(((double)x - (double)max_x) * c64); }
};

__device__ __forceinline__ uint32_t key_part(unsigned long long e) { return (uint32_t)(e >> 32); }
__device__ __forceinline__ int id_part(unsigned long long e) { return (int)~(uint32_t)e; }

// The leader's candidates in order of value, their weights, and their places in the order of ids.
__device__ void order_list(const SampleRow& r, int n) {
  SampleShared& sh = r.sh;
  const int quarter = r.t & 3;
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += SG_THREADS / 4) {
    const int i = i0 + r.t / 4;
    const unsigned long long mine = i < n ? sh.list[i] : 0;
    int above = 0, earlier = 0;
#pragma unroll 4
    for (int l = quarter; l < n; l += 4) {
      const unsigned long long other = sh.list[l];
      above += other > mine;
      earlier += (uint32_t)other > (uint32_t)mine;  // complements of ids
    }
    above += __shfl_xor_sync(0xffffffff, above, 1);
    above += __shfl_xor_sync(0xffffffff, above, 2);
    earlier += __shfl_xor_sync(0xffffffff, earlier, 1);
    earlier += __shfl_xor_sync(0xffffffff, earlier, 2);
    if (i < n && quarter == 0) {
      sh.sorted[above] = mine;
      sh.weight[above] = r.weight(of_key(key_part(mine)));
      sh.by_id[earlier] = (uint16_t)above;
    }
  }
  __syncthreads();
}

// For warp 0 of the leader: the running sums of v(i), i < n, each lane its own part of them; before(i, sum before i, v(i)).
template <typename V, typename F>
__device__ __forceinline__ double running_sums(int lane, int n, V v, F before) {
  const int each = (n + 31) / 32, a = min(n, lane * each), b = min(n, a + each);
  double s = 0.;
  for (int i = a; i < b; ++i) s += v(i);
  double scan = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffff, scan, o);
    if (lane >= o) scan += up;
  }
  const double total = __shfl_sync(0xffffffff, scan, 31);
  double run = scan - s;
  for (int i = a; i < b; ++i) {
    const double one = v(i);
    before(i, run, one);
    run += one;
  }
  return total;
}

// Where the value of the sorted candidate i begins.
__device__ __forceinline__ int first_of_value(const SampleShared& sh, int i) {
  int first = 0, last = i;
  const uint32_t key = key_part(sh.sorted[i]);
  while (first < last) {
    const int mid = (first + last) / 2;
    if (key_part(sh.sorted[mid]) == key) last = mid;
    else first = mid + 1;
  }
  return first;
}

// The leader's answer from its candidates, by its first warp. `total` +- `error` is the mass of the row that top-p takes a
// share of, where top-k is off; `complete`: no token below the candidates can be kept.
__device__ void answer_from_list(const SampleRow& r, int n, bool complete, uint32_t low_m, double total, double error,
                                 long long* token, float* logprob) {
  SampleShared& sh = r.sh;
  const int lane = r.lane;
  const double all = running_sums(lane, n, [&](int i) { return sh.weight[i]; },
                                  [&](int i, double run, double) { sh.before[i] = run; });
  __syncwarp();
  int nk = n;
  if (r.use_k) {
    const uint32_t kth = r.k <= n ? key_part(sh.sorted[r.k - 1]) : 0;
    nk = 0;
    for (int i = lane; i < n; i += 32) nk += key_part(sh.sorted[i]) >= kth;
    nk = __reduce_add_sync(0xffffffff, nk);
    total = nk < n ? sh.before[nk] : all;
    error = 0.;
  }
  const double share = r.p * total, blur = r.p * error;
  bool unsure = false;
  int kept = 0;
  for (int i = lane; i < nk; i += 32) {
    bool keep = !r.use_m || key_part(sh.sorted[i]) >= low_m;
    if (r.use_p && i > 0) {
      const int first = first_of_value(sh, i);
      unsure |= first > 0 && blur > 0. && fabs(sh.before[first] - share) <= blur;
      keep &= first == 0 || !(sh.before[first] > share);
    }
    kept += keep;
  }
  kept = __reduce_add_sync(0xffffffff, kept);
  int verdict = kDone;
  if (!complete && r.use_p) {  // is the bound of top-p among the candidates?
    unsure |= blur > 0. && fabs(all - share) <= blur;
    if (!(all > share)) verdict = kIncomplete;
  }
  if (__any_sync(0xffffffff, unsure)) verdict = kAmbiguous;
  if (verdict == kDone) {
    const double mass = kept < n ? sh.before[kept] : all, target = r.draw * mass;
    int hit = n, last = -1;  // in the order of ids: the first at which the running sum is above the target, the last with mass
    running_sums(lane, n, [&](int q) { return sh.by_id[q] < kept ? sh.weight[sh.by_id[q]] : 0.; },
                 [&](int q, double run, double one) {
                   if (one > 0.) last = q;
                   if (one > 0. && run + one > target) hit = min(hit, q);
                 });
    hit = __reduce_min_sync(0xffffffff, hit);
    last = __reduce_max_sync(0xffffffff, last);
    if (lane == 0) {
      const int i = sh.by_id[hit < n ? hit : last];
      *token = id_part(sh.sorted[i]);
      if (logprob) *logprob = (float)log(sh.weight[i] / mass);
    }
  }
  if (lane == 0) sh.verdict = verdict;
}

// The leader's bound of top-p, by its first warp, among the candidates of a few steps of the histogram, above which lies
// `above` +- `error`; `end`: no logit lies below them. The mass of strictly larger logits must be known to lie below or above
// the share.
__device__ void bound_from_list(const SampleRow& r, int n, bool end, double above, double error, double share, double blur) {
  SampleShared& sh = r.sh;
  const double doubt = error + blur;
  const double all = above + running_sums(r.lane, n, [&](int i) { return sh.weight[i]; },
                                          [&](int i, double run, double) { sh.before[i] = run; });
  __syncwarp();
  bool unsure = !end && doubt > 0. && fabs(all - share) <= doubt;
  int kept = 0;
  for (int i = r.lane; i < n; i += 32) {
    const double larger = above + sh.before[first_of_value(sh, i)];
    kept += !(larger > share);
    unsure |= larger > 0. && doubt > 0. && fabs(larger - share) <= doubt;
  }
  kept = __reduce_add_sync(0xffffffff, kept);
  unsure = __any_sync(0xffffffff, unsure);
  if (r.lane == 0) {
    sh.verdict = unsure ? kAmbiguous : (kept == 0 || (!end && !(all > share)) ? kIncomplete : kDone);
    sh.low = kept > 0 ? key_part(sh.sorted[kept - 1]) : 0;
  }
}

// HELD: the CTA's part of the row lies in shared memory.
template <typename T, bool HELD>
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
#pragma unroll 1
  for (int i0 = 0; i0 < mine; i0 += SG_VECS) {
    uint4 u[SG_VECS];
#pragma unroll
    for (int i = 0; i < SG_VECS; ++i) u[i] = i0 + i < mine ? vecs.load(w0 + (i0 + i) * 32 + lane) : vec_neg_inf<T>();
#pragma unroll
    for (int i = 0; i < SG_VECS; ++i) {
      if (HELD && i0 + i < mine) held[(i0 + i) * SG_THREADS + t] = u[i];
      const float most = vec_max<T>(u[i]);
      nan |= most != most;
      top = fmaxf(top, most);
    }
  }
  const auto vec = [&](int i) { return HELD ? held[i * SG_THREADS + t] : vecs.load(w0 + i * 32 + lane); };
  // f(vector, its number) over this thread's vectors, several in flight
  const auto for_vecs = [&](auto f) {
    constexpr int kBatch = HELD ? 2 : 4;
    int i = 0;
#pragma unroll 1
    for (; i + kBatch <= mine; i += kBatch) {
      uint4 u[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) u[j] = vec(i + j);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) f(u[j], i + j);
    }
#pragma unroll 1
    for (; i < mine; ++i) f(vec(i), i);
  };
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
  long long* const token = a.token + row;
  float* const logprob = a.logprob ? a.logprob + row : nullptr;
  SampleShared* lead = &sh;
  if (cs > 1) lead = cg::this_cluster().map_shared_rank(&sh, 0);
  if (t == 0) sh.n = 0;
  r.c64 = 1.4426950408889634 / r.T64;
  const float c = (float)r.c64;
  r.max_x = of_key(r.max_key(key_of(nan ? of_key(0xFFFFFFFFu) : top)));

  // f(element, id) over this thread's elements
  const auto each = [&](auto f) {
    for_vecs([&](const uint4& u, int i) {
      const int at = vecs.first(w0 + i * 32 + lane);
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at + e >= 0 && at + e < a.V) f(x[e], at + e);
    });
  };
  // Mass of a vector's logits from `low` on. In 32 bits each exponential is within 2^-22 of itself and 3 |t| 2^-24 ln 2 for
  // the roundings of t = (x - max) c, and eight of them are added in a tree.
  const Pair ref2(-r.max_x, -r.max_x), c2(c, c);
  const auto vec_mass = [&](const uint4& u, bool precise, float low) -> double {
    float x[E];
    vec_floats<T>(u, x);
    if (precise) {
      double s = 0.;
#pragma unroll
      for (int e = 0; e < E; ++e) s += x[e] >= low ? r.weight(x[e]) : 0.;
      return s;
    }
    Pair q[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e)
      q[e] = exp2_fast((Pair(x[2 * e] >= low ? x[2 * e] : -INFINITY, x[2 * e + 1] >= low ? x[2 * e + 1] : -INFINITY) + ref2) * c2);
#pragma unroll
    for (int o = E / 4; o > 0; o >>= 1)
#pragma unroll
      for (int e = 0; e < o; ++e) q[e] = q[e] + q[e + o];
    return (double)q[0].sum();
  };
  // Over the row, with a bound on its error: the mass' average |t| is the entropy of its shares less log2 of it (the largest
  // weight is 1), at most log2 V - log2 total.
  double error = 0.;
  const float log_v = log2f((float)a.V);
  const auto masses = [&](bool precise, float low) {
    double s = 0.;
    if (precise) {
#pragma unroll 1
      for (int i = 0; i < mine; ++i) s += vec_mass(vec(i), true, low);
    } else {
      for_vecs([&](const uint4& u, int) { s += vec_mass(u, false, low); });
    }
    const SampleRow::Part part = r.sum(s);
    error = precise ? 0. : part.total * (4.5e-7 + 1.3e-7 * fmaxf(log_v - log2f((float)part.total), 0.f));
    return part;
  };
  // Draws among the logits from `low` on.
  const auto draw = [&](float low) {
#pragma unroll 1
    for (int precise = 0; precise < 2; ++precise) {
      if (rank == 0 && t == 0) sh.verdict = kDone;
      const SampleRow::Part part = masses(precise, low);
      // The CTA in whose part the target lies, and there, counted from its start, the warp. Should rounding leave the
      // target at the very end, the last one with any mass takes it.
      double target = r.draw * part.total;
      const bool here = part.here > 0. && part.before <= target && (target < part.before + part.here || part.last);
      target -= part.before;
      double before = part.warp_before;
      if (here && part.warp > 0. && before <= target && (target < before + part.warp || part.warp_last)) {
        int at_i = 0, last_i = 0;
        double at_before = -1., last_before = before, s;
#pragma unroll 1
        for (int i0 = 0; i0 < chunk / 32; i0 += 4) {
          double part4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) part4[i] = i0 + i < mine ? vec_mass(vec(i0 + i), precise, low) : 0.;
#pragma unroll
          for (int i = 0; i < 4; ++i) part4[i] = SampleRow::warp_add(part4[i]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s = part4[i];
            if (s > 0.) last_i = i0 + i, last_before = before;
            if (at_before < 0. && before + s > target) at_i = i0 + i, at_before = before;
            before += s;
          }
          if (at_before >= 0.) break;
        }
        if (at_before < 0.) at_i = last_i, at_before = last_before;
        s = at_i < mine ? vec_mass(vec(at_i), precise, low) : 0.;
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
          vec_floats<T>(vec(at_i), x);
          const int at = vecs.first(w0 + at_i * 32 + lane);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            if (!(x[e] >= low)) continue;
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
            *token = id;
            if (logprob) *logprob = (float)log(r.weight(chosen) / part.total);
          }
        }
      }
      r.sync();
      const int verdict = lead->verdict;
      r.sync();
      if (verdict == kDone) return;
    }
  };
  // Candidates: logits from `low` on for which `in` holds, into the leader's list.
  const auto gather = [&](float low, auto in) {
    for_vecs([&](const uint4& u, int i) {
      if (!(vec_max<T>(u) >= low)) return;
      const int at = vecs.first(w0 + i * 32 + lane);
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (!(x[e] >= low) || !in(x[e])) continue;
        const int slot = atomicAdd(&lead->n, 1);
        if (slot < SG_CAP) lead->list[slot] = (unsigned long long)key_of(x[e]) << 32 | (uint32_t)~(at + e);
      }
    });
    r.sync();
    return lead->n;
  };

  const auto run = [&] {
    if (!(fabsf(r.max_x) < INFINITY)) {  // a NaN, an infinity or nothing allowed: no distribution; the largest number
      uint32_t key = 0;
      each([&](float x, int) { if (x == x) key = max(key, key_of(x)); });
      key = r.max_key(key);
      uint32_t first = 0;
      each([&](float x, int id) { if (x == x && key_of(x) == key) first = max(first, ~(uint32_t)id); });
      first = r.max_key(first);
      if (rank == 0 && t == 0) {
        *token = key ? (int)~first : 0;
        if (logprob) *logprob = __int_as_float(0x7FC00000);
      }
      return;
    }
    if (greedy) {
      uint32_t first = 0;
      if (top == r.max_x) each([&](float x, int id) { if (x == r.max_x) first = max(first, ~(uint32_t)id); });
      first = r.max_key(first);
      const double total = logprob ? masses(false, -INFINITY).total : 1.;
      if (rank == 0 && t == 0) {
        *token = (int)~first;
        if (logprob) *logprob = (float)-log(total);
      }
      return;
    }

    // min-p as a bound on the key: the least whose weight reaches it, among the 32 around max + T ln m, or where that window
    // lies above it (temperatures at which neighbours have the same weight) by a search in 32 parts.
    if (r.use_m && w == 0) {
      const uint32_t max_key = key_of(r.max_x);
      const auto reaches = [&](uint32_t key) {
        return __ballot_sync(0xffffffff, key == max_key || (key < max_key && r.weight(of_key(key)) >= r.m));
      };
      uint32_t lo = key_of(-3.4028235e38f), step = 1;
      uint32_t from = max(key_of((float)fmax(r.max_x + r.T64 * log(r.m), -3.4e38)), lo + 16) - 16;
      uint32_t ok = reaches(from + lane), hi = ok ? from + __ffs(ok) - 1 : max_key;
      if (ok & 1) {
        while (lo < hi) {
          step = (hi - lo) / 32 + 1;
          ok = reaches(min(lo + lane * step, hi));  // the last one does
          const int i = __ffs(ok) - 1;
          hi = min(lo + i * step, hi);
          if (i > 0) lo = lo + (i - 1) * step + 1;
          else break;
        }
      }
      if (lane == 0) sh.low = hi;
    }
    const bool by_k = r.use_k && r.k <= SG_LIST_K;
    const bool by_list = by_k || (!r.use_k && (r.use_p || r.use_m));
    // A bound that all candidates of top-k, or the SG_LIST_K largest logits, reach.
    uint32_t low = 0xFFFFFFFFu;
    if (by_k || (r.use_p && !r.use_k)) {
      const auto full = [&](int n) { return n < 32 ? 0 : min((n - 32) / chunk + 1, SG_WARPS); };  // warps without an idle lane
      const int warps = (cs - 1) * full(per) + full(vecs.n - (cs - 1) * per);
      const int j = warps > 0 ? ((by_k ? r.k : SG_LIST_K) + warps - 1) / warps : 33;
      uint32_t key = key_of(top);
      if (j > 32) {
        low = 0;
      } else if (w < full(v1 - v0)) {
        for (int i = 0;; ++i) {
          low = __reduce_max_sync(0xffffffff, key);
          if (i == j - 1) break;
          if (lane == __ffs(__ballot_sync(0xffffffff, key == low)) - 1) key = 0;
        }
      }
    }
    low = r.min_key(low);  // and its barrier for sh.low
    const uint32_t low_m = r.use_m ? sh.low : 0;
    double total = 0.;
    if (r.use_p && !by_k && !r.use_k) total = masses(false, -INFINITY).total;
    double total_error = error;
    if (by_list) {
      uint32_t bound = by_k || r.use_p ? low : 0;
      bool complete = by_k || bound == 0;
      if (r.use_m && !(by_k && r.use_p) && low_m >= bound) bound = low_m, complete = true;
      // below all numbers: -inf and the padding have no mass
      const float reach = bound <= key_of(-INFINITY) ? -3.4028235e38f : of_key(bound);
      const bool hopeless = !complete && masses(false, reach).total < 0.999 * r.p * total;
      const int n = hopeless ? SG_CAP + 1 : gather(reach, [](float) { return true; });
      if (n <= SG_CAP) {
        if (rank == 0) order_list(r, n);
        for (int precise = 0;; ++precise) {
          if (rank == 0 && w == 0) answer_from_list(r, n, complete, low_m, total, total_error, token, logprob);
          r.sync();
          const int verdict = lead->verdict;
          r.sync();
          if (verdict == kDone) return;
          if (verdict == kIncomplete) break;
          total = masses(true, -INFINITY).total;
          total_error = 0.;
        }
      } else {
        r.sync();  // the leader's count has been read
      }
    }

    // Many tokens stay. A histogram of the logits over equal steps down from the largest.
    float least = INFINITY;
    for_vecs([&](const uint4& u, int) {
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) least = fminf(least, x[e] > -INFINITY ? x[e] : least);
    });
    least = of_key(r.min_key(key_of(least)));
    float range = r.max_x - least;
    if (r.use_p && !r.use_k) range = fminf(range, 24.f * (float)r.T64);
    const bool flat = !(range > 0.f);  // all numbers are equal
    const float scale = flat ? 0.f : (SG_BINS - 1) / range;
    const auto bin_of = [&](float x) { return min((int)((r.max_x - x) * scale), SG_BINS - 1); };
    constexpr int kEach = SG_BINS / SG_THREADS;
    uint32_t count[kEach];  // of this thread's bins, over the row
    const bool by_bins = scale > 0.f && isfinite(scale) && (r.use_p || r.use_k);
    if (by_bins) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) sh.bins[t * kEach + i] = 0;
      __syncthreads();
      for_vecs([&](const uint4& u, int) {
        float x[E];
        vec_floats<T>(u, x);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (x[e] > -INFINITY) atomicAdd(&sh.bins[bin_of(x[e])], 1u);
      });
      r.sync();
#pragma unroll
      for (int i = 0; i < kEach; ++i) count[i] = 0;
      for (int o = 0; o < cs; ++o) {
        const uint32_t* theirs = cs > 1 ? cg::this_cluster().map_shared_rank(sh.bins, o) : sh.bins;
#pragma unroll
        for (int i = 0; i < kEach; ++i) count[i] += theirs[t * kEach + i];
      }
      r.sync();  // the bins give way to the list's weights
    }
    // The first bin at which the running sum of `of`(bin, count) exceeds `share`, SG_BINS if none does; `above`: the sum
    // before it.
    const auto find_bin = [&](double share, auto of, double& above) {
      double s = 0.;
#pragma unroll
      for (int i = 0; i < kEach; ++i) s += of(t * kEach + i, count[i]);
      double scan = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffff, scan, o);
        if (lane >= o) scan += up;
      }
      if (t == 0) sh.found = SG_BINS;
      if (lane == 31) sh.scan64[w] = scan;
      __syncthreads();
      double base = 0.;
      for (int i = 0; i < w; ++i) base += sh.scan64[i];
      double before = base + scan - s;
      if (before <= share && base + scan > share) {
        bool done = false;
        for (int i = 0; i < kEach; ++i) {
          const double one = of(t * kEach + i, count[i]);
          if (!done && before + one > share) {
            atomicMin(&sh.found, t * kEach + i);
            done = true;
          }
          if (!done) before += one;
        }
      }
      __syncthreads();
      const int bin = sh.found;
      if (bin / kEach == t) sh.scan64[0] = before;
      __syncthreads();
      above = sh.scan64[0];
      __syncthreads();
      return bin;
    };

    uint32_t kth = 0;  // top-k's bound
    if (r.use_k && flat) {
      kth = key_of(r.max_x);
    } else if (r.use_k) {
      bool found = false;
      if (by_bins) {
        double above;
        const int bin = find_bin(r.k - 0.5, [](int, uint32_t n) { return (double)n; }, above);
        if (bin == SG_BINS) {
          found = true;  // fewer numbers than k
        } else {
          if (rank == 0 && t == 0) sh.n = 0;
          r.sync();
          const int n = gather(-3.4028235e38f, [&](float x) { return bin_of(x) == bin; });
          if (n <= SG_CAP) {
            if (rank == 0) {
              order_list(r, n);
              if (t == 0) sh.low = key_part(sh.sorted[min(max(r.k - (int)above - 1, 0), n - 1)]);
            }
            found = true;
          }
          r.sync();
          kth = lead->low;
          r.sync();
          if (!found) kth = 0;
        }
      }
      if (!found) {  // ties, or outliers that leave too few steps for the rest: bisection of the key
#pragma unroll 1
        for (int b = 31; b >= 0; --b) {
          const uint32_t next = kth | 1u << b;
          int n = 0;
          each([&](float x, int) { n += key_of(x) >= next; });
          if (r.count(n) >= r.k) kth = next;
        }
      }
    }
    const auto from = [&](uint32_t key) { return key <= key_of(-3.4028235e38f) ? -3.4028235e38f : of_key(key); };
    uint32_t cut = 0;  // top-p's bound
    if (r.use_p && flat) {
      cut = key_of(r.max_x);
    } else if (r.use_p) {
      bool found = false;
      if (r.use_k) {
        total = masses(false, from(kth)).total;
        total_error = error;
      }
      int first = 0, last = -1, n = 0;
      if (by_bins) {
        // the steps around the one that the weights at their middles point to
        double above;
        const int bin = find_bin(r.p * total, [&](int b, uint32_t n) {
          return n ? n * (double)exp2_fast(-((float)b + 0.5f) / scale * c) : 0.;
        }, above);
        first = max(bin - 2, 0);
        last = min(bin + 2, SG_BINS - 1);
        if (rank == 0 && t == 0) sh.n = 0;
        r.sync();
        n = gather(from(kth), [&](float x) {
          const int b = bin_of(x);
          return b >= first && b <= last;
        });
        if (n <= SG_CAP && rank == 0) order_list(r, n);
        r.sync();
      }
#pragma unroll 1
      for (int precise = 0; precise < 2 && !found; ++precise) {
        if (precise) {
          total = masses(true, from(kth)).total;
          total_error = 0.;
        }
        const double share = r.p * total, blur = r.p * total_error;
        if (by_bins && n <= SG_CAP) {
          // the least number of the steps above: a bound between them and those gathered
          float edge = INFINITY;
          each([&](float x, int) { if (x > -INFINITY && bin_of(x) < first) edge = fminf(edge, x); });
          edge = of_key(r.min_key(key_of(edge)));
          const double above = edge < INFINITY ? masses(precise, fmaxf(edge, from(kth))).total : (error = 0., 0.);
          if (rank == 0 && w == 0) bound_from_list(r, n, last == SG_BINS - 1, above, error, share, blur);
          r.sync();
          const int verdict = lead->verdict;
          cut = lead->low;
          r.sync();
          if (verdict == kDone) break;
          if (verdict == kAmbiguous) continue;
        }
        // Bisection: the largest key such that it and those above hold more than the share.
        bool unsure = false;
        cut = 0;
#pragma unroll 1
        for (int b = 31; b >= 0; --b) {
          const uint32_t next = cut | 1u << b;
          const double s = next > key_of(r.max_x) ? (error = 0., 0.) : masses(precise, from(max(next, kth))).total;
          unsure |= error + blur > 0. && fabs(s - share) <= error + blur;
          if (s > share) cut = next;
        }
        found = !unsure;
      }
    }
    draw(from(max(max(kth, cut), low_m)));
  };
  run();
  if (cs > 1) cg::this_cluster().sync();  // no CTA leaves while others read its memory
}

template <typename T, bool HELD>
void sample_given_launch(const SampleGivenArgs& a, int smem, int device, cudaStream_t s) {
  auto* kernel = sample_given_kernel<T, HELD>;
  static bool ready[64] = {};  // per device
  if (device < 0 || device >= 64 || !ready[device]) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SG_VECS * SG_THREADS * 16);
    if (device >= 0 && device < 64) ready[device] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a.rows * a.cluster);
  cfg.blockDim = dim3(SG_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = a.cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = a.cluster > 1 ? 2 : 1;
  note_launch();
  cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T>
void sample_given_sized(SampleGivenArgs a, int device, cudaStream_t s) {
  constexpr int E = LogitType<T>::E;
  const int vecs = (a.V + E - 1) / E + 1;  // one more where a row starts off the grid
  const int sms = astrai_host::num_sms(device);
  const char* env = getenv("SG_CS");
  int cs = 1;
  while (cs < SG_MAX_CLUSTER && (long long)a.rows * cs * 2 <= sms && vecs >= cs * 2 * SG_THREADS) cs *= 2;
  if (env) cs = atoi(env);
  a.cluster = cs;
  const int each = ((vecs + cs - 1) / cs + SG_THREADS - 1) / SG_THREADS;  // vectors of a thread
  if (each <= SG_VECS) sample_given_launch<T, true>(a, each * SG_THREADS * 16, device, s);
  else sample_given_launch<T, false>(a, 0, device, s);
}

}  // namespace astrai

namespace astrai_host {
using namespace astrai;

void sample_given(const void* x, long long ldx, int rows, int V, const void* uniform, bool uniform64,
                  const float* temperature, const int* top_k, const float* top_p, const float* min_p, long long* token,
                  float* logprob, int dtype, int device, cudaStream_t s) {
  const SampleGivenArgs a{x, ldx, rows, V, 1, uniform, uniform64, temperature, top_k, top_p, min_p, token, logprob};
  if (dtype == 0) sample_given_sized<__nv_bfloat16>(a, device, s);
  else if (dtype == 1) sample_given_sized<__half>(a, device, s);
  else sample_given_sized<float>(a, device, s);
}

}  // namespace astrai_host
