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
// A CTA of 512 threads takes a row, two on an SM. Logits that fit stay in its shared memory between the passes over them,
// others come from L2 again. (In an earlier form, whose passes were inlined and waited for their instructions, 64 rows of 32000
// with k = 50 took 13.9 us, 15.4 with 1024 threads and more with clusters of CTAs for a row; not measured again since.) The
// bound that gathers the candidates is the one of the top logits: the smallest, over the warps, of each warp's j-th largest
// thread maximum. Where top-p reaches below them (flat rows) or k is large, a histogram over 4096 equal steps of the logits
// shows in which steps the bound must lie, and the few logits there are ordered and decided exactly.
//
// What bounds it is the chain of a row's steps, of 1000 to 5000 clocks each with their barriers (64 rows of 32000, k = 50:
// load 2100, largest 1400, bound 1600, gather 3800, sort 2800, draw 5600), and for flat rows the 13 operations in 64 bits a logit
// where the 32-bit sums leave doubt: 64 rows of 32000 take 10 us with k = 50, 12.5 with k = 50 and p = 0.95, 50 to 65 with
// p = 0.9 or 0.98 alone, 27 with no filter at all.
//
// A row takes each step once, so that the time to fetch instructions counts: inlined into each other, the passes were 430 KB
// of code, a third of all stalls waited for it (64 rows of 32000, k = 50: 15 us), hence functions that are called.
#include "launch.cuh"
#include "logits.cuh"

namespace astrai {

constexpr int SG_THREADS = 512;
constexpr int SG_VECS = 8;      // 16-byte vectors that a thread loads at once
constexpr int SG_LIST_K = 256;  // top-k up to here, and the largest logits looked at for top-p, go by the list
constexpr int SG_CAP = 2 * SG_THREADS;  // candidates
constexpr int SG_BINS = 4096;
constexpr int SG_GROUPS = 8;    // of a thread's vectors: each with its maximum
constexpr uint32_t kLowest = 0x00800000u;  // the key of the lowest finite number

struct SampleGivenArgs {
  const void* x;
  long long ldx;
  int rows, V;
  const void* uniform;  // [rows] fp32 or fp64
  int uniform64;
  const float* temperature;  // [rows]
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* token;  // [rows]
  float* logprob;    // [rows] or null
};

// 2^(k / 16), in shared memory: a warp's 32 reads of these 16 words meet no bank twice.
struct Powers {
  double at[16];
};
// 2^(t / 16) for N values t <= 0 in 64 bits, within 2^-42 of themselves (below 2^-1000: zero): a power of two, one of `pow`
// and e^z = sum z^n / n! at |z| <= ln 2 / 32, whose sixth term is below 2^-42. Step by step for all of them, as each step
// waits for the last.
template <int N>
__device__ __forceinline__ void exp2_16th(double (&t)[N], const Powers& pow) {
  constexpr double kRound = 6755399441055744.;  // 1.5 * 2^52: adding it rounds to a whole number
  constexpr double a = 0.6931471805599453 / 16.;
  constexpr double kTerms[] = {a * a * a * a / 24., a * a * a / 6., a * a / 2., a, 1.};
  int n[N], live[N];
  double e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    live[i] = t[i] > -16000. ? -1 : 0;
    const double whole = t[i] + kRound;
    n[i] = __double2loint(whole);
    t[i] -= whole - kRound;
    e[i] = a * a * a * a * a / 120.;
  }
#pragma unroll
  for (const double term : kTerms)
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = fma(e[i], t[i], term);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    e[i] *= pow.at[n[i] & 15];
    t[i] = __hiloint2double((__double2hiint(e[i]) + (n[i] >> 4 << 20)) & live[i], __double2loint(e[i]) & live[i]);
  }
}

// The least key in lo .. hi for which `reaches` holds, in all lanes: it holds from some key on, at hi at the latest.
template <typename F>
__device__ __forceinline__ uint32_t least_key(int lane, uint32_t lo, uint32_t hi, F reaches) {
#pragma unroll 1
  while (lo < hi) {
    const uint32_t step = (hi - lo + 30) / 31;  // the last lane takes hi
    const int i = __ffs(__ballot_sync(0xffffffff, reaches(min(lo + lane * step, hi)))) - 1;
    hi = min(lo + i * step, hi);
    if (i == 0) break;
    lo += (i - 1) * step + 1;
  }
  return hi;
}

enum Verdict { kDone = 0, kAmbiguous = 1, kIncomplete = 2 };

struct SampleShared {
  // candidates in no order; some of their numbers in descending order
  uint32_t key[SG_CAP], id[SG_CAP], sorted[SG_CAP];
  union {
    double before[SG_CAP];     // mass before a sorted one
    uint32_t swap[2][SG_CAP];  // for sorting
    uint32_t bins[SG_BINS];
  };
  double warp_sum[SG_THREADS / 32];
  double group_sum[SG_THREADS / 32][SG_GROUPS];  // a warp's mass by groups of vectors
  uint32_t warp_key[SG_THREADS / 32];
  // the row and its settings
  const void* row;
  int V, chunk, group;  // chunk: vectors of a warp, one after another, so that sums over warps are sums over ids
  float max_x, c;       // c = log2(e) / T
  double T64, c64, p, m, draw;  // c64 = 16 log2(e) / T
  Powers pow;
  int k;
  bool use_k, use_p, use_m;
  long long* token;
  float* logprob;
  // results
  int n;           // candidates
  uint32_t low;    // the least key that min-p keeps, later of a bound
  int hit, last;
  int bin;
  float above;     // the histogram's sum before `bin`
};

template <typename T, bool HELD>
struct Sampler {
  static constexpr int E = LogitType<T>::E, NT = SG_THREADS, kWarps = NT / 32;

  static __device__ __forceinline__ SampleShared& shared() {
    extern __shared__ __align__(16) unsigned char sample_smem[];
    return *reinterpret_cast<SampleShared*>(sample_smem);
  }
  // the held vectors: i of thread t at i * NT + t; if they are not held, the maxima of their groups
  static __device__ __forceinline__ uint4* held() {
    extern __shared__ __align__(16) unsigned char sample_smem[];
    return reinterpret_cast<uint4*>(sample_smem + (sizeof(SampleShared) + 15) / 16 * 16);
  }
  static __device__ __forceinline__ float* tops() { return reinterpret_cast<float*>(held()); }

  // This thread's vectors: w0 + i * 32 + lane, i < mine.
  struct Mine {
    RowVecs<T> vecs;
    int w0, mine;
    __device__ Mine(const SampleShared& sh) : vecs(static_cast<const T*>(sh.row), sh.V) {
      const int t = threadIdx.x;
      w0 = t / 32 * sh.chunk;
      mine = max(0, min(sh.chunk / 32, (min(w0 + sh.chunk, vecs.n) - w0 - (t & 31) + 31) / 32));
    }
    __device__ __forceinline__ int first(int i) const { return vecs.first(w0 + i * 32 + (threadIdx.x & 31)); }
    __device__ __forceinline__ uint4 vec(int i) const {
      if (i >= mine) return vec_neg_inf<T>();
      return HELD ? held()[i * NT + threadIdx.x] : vecs.load(w0 + i * 32 + (threadIdx.x & 31));
    }
    __device__ __forceinline__ void four(int i, uint4 (&u)[4]) const {
      if constexpr (HELD) {
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = vec(i + j);
      } else {
        vecs.load(w0 + i * 32, shared().chunk / 32 - i, mine - i, u);
      }
    }
  };
  // f(vector, its number) over this thread's vectors of the groups that reach `low`, four in flight (with some behind the
  // last that read as -inf); g(group) after each
  template <typename F, typename G>
  static __device__ __forceinline__ void for_vecs(const SampleShared& sh, const Mine& me, float low, F f, G g) {
#pragma unroll 1
    for (int i0 = 0, at = 0; i0 < sh.chunk / 32; i0 += sh.group, ++at) {
      const int end = min(i0 + sh.group, me.mine);
      if (i0 < end && tops()[at * NT + threadIdx.x + (HELD ? sh.chunk / 32 * NT * 4 : 0)] >= low) {
#pragma unroll 1
        for (int i = i0; i < end; i += 4) {
          uint4 u[4];
          me.four(i, u);
#pragma unroll
          for (int j = 0; j < 4; ++j) f(u[j], i + j);
        }
      }
      g(at);
    }
  }
  template <typename F>
  static __device__ __forceinline__ void for_vecs(const SampleShared& sh, const Mine& me, float low, F f) {
    for_vecs(sh, me, low, f, [](int) {});
  }

  // ---------------------------------------------------------------- reductions: the same result in all threads
  template <typename F>
  static __device__ __forceinline__ uint32_t reduce(uint32_t v, uint32_t none, F f) {
    SampleShared& sh = shared();
    v = f(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.warp_key[threadIdx.x / 32] = v;
    __syncthreads();
    return f((threadIdx.x & 31) < kWarps ? sh.warp_key[threadIdx.x & 31] : none);
  }
  static __device__ __noinline__ uint32_t max_of(uint32_t v) {
    return reduce(v, 0, [](uint32_t x) { return __reduce_max_sync(0xffffffff, x); });
  }
  static __device__ __noinline__ uint32_t min_of(uint32_t v) { return ~max_of(~v); }
  static __device__ __noinline__ uint32_t sum_of(uint32_t v) {
    return reduce(v, 0, [](uint32_t x) { return __reduce_add_sync(0xffffffff, x); });
  }
  static __device__ __forceinline__ double warp_add(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
    return v;
  }
  static __device__ __forceinline__ double lanes_before(double v) {  // running sum over the lanes, v included
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffff, v, o);
      if ((threadIdx.x & 31) >= o) v += up;
    }
    return v;
  }
  // The sum over the threads before this one, and over all. The warps' sums stay in sh.warp_sum.
  static __device__ __noinline__ double2 scan(double s) {
    SampleShared& sh = shared();
    const int lane = threadIdx.x & 31, w = threadIdx.x / 32;
    const double run = lanes_before(s);
    __syncthreads();
    if (lane == 31) sh.warp_sum[w] = run;
    __syncthreads();
    const double warps = lanes_before(lane < kWarps ? sh.warp_sum[lane] : 0.);
    const double base = __shfl_sync(0xffffffff, warps, max(w - 1, 0));
    return make_double2((w > 0 ? base : 0.) + (run - s), __shfl_sync(0xffffffff, warps, 31));
  }

  // ---------------------------------------------------------------- passes over the row
  static __device__ __noinline__ double weight(float x) {
    const SampleShared& sh = shared();
    double t[1] = {((double)x - (double)sh.max_x) * sh.c64};
    exp2_16th(t, sh.pow);
    return t[0];
  }
  // ln x within 2^-40, for x >= 1: the fp32 logarithm and one step of Newton's method for e^y = x.
  static __device__ __forceinline__ double log_64(double x) {
    const double y = (double)logf((float)x);
    double t[1] = {-y * (16. * 1.4426950408889634)};
    exp2_16th(t, shared().pow);
    return y + (x * t[0] - 1.);
  }
  // Mass of a vector's logits from `low` on. In 32 bits each exponential is within 2^-22 of itself and 3 |t| 2^-24 ln 2 for
  // the roundings of t = (x - max) c, and eight of them are added in a tree.
  static __device__ __forceinline__ double vec_mass(const uint4& u, float low, Pair ref2, Pair c2) {
    float x[E];
    vec_floats<T>(u, x);
    Pair q[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e)
      q[e] = exp2_fast((Pair(x[2 * e] >= low ? x[2 * e] : -INFINITY, x[2 * e + 1] >= low ? x[2 * e + 1] : -INFINITY) + ref2) * c2);
#pragma unroll
    for (int o = E / 4; o > 0; o >>= 1)
#pragma unroll
      for (int e = 0; e < o; ++e) q[e] = q[e] + q[e + o];
    return (double)q[0].sum();
  }
  // In 64 bits, and that of the logits from `high` on added to `above`.
  static __device__ __forceinline__ double vec_mass_64(const uint4& u, float low, double max_x, double c64, float high, double& above) {
    float x[E];
    vec_floats<T>(u, x);
    double sum = 0.;
#pragma unroll
    for (int e0 = 0; e0 < E; e0 += 4) {
      double s[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = x[e0 + e] >= low ? ((double)x[e0 + e] - max_x) * c64 : -INFINITY;
      exp2_16th(s, shared().pow);
      sum += (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x[e0 + e] >= high) above += s[e];
    }
    return sum;
  }
  // This warp's mass of vectors i .. i + 3 each.
  static __device__ __noinline__ void warp_masses(bool precise, float low, int i, int end, double (&s)[4], double& mine, int which) {
    const SampleShared& sh = shared();
    const Mine me(sh);
    const Pair ref2(-sh.max_x, -sh.max_x), c2(sh.c, sh.c);
    double none = 0.;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 u = i + j < end ? me.vec(i + j) : vec_neg_inf<T>();
      s[j] = precise ? vec_mass_64(u, low, sh.max_x, sh.c64, INFINITY, none) : vec_mass(u, low, ref2, c2);
      if (j == which) mine = s[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = warp_add(s[j]);
  }
  // The row's mass from `low` on; by warps in sh.warp_sum, by their groups in sh.group_sum. That from `high` on in `above`: both
  // in one pass, as 13 operations of 64 bits a logit bound it (32000 logits: 12000 clocks).
  static __device__ __noinline__ double mass_64(float low, float high, double& above) {
    SampleShared& sh = shared();
    const Mine me(sh);
    const double max_x = sh.max_x, c64 = sh.c64;
    double s = 0., s_high = 0.;
#pragma unroll 1
    for (int i0 = 0, at = 0; i0 < sh.chunk / 32; i0 += sh.group, ++at) {
      double part = 0.;
#pragma unroll 1
      for (int i = i0; i < min(i0 + sh.group, me.mine); ++i) part += vec_mass_64(me.vec(i), low, max_x, c64, high, s_high);
      s += part;
      if (!HELD) {
        part = warp_add(part);
        if ((threadIdx.x & 31) == 0) sh.group_sum[threadIdx.x / 32][at] = part;
      }
    }
    if (high < INFINITY) above = scan(s_high).y;
    return scan(s).y;
  }
  static __device__ __noinline__ double mass_32(float low) {
    SampleShared& sh = shared();
    const Mine me(sh);
    const Pair ref2(-sh.max_x, -sh.max_x), c2(sh.c, sh.c);
    double s = 0., part = 0.;
    for_vecs(sh, me, low, [&](const uint4& u, int) { part += vec_mass(u, low, ref2, c2); },
             [&](int at) {
               s += part;
               if (!HELD) {
                 part = warp_add(part);
                 if ((threadIdx.x & 31) == 0) sh.group_sum[threadIdx.x / 32][at] = part;
               }
               part = 0.;
             });
    return scan(s).y;
  }
  // With a bound on its error: the mass' average |t| is the entropy of its shares less log2 of it (the largest weight is 1),
  // at most log2 V - log2 total.
  static __device__ __forceinline__ double mass(bool precise, float low, double& error) {
    double none;
    const double total = precise ? mass_64(low, INFINITY, none) : mass_32(low);
    error = precise || total == 0. ? 0. : total * (4.5e-7 + 1.3e-7 * fmaxf(log2f((float)shared().V) - log2f((float)total), 0.f));
    return total;
  }
  // The place of this lane's `mine` entries in a list, behind those that it has: one atomic a warp.
  static __device__ __forceinline__ int place(int* n, int mine) {
    const int lane = threadIdx.x & 31;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffff, upto, o);
      if (lane >= o) upto += up;
    }
    int at = 0;
    if (lane == 31 && upto > 0) at = atomicAdd(n, upto);
    return __shfl_sync(0xffffffff, at, 31) + upto - mine;
  }
  // Candidates: the logits from `low` on, if they are not too many; their number. First the vectors that hold any, marked in a
  // word for up to 32 of a thread's, then those vectors' elements, a vector a thread: a warp in which a few lanes look at eight
  // elements each takes as long as if all did.
  static __device__ __noinline__ int gather_top(float low) {
    SampleShared& sh = shared();
    const Mine me(sh);
    const int t = threadIdx.x;
    __syncthreads();
    if (t == 0) sh.n = sh.hit = 0;
    __syncthreads();
#pragma unroll 1
    for (int i0 = 0, at = 0; i0 < sh.chunk / 32; i0 += sh.group, ++at) {
      const int end = min(i0 + sh.group, me.mine);
      const bool may = i0 < end && tops()[at * NT + t + (HELD ? sh.chunk / 32 * NT * 4 : 0)] >= low;
      if (!__any_sync(0xffffffff, may)) continue;
#pragma unroll 1
      for (int i1 = i0; i1 < min(i0 + sh.group, sh.chunk / 32); i1 += 32) {
        uint32_t marks = 0;
        if (may) {
#pragma unroll 1
          for (int i = i1; i < min(i1 + 32, end); i += 4) {
            uint4 u[4];
            me.four(i, u);
            uint32_t some = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) some |= (uint32_t)(i + j < end && vec_max<T>(u[j]) >= low) << j;
            marks |= some << (i - i1);
          }
        }
        __syncwarp();
        int to = place(&sh.hit, __popc(marks));
#pragma unroll 1
        for (; marks && to < SG_CAP; marks &= marks - 1) sh.sorted[to++] = (i1 + __ffs(marks) - 1) * NT + t;
      }
    }
    __syncthreads();
    const int n = sh.hit;
    if (n > SG_CAP) return SG_CAP + 1;
#pragma unroll 1
    for (int q0 = 0; q0 < n; q0 += NT) {
      const int q = q0 + t;
      uint32_t marks = 0;
      int first = 0;
      float x[E];
      if (q < n) {
        const int v = sh.sorted[q], of = v % NT, number = of / 32 * sh.chunk + v / NT * 32 + of % 32;
        first = me.vecs.first(number);
        vec_floats<T>(HELD ? held()[v] : me.vecs.load(number), x);
#pragma unroll
        for (int e = 0; e < E; ++e) marks |= (uint32_t)(x[e] >= low && first + e >= 0 && first + e < sh.V) << e;
      }
      __syncwarp();
      int to = place(&sh.n, __popc(marks));
#pragma unroll 1
      for (; marks && to < SG_CAP; marks &= marks - 1, ++to) {
        const int e = __ffs(marks) - 1;
        float one = x[0];
#pragma unroll
        for (int j = 1; j < E; ++j) one = e == j ? x[j] : one;
        sh.key[to] = key_of(one);
        sh.id[to] = first + e;
      }
    }
    __syncthreads();
    return sh.n;
  }
  // Candidates: the logits in low .. high (exclusive), if they are not too many; their number.
  static __device__ __noinline__ int gather(float low, float high) {
    SampleShared& sh = shared();
    const Mine me(sh);
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    for_vecs(sh, me, low, [&](const uint4& u, int i) {
      if (!(vec_max<T>(u) >= low)) return;
      float x[E];
      vec_floats<T>(u, x);
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) bits |= (uint32_t)(x[e] >= low && x[e] < high) << e;
      if (!bits) return;
      int to = atomicAdd(&sh.n, __popc(bits));
      const int at = me.first(i);
#pragma unroll 1
      for (; bits; bits &= bits - 1, ++to) {
        const int e = __ffs(bits) - 1;
        float one = x[0];
#pragma unroll
        for (int j = 1; j < E; ++j) one = e == j ? x[j] : one;
        if (to < SG_CAP) sh.key[to] = key_of(one), sh.id[to] = at + e;
      }
    });
    __syncthreads();
    return sh.n;
  }
  // The number of logits from `low` on by steps down from the largest; those in the last step, or beyond it, are not counted.
  static __device__ __forceinline__ int bin_of(float x, float max_x, float scale) {
    return min((int)((max_x - x) * scale), SG_BINS - 1);
  }
  static __device__ __noinline__ void histogram(float scale, float low) {
    SampleShared& sh = shared();
    const Mine me(sh);
    __syncthreads();
    for (int i = threadIdx.x; i < SG_BINS; i += NT) sh.bins[i] = 0;
    __syncthreads();
    const float max_x = sh.max_x;
    for_vecs(sh, me, low, [&](const uint4& u, int) {
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int bin = bin_of(x[e], max_x, scale);
        if (x[e] >= low && bin < SG_BINS - 1) atomicAdd(&sh.bins[bin], 1u);
      }
    });
    __syncthreads();
  }
  // The first bin at which the running sum exceeds `target` (SG_BINS: none) and the sum before it: of the logits' number, or
  // of their mass with each taken at the middle of its step (fp32, sums of whole numbers up to 2^22 are exact).
  static __device__ __noinline__ int find_bin(float target, float scale, bool mass, float& above) {
    SampleShared& sh = shared();
    constexpr int kEach = SG_BINS / NT;
    const int t = threadIdx.x, lane = t & 31, w = t / 32;
    float bins[kEach], s = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      bins[i] = (float)sh.bins[t * kEach + i];
      if (mass) bins[i] *= exp2_fast(-((float)(t * kEach + i) + 0.5f) / scale * sh.c);
      s += bins[i];
    }
    float run = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float up = __shfl_up_sync(0xffffffff, run, o);
      if (lane >= o) run += up;
    }
    __syncthreads();
    if (lane == 31) sh.warp_key[w] = __float_as_uint(run);
    if (t == 0) sh.bin = SG_BINS;
    __syncthreads();
    float warps = lane < kWarps ? __uint_as_float(sh.warp_key[lane]) : 0.f;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float up = __shfl_up_sync(0xffffffff, warps, o);
      if (lane >= o) warps += up;
    }
    const float base = __shfl_sync(0xffffffff, warps, max(w - 1, 0));
    float before = (w > 0 ? base : 0.f) + (run - s);
    if (before <= target && before + s > target) {  // two threads where rounding lets their parts overlap: the first
      int i = 0;
#pragma unroll
      for (int b = 0; b < kEach; ++b)
        if (i == b && b + 1 < kEach && before + bins[b] <= target) before += bins[b], ++i;
      atomicMin(&sh.bin, t * kEach + i);
    }
    __syncthreads();
    const int bin = sh.bin;
    if (bin / kEach == t) sh.above = before;
    __syncthreads();
    above = sh.above;
    return bin;
  }
  // That running sum before bin `end`.
  static __device__ __noinline__ double mass_of_bins(int end, float scale) {
    const SampleShared& sh = shared();
    float s = 0.f;
    for (int i = threadIdx.x; i < end; i += NT) s += (float)sh.bins[i] * exp2_fast(-((float)i + 0.5f) / scale * sh.c);
    return scan((double)s).y;
  }
  // The least key in a bin before this one.
  static __device__ __noinline__ uint32_t edge_of(int bin, float scale) {
    const float max_x = shared().max_x;
    const auto before = [&](uint32_t key) { return bin_of(of_key(key), max_x, scale) < bin; };
    uint32_t lo = kLowest, hi = key_of(max_x);
    const float x = max_x - (float)bin / scale, near = 1e-6f * (fabsf(max_x) + fabsf(x));  // a window around it
    const uint32_t a = key_of(x - near), b = key_of(x + near);
    if (a > lo && b < hi && !before(a) && before(b)) lo = a, hi = b;
    return least_key(threadIdx.x & 31, lo, hi, before);
  }
  static __device__ __noinline__ float least() {
    const SampleShared& sh = shared();
    const Mine me(sh);
    float least = INFINITY;
    for_vecs(sh, me, -INFINITY, [&](const uint4& u, int) {
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) least = fminf(least, x[e] > -INFINITY ? x[e] : least);
    });
    return of_key(min_of(key_of(least)));
  }
  static __device__ __noinline__ int count_from(float low) {
    const SampleShared& sh = shared();
    const Mine me(sh);
    int n = 0;
    for_vecs(sh, me, low, [&](const uint4& u, int) {
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) n += x[e] >= low;
    });
    return sum_of(n);
  }
  // The largest number of a row with NaN (`tops` leave out the vectors that hold one); -inf where there is none.
  static __device__ __noinline__ float largest_number() {
    const SampleShared& sh = shared();
    const Mine me(sh);
    float most = -INFINITY;
    for_vecs(sh, me, -INFINITY, [&](const uint4& u, int) { most = fmaxf(most, vec_max_number<T>(u)); });
    return of_key(max_of(key_of(most)));
  }
  // The lowest id of a number equal to `value`, looked for where `tops` reach `from`.
  static __device__ __noinline__ uint32_t first_id(float value, float from) {
    const SampleShared& sh = shared();
    const Mine me(sh);
    uint32_t first = 0;  // complement
    for_vecs(sh, me, from, [&](const uint4& u, int i) {
      float x[E];
      vec_floats<T>(u, x);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int id = me.first(i) + e;
        if (i < me.mine && x[e] == value && id >= 0 && id < sh.V) first = max(first, ~(uint32_t)id);
      }
    });
    return ~max_of(first);
  }

  // ---------------------------------------------------------------- candidates
  // `n` numbers of sh (at `from`) in descending order into sh.sorted: a bitonic sort, one or two numbers a thread,
  // within a warp by shuffles. Written out: as a loop its branches took most of the time (128 numbers: 7000 clocks, now about 2700).
  template <bool TWO>
  static __device__ __noinline__ void sort_by(int n, uint32_t v0, uint32_t v1) {
    SampleShared& sh = shared();
    const int t = threadIdx.x;
    int turn = 0;
#pragma unroll
    for (int k = 2; k <= (TWO ? 2 * SG_THREADS : SG_THREADS); k <<= 1) {
      if (k / 2 >= n) break;
#pragma unroll
      for (int j = k >> 1; j > 0; j >>= 1) {
        if (j == SG_THREADS) {  // the two numbers of a thread
          const uint32_t a = max(v0, v1);
          v1 = min(v0, v1);
          v0 = a;
          continue;
        }
        uint32_t o0, o1 = 0;
        if (j >= 32) {
          sh.swap[turn][t] = v0;
          if (TWO) sh.swap[turn][t + SG_THREADS] = v1;
          __syncthreads();
          o0 = sh.swap[turn][t ^ j];
          if (TWO) o1 = sh.swap[turn][(t ^ j) + SG_THREADS];
          turn ^= 1;
        } else {
          o0 = __shfl_xor_sync(0xffffffff, v0, j);
          if (TWO) o1 = __shfl_xor_sync(0xffffffff, v1, j);
        }
        const bool lower = (t & j) == 0;
        v0 = ((t & k) == 0) == lower ? max(v0, o0) : min(v0, o0);
        if (TWO) v1 = (((t + SG_THREADS) & k) == 0) == lower ? max(v1, o1) : min(v1, o1);
      }
    }
    if (t < n) sh.sorted[t] = v0;
    if (TWO && t + SG_THREADS < n) sh.sorted[t + SG_THREADS] = v1;
  }
  static __device__ __noinline__ void sort(int n, const uint32_t* from) {
    const int t = threadIdx.x;
    const uint32_t v0 = t < n ? from[t] : 0, v1 = t + SG_THREADS < n ? from[t + SG_THREADS] : 0;
    __syncthreads();
    if (n > SG_THREADS) sort_by<true>(n, v0, v1);
    else sort_by<false>(n, v0, v1);
    __syncthreads();
  }
  // Where the value of the sorted candidate i begins.
  static __device__ __forceinline__ int first_of_value(const SampleShared& sh, int i) {
    const uint32_t key = sh.sorted[i];
    if (i == 0 || sh.sorted[i - 1] != key) return i;
    int first = 0, last = i - 1;
#pragma unroll 1
    while (first < last) {
      const int mid = (first + last) / 2;
      if (sh.sorted[mid] == key) last = mid;
      else first = mid + 1;
    }
    return first;
  }
  // The mass before each of the sorted candidates, and of all.
  static __device__ __noinline__ double mass_before(int n) {
    SampleShared& sh = shared();
    const int each = n > NT ? 2 : 1, i = threadIdx.x * each;
    double a = 0., b = 0.;
    if (i < n) a = weight(of_key(sh.sorted[i]));
    if (each == 2 && i + 1 < n) b = weight(of_key(sh.sorted[i + 1]));
    const double2 run = scan(a + b);
    if (i < n) sh.before[i] = run.x;
    if (each == 2 && i + 1 < n) sh.before[i + 1] = run.x + a;
    __syncthreads();
    return run.y;
  }
  // Top-p's bound among the sorted candidates, above which lies the mass `above`: keeps those whose strictly larger logits
  // hold at most `share`; `doubt`: how near to it that is not known; `end`: no logit that could be kept lies below them.
  // The least key that is kept in sh.low.
  static __device__ __noinline__ Verdict bound(int n, double above, double share, double doubt, bool end) {
    SampleShared& sh = shared();
    const double all = above + mass_before(n);
    bool unsure = !end && doubt > 0. && fabs(all - share) <= doubt;
    int kept = 0;
#pragma unroll 1
    for (int i = threadIdx.x; i - (int)threadIdx.x < n; i += NT) {
      bool keep = false;
      if (i < n) {
        const double larger = above + sh.before[first_of_value(sh, i)];
        keep = larger == 0. || !(larger > share);
        unsure |= larger > 0. && doubt > 0. && fabs(larger - share) <= doubt;
      }
      kept += __syncthreads_count(keep);
    }
    unsure = __syncthreads_or(unsure);
    if (threadIdx.x == 0) sh.low = kept > 0 ? sh.sorted[kept - 1] : 0;
    __syncthreads();
    return unsure ? kAmbiguous : kept == 0 || (!end && !(all > share)) ? kIncomplete : kDone;
  }
  // The draw among the candidates from the key `low` on, in the order of ids: an id and a place in the list make one number.
  static __device__ __noinline__ void draw_from_list(int n, uint32_t low) {
    SampleShared& sh = shared();
    const int t = threadIdx.x;
    __syncthreads();
    for (int i = t; i < n; i += NT) sh.swap[1][i] = ~(sh.id[i] << 10 | i);
    __syncthreads();
    sort(n, sh.swap[1]);
    if (t == 0) sh.hit = SG_CAP, sh.last = -1;
    const int each = n > NT ? 2 : 1, i = t * each;
    double w0 = 0., w1 = 0.;
    if (i < n && sh.key[~sh.sorted[i] & 1023] >= low) w0 = weight(of_key(sh.key[~sh.sorted[i] & 1023]));
    if (each == 2 && i + 1 < n && sh.key[~sh.sorted[i + 1] & 1023] >= low) w1 = weight(of_key(sh.key[~sh.sorted[i + 1] & 1023]));
    const double2 run = scan(w0 + w1);  // with its barriers for hit and last
    const double target = sh.draw * run.y;
    int hit = SG_CAP;  // the first at which the running sum is above the target, or the last with any mass
    if (w1 > 0. && run.x + w0 + w1 > target) hit = i + 1;
    if (w0 > 0. && run.x + w0 > target) hit = i;
    hit = __reduce_min_sync(0xffffffff, hit);
    const int last = __reduce_max_sync(0xffffffff, w1 > 0. ? i + 1 : w0 > 0. ? i : -1);
    if ((t & 31) == 0 && hit < SG_CAP) atomicMin(&sh.hit, hit);
    if ((t & 31) == 0 && last >= 0) atomicMax(&sh.last, last);
    __syncthreads();
    if (t == 0) answer(~sh.sorted[sh.hit < n ? sh.hit : sh.last] & 1023, run.y);
  }
  static __device__ __noinline__ void answer(int place, double total) { answer(shared().id[place], of_key(shared().key[place]), total); }
  static __device__ __noinline__ void answer(int id, float x, double total) {
    const SampleShared& sh = shared();
    *sh.token = id;
    if (sh.logprob) *sh.logprob = (float)(((double)x - (double)sh.max_x) / sh.T64 - log_64(total));
  }
  // The draw among all logits from `low` on.
  static __device__ __noinline__ void draw(float low) {
    SampleShared& sh = shared();
    const int lane = threadIdx.x & 31, w = threadIdx.x / 32;
#pragma unroll 1
    for (int precise = 0; precise < 2; ++precise) {
      double error;
      const double total = mass(precise, low, error), target = sh.draw * total;
      if (threadIdx.x == 0) sh.hit = kDone;
      // The warp in whose part the target lies: the first whose end in the running sum is above it. Should rounding leave the
      // target at the very end, the last one with any mass takes it. All warps see the same sums, so that one takes it.
      const double theirs = lane < kWarps ? sh.warp_sum[lane] : 0., upto = lanes_before(theirs);
      const uint32_t full = __ballot_sync(0xffffffff, theirs > 0.), ends = __ballot_sync(0xffffffff, theirs > 0. && upto > target);
      double before = __shfl_sync(0xffffffff, upto, max(w - 1, 0));
      if (w == 0) before = 0.;
      __syncthreads();
      if (w == (ends ? __ffs(ends) - 1 : 31 - __clz(full))) {
        int begin = 0, end = sh.chunk / 32;
        if (!HELD) {  // the group
          double run = before;
          bool found = false;
          for (int g = 0; g * sh.group < sh.chunk / 32; ++g) {
            const double one = sh.group_sum[w][g];
            if (!found && one > 0.) begin = g * sh.group, before = run, found = run + one > target;
            run += one;
          }
          end = min(begin + sh.group, sh.chunk / 32);
        }
        // four rows of vectors at a time, then the row
        int at_i = -1, last_i = begin;
        double at_before = 0., last_before = before, s[4], mine;
#pragma unroll 1
        for (int i0 = begin; i0 < end && at_i < 0; i0 += 4) {
          warp_masses(precise, low, i0, end, s, mine, -1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (s[i] > 0.) last_i = i0 + i, last_before = before;
            if (at_i < 0 && s[i] > 0. && before + s[i] > target) at_i = i0 + i, at_before = before;
            before += s[i];
          }
        }
        if (at_i < 0) at_i = last_i, at_before = last_before;
        warp_masses(precise, low, at_i, at_i + 1, s, mine, 0);
        const double run = lanes_before(mine);
        const uint32_t above = __ballot_sync(0xffffffff, mine > 0. && at_before + run > target);
        const uint32_t some = __ballot_sync(0xffffffff, mine > 0.);
        if (lane == (above ? __ffs(above) - 1 : 31 - __clz(some))) {
          const Mine me(sh);
          double upto = at_before + (run - mine), c0 = upto, c1 = upto;
          int id = -1;
          float chosen = 0.f, x[E];
          vec_floats<T>(me.vec(at_i), x);
#pragma unroll 1
          for (int e = 0; e < E; ++e) {
            float one_x = x[0];
#pragma unroll
            for (int j = 1; j < E; ++j) one_x = e == j ? x[j] : one_x;
            if (!(one_x >= low)) continue;
            const double one = precise ? weight(one_x) : (double)exp2_fast((one_x - sh.max_x) * sh.c);
            if (one > 0. && (id < 0 || !(c1 > target))) {  // the first above the target, or the last with any mass
              id = me.first(at_i) + e;
              chosen = one_x;
              c0 = upto;
              c1 = upto + one;
            }
            upto += one;
          }
          if (!precise && (target - c0 <= 2. * error || c1 - target <= 2. * error)) sh.hit = kAmbiguous;
          else answer(id, chosen, total);
        }
      }
      __syncthreads();
      if (sh.hit == kDone) return;
    }
  }

  // ---------------------------------------------------------------- bounds where many tokens stay
  static __device__ __forceinline__ float from(uint32_t key) { return of_key(max(key, kLowest)); }
  static __device__ __forceinline__ bool usable(float range) {
    return range > 0.f && range < 1e37f && (SG_BINS - 1) / range < 1e37f;
  }
  // The histogram's range is `near` first (four times from the largest to a logit that SG_LIST_K logits reach); if that is too
  // short, down to the least.
  static __device__ __noinline__ uint32_t top_k_bound(int k, float near) {
    SampleShared& sh = shared();
#pragma unroll 1
    for (int attempt = 0; attempt < 2; ++attempt) {
      const float range = attempt == 0 ? near : sh.max_x - least();
      if (!usable(range)) continue;
      const float scale = (SG_BINS - 1) / range;
      histogram(scale, of_key(kLowest));
      float above;
      const int bin = find_bin((float)(k - 1), scale, false, above);
      if (bin == SG_BINS && attempt == 1 && count_from(of_key(kLowest)) < k) return 0;  // fewer numbers than k
      if (bin == SG_BINS) continue;
      const float high = bin > 0 ? of_key(edge_of(bin, scale)) : INFINITY;
      const int n = gather(of_key(edge_of(bin + 1, scale)), high);
      if (n > SG_CAP) continue;
      sort(n, sh.key);
      return sh.sorted[min(max(k - (int)above - 1, 0), n - 1)];
    }
    // ties, or outliers that leave too few steps for the rest: bisection of the key
    uint32_t kth = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
      const uint32_t next = kth | 1u << b;
      if (next <= key_of(sh.max_x) && (next < kLowest || count_from(of_key(next)) >= k)) kth = next;
    }
    return kth < kLowest ? 0 : kth;
  }
  // `total` +- `error`: the mass from top-k's bound `kth` on.
  static __device__ __noinline__ uint32_t top_p_bound(uint32_t kth, double total, double error, float near) {
    SampleShared& sh = shared();
    int precise = 0;
#pragma unroll 1
    for (int attempt = 0; attempt < 2; ++attempt) {
      const float range = fminf(24.f * (float)sh.T64, attempt == 0 ? near : sh.max_x - least());
      if (!usable(range)) continue;
      const float scale = (SG_BINS - 1) / range;
      double off = 0.;
      // Where the steps' masses point to; if the bound does not lie there, as far on as their sum was off at that side.
#pragma unroll 1
      for (int turn = 0; turn < 4; ++turn) {
        histogram(scale, from(kth));
        float unused;
        const int bin = find_bin((float)fmax(sh.p * total - off, 0.), scale, true, unused);
        if (bin >= SG_BINS - 1 && attempt == 0) break;
        const int first = min(max(bin - 2, 0), SG_BINS - 1), last = min(bin + 2, SG_BINS - 1);
        const double guess = mass_of_bins(first, scale);
        double guess_last = guess;
        for (int i = first; i <= last; ++i) guess_last += (double)((float)sh.bins[i] * exp2_fast(-((float)i + 0.5f) / scale * sh.c));
        const float high = first > 0 ? of_key(edge_of(first, scale)) : INFINITY;
        const uint32_t low = max(last == SG_BINS - 1 ? kLowest : edge_of(last + 1, scale), kth);
        const int n = gather(from(low), high);
        if (n > SG_CAP) break;
        if (n > 0) sort(n, sh.key);
        Verdict verdict;
        double above;
#pragma unroll 1
        for (;; precise = 1) {
          double blur = 0.;
          above = 0.;
          if (precise) total = mass_64(from(kth), fmaxf(high, from(kth)), above), error = 0.;
          else if (first > 0) above = mass(false, fmaxf(high, from(kth)), blur);
          verdict = bound(n, above, sh.p * total, blur + sh.p * error, last == SG_BINS - 1 || low == kth);
          if (verdict != kAmbiguous) break;
        }
        if (verdict == kDone) return sh.low;
        // The next turn's target is then below what the steps hold before `first`, or not below what they hold up to `last`.
        if (above > sh.p * total || n == 0) off = above - guess;
        else off = above + mass_before(n) - guess_last;
      }
    }
#pragma unroll 1
    for (;; precise = 1) {  // bisection: the largest key such that it and those above hold more than the share
      if (precise && error > 0.) total = mass(true, from(kth), error);
      const double share = sh.p * total;
      bool unsure = false;
      uint32_t cut = 0;
#pragma unroll 1
      for (int b = 31; b >= 0; --b) {
        const uint32_t next = cut | 1u << b;
        double blur = 0., s = 0.;
        if (next <= key_of(sh.max_x)) s = mass(precise, from(max(next, kth)), blur);
        blur += sh.p * error;
        unsure |= blur > 0. && fabs(s - share) <= blur;
        if (s > share) cut = next;
      }
      if (!unsure) return cut;
    }
  }

  // ---------------------------------------------------------------- the row
  static __device__ __forceinline__ void run(float top) {
    SampleShared& sh = shared();
    const int t = threadIdx.x, lane = t & 31, w = t / 32;
    const float max_x = sh.max_x;
    // min-p as a bound on the key: the least whose weight reaches it, among the 32 around max + T ln m, or by a search where
    // that window lies above it (temperatures at which neighbours have the same weight) or below it (next to zero, where 32
    // keys are less apart than the weight's error of 2^-42).
    if (sh.use_m && w == 0) {
      const uint32_t max_key = key_of(max_x);
      const auto reaches = [&](uint32_t key) { return weight(of_key(key)) >= sh.m || key >= max_key; };
      const uint32_t mid = key_of((float)fmax(max_x + sh.T64 * log(sh.m), -3.4e38)), low = max(mid, kLowest + 16) - 16;
      const uint32_t ok = __ballot_sync(0xffffffff, reaches(low + lane));
      uint32_t key = ok ? min(low + __ffs(ok) - 1, max_key) : max_key;
      if (ok & 1) key = least_key(lane, kLowest, key, reaches);
      if (!ok) key = least_key(lane, low + 32, max_key, reaches);
      if (lane == 0) sh.low = key;
    }
    const bool by_k = sh.use_k && sh.k <= SG_LIST_K;
    // A bound that all candidates of top-k, or the SG_LIST_K largest logits, reach.
    uint32_t low = 0xFFFFFFFFu;
    if (sh.use_k || sh.use_p) {
      const int chunk = sh.chunk, n = RowVecs<T>(static_cast<const T*>(sh.row), sh.V).n;
      const int warps = n < 32 ? 0 : min((n - 32) / chunk + 1, kWarps);  // without an idle lane
      const int j = warps > 0 ? ((by_k ? sh.k : SG_LIST_K) + warps - 1) / warps : 33;
      uint32_t key = key_of(top);
      if (j > 32) {
        low = 0;
      } else if (w < warps) {
#pragma unroll 1
        for (int i = 0;; ++i) {
          low = __reduce_max_sync(0xffffffff, key);
          if (i == j - 1) break;
          if (lane == __ffs(__ballot_sync(0xffffffff, key == low)) - 1) key = 0;
        }
      }
    }
    low = min_of(low);  // and its barrier for sh.low
    const uint32_t low_m = sh.use_m ? sh.low : 0;
    double total = 0., error = 0.;
    if (sh.use_p && !sh.use_k) total = mass(false, -INFINITY, error);
    if (by_k || (!sh.use_k && (sh.use_p || sh.use_m))) {
      uint32_t least = by_k || sh.use_p ? low : 0;
      bool complete = by_k || least == 0;  // no token below the candidates can be kept
      if (sh.use_m && !(by_k && sh.use_p) && low_m >= least) least = low_m, complete = true;
      const int n = gather_top(from(least));
      bool may = n <= SG_CAP;
      if (may && !complete) {  // where the candidates' mass cannot reach top-p's bound they need no order
        float s = 0.f;
        for (int i = t; i < n; i += NT) s += exp2_fast((of_key(sh.key[i]) - max_x) * sh.c);
        may = !(scan((double)s).y < 0.999 * sh.p * total);
      }
      if (may) {
        if (sh.use_k || sh.use_p) sort(n, sh.key);
        uint32_t cut = low_m;
        Verdict verdict = kDone;
        int members = n;
        if (by_k) {
          const uint32_t kth = sh.k <= n ? sh.sorted[sh.k - 1] : 0;
          cut = max(cut, kth);
          if (sh.use_p) {
            members = 0;
#pragma unroll 1
            for (int i = t; i - t < n; i += NT) members += __syncthreads_count(i < n && sh.sorted[i] >= kth);
          }
        }
        if (sh.use_p) {
#pragma unroll 1
          for (;;) {
            if (by_k) total = mass_before(members);
            verdict = bound(members, 0., sh.p * total, sh.p * error, complete);
            if (verdict != kAmbiguous) break;
            total = mass(true, -INFINITY, error);
          }
          cut = max(cut, sh.low);
        }
        if (verdict == kDone) {
          draw_from_list(n, cut);
          return;
        }
      }
    }
    const float near = low < kLowest || low > key_of(max_x) ? 0.f : 4.f * (max_x - of_key(low));
    uint32_t cut = low_m;
    if (sh.use_k) {
      const uint32_t kth = top_k_bound(sh.k, near);
      if (sh.use_p) total = mass(false, from(kth), error);
      cut = max(cut, sh.use_p ? max(kth, top_p_bound(kth, total, error, near)) : kth);
    } else if (sh.use_p) {
      cut = max(cut, top_p_bound(0, total, error, near));
    }
    draw(from(cut));
  }
};

// HELD: the logits stay in shared memory.
template <typename T, bool HELD>
__global__ void __launch_bounds__(SG_THREADS, 2) sample_given_kernel(const SampleGivenArgs a) {
  constexpr int NT = SG_THREADS;
  using S = Sampler<T, HELD>;
  SampleShared& sh = S::shared();
  const int t = threadIdx.x, lane = t & 31, row = blockIdx.x;
  begin_early();
  const T* x = static_cast<const T*>(a.x) + (long long)row * a.ldx;
  const RowVecs<T> vecs(x, a.V);
  const int chunk = (vecs.n + NT - 1) / NT * 32;
  const int group = HELD ? chunk / 32 : ((chunk / 32 + SG_GROUPS - 1) / SG_GROUPS + SG_VECS - 1) / SG_VECS * SG_VECS;
  const int w0 = t / 32 * chunk, mine = max(0, min(chunk / 32, (min(w0 + chunk, vecs.n) - w0 - lane + 31) / 32));
  float top = -INFINITY, top_here = -INFINITY;
  bool nan = false;
#pragma unroll 1
  for (int i0 = 0; i0 < mine; i0 += SG_VECS) {
    uint4 u[SG_VECS];
    vecs.load(w0 + i0 * 32, chunk / 32 - i0, mine - i0, u);
#pragma unroll
    for (int i = 0; i < SG_VECS; ++i) {
      if (HELD && i0 + i < mine) S::held()[(i0 + i) * NT + t] = u[i];
      const float most = vec_max<T>(u[i]);
      nan |= most != most;
      top_here = fmaxf(top_here, most);
    }
    if (!HELD && ((i0 + SG_VECS) % group == 0 || i0 + SG_VECS >= mine)) {
      S::tops()[i0 / group * NT + t] = top_here;
      top = fmaxf(top, top_here);
      top_here = -INFINITY;
    }
  }
  if (HELD) S::tops()[chunk / 32 * NT * 4 + t] = top = top_here;  // behind the vectors
  const float temperature = a.temperature[row];
  const bool greedy = !(temperature > 0.f);
  if (t == 0) {
    sh.row = x;
    sh.V = a.V, sh.chunk = chunk, sh.group = group;
    sh.T64 = (double)(greedy ? 1.f : fminf(fmaxf(temperature, 1e-8f), 3.4e38f));
    sh.c64 = 16. * 1.4426950408889634 / sh.T64;
    sh.c = (float)(1.4426950408889634 / sh.T64);
    sh.k = a.top_k[row];
    sh.use_k = !greedy && sh.k > 0 && sh.k < a.V;
    const float p = a.top_p[row], m = a.min_p[row];
    sh.use_p = !greedy && p < 1.f;
    sh.use_m = !greedy && m > 0.f;
    sh.p = sh.use_p ? fmax((double)p, 0.) : 1.;
    sh.m = sh.use_m ? fmin((double)m, 1.) : 0.;
    const double u = a.uniform64 ? static_cast<const double*>(a.uniform)[row] : (double)static_cast<const float*>(a.uniform)[row];
    sh.draw = fmin(fmax(u, 0.), 1.);  // a NaN becomes 0
    sh.token = a.token + row;
    sh.logprob = a.logprob ? a.logprob + row : nullptr;
  }
  if (t >= 32 && t < 48) sh.pow.at[t - 32] = exp2((t - 32) / 16.);
  const uint32_t max_key = S::max_of(key_of(nan ? of_key(0xFFFFFFFFu) : top));
  if (t == 0) sh.max_x = of_key(max_key);
  __syncthreads();
  if (!(fabsf(of_key(max_key)) < INFINITY)) {  // a NaN, an infinity or nothing allowed: no distribution; the largest number
    const float most = S::largest_number();
    const uint32_t id = S::first_id(most, -INFINITY);
    if (t == 0) {
      *sh.token = id < (uint32_t)a.V ? id : 0;
      if (sh.logprob) *sh.logprob = __int_as_float(0x7FC00000);
    }
  } else if (greedy) {
    const uint32_t id = S::first_id(of_key(max_key), of_key(max_key));
    const double total = sh.logprob ? S::mass_32(-INFINITY) : 1.;
    if (t == 0) S::answer((int)id, of_key(max_key), total);
  } else {
    S::run(top);
  }
}

constexpr int SG_MAX_SMEM = 113 * 1024;  // two CTAs on an SM

template <typename T, bool HELD>
void sample_given_launch(const SampleGivenArgs& a, int smem, int device, cudaStream_t s) {
  auto* kernel = sample_given_kernel<T, HELD>;
  static bool ready[64] = {};  // per device
  if (device < 0 || device >= 64 || !ready[device]) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SG_MAX_SMEM);
    if (device >= 0 && device < 64) ready[device] = true;
  }
  launch_early(kernel, dim3((unsigned)a.rows), dim3(SG_THREADS), smem, s, a);
}

template <typename T>
void sample_given_typed(const SampleGivenArgs& a, int device, cudaStream_t s) {
  constexpr int E = LogitType<T>::E;
  const int vecs = (a.V + E - 1) / E + 1;  // one more where a row starts off the grid
  const int state = ((int)sizeof(SampleShared) + 15) / 16 * 16;
  const int held = (vecs + SG_THREADS - 1) / SG_THREADS * SG_THREADS * 16 + SG_THREADS * 4;
  if (held <= SG_MAX_SMEM - state) sample_given_launch<T, true>(a, state + held, device, s);
  else sample_given_launch<T, false>(a, state + SG_GROUPS * SG_THREADS * 4, device, s);
}

}  // namespace astrai

namespace astrai_host {
using namespace astrai;

void sample_given(const void* x, long long ldx, int rows, int V, const void* uniform, bool uniform64,
                  const float* temperature, const int* top_k, const float* top_p, const float* min_p, long long* token,
                  float* logprob, int dtype, int device, cudaStream_t s) {
  const SampleGivenArgs a{x, ldx, rows, V, uniform, uniform64, temperature, top_k, top_p, min_p, token, logprob};
  if (dtype == 0) sample_given_typed<__nv_bfloat16>(a, device, s);
  else if (dtype == 1) sample_given_typed<__half>(a, device, s);
  else sample_given_typed<float>(a, device, s);
}

}  // namespace astrai_host
