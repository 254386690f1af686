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
// The sums run over the tokens outside J and over J apart: q_0 as 1 - sum q_jk would lose what a good student leaves to the
// others. They are joined at the greater of their two references (each part's largest logit; on a cluster the row's), so that
// tokens masked with large finite numbers, in one part of the row or in all of it, neither overflow nor cost digits. The tokens
// of J are overwritten with -inf in the CTA's copy of the row, which leaves their base gradient at zero; their own gradients
// are written over it.
//
// Persistent CTAs take row after row: a bulk copy brings the row into shared memory, NT threads take the maximum, the sum and
// the gradient from there, and one more warp does what is small: the sums over J, the row's coefficients and loss, the copy of
// the next row. A warp that works alone spends about 15 clocks on an instruction, so that the marks and gradients of J are
// spread over all threads. Three CTAs share an SM, so that one row is copied or written while others are computed. (With the row in
// registers and J spread over 512 threads, 60 % of the instructions were the same few for every thread.) A row that does not fit
// is shared by a cluster, whose extra warps exchange the sums through distributed shared memory.
//
// Measured (inputs not in L2): 8192 rows of 32000 bf16, k = 64: loss and gradient 236 us (4.4 TB/s of what has to be read and
// written), the loss alone 130 us (4.0 TB/s). With tau other than 1 and h > 0 a logit takes two exponentials for the sums and two
// for the gradient: 350 us, of which 233 are 16 exponentials a clock and SM. 768 rows of 131072 fp32 on clusters: 210 us (3.8 TB/s).
// The loss, in 150 cases of up to 2^24 logits: 5.8e-8 off in the root mean square and 2.1e-7 at most.
#include <cooperative_groups.h>

#include <algorithm>

#include "launch.cuh"
#include "logits.cuh"

namespace astrai {

namespace cg = cooperative_groups;

constexpr int DST_MAX_K = 1024;
constexpr int DST_MAX_CLUSTER = 16;
constexpr int DST_VECS = 4352;  // vectors of a row in one CTA: 68 KB, three CTAs on an SM
constexpr int DST_MAX_SMEM = 224 * 1024;
constexpr float LOG2E = 1.4426950408889634f;

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
  float inv_tau, inv_tau_rest;       // 1 / tau, and what its rounding left out
  float c, kl_loss, kl_grad, hard;   // log2(e) / tau, (1 - h) tau^2, (1 - h) tau, h
  int two;                           // the labels' part has a temperature of its own
  const float* count;     // rows that count, null: all
  const float* grad;      // gradient of the loss, null: `expected`
  float expected;
  int unless_expected;    // nothing is done if *grad == expected
  float* row_loss;        // null: not wanted
  int* err;
};

__device__ __forceinline__ bool label_counts(long long y, long long ignore, int V) { return y != ignore && y >= 0 && y < V; }

__device__ __forceinline__ float teacher_value(const DistillArgs& a, long long i) {
  if (a.values_type == 0) return __bfloat162float(static_cast<const __nv_bfloat16*>(a.values)[i]);
  if (a.values_type == 1) return __half2float(static_cast<const __half*>(a.values)[i]);
  return static_cast<const float*>(a.values)[i];
}

// a finite reference for a maximum
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }

// The student's mass at one temperature: outside J and on J as sums of 2^((x - ref) c), joined. `gap` is J's reference less
// that outside (-inf: nothing on J). `sum` is all of it relative to the greater reference, so that neither part overflows.
struct Mass {
  float up, down;  // a weight of one at the reference outside J, and at J's, relative to the greater
  float sum;
  __device__ Mass(float outside, float on, float gap, float c) {
    up = exp2_fast(fminf(-gap * c, 0.f));
    down = exp2_fast(fminf(gap * c, 0.f));
    sum = fmaf(on, down, outside * up);  // (as below, fused by hand: the loss has the same bits with and without a gradient)
  }
  __device__ float inv_rel_outside() const { return up / sum; }  // 1 / all of it, relative to each reference
  __device__ float inv_rel_on() const { return down / sum; }
};

// One entry of the teacher in shared memory.
struct Entry {
  int id;       // -1: none
  float value;  // the teacher's logit; then its mass
  float x;      // the student's logit, in this CTA's part of the row
  int here;     // it lies there
};

// What the extra warp tells the others about a row: gradients outside J are base 2^((x - ref) c) + base1 2^((x - ref) log2 e).
struct Coefficients {
  float ref, base, base1;
  float kl, ce, inv, all, mj, inv_on, inv_on1;
};

__device__ __forceinline__ uint32_t remote(const void* p, int rank) {  // the same place in another CTA of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, int* err) {
  const uint64_t t0 = globaltimer();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(0x989680u)
        : "memory");
    if (ok) return true;
    if (globaltimer() - t0 > ASTRAI_WAIT_NS) {
      set_error(err, kErrWaitPeer);
      return false;
    }
  }
}

// f(vector number) for this thread's vectors, four at a time
template <int NT, typename F>
__device__ __forceinline__ void each_vec(int n, F f) {
  int v = threadIdx.x;
#pragma unroll 1
  for (; v + 3 * NT < n; v += 4 * NT) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f(v + i * NT);
  }
#pragma unroll 1
  for (; v < n; v += NT) f(v);
}

// (3: 72 registers; left to itself the compiler takes 56 for some types, and spills: 245 us for 8192 rows of 32000 instead of 236)
template <typename T, int NT, bool TRAIN, bool TWO>
__global__ void __launch_bounds__(NT + 32, NT == 256 && TRAIN ? 3 : 0) distill_kernel(const DistillArgs a, int held) {
  constexpr int E = LogitType<T>::E, W = NT / 32;
  using Bits = typename std::conditional<E == 4, uint32_t, uint16_t>::type;
  extern __shared__ __align__(128) unsigned char distill_smem[];  // the row's vectors, then the entries
  uint4* const buffer = reinterpret_cast<uint4*>(distill_smem);
  Bits* const elements = reinterpret_cast<Bits*>(distill_smem);
  Entry* const entries_of[2] = {reinterpret_cast<Entry*>(distill_smem + held),
                                reinterpret_cast<Entry*>(distill_smem + held) + a.K};
  __shared__ float part_max[W], part_sum[2 * W];
  __shared__ Coefficients coefs;
  __shared__ float theirs[2][DST_MAX_CLUSTER][8];
  __shared__ int twice[2];
  // Two barriers in turn for the exchange of sums: one counts arrivals, not senders, and a CTA that is done with a row might
  // arrive for the next one before another's arrival for this row has come. For the row after next it cannot: then it has seen
  // that one's arrival for the next row, which follows the one for this.
  __shared__ uint64_t full, told[2];
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int cs = a.cluster, rank = cs > 1 ? (int)cg::this_cluster().block_rank() : 0;
  const int stride = gridDim.x / cs;
  begin_early();
  float g = a.expected;
  if (a.grad) {
    g = *a.grad;
    if (a.unless_expected && g == a.expected) return;
  }
  if (t < 2) twice[t] = 0;
  if (t == 0) {
    mbar_init(&full, 2);  // the copy, and the cut vectors
    mbar_init(&told[0], cs);
    mbar_init(&told[1], cs);
    fence_mbar_init();
  }
  if (cs > 1) cg::this_cluster().sync();
  else __syncthreads();

  const bool extra = w == W;
  const float c = a.c;
  const float scale = TRAIN ? g / (a.count ? fmaxf(*a.count, 1.f) : (float)max(a.rows, 1)) : 0.f;
  const auto row_vecs = [&](int row) { return RowVecs<T>(static_cast<const T*>(a.x) + (long long)row * a.ldx, a.V); };
  // The extra warp: the whole vectors of this CTA's part of a row by the copy, a cut first or last one by element; finish()
  // has what begin() loaded.
  const auto begin = [&](int row, uint4& cut) {
    const RowVecs<T> v = row_vecs(row);
    const int per = (v.n + cs - 1) / cs, v0 = rank * per, v1 = min(v0 + per, v.n);
    const int b = v0 + (v0 < v1 && !v.whole(v0)), e = v1 - (v0 < v1 && !v.whole(v1 - 1));
    if (lane == 0) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // behind the marks in the row before
      if (b < e) {
        mbar_expect_tx(&full, (uint32_t)(e - b) * 16);
        bulk_load(buffer + (b - v0), v.row + v.first(b), (uint32_t)(e - b) * 16, &full);
      } else {
        mbar_arrive(&full);
      }
    }
    const int mine = lane == 0 ? v0 : v1 - 1;
    if (lane < 2 && v0 < v1 && !v.whole(mine)) cut = v.load(mine);
  };
  const auto finish = [&](int row, const uint4& cut) {
    const RowVecs<T> v = row_vecs(row);
    const int per = (v.n + cs - 1) / cs, v0 = rank * per, v1 = min(v0 + per, v.n), mine = lane == 0 ? v0 : v1 - 1;
    if (lane < 2 && v0 < v1 && !v.whole(mine)) buffer[mine - v0] = cut;
    __syncwarp();
    if (lane == 0) mbar_arrive(&full);
  };
  const auto id_at = [&](int row, int k) -> long long {
    const long long at = (long long)row * a.K + k;
    return a.ids64 ? static_cast<const long long*>(a.ids)[at] : static_cast<const int*>(a.ids)[at];
  };
  // Labels are read two rows ahead, the entries one.
  const auto label_of = [&](int row) -> long long { return a.target && row < a.rows ? a.target[row] : -1; };
  const auto counts = [&](int row, long long y) { return row < a.rows && (!a.target || label_counts(y, a.ignore, a.V)); };
  // entry k of a row, the logit left out
  const auto read_entry = [&](int row, int k, long long j, float value) {
    Entry n{-1, -INFINITY, -INFINITY, 0};
    if (j >= 0 && j < a.V) {
      const RowVecs<T> v = row_vecs(row);
      const int per = (v.n + cs - 1) / cs, v0 = rank * per, v1 = min(v0 + per, v.n), at = ((int)j + v.head) / E;
      n.id = (int)j;
      n.value = value;
      n.here = at >= v0 && at < v1;
    }
    return n;
  };
  const auto fill_entries = [&](int row, Entry* entries, int from) {
    for (int k = from; k < a.K; k += NT) entries[k] = read_entry(row, k, id_at(row, k), teacher_value(a, (long long)row * a.K + k));
  };
  int row = blockIdx.x / cs, turn = 0;
  uint32_t phase = 0, told_phase = 0;
  long long y = label_of(row), y_next = label_of(row + stride), y_after;
  uint4 cut = make_uint4(0, 0, 0, 0);
  if (counts(row, y)) {
    if (extra) {
      begin(row, cut);
      finish(row, cut);
    } else {
      fill_entries(row, entries_of[0], t);
    }
  }

#pragma unroll 1
  for (; row < a.rows; row += stride, y = y_next, y_next = y_after) {
    y_after = label_of(row + 2 * stride);
    const bool counted = counts(row, y), counted_next = counts(row + stride, y_next);
    // this thread's first entry of the next row, on its way until the end of this one
    const bool ahead = counted && counted_next && !extra && t < a.K;
    long long id_next = -1;
    float value_next = 0.f;
    if (ahead) {
      id_next = id_at(row + stride, t);
      value_next = teacher_value(a, (long long)(row + stride) * a.K + t);
    }
    const RowVecs<T> vecs = row_vecs(row);
    T* const dx = TRAIN ? static_cast<T*>(a.dx) + (long long)row * a.lddx : nullptr;
    const int per = (vecs.n + cs - 1) / cs, v0 = rank * per, v1 = min(v0 + per, vecs.n), nv = max(v1 - v0, 0);
    if (!counted) {  // the same for the whole cluster
      if constexpr (TRAIN)
        for (int v = v0 + t; v < v1; v += NT + 32) vecs.store(dx, v, make_uint4(0, 0, 0, 0));
      if (a.row_loss && rank == 0 && t == 0) a.row_loss[row] = 0.f;
      if (counted_next) {
        if (extra) {
          begin(row + stride, cut);
          finish(row + stride, cut);
        } else {
          fill_entries(row + stride, entries_of[turn], t);
        }
      }
      continue;
    }
    Entry* const entries = entries_of[turn];
    if (!mbar_wait(&full, phase, a.err, kErrWaitFull)) return;  // (then all threads run out of time)
    phase ^= 1;
    // ---- the logits of J, and -inf in their places; every entry leaves its number in between: one that does not find it has
    // an id that comes again
    const int base_id = vecs.first(v0);  // the id of the buffer's first element
    if (!extra)
      for (int k = t; k < a.K; k += NT)
        if (entries[k].here) {
          const int at = entries[k].id - base_id;
          entries[k].x = LogitType<T>::one(reinterpret_cast<const T*>(elements)[at]);
          elements[at] = (Bits)k;
        }
    __syncthreads();
    if (!extra)
      for (int k = t; k < a.K; k += NT)
        if (entries[k].here) {
          const int at = entries[k].id - base_id;
          if (elements[at] != (Bits)k) twice[turn] = 1;
          elements[at] = (Bits)LogitType<T>::kNegInf;
        }
    __syncthreads();
    const bool repeated = twice[turn];

    // ---- the largest logit outside J
    if (!extra) {
      float m0 = -INFINITY;
      each_vec<NT>(nv, [&](int v) { m0 = fmaxf(m0, vec_max_number<T>(buffer[v])); });
      m0 = of_key(__reduce_max_sync(0xffffffff, key_of(m0)));
      if (lane == 0) part_max[w] = m0;
    }
    __syncthreads();

    // ---- the extra warp: the sums over J
    // the teacher's largest logit and its mass on J relative to that; of it that with a logit here; the sum of mass * (the
    // teacher's logit - the student's), each relative to its largest (in this CTA): one small number a token, as both logarithms'
    // sums would be far larger than their difference; the student's sums here, over tau and at 1
    float rest = -INFINITY, vt = -INFINITY, mj = -INFINITY, teach = 0.f, cross = 0.f, own = 0.f, on = 0.f, on1 = 0.f;
    bool label = false;  // it is one of the entries
    if (extra) {
      if (a.rest) rest = a.rest[row];
#pragma unroll 2
      for (int k = lane; k < a.K; k += 32) {
        const Entry n = entries[k];
        if (repeated && n.here) entries[k].x = LogitType<T>::one(vecs.row[n.id]);  // another's number may have been read
        vt = fmaxf(vt, n.value);
        mj = fmaxf(mj, n.here ? entries[k].x : -INFINITY);
        label |= n.id >= 0 && n.id == y;
      }
      label = __any_sync(0xffffffff, label);
      vt = of_key(__reduce_max_sync(0xffffffff, key_of(vt)));
      mj = of_key(__reduce_max_sync(0xffffffff, key_of(mj)));
      const float vref = ref_of(vt), ref = ref_of(mj);
#pragma unroll 2
      for (int k = lane; k < a.K; k += 32) {
        const Entry n = entries[k];
        const float th = n.value - vref, zh = n.x - ref, e = n.id >= 0 ? exp2_fast(th * c) : 0.f;
        entries[k].value = e;
        teach += e;
        if (!n.here) continue;
        if (e != 0.f) cross += e * (th - zh), own += e;
        bool first = true;  // the student's mass at an id that comes again counts once, with the first of its entries
        for (int l = 0; repeated && first && l < k; ++l) first = entries[l].id != n.id;
        if (first) {
          on += exp2_fast(zh * c);
          if constexpr (TWO) on1 += exp2_fast(zh * LOG2E);
        }
      }
      teach = warp_sum(teach);
      cross = warp_sum(cross);
      on = warp_sum(on);
      if constexpr (TWO) on1 = warp_sum(on1);
      if (cs > 1) own = warp_sum(own);
    }
    // ---- sums outside J, over tau and at 1
    float most = part_max[lane & (W - 1)];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffff, most, o));
    const Pair c2(c, c), log2e2(LOG2E, LOG2E);
    if (!extra) {
      const Pair ref2(-ref_of(most), -ref_of(most));
      Pair s2(0.f, 0.f), s1(0.f, 0.f);
      each_vec<NT>(nv, [&](int v) {
        Pair p[E / 2];
        vec_pairs<T>(buffer[v], p);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          const Pair d = p[e] + ref2;
          s2 = s2 + exp2_fast(d * c2);
          if constexpr (TWO) s1 = s1 + exp2_fast(d * log2e2);
        }
      });
      const float a2 = warp_sum(s2.sum()), a1 = TWO ? warp_sum(s1.sum()) : 0.f;
      if (lane == 0) part_sum[w] = a2, part_sum[W + w] = a1;
    }
    __syncthreads();
    if (!TRAIN && extra && counted_next) begin(row + stride, cut);  // the buffer has been read

    // ---- the extra warp: the row's coefficients and loss
    if (extra) {
      float mo = ref_of(most);  // the logit that the sums outside J are relative to
      float out = warp_sum(lane < W ? part_sum[lane] : 0.f), out1 = TWO ? warp_sum(lane < W ? part_sum[W + lane] : 0.f) : 0.f;
      if (cs > 1) {  // of all CTAs, relative to one reference
        if (lane < cs) {
          const float mine[8] = {most, out, out1, mj, on, on1, cross, own};
          const uint32_t to = remote(&theirs[turn][rank][0], lane);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4 * i), "f"(mine[i]) : "memory");
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote(&told[turn], lane)) : "memory");
        }
        __syncwarp();
        if (!wait_cluster(&told[turn], told_phase >> turn & 1, a.err)) return;  // (no copy follows: the others run out of time)
        told_phase ^= 1u << turn;
        const float* their = theirs[turn][lane < cs ? lane : 0];
        const float m = lane < cs ? their[0] : -INFINITY, m_on = lane < cs ? their[3] : -INFINITY;
        mo = ref_of(warp_max(m));  // the row's: another part's sum may be any distance above this one's own largest
        const bool some = m != -INFINITY;
        out = warp_sum(some ? their[1] * exp2_fast((m - mo) * c) : 0.f);
        if constexpr (TWO) out1 = warp_sum(some ? their[2] * exp2_fast((m - mo) * LOG2E) : 0.f);
        mj = ref_of(warp_max(m_on));
        const bool some_on = m_on != -INFINITY;
        on = warp_sum(some_on ? their[4] * exp2_fast((m_on - mj) * c) : 0.f);
        if constexpr (TWO) on1 = warp_sum(some_on ? their[5] * exp2_fast((m_on - mj) * LOG2E) : 0.f);
        // (m_on - mj may be out of range where this part gives the teacher's tokens no mass)
        cross = warp_sum(lane < cs ? their[6] - (some_on && their[7] != 0.f ? their[7] * (m_on - mj) : 0.f) : 0.f);
      } else {
        mj = ref_of(mj);
      }
      if (out == 0.f) mo = mj;  // nothing outside J
      const float gap = on == 0.f ? -INFINITY : mj - mo;
      const Mass z(out, on, gap, c);
      const Mass z1 = TWO ? Mass(out1, on1, gap, LOG2E) : z;
      // the teacher's share outside J: its logarithm over the largest entry's, and the masses relative to the greater of both
      const float over = vt == -INFINITY ? rest == -INFINITY ? -INFINITY : rest - rest
                                         : fmaf(-vt, a.inv_tau_rest, fmaf(-vt, a.inv_tau, rest));
      const float top = fmaxf(over, 0.f), pr = exp2_fast((over - top) * LOG2E), shrink = exp2_fast(-top * LOG2E);
      const float on_j = __fmul_rn(teach, shrink), mass = on_j + pr, inv = mass != 0.f ? 1.f / mass : 0.f, p0 = pr * inv;
      if constexpr (TRAIN) {
        const float all = mass != 0.f ? 1.f : 0.f, kl = scale * a.kl_grad, ce = scale * a.hard;
        const float share = out != 0.f ? p0 / out : 0.f;
        if (lane == 0) {
          coefs.ref = mo;
          coefs.base = kl * (all * z.inv_rel_outside() - share) + (TWO ? 0.f : ce * z.inv_rel_outside());
          coefs.base1 = TWO ? ce * z1.inv_rel_outside() : 0.f;
          coefs.kl = kl, coefs.ce = ce, coefs.inv = inv * shrink, coefs.all = all;
          coefs.mj = mj, coefs.inv_on = z.inv_rel_on(), coefs.inv_on1 = TWO ? z1.inv_rel_on() : z.inv_rel_on();
        }
        __syncthreads();
      }
      if (a.row_loss && rank == 0) {
        // The divergence may be far smaller than the logarithms of the masses. Of the largest of J (lane 0) and of the share
        // outside (lane 1) it takes the logarithm of the teacher's probability over the student's, from masses joined in 64 bits.
        // What the factors up, down, shrink and pr are off by is then in both distributions' sums too, and counts only as much
        // as the two differ.
        const bool o = lane == 1;
        const float part = o ? pr : on_j, apart = __fmul_rn(gap, a.inv_tau);
        const double sum = fma((double)on, (double)z.down, (double)out * z.up);
        const double of_teacher = fma((double)teach, (double)shrink, (double)pr);
        const double den = of_teacher * (o ? (double)z.up * out : (double)z.down);
        float ln, more = 0.f;
        if (fminf(o ? z.up : z.down, o ? pr : shrink) > 1e-30f && den > 0.) {
          double per = __fdividef(1.f, (float)den);
          per *= fma(-den, per, 2.);
          const double ratio = sum * (o ? pr : shrink) * per;
          const float near = (float)ratio;
          ln = logf(near);
          more = __fdividef((float)(ratio - near), near);
        } else {  // far from each other, or nothing there
          ln = (o ? over - top + fmaxf(apart, 0.f) - logf(out) : fmaxf(-apart, 0.f) - top) + logf(z.sum / mass);
        }
        const float term = part != 0.f ? __fmul_rn(part, ln) : 0.f, add = part != 0.f ? __fmul_rn(part, more) : 0.f;
        const float crossed = shrink != 0.f ? __fmul_rn(cross * shrink, a.inv_tau) : 0.f;
        const float terms = term + __shfl_sync(0xffffffff, term, 1) + crossed + (add + __shfl_sync(0xffffffff, add, 1));
        float loss = mass != 0.f ? __fmul_rn(terms * inv, a.kl_loss) : 0.f;
        // relative to the greater reference: the label lies there unless its logit is far below, so that nothing large cancels
        if (a.hard > 0.f && lane == 0)
          loss = fmaf(a.hard, ((gap > 0.f ? mj : mo) - LogitType<T>::one(vecs.row[y])) + logf(z1.sum), loss);
        if (lane == 0) a.row_loss[row] = loss;
      }
    } else if constexpr (TRAIN) {
      __syncthreads();
    }
    // ---- the gradient outside J
    const auto outside = [&](Pair p, const Coefficients& k) {
      p = p + Pair(-k.ref, -k.ref);
      const Pair d = Pair(k.base, k.base) * exp2_fast(p * c2);
      if constexpr (TWO) return fma2(Pair(k.base1, k.base1), exp2_fast(p * log2e2), d);
      return d;
    };
    if constexpr (TRAIN) {
      if (!extra) {
        const Coefficients k = coefs;
        const int b = v0 < v1 && !vecs.whole(v0) ? 1 : 0, e = nv - (nv > 0 && !vecs.whole(v1 - 1));
        T* const to = dx + base_id;
        each_vec<NT>(nv, [&](int v) {
          Pair p[E / 2];
          vec_pairs<T>(buffer[v], p);
#pragma unroll
          for (int e = 0; e < E / 2; ++e) p[e] = outside(p[e], k);
          const uint4 u = pairs_round<T>(p);
          if (v >= b && v < e) *reinterpret_cast<uint4*>(to + v * E) = u;
          else vecs.store(dx, v0 + v, u);
        });
      }
    }
    if constexpr (TRAIN) {
      __syncthreads();  // the base gradient lies before the entries'; the buffer has been read
      const Coefficients k = coefs;
      if (extra) {
        if (counted_next) begin(row + stride, cut);
        if (lane == 0 && y >= 0 && k.ce != 0.f && !label && y >= base_id && y - base_id < nv * E) {
          const float xy = LogitType<T>::one(vecs.row[y]);
          dx[y] = LogitType<T>::round(outside(Pair(xy, xy), k).get().x - k.ce);
        }
      } else {
        for (int i = t; i < a.K; i += NT) {
          const Entry n = entries[i];
          if (!n.here) continue;
          float p = n.value * k.inv;
          if (repeated) {  // the teacher's mass of all entries with this id, the same whichever of them writes it
            p = 0.f;
            for (int l = 0; l < a.K; ++l)
              if (entries[l].id == n.id) p += entries[l].value * k.inv;
          }
          const float q = exp2_fast((n.x - k.mj) * c) * k.inv_on;
          const float q1 = TWO ? exp2_fast((n.x - k.mj) * LOG2E) * k.inv_on1 : q;
          dx[n.id] = LogitType<T>::round(k.kl * (q * k.all - p) + k.ce * (q1 - (n.id == y ? 1.f : 0.f)));
        }
      }
    }
    if (counted_next) {
      if (extra) {
        finish(row + stride, cut);
      } else {
        if (ahead) entries_of[turn ^ 1][t] = read_entry(row + stride, t, id_next, value_next);
        fill_entries(row + stride, entries_of[turn ^ 1], t + NT);
      }
    }
    if (t == 0) twice[turn ^ 1] = 0;  // last read a row ago
    turn ^= 1;
  }
  if (cs > 1) cg::this_cluster().sync();  // others may still write here
}

// count[0] = rows that count
__global__ void __launch_bounds__(1024) distill_count_kernel(const long long* target, long long ignore, int rows, int V,
                                                             float* count) {
  __shared__ int part[32];
  begin_early();
  int n = 0;
  for (int r = threadIdx.x; r < rows; r += 1024) n += label_counts(target[r], ignore, V);
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

template <typename T, int NT, bool TRAIN, bool TWO>
void distill_launch(const DistillArgs& a, int vecs, int device, cudaStream_t s) {
  auto* kernel = distill_kernel<T, NT, TRAIN, TWO>;
  const int held = (vecs * 16 + 127) / 128 * 128, smem = held + 2 * a.K * (int)sizeof(Entry);
  static bool ready[64] = {};  // per device
  if (device < 0 || device >= 64 || !ready[device]) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DST_MAX_SMEM);
    cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (device >= 0 && device < 64) ready[device] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.cluster);
  cfg.blockDim = dim3(NT + 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2]{};
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  // as many clusters as run at once, each with rows of its own; asked again when the sizes change
  static thread_local struct {
    int device = -1, smem, cluster, most;
  } fit;
  if (fit.device != device || fit.smem != (int)smem || fit.cluster != a.cluster) {
    int most = 0;
    if (a.cluster > 1) {
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess) most = 0;
    } else if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&most, kernel, NT + 32, smem) != cudaSuccess) {
      most = 0;
    } else {
      most *= astrai_host::num_sms(device);
    }
    fit.device = device, fit.smem = (int)smem, fit.cluster = a.cluster, fit.most = std::max(most, 1);
  }
  cfg.gridDim = dim3((unsigned)(std::min(a.rows, fit.most) * a.cluster));
  cfg.numAttrs = 2;
  if (a.cluster == 1) cfg.attrs = at + 1, cfg.numAttrs = 1;
  note_launch();
  cudaLaunchKernelEx(&cfg, kernel, a, held);
}

template <typename T, bool TRAIN, bool TWO>
void distill_sized(DistillArgs a, int device, cudaStream_t s) {
  constexpr int E = LogitType<T>::E;
  const int vecs = (a.V + E - 1) / E + 1;  // one more where a row starts off the grid
  int cs = 1;
  while ((vecs + cs - 1) / cs > DST_VECS) cs *= 2;
  a.cluster = cs;
  const int per = (vecs + cs - 1) / cs;
  // Short rows go to small CTAs, of which more share an SM: 8192 rows, k = 64, loss and gradient with 128 and with 256 threads:
  // 53 and 86 us at 1000 tokens in bf16, 68 and 97 at 4096, 88 and 113 at 8192 (1024 vectors), 131 and 162 at 16000, 252 and 238
  // at 32000; fp32 80 and 110 at 4096. So between 1025 and some 3000 vectors this takes the slower side.
  if (per <= 1024) return distill_launch<T, 128, TRAIN, TWO>(a, per, device, s);
  distill_launch<T, 256, TRAIN, TWO>(a, per, device, s);
}

template <typename T>
void distill_typed(const DistillArgs& a, int device, cudaStream_t s) {
  const bool two = a.two;
  if (a.dx)
    two ? distill_sized<T, true, true>(a, device, s) : distill_sized<T, true, false>(a, device, s);
  else
    two ? distill_sized<T, false, true>(a, device, s) : distill_sized<T, false, false>(a, device, s);
}

}  // namespace astrai

namespace astrai_host {
using namespace astrai;

int distill_max_k() { return DST_MAX_K; }
// longest row for elements of this size
int distill_max_vocab(int elem) { return DST_MAX_CLUSTER * DST_VECS * (16 / elem) - 16 / elem; }

void distill(const void* x, long long ldx, void* dx, long long lddx, const void* ids, bool ids64, const void* values,
             int values_type, const float* rest, const long long* target, long long ignore, int rows, int V, int K,
             double tau, double hard, const float* grad, float expected, bool unless_expected, float* row_loss,
             float* count, bool have_count, float* loss, int dtype, int device, cudaStream_t s) {
  if (target && !have_count)
    launch_early(distill_count_kernel, dim3(1), dim3(1024), 0, s, target, ignore, rows, V, count);
  const double per = std::min(1. / tau, 1e38), soft = 1. - hard;
  DistillArgs a{x, ldx, dx, lddx, ids, ids64, values, values_type, rest, target, ignore, rows, V, K, 1, (float)per,
                (float)(per - (float)per), (float)std::min(1.4426950408889634 * per, 1e38), (float)(soft * tau * tau),
                (float)(soft * tau), (float)hard, hard > 0. && tau != 1., target ? count : nullptr, grad, expected,
                unless_expected, row_loss, astrai_host::error_word(device)};
  if (rows > 0) {
    if (dtype == 0) distill_typed<__nv_bfloat16>(a, device, s);
    else if (dtype == 1) distill_typed<__half>(a, device, s);
    else distill_typed<float>(a, device, s);
  }
  if (loss)
    launch_early(distill_mean_kernel, dim3(1), dim3(1024), 0, s, (const float*)row_loss, rows,
                 (const float*)(target ? count : nullptr), loss);
}

}  // namespace astrai_host
