// RMS norm of every query and key head with the rotation of its position in the same pass, forward
// and backward (sm_100a). No counterpart as one operation in the reference project, which rotates
// with elementwise ops (astrai/model/components/rope.py:26-33) and then normalises each head
// (astrai/model/components/attention.py:79-84).
//
// With z a head's D channels, R the rotation of rot of them by the position's (cos, sin) row, and
// n(z) = z / sqrt(mean z^2 + eps) * w:
//   after : y = n(R x)      before: y = R n(x)      none: y = R x
// R need not be a pure rotation: a table scaled for long contexts carries a factor, and the backward
// applies R^T, not R^-1. Backward, with u = z / rms (z = R x for after, x for before), g the gradient
// that reaches n's output (dy, or R^T dy for before):
//   dw += g u      dz = (g w - u mean(g w u)) / rms      dx = R^T dz (after) or dz (before)
// The statistics are recomputed from x, so the forward saves nothing but its inputs.
//
// A head belongs to LPH lanes (a power of two) of 8 channels each, held as four pairs that rotate
// together: neighbouring channels in the interleaved layout; in the half layout two runs of four
// channels rot / 2 apart, so that no channel has to change lanes. Everything is fp32 in registers;
// outputs are rounded once.
#include <algorithm>
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.cuh"

namespace astrai {
namespace {

enum NormMode { kNone = 0, kAfter = 1, kBefore = 2 };

struct QkNormParams {
  const void* x;
  const void* dy;   // backward only
  void* out;        // y, or dx in the backward
  long long ldx, lddy, ldo;
  const void* wq;
  const void* wk;
  const float2* table;
  const int* pos;   // null: row % seq_len
  float* dw_part;   // backward: [blocks][2][D]
  int* err;
  int rows, hq, hkv, D, rot, rot_off, seq_len, max_pos;
  int q_parts;      // warps of a row that share its query heads; the others share its key heads
  int warps_per_row, rows_at_once;  // of a CTA's consumers in qk_norm_rows_kernel
  float eps, inv_d;
  bool inverse;     // without a norm: the transposed rotation
};

template <typename T>
__device__ __forceinline__ T round_to(float x) {
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
  else return x;
}
// Two fp32 numbers in one 64-bit register: sm_100's packed instructions work on both at once.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum(F2 a) {
  const float2 f = split(a);
  return f.x + f.y;
}
// two neighbours of T, as loaded
template <typename T>
__device__ __forceinline__ float2 unpack2(const T* v) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(v[0], v[1]);
  } else if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2*>(v));
  } else {
    const unsigned u = *reinterpret_cast<const unsigned*>(v);
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
}
template <typename T>
__device__ __forceinline__ void pack2(T* v, float a, float b) {
  if constexpr (sizeof(T) == 4) v[0] = a, v[1] = b;
  else if constexpr (std::is_same<T, __half>::value) *reinterpret_cast<__half2*>(v) = __floats2half2_rn(a, b);
  else *reinterpret_cast<unsigned*>(v) = pack_bf16(a, b);
}
template <typename T>
struct alignas(sizeof(T) * 4) Four {
  T v[4];
};
template <typename T>
struct alignas(16) Raw8 {  // a lane's 8 channels as loaded
  Four<T> c[2];
};

// Where a lane's channels lie in its head. Interleaved: 8 neighbours, pairs (2i, 2i + 1). Half:
// lanes below rot / 8 hold channels j .. j + 3 of both halves of the rotated part, pairs
// (i, i + rot / 2); the others 8 neighbours of the rest, in order.
template <bool HALF>
struct Place {
  int c0, c1;    // first channels of the two runs of four
  int cs;        // first (cos, sin) pair, or -1: not rotated
  bool on;
  __device__ __forceinline__ Place(int l, const QkNormParams& p) {
    on = l * 8 < p.D;
    if constexpr (HALF) {
      if (l * 8 < p.rot) {
        c0 = p.rot_off + l * 4;
        c1 = c0 + p.rot / 2;
        cs = l * 4;
      } else {
        c0 = l * 8 - p.rot;
        if (c0 >= p.rot_off) c0 += p.rot;
        c1 = c0 + 4;
        cs = -1;
      }
    } else {
      c0 = l * 8;
      c1 = c0 + 4;
      cs = c0 >= p.rot_off && c0 < p.rot_off + p.rot ? (c0 - p.rot_off) / 2 : -1;
    }
  }
};

template <bool HALF, typename T>
__device__ __forceinline__ Raw8<T> load_raw(const T* head, const Place<HALF>& at) {
  Raw8<T> r;
  if constexpr (HALF || sizeof(T) == 4) {
    r.c[0] = *reinterpret_cast<const Four<T>*>(head + at.c0);
    r.c[1] = *reinterpret_cast<const Four<T>*>(head + at.c1);
  } else {
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(head + at.c0);
  }
  return r;
}
// A lane's channels in registers: the first members of its four pairs and the second ones, two to a register.
struct Head {
  F2 a[2], b[2];
};
template <bool HALF, typename T>
__device__ __forceinline__ Head to_head(const Raw8<T>& r) {
  Head z;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (HALF) {
      const float2 u = unpack2(r.c[0].v + 2 * i), v = unpack2(r.c[1].v + 2 * i);
      z.a[i] = f2(u.x, u.y), z.b[i] = f2(v.x, v.y);
    } else {
      const float2 u = unpack2(r.c[i].v), v = unpack2(r.c[i].v + 2);
      z.a[i] = f2(u.x, v.x), z.b[i] = f2(u.y, v.y);
    }
  }
  return z;
}
template <bool HALF, typename T>
__device__ __forceinline__ void store_head(T* head, const Place<HALF>& at, const Head& z) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = split(z.a[i]), b = split(z.b[i]);
    if constexpr (HALF) {
      pack2(r.c[0].v + 2 * i, a.x, a.y);
      pack2(r.c[1].v + 2 * i, b.x, b.y);
    } else {
      pack2(r.c[i].v, a.x, b.x);
      pack2(r.c[i].v + 2, a.y, b.y);
    }
  }
  if constexpr (HALF || sizeof(T) == 4) {
    *reinterpret_cast<Four<T>*>(head + at.c0) = r.c[0];
    *reinterpret_cast<Four<T>*>(head + at.c1) = r.c[1];
  } else {
    *reinterpret_cast<uint4*>(head + at.c0) = *reinterpret_cast<const uint4*>(&r);
  }
}
__device__ __forceinline__ Head zero_head() {
  Head z;
#pragma unroll
  for (int i = 0; i < 2; ++i) z.a[i] = z.b[i] = f2(0.f, 0.f);
  return z;
}
struct Turn {  // cos, sin and -sin of a lane's four pairs
  F2 c[2], s[2], n[2];
};
__device__ __forceinline__ Turn no_turn() {
  Turn t;
#pragma unroll
  for (int i = 0; i < 2; ++i) t.c[i] = f2(1.f, 1.f), t.s[i] = t.n[i] = f2(0.f, 0.f);
  return t;
}
__device__ __forceinline__ Turn to_turn(const float4* q) {
  Turn t;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 u = q[i];
    t.c[i] = f2(u.x, u.z);
    t.s[i] = f2(u.y, u.w);
    t.n[i] = f2(-u.y, -u.w);
  }
  return t;
}
__device__ __forceinline__ void rotate(Head& z, const Turn& t) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const F2 a = z.a[i];
    z.a[i] = fma2(a, t.c[i], mul(z.b[i], t.n[i]));
    z.b[i] = fma2(a, t.s[i], mul(z.b[i], t.c[i]));
  }
}
__device__ __forceinline__ void rotate_back(Head& z, const Turn& t) {  // by the transpose
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const F2 a = z.a[i];
    z.a[i] = fma2(a, t.c[i], mul(z.b[i], t.s[i]));
    z.b[i] = fma2(a, t.n[i], mul(z.b[i], t.c[i]));
  }
}
// A lane's four (cos, sin) pairs of a row. A position outside the table records kErrBadArg and leaves
// the row unrotated.
template <bool HALF>
__device__ __forceinline__ Turn load_turn(const QkNormParams& p, int row, const Place<HALF>& at) {
  if (!at.on || at.cs < 0) return no_turn();
  const int t = p.pos ? p.pos[row] : row % p.seq_len;
  if (t < 0 || t >= p.max_pos) {
    set_error(p.err, kErrBadArg);
    return no_turn();
  }
  return to_turn(reinterpret_cast<const float4*>(p.table + (long long)t * (p.rot / 2) + at.cs));
}
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  return v;
}

// The heads of a row that a warp owns: only query heads or only key heads, so that one weight and one sum of
// weight gradients stay in its registers. It takes them in steps of 32 / LPH, `stride` steps apart.
struct Share {
  int part, stride, col0, heads;
  bool key;
  __device__ __forceinline__ Share(const QkNormParams& p, int w, int warps) {
    key = w >= p.q_parts;
    part = key ? w - p.q_parts : w;
    stride = key ? warps - p.q_parts : p.q_parts;
    col0 = key ? p.hq * p.D : 0;
    heads = key ? p.hkv : p.hq;
  }
};

// One head in a lane group's registers, forward.
template <int LPH, int NORM>
__device__ __forceinline__ void head_forward(Head& z, const Turn& t, const Head& w, const QkNormParams& p) {
  if (NORM == kNone && p.inverse) {
    rotate_back(z, t);
    return;
  }
  if (NORM != kBefore) rotate(z, t);
  if (NORM != kNone) {
    F2 ss = mul(z.a[0], z.a[0]);
    ss = fma2(z.b[0], z.b[0], ss);
    ss = fma2(z.a[1], z.a[1], ss);
    ss = fma2(z.b[1], z.b[1], ss);
    const float r = rsqrtf(fmaf(head_sum<LPH>(sum(ss)), p.inv_d, p.eps));
    const F2 rr = f2(r, r);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      z.a[i] = mul(z.a[i], mul(rr, w.a[i]));
      z.b[i] = mul(z.b[i], mul(rr, w.b[i]));
    }
  }
  if (NORM == kBefore) rotate(z, t);
}
// and backward: z of x becomes dx, dw gains g u
template <int LPH, int NORM>
__device__ __forceinline__ void head_backward(Head& z, Head& g, const Turn& t, const Head& w, Head& dw,
                                              const QkNormParams& p) {
  if (NORM == kAfter) rotate(z, t);
  if (NORM == kBefore) rotate_back(g, t);
  F2 ss = mul(z.a[0], z.a[0]), gz = mul(mul(g.a[0], w.a[0]), z.a[0]);
  ss = fma2(z.b[0], z.b[0], ss), gz = fma2(mul(g.b[0], w.b[0]), z.b[0], gz);
  ss = fma2(z.a[1], z.a[1], ss), gz = fma2(mul(g.a[1], w.a[1]), z.a[1], gz);
  ss = fma2(z.b[1], z.b[1], ss), gz = fma2(mul(g.b[1], w.b[1]), z.b[1], gz);
  const float r = rsqrtf(fmaf(head_sum<LPH>(sum(ss)), p.inv_d, p.eps));
  const float m = -head_sum<LPH>(sum(gz)) * p.inv_d * r * r * r;  // -mean(g w u) / rms^2: times z, -u mean(g w u) / rms
  const F2 rr = f2(r, r), mm = f2(m, m);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const F2 ta = mul(g.a[i], rr), tb = mul(g.b[i], rr);
    dw.a[i] = fma2(ta, z.a[i], dw.a[i]);
    dw.b[i] = fma2(tb, z.b[i], dw.b[i]);
    z.a[i] = fma2(ta, w.a[i], mul(z.a[i], mm));
    z.b[i] = fma2(tb, w.b[i], mul(z.b[i], mm));
  }
  if (NORM == kAfter) rotate_back(z, t);
}

constexpr int kSteps = 4;  // steps of a warp whose loads are in flight together

// Few rows: block (32, warps per row, rows), straight from global memory.
template <typename T, int LPH, bool HALF, int NORM>
__global__ void __launch_bounds__(384, 2) qk_norm_fwd_kernel(const QkNormParams p) {
  constexpr int HPW = 32 / LPH, U = sizeof(T) == 4 ? kSteps / 2 : kSteps;
  const int lane = threadIdx.x, sub = lane / LPH;
  const Place<HALF> at(lane % LPH, p);
  const Share sh(p, threadIdx.y, blockDim.y);
  begin_early();
  const int row = blockIdx.x * blockDim.z + threadIdx.z;
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + (long long)row * p.ldx + sh.col0 + sub * p.D;
  T* y = static_cast<T*>(p.out) + (long long)row * p.ldo + sh.col0 + sub * p.D;
  const int step = HPW * p.D;
  Turn turn;
  Head w = zero_head();
  for (int s0 = sh.part; s0 * HPW < sh.heads; s0 += U * sh.stride) {
    Raw8<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * sh.stride;
      if (s * HPW + sub < sh.heads && at.on) raw[u] = load_raw<HALF>(x + s * step, at);
    }
    if (s0 == sh.part) {  // behind the first loads
      turn = load_turn<HALF>(p, row, at);
      if (NORM != kNone && at.on) w = to_head<HALF>(load_raw<HALF>(static_cast<const T*>(sh.key ? p.wk : p.wq), at));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * sh.stride;
      if (s * HPW >= sh.heads) break;  // the same for the whole warp
      const bool on = s * HPW + sub < sh.heads && at.on;
      Head z = on ? to_head<HALF>(raw[u]) : zero_head();
      head_forward<LPH, NORM>(z, turn, w, p);
      if (on) store_head<HALF>(y + s * step, at, z);
    }
  }
}

// Many rows, both directions: a producer warp keeps STAGES chunks of `chunk` rows (x, dy in the backward, and
// their (cos, sin) rows) on their way into shared memory with bulk copies, so that the loads in flight do not
// depend on registers or occupancy; the other warps take their heads of each row out of it. CTA c has the
// chunks c, c + grid, ... In the backward the sums of g u stay in registers and go to the CTA's own row of dw_part,
// so the result does not depend on any order in time.
// Forward nearly bound by HBM, backward by latency: 8192 rows of 20 heads of 128 in bfloat16 take 15.5 us forward (84
// MB, 0.83 of the copy rate) and 29 us backward (126 MB, 0.66), where 30 % of the warps an SM can hold issue in 54 %
// of its slots, waiting for the instruction before (105 per two heads forward, 190 backward), for the two sums over
// a head's lanes and for shared memory.
constexpr int kStages = 4;
// consumer warps of a CTA at most: 10 leave the backward of 16-bit types enough registers not to spill (33.7 -> 30 us at
// 8192 rows of 20 heads of 128), 4-byte rows are so wide that often only one is in a chunk and all warps share it
__host__ __device__ constexpr int max_warps(int elem) { return elem == 4 ? 12 : 10; }
constexpr int kRowsSmem = 100 * 1024;  // of which an SM holds two
// Input bytes from which the forward takes qk_norm_rows_kernel. Measured on B200, 20 heads of 128 in bfloat16: 148
// rows (0.8 MB) 2.08 us straight from global memory and 2.13 through shared memory, 300 rows 3.19 and 2.67, 8192 rows
// 45.8 and 15.5; 9 heads of 64: 600 rows (0.7 MB) 2.30 and 2.39, 2048 rows (2.4 MB) 3.69 and 3.46.
constexpr long long kFewBytes = 1400000;

// EVEN: every lane group of every step has a whole head (D = 8 LPH, head counts multiples of 32 / LPH).
template <typename T, int LPH, bool HALF, int NORM, bool EVEN, bool BWD>
__global__ void __launch_bounds__(32 * (max_warps(sizeof(T)) + 1), 2) qk_norm_rows_kernel(const QkNormParams p, int chunk) {
  constexpr int HPW = 32 / LPH;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint64_t full[kStages], empty[kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (blockDim.x >> 5) - 1;
  const int row_bytes = (p.hq + p.hkv) * p.D * (int)sizeof(T), cs_bytes = p.rot * 4;
  const int per_row = row_bytes * (BWD ? 2 : 1) + cs_bytes, stage_bytes = per_row * chunk;
  const int chunks = (p.rows + chunk - 1) / chunk;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], warps);
    }
    fence_mbar_init();
  }
  begin_early();
  __syncthreads();
  Head dw = zero_head();
  Place<HALF> at(lane % LPH, p);
  if (EVEN) at.on = true;
  const int sub = lane / LPH;

  if (warp == warps) {  // producer: lane r copies row r of the chunk
    int n = 0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x, ++n) {
      const int st = n % kStages, row = c * chunk + lane, live = min(chunk, p.rows - c * chunk);
      int pos = 0;
      if (lane < live) pos = p.pos ? p.pos[row] : row % p.seq_len;
      const bool in_table = pos >= 0 && pos < p.max_pos;
      if (n >= kStages && !mbar_wait(&empty[st], (n / kStages - 1) & 1, p.err, kErrWaitEmpty)) break;
      unsigned char* at_row = smem + st * stage_bytes + lane * per_row;
      if (lane < live && !in_table) {  // left unrotated
        set_error(p.err, kErrBadArg);
        for (int i = 0; i < p.rot / 2; ++i)
          reinterpret_cast<float2*>(at_row + per_row - cs_bytes)[i] = make_float2(1.f, 0.f);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before a later copy into the same place
      }
      const int tables = __popc(__ballot_sync(0xffffffff, lane < live && in_table));
      __syncwarp();  // rows written here are visible to the lane that arrives
      if (lane == 0) mbar_expect_tx(&full[st], live * (per_row - cs_bytes) + tables * cs_bytes);
      __syncwarp();
      if (lane < live) {
        bulk_load(at_row, static_cast<const T*>(p.x) + (long long)row * p.ldx, row_bytes, &full[st]);
        if (BWD)
          bulk_load(at_row + row_bytes, static_cast<const T*>(p.dy) + (long long)row * p.lddy, row_bytes, &full[st]);
        if (in_table)
          bulk_load(at_row + per_row - cs_bytes, p.table + (long long)pos * (p.rot / 2), cs_bytes, &full[st]);
      }
    }
    // no copy outlives the CTA, should its consumers have given up
    for (int i = max(0, n - kStages); i < n; ++i) mbar_wait(&full[i % kStages], (i / kStages) & 1, p.err, kErrWaitFull);
  } else {
    const int z = warp / p.warps_per_row;  // of every p.rows_at_once rows, this warp has the z-th
    const Share sh(p, warp - z * p.warps_per_row, p.warps_per_row);
    const Head w = NORM != kNone && at.on
                       ? to_head<HALF>(load_raw<HALF>(static_cast<const T*>(sh.key ? p.wk : p.wq), at)) : zero_head();
    const int stride = sh.stride * HPW * p.D, col = sh.col0 + (sh.part * HPW + sub) * p.D;
    const int left = sh.heads - sh.part * HPW;  // heads from the warp's first on
    const int steps = left > 0 ? (left + sh.stride * HPW - 1) / (sh.stride * HPW) : 0;
    // a lane group behind the last head has a step less, lanes without channels have none
    const int mine = EVEN ? steps : at.on ? max(0, (left - sub + sh.stride * HPW - 1) / (sh.stride * HPW)) : 0;
    int n = 0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x, ++n) {
      const int st = n % kStages, live = min(chunk, p.rows - c * chunk);
      if (!mbar_wait(&full[st], (n / kStages) & 1, p.err, kErrWaitFull)) break;
      const unsigned char* src = smem + st * stage_bytes + z * per_row;
      T* out = static_cast<T*>(p.out) + ((long long)c * chunk + z) * p.ldo + col;
      for (int r = z; r < live; r += p.rows_at_once, src += p.rows_at_once * per_row, out += p.rows_at_once * p.ldo) {
        const Turn turn = at.on && at.cs >= 0
                              ? to_turn(reinterpret_cast<const float4*>(src + per_row - cs_bytes + at.cs * 8)) : no_turn();
        const T* x = reinterpret_cast<const T*>(src) + col;
        T* y = out;
#pragma unroll(BWD || sizeof(T) == 4 ? 1 : 2)
        for (int s = 0; s < steps; ++s, x += stride, y += stride) {
          const bool on = EVEN || s < mine;
          Head v = on ? to_head<HALF>(load_raw<HALF>(x, at)) : zero_head();
          if (BWD) {
            const T* dy = reinterpret_cast<const T*>(reinterpret_cast<const unsigned char*>(x) + row_bytes);
            Head g = on ? to_head<HALF>(load_raw<HALF>(dy, at)) : zero_head();
            head_backward<LPH, NORM>(v, g, turn, w, dw, p);
          } else {
            head_forward<LPH, NORM>(v, turn, w, p);
          }
          if (on) store_head<HALF>(y, at, v);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
  }
  if (!BWD) return;
  // lanes of a warp that hold the same channels, then the CTA's warps of each weight in order
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);  // [warp][D]; every copy has been waited for
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float2 a = split(dw.a[i]), b = split(dw.b[i]);
#pragma unroll
    for (int o = 16; o >= LPH; o >>= 1) {
      a.x += __shfl_xor_sync(0xffffffff, a.x, o), a.y += __shfl_xor_sync(0xffffffff, a.y, o);
      b.x += __shfl_xor_sync(0xffffffff, b.x, o), b.y += __shfl_xor_sync(0xffffffff, b.y, o);
    }
    if (warp < warps && sub == 0 && at.on) {
      float* to = red + warp * p.D;
      if (HALF) to[at.c0 + 2 * i] = a.x, to[at.c0 + 2 * i + 1] = a.y, to[at.c1 + 2 * i] = b.x, to[at.c1 + 2 * i + 1] = b.y;
      else to[at.c0 + 4 * i] = a.x, to[at.c0 + 4 * i + 1] = b.x, to[at.c0 + 4 * i + 2] = a.y, to[at.c0 + 4 * i + 3] = b.y;
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.D; c += blockDim.x) {
    const bool key = c >= p.D;
    float s = 0.f;
    for (int w = 0; w < warps; ++w)
      if ((w % p.warps_per_row >= p.q_parts) == key) s += red[w * p.D + c - key * p.D];
    p.dw_part[(long long)blockIdx.x * 2 * p.D + c] = s;
  }
}

// dw[c] = sum over blocks of part[block][c], c over both weights: 8 columns (one sector of each
// partial row) per CTA, 32 rows of threads.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_dw_kernel(const float* part, int blocks, int D, T* dwq, T* dwk) {
  begin_early();
  __shared__ float s[8][8];
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  const int c = blockIdx.x * 8 + tx;
  float a = 0.f;
#pragma unroll 10
  for (int b = ty; b < blocks; b += 32) a += part[(long long)b * 2 * D + c];
  a += __shfl_xor_sync(0xffffffff, a, 8);
  a += __shfl_xor_sync(0xffffffff, a, 16);
  if ((threadIdx.x & 31) < 8) s[threadIdx.x >> 5][tx] = a;
  __syncthreads();
  if (threadIdx.x < 8) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += s[i][tx];
    T* o = c < D ? dwq + c : dwk + (c - D);
    *o = round_to<T>(t);
  }
}

// How a call runs. chunk 0: qk_norm_fwd_kernel with `block`; else qk_norm_rows_kernel.
struct Launch {
  int lph, blocks, chunk, smem;
  dim3 block;
};

template <typename K>
void allow_smem(K kernel, int smem, bool* set) {  // the attribute belongs to the device that is current
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && set[dev]) return;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (dev >= 0 && dev < 64) set[dev] = true;
}
template <typename T, int LPH, bool HALF, int NORM, bool EVEN, bool BWD>
void launch_rows(const QkNormParams& p, const Launch& l, cudaStream_t s) {
  auto kernel = qk_norm_rows_kernel<T, LPH, HALF, NORM, EVEN, BWD>;
  static bool set[64] = {};
  allow_smem(kernel, kRowsSmem, set);
  launch_early(kernel, dim3(l.blocks), l.block, l.smem, s, p, l.chunk);
}
template <typename T, int LPH, bool HALF, int NORM, bool BWD>
void launch(const QkNormParams& p, const Launch& l, cudaStream_t s) {
  constexpr int HPW = 32 / LPH;
  if constexpr (BWD && NORM == kNone) return;  // the transposed rotation is a forward call
  if (!BWD && l.chunk == 0)
    launch_early(qk_norm_fwd_kernel<T, LPH, HALF, NORM>, dim3(l.blocks), l.block, 0, s, p);
  else if (p.D == 8 * LPH && p.hq % HPW == 0 && p.hkv % HPW == 0) launch_rows<T, LPH, HALF, NORM, true, BWD>(p, l, s);
  else launch_rows<T, LPH, HALF, NORM, false, BWD>(p, l, s);
}
template <typename T, bool HALF, int NORM, bool BWD>
void by_heads(const QkNormParams& p, const Launch& l, cudaStream_t s) {
  if (l.lph == 8) launch<T, 8, HALF, NORM, BWD>(p, l, s);
  else if (l.lph == 16) launch<T, 16, HALF, NORM, BWD>(p, l, s);
  else launch<T, 32, HALF, NORM, BWD>(p, l, s);
}
template <typename T, bool BWD>
void by_mode(const QkNormParams& p, const Launch& l, bool half_layout, int norm, cudaStream_t s) {
  if (half_layout) {
    if (norm == kNone) by_heads<T, true, kNone, BWD>(p, l, s);
    else if (norm == kAfter) by_heads<T, true, kAfter, BWD>(p, l, s);
    else by_heads<T, true, kBefore, BWD>(p, l, s);
  } else {
    if (norm == kNone) by_heads<T, false, kNone, BWD>(p, l, s);
    else if (norm == kAfter) by_heads<T, false, kAfter, BWD>(p, l, s);
    else by_heads<T, false, kBefore, BWD>(p, l, s);
  }
}
template <typename T>
void sum_dw(const QkNormParams& p, int blocks, void* dwq, void* dwk, cudaStream_t s) {
  launch_early(qk_norm_dw_kernel<T>, dim3(2 * p.D / 8), dim3(256), 0, s, (const float*)p.dw_part, blocks, p.D,
               static_cast<T*>(dwq), static_cast<T*>(dwk));
}

}  // namespace
}  // namespace astrai

namespace astrai_host {

namespace {

int lanes_per_head(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// Few rows: one step per warp at most 12 warps a row. A row's warps sit in one block, so its (cos, sin) pairs
// come from L2 once.
astrai::Launch few_rows(astrai::QkNormParams& p) {
  astrai::Launch l{};
  l.lph = lanes_per_head(p.D);
  const int hpw = 32 / l.lph, sq = (p.hq + hpw - 1) / hpw, sk = (p.hkv + hpw - 1) / hpw;
  p.q_parts = std::min(8, sq);
  const int warps = p.q_parts + std::min(4, sk);
  l.block = dim3(32, warps, std::max(1, 8 / warps));
  l.blocks = (p.rows + (int)l.block.z - 1) / (int)l.block.z;
  return l;
}

// Heads of a row that qk_norm_rows_kernel can take at a time: kStages of them fit half an SM's shared memory.
int heads_that_fit(int D, int rot, int elem, bool bwd) {
  return (astrai::kRowsSmem / astrai::kStages - rot * 4) / (D * elem * (bwd ? 2 : 1));
}
int launches_of_rows(int heads, int D, int rot, int elem, bool bwd) {
  const int n = heads_that_fit(D, rot, elem, bwd);
  return (heads + n - 1) / n;
}

// Many rows: consumer warps in the ratio of query to key heads, chunks of at most 4 rows (more even shares).
astrai::Launch many_rows(astrai::QkNormParams& p, int elem, bool bwd, int sms) {
  using namespace astrai;
  Launch l{};
  l.lph = lanes_per_head(p.D);
  const int hpw = 32 / l.lph, sq = (p.hq + hpw - 1) / hpw, sk = (p.hkv + hpw - 1) / hpw;
  const int per_row = (p.hq + p.hkv) * p.D * elem * (bwd ? 2 : 1) + p.rot * 4;
  l.chunk = std::min(std::min(4, (p.rows + 2 * sms - 1) / (2 * sms)), kRowsSmem / (kStages * per_row));
  // `turns` steps of a warp per row and as many rows at once as there are warps for: the most rows per step, and of
  // equals two turns, which share a row's (cos, sin) pairs (24 + 4 heads of 64, 2048 rows: 2 turns 4.8 us, 3 turns 5.3)
  double best = 0;
  for (int turns = 1; turns <= std::max(sq, sk); ++turns) {
    const int q = (sq + turns - 1) / turns, w = q + (sk + turns - 1) / turns;
    if (w > max_warps(elem)) continue;
    const int rows = std::min(max_warps(elem) / w, l.chunk);
    if ((double)rows / turns < best || ((double)rows / turns == best && turns > 2)) continue;
    best = (double)rows / turns;
    p.q_parts = q, p.warps_per_row = w, p.rows_at_once = rows;
  }
  const int warps = p.warps_per_row * p.rows_at_once;
  l.smem = std::max(per_row * l.chunk * kStages, bwd ? warps * p.D * 4 : 0);
  l.block = dim3(32 * (warps + 1));
  l.blocks = std::min(2 * sms, (p.rows + l.chunk - 1) / l.chunk);
  return l;
}

// The heads [h0, h0 + n) of a call as a call of its own.
astrai::QkNormParams some_heads(const astrai::QkNormParams& p, int h0, int n, int elem) {
  astrai::QkNormParams r = p;
  const long long off = (long long)h0 * p.D * elem;
  r.x = static_cast<const char*>(p.x) + off;
  if (p.dy) r.dy = static_cast<const char*>(p.dy) + off;
  r.out = static_cast<char*>(p.out) + off;
  r.hq = std::max(0, std::min(p.hq - h0, n));
  r.hkv = n - r.hq;
  return r;
}

}  // namespace

// dtype: 0 bf16, 1 fp16, 2 fp32. norm: 0 none, 1 after the rotation, 2 before it.
void qk_norm_fwd(const void* x, long long ldx, void* y, long long ldy, int rows, int hq, int hkv, int D,
                 const void* table, int max_pos, const int* pos, int seq_len, const void* wq, const void* wk, int rot,
                 int rot_off, bool half_layout, int norm, int inverse, float eps, int dtype, int device,
                 cudaStream_t s) {
  using namespace astrai;
  if (rows <= 0) return;
  QkNormParams p{};
  p.x = x, p.out = y, p.ldx = ldx, p.ldo = ldy, p.wq = wq, p.wk = wk;
  p.table = static_cast<const float2*>(table), p.pos = pos, p.err = error_word(device);
  p.rows = rows, p.hq = hq, p.hkv = hkv, p.D = D, p.rot = rot, p.rot_off = rot_off;
  p.seq_len = seq_len, p.max_pos = max_pos, p.inverse = inverse != 0, p.eps = eps, p.inv_d = 1.f / D;
  const int sms = num_sms(device), elem = dtype == 2 ? 4 : 2, heads = hq + hkv;
  const auto run = [&](const QkNormParams& part, const Launch& l) {
    if (dtype == 0) by_mode<__nv_bfloat16, false>(part, l, half_layout, norm, s);
    else if (dtype == 1) by_mode<__half, false>(part, l, half_layout, norm, s);
    else by_mode<float, false>(part, l, half_layout, norm, s);
  };
  if ((long long)rows * heads * D * elem < kFewBytes) {
    const Launch l = few_rows(p);
    run(p, l);
    return;
  }
  const int n = launches_of_rows(heads, D, rot, elem, false), per = (heads + n - 1) / n;
  for (int h0 = 0; h0 < heads; h0 += per) {
    QkNormParams part = some_heads(p, h0, std::min(per, heads - h0), elem);
    const Launch l = many_rows(part, elem, false, sms);
    run(part, l);
  }
}

// fp32 elements of scratch that the backward needs: 2 * D for each CTA of each of its launches.
long long qk_norm_bwd_scratch(int rows, int heads, int D, int rot, int elem, int device) {
  return 2LL * D * std::min(rows, num_sms(device) * 2) * launches_of_rows(heads, D, rot, elem, true);
}

void qk_norm_bwd(const void* dy, long long lddy, const void* x, long long ldx, void* dx, long long lddx, int rows,
                 int hq, int hkv, int D, const void* table, int max_pos, const int* pos, int seq_len, const void* wq,
                 const void* wk, int rot, int rot_off, bool half_layout, int norm, float eps, void* dwq, void* dwk,
                 float* scratch, int dtype, int device, cudaStream_t s) {
  using namespace astrai;
  if (rows <= 0) return;
  QkNormParams p{};
  p.x = x, p.dy = dy, p.out = dx, p.ldx = ldx, p.lddy = lddy, p.ldo = lddx, p.wq = wq, p.wk = wk;
  p.table = static_cast<const float2*>(table), p.pos = pos, p.dw_part = scratch, p.err = error_word(device);
  p.rows = rows, p.hq = hq, p.hkv = hkv, p.D = D, p.rot = rot, p.rot_off = rot_off;
  p.seq_len = seq_len, p.max_pos = max_pos, p.eps = eps, p.inv_d = 1.f / D;
  const int sms = num_sms(device), elem = dtype == 2 ? 4 : 2, heads = hq + hkv;
  const int n = launches_of_rows(heads, D, rot, elem, true), per = (heads + n - 1) / n;
  int parts = 0;
  for (int h0 = 0; h0 < heads; h0 += per) {
    QkNormParams part = some_heads(p, h0, std::min(per, heads - h0), elem);
    const Launch l = many_rows(part, elem, true, sms);
    part.dw_part = scratch + 2LL * D * parts;
    parts += l.blocks;
    if (dtype == 0) by_mode<__nv_bfloat16, true>(part, l, half_layout, norm, s);
    else if (dtype == 1) by_mode<__half, true>(part, l, half_layout, norm, s);
    else by_mode<float, true>(part, l, half_layout, norm, s);
  }
  if (dtype == 0) sum_dw<__nv_bfloat16>(p, parts, dwq, dwk, s);
  else if (dtype == 1) sum_dw<__half>(p, parts, dwq, dwk, s);
  else sum_dw<float>(p, parts, dwq, dwk, s);
}

}  // namespace astrai_host
