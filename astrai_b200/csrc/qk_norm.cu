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
  int rows, hq, heads, D, rot, rot_off, seq_len, max_pos, parts;
  float sign, eps;
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, float* o) {
  if constexpr (sizeof(T) == 4) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same<T, __half>::value) o[j] = __half2float(e[j]);
      else o[j] = __bfloat162float(e[j]);
    }
  }
}
template <typename T>
__device__ __forceinline__ T round_to(float x) {
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(x);
  else return x;
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
// raw channels -> the pairs' first and second members
template <bool HALF, typename T>
__device__ __forceinline__ void to_pairs(const Raw8<T>& r, float* a, float* b) {
  float f[8];
  load4(r.c[0].v, f);
  load4(r.c[1].v, f + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = HALF ? f[i] : f[2 * i];
    b[i] = HALF ? f[4 + i] : f[2 * i + 1];
  }
}
template <bool HALF, typename T>
__device__ __forceinline__ void store_pairs(T* head, const Place<HALF>& at, const float* a, const float* b) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (HALF) {
      r.c[0].v[i] = round_to<T>(a[i]);
      r.c[1].v[i] = round_to<T>(b[i]);
    } else {
      r.c[i / 2].v[i % 2 * 2] = round_to<T>(a[i]);
      r.c[i / 2].v[i % 2 * 2 + 1] = round_to<T>(b[i]);
    }
  }
  if constexpr (HALF || sizeof(T) == 4) {
    *reinterpret_cast<Four<T>*>(head + at.c0) = r.c[0];
    *reinterpret_cast<Four<T>*>(head + at.c1) = r.c[1];
  } else {
    *reinterpret_cast<uint4*>(head + at.c0) = *reinterpret_cast<const uint4*>(&r);
  }
}
__device__ __forceinline__ void rotate(float* a, float* b, const float2* cs, float sign) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float s = sign * cs[i].y, x = a[i];
    a[i] = x * cs[i].x - b[i] * s;
    b[i] = x * s + b[i] * cs[i].x;
  }
}
// A lane's four (cos, sin) pairs of a row. A position outside the table records kErrBadArg and leaves
// the row unrotated.
template <bool HALF>
__device__ __forceinline__ void load_cs(const QkNormParams& p, int row, const Place<HALF>& at, float2* cs) {
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = make_float2(1.f, 0.f);
  if (!at.on || at.cs < 0) return;
  const int t = p.pos ? p.pos[row] : row % p.seq_len;
  if (t < 0 || t >= p.max_pos) {
    set_error(p.err, kErrBadArg);
    return;
  }
  const float4* c = reinterpret_cast<const float4*>(p.table + (long long)t * (p.rot / 2) + at.cs);
  const float4 u = c[0], v = c[1];
  cs[0] = make_float2(u.x, u.y), cs[1] = make_float2(u.z, u.w);
  cs[2] = make_float2(v.x, v.y), cs[3] = make_float2(v.z, v.w);
}
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  return v;
}

constexpr int kUnroll = 4;  // heads per lane group and warp item: their loads are in flight together

// One warp per (row, part): the row's heads in steps of 32 / LPH are dealt out to `parts` warps.
template <typename T, int LPH, bool HALF, int NORM>
__global__ void __launch_bounds__(256) qk_norm_fwd_kernel(const QkNormParams p) {
  constexpr int HPW = 32 / LPH;
  const int lane = threadIdx.x & 31, sub = lane / LPH;
  const Place<HALF> at(lane % LPH, p);
  const long long item = blockIdx.x * 8LL + (threadIdx.x >> 5);
  const int row = (int)(item / p.parts), part = (int)(item % p.parts);
  if (row >= p.rows) return;
  const T* x = static_cast<const T*>(p.x) + (long long)row * p.ldx;
  T* y = static_cast<T*>(p.out) + (long long)row * p.ldo;
  Raw8<T> raw[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int h = (part + u * p.parts) * HPW + sub;
    if (h < p.heads && at.on) raw[u] = load_raw<HALF>(x + h * p.D, at);
  }
  float2 cs[4];
  load_cs<HALF>(p, row, at, cs);
  float w[2][8];
  if (NORM != kNone && at.on) {
    to_pairs<HALF>(load_raw<HALF>(static_cast<const T*>(p.wq), at), w[0], w[0] + 4);
    to_pairs<HALF>(load_raw<HALF>(static_cast<const T*>(p.wk), at), w[1], w[1] + 4);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int h = (part + u * p.parts) * HPW + sub;
    const bool on = h < p.heads && at.on;
    if ((part + u * p.parts) * HPW >= p.heads) break;  // the same for the whole warp
    float a[4], b[4];
    if (on) to_pairs<HALF>(raw[u], a, b);
    if (NORM != kBefore && on) rotate(a, b, cs, p.sign);
    if (NORM != kNone) {
      float ss = 0.f;
      if (on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += a[i] * a[i] + b[i] * b[i];
      }
      const float r = rsqrtf(head_sum<LPH>(ss) / (float)p.D + p.eps);
      if (on) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a[i] *= r * (h < p.hq ? w[0][i] : w[1][i]);
          b[i] *= r * (h < p.hq ? w[0][4 + i] : w[1][4 + i]);
        }
      }
    }
    if (NORM == kBefore && on) rotate(a, b, cs, p.sign);
    if (on) store_pairs<HALF>(y + h * p.D, at, a, b);
  }
}

// Backward: a warp walks items of the same shape, keeping its lanes' sums of g u in registers; a
// block's sums go to its own row of dw_part, so the result does not depend on any order in time.
template <typename T, int LPH, bool HALF, int NORM>
__global__ void __launch_bounds__(256) qk_norm_bwd_kernel(const QkNormParams p) {
  constexpr int HPW = 32 / LPH, U = 2;
  const int lane = threadIdx.x & 31, sub = lane / LPH, warp = threadIdx.x >> 5;
  const Place<HALF> at(lane % LPH, p);
  float w[2][8], dw[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[0][i] = w[1][i] = dw[0][i] = dw[1][i] = 0.f;
  if (at.on) {
    to_pairs<HALF>(load_raw<HALF>(static_cast<const T*>(p.wq), at), w[0], w[0] + 4);
    to_pairs<HALF>(load_raw<HALF>(static_cast<const T*>(p.wk), at), w[1], w[1] + 4);
  }
  const long long items = (long long)p.rows * p.parts;
  for (long long item = blockIdx.x * 8LL + warp; item < items; item += gridDim.x * 8LL) {
    const int row = (int)(item / p.parts), part = (int)(item % p.parts);
    const T* x = static_cast<const T*>(p.x) + (long long)row * p.ldx;
    const T* dy = static_cast<const T*>(p.dy) + (long long)row * p.lddy;
    T* dx = static_cast<T*>(p.out) + (long long)row * p.ldo;
    float2 cs[4];
    load_cs<HALF>(p, row, at, cs);
    for (int s0 = part; s0 * HPW < p.heads; s0 += U * p.parts) {
      Raw8<T> rx[U], rg[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = (s0 + u * p.parts) * HPW + sub;
        if (h < p.heads && at.on) {
          rx[u] = load_raw<HALF>(x + h * p.D, at);
          rg[u] = load_raw<HALF>(dy + h * p.D, at);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = (s0 + u * p.parts) * HPW + sub;
        const bool on = h < p.heads && at.on, isq = h < p.hq;
        float a[4], b[4], ga[4], gb[4], ss = 0.f, gz = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = b[i] = ga[i] = gb[i] = 0.f;
        if (on) {
          to_pairs<HALF>(rx[u], a, b);
          to_pairs<HALF>(rg[u], ga, gb);
          if (NORM == kAfter) rotate(a, b, cs, 1.f);
          if (NORM == kBefore) rotate(ga, gb, cs, -1.f);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            ss += a[i] * a[i] + b[i] * b[i];
            gz += ga[i] * (isq ? w[0][i] : w[1][i]) * a[i] + gb[i] * (isq ? w[0][4 + i] : w[1][4 + i]) * b[i];
          }
        }
        ss = head_sum<LPH>(ss);
        gz = head_sum<LPH>(gz);
        const float r = rsqrtf(ss / (float)p.D + p.eps);
        const float m = gz * r * r / (float)p.D;  // mean(g w u) / rms: times z it is u mean(g w u)
        if (on) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float ta = ga[i] * a[i] * r, tb = gb[i] * b[i] * r;
            dw[0][i] += isq ? ta : 0.f;
            dw[1][i] += isq ? 0.f : ta;
            dw[0][4 + i] += isq ? tb : 0.f;
            dw[1][4 + i] += isq ? 0.f : tb;
            a[i] = r * (ga[i] * (isq ? w[0][i] : w[1][i]) - a[i] * m);
            b[i] = r * (gb[i] * (isq ? w[0][4 + i] : w[1][4 + i]) - b[i] * m);
          }
          if (NORM == kAfter) rotate(a, b, cs, -1.f);
          store_pairs<HALF>(dx + h * p.D, at, a, b);
        }
      }
    }
  }
  // lanes of the warp that hold the same channels, then the block's warps in order
  __shared__ float red[8][2][256];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int o = 16; o >= LPH; o >>= 1) dw[k][i] += __shfl_xor_sync(0xffffffff, dw[k][i], o);
  if (sub == 0 && at.on) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int ca = HALF ? at.c0 + i : at.c0 + 2 * i, cb = HALF ? at.c1 + i : at.c0 + 2 * i + 1;
        red[warp][k][ca] = dw[k][i];
        red[warp][k][cb] = dw[k][4 + i];
      }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.D; c += 256) {
    const int k = c >= p.D, ch = c - k * p.D;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += red[i][k][ch];
    p.dw_part[(long long)blockIdx.x * 2 * p.D + c] = s;
  }
}

// dw[c] = sum over blocks of part[block][c], c over both weights: 8 columns (one sector of each
// partial row) per CTA, 32 rows of threads, then a tree through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_dw_kernel(const float* __restrict__ part, int blocks, int D,
                                                         T* __restrict__ dwq, T* __restrict__ dwk) {
  __shared__ float s[32][9];
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  const int c = blockIdx.x * 8 + tx;
  float a = 0.f;
#pragma unroll 4
  for (int b = ty; b < blocks; b += 32) a += part[(long long)b * 2 * D + c];
  s[ty][tx] = a;
  __syncthreads();
#pragma unroll
  for (int h = 16; h > 0; h >>= 1) {
    if (ty < h) s[ty][tx] += s[ty + h][tx];
    __syncthreads();
  }
  if (ty == 0) {
    T* o = c < D ? dwq + c : dwk + (c - D);
    *o = round_to<T>(s[0][tx]);
  }
}

template <typename T, bool HALF, int NORM>
void launch_fwd(const QkNormParams& p, int lph, int blocks, cudaStream_t s) {
  switch (lph) {
    case 8: (note_launch(), qk_norm_fwd_kernel<T, 8, HALF, NORM><<<blocks, 256, 0, s>>>(p)); break;
    case 16: (note_launch(), qk_norm_fwd_kernel<T, 16, HALF, NORM><<<blocks, 256, 0, s>>>(p)); break;
    default: (note_launch(), qk_norm_fwd_kernel<T, 32, HALF, NORM><<<blocks, 256, 0, s>>>(p)); break;
  }
}
template <typename T, bool HALF, int NORM>
void launch_bwd(const QkNormParams& p, int lph, int blocks, cudaStream_t s) {
  switch (lph) {
    case 8: (note_launch(), qk_norm_bwd_kernel<T, 8, HALF, NORM><<<blocks, 256, 0, s>>>(p)); break;
    case 16: (note_launch(), qk_norm_bwd_kernel<T, 16, HALF, NORM><<<blocks, 256, 0, s>>>(p)); break;
    default: (note_launch(), qk_norm_bwd_kernel<T, 32, HALF, NORM><<<blocks, 256, 0, s>>>(p)); break;
  }
}
template <typename T>
void fwd_typed(const QkNormParams& p, int lph, int blocks, bool half_layout, int norm, cudaStream_t s) {
  if (half_layout) {
    if (norm == kNone) launch_fwd<T, true, kNone>(p, lph, blocks, s);
    else if (norm == kAfter) launch_fwd<T, true, kAfter>(p, lph, blocks, s);
    else launch_fwd<T, true, kBefore>(p, lph, blocks, s);
  } else {
    if (norm == kNone) launch_fwd<T, false, kNone>(p, lph, blocks, s);
    else if (norm == kAfter) launch_fwd<T, false, kAfter>(p, lph, blocks, s);
    else launch_fwd<T, false, kBefore>(p, lph, blocks, s);
  }
}
template <typename T>
void bwd_typed(const QkNormParams& p, int lph, int blocks, bool half_layout, int norm, void* dwq, void* dwk,
               cudaStream_t s) {
  if (half_layout) {
    if (norm == kAfter) launch_bwd<T, true, kAfter>(p, lph, blocks, s);
    else launch_bwd<T, true, kBefore>(p, lph, blocks, s);
  } else {
    if (norm == kAfter) launch_bwd<T, false, kAfter>(p, lph, blocks, s);
    else launch_bwd<T, false, kBefore>(p, lph, blocks, s);
  }
  (note_launch(), qk_norm_dw_kernel<T><<<2 * p.D / 8, 256, 0, s>>>(p.dw_part, blocks, p.D, static_cast<T*>(dwq),
                                                                   static_cast<T*>(dwk)));
}

int lanes_per_head(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

}  // namespace
}  // namespace astrai

namespace astrai_host {

// dtype: 0 bf16, 1 fp16, 2 fp32. norm: 0 none, 1 after the rotation, 2 before it.
void qk_norm_fwd(const void* x, long long ldx, void* y, long long ldy, int rows, int hq, int hkv, int D,
                 const void* table, int max_pos, const int* pos, int seq_len, const void* wq, const void* wk, int rot,
                 int rot_off, bool half_layout, int norm, int inverse, float eps, int dtype, int device,
                 cudaStream_t s) {
  using namespace astrai;
  if (rows <= 0) return;
  const int lph = lanes_per_head(D), steps = (hq + hkv + 32 / lph - 1) / (32 / lph);
  QkNormParams p{};
  p.x = x, p.out = y, p.ldx = ldx, p.ldo = ldy, p.wq = wq, p.wk = wk;
  p.table = static_cast<const float2*>(table), p.pos = pos, p.err = error_word(device);
  p.rows = rows, p.hq = hq, p.heads = hq + hkv, p.D = D, p.rot = rot, p.rot_off = rot_off;
  p.seq_len = seq_len, p.max_pos = max_pos, p.sign = inverse ? -1.f : 1.f, p.eps = eps;
  p.parts = (steps + kUnroll - 1) / kUnroll;
  const int blocks = (int)(((long long)rows * p.parts + 7) / 8);
  if (dtype == 0) fwd_typed<__nv_bfloat16>(p, lph, blocks, half_layout, norm, s);
  else if (dtype == 1) fwd_typed<__half>(p, lph, blocks, half_layout, norm, s);
  else fwd_typed<float>(p, lph, blocks, half_layout, norm, s);
}

// Blocks of the backward launch, each with 2 * D floats of scratch.
int qk_norm_bwd_blocks(int rows, int device) {
  return std::max(1, std::min((rows + 7) / 8, num_sms(device) * 3));
}

void qk_norm_bwd(const void* dy, long long lddy, const void* x, long long ldx, void* dx, long long lddx, int rows,
                 int hq, int hkv, int D, const void* table, int max_pos, const int* pos, int seq_len, const void* wq,
                 const void* wk, int rot, int rot_off, bool half_layout, int norm, float eps, void* dwq, void* dwk,
                 float* scratch, int dtype, int device, cudaStream_t s) {
  using namespace astrai;
  QkNormParams p{};
  p.x = x, p.dy = dy, p.out = dx, p.ldx = ldx, p.lddy = lddy, p.ldo = lddx, p.wq = wq, p.wk = wk;
  p.table = static_cast<const float2*>(table), p.pos = pos, p.dw_part = scratch, p.err = error_word(device);
  p.rows = rows, p.hq = hq, p.heads = hq + hkv, p.D = D, p.rot = rot, p.rot_off = rot_off;
  p.seq_len = seq_len, p.max_pos = max_pos, p.sign = 1.f, p.eps = eps, p.parts = 1;
  const int lph = lanes_per_head(D), blocks = qk_norm_bwd_blocks(rows, device);
  if (dtype == 0) bwd_typed<__nv_bfloat16>(p, lph, blocks, half_layout, norm, dwq, dwk, s);
  else if (dtype == 1) bwd_typed<__half>(p, lph, blocks, half_layout, norm, dwq, dwk, s);
  else bwd_typed<float>(p, lph, blocks, half_layout, norm, dwq, dwk, s);
}

}  // namespace astrai_host
