// Paged KV cache in 8-bit integers (sm_100a): append with quantisation, read-back, and causal
// attention of one or a few new tokens over it. No counterpart in the reference project, whose cache
// holds the model's type (astrai/inference/core/cache.py:189-276).
//
// Layout per layer: values int8 [page][kv_head][slot][D], and one fp32 magnitude for each block of
// `block` tokens and head, [page][kv_head][page_size / block]. A stored integer q stands for
// q * absmax / 127. Keeping the magnitude itself instead of the step absmax / 127 makes quantisation
// exact to describe: q = rint(127 x / absmax), with 127 x exact in fp32 for 16-bit inputs and the
// division correctly rounded, so ties fall where the real quotient has them.
//
// Attention holds the integers as fp16 (exact) on the tensor cores' mma.m16n8k16: the work is one
// pass over the cache at a few operations per byte, bound by HBM, and fragments straight from
// converted registers spare the second trip through shared memory that tcgen05 operands would need.
// S^T = K Q^T and O^T = V^T P^T put the tokens (then the channels) on the 16-row side and the query
// rows that share a KV head on the 8-column side, so a group of 4 query heads wastes half a tile and
// not three quarters.
#include <algorithm>
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.cuh"

namespace astrai {
namespace {

// ------------------------------------------------------------------ append
struct AppendParams {
  const void* src[2];           // k, v [B, S, Hkv, D]
  long long sb[2], st[2], sh[2];  // their strides (elements)
  signed char* cache[2];
  float* absmax[2];
  const int* table;
  const int* starts;
  const int* lens;
  int B, S, Hkv, page_size, n_pages, max_pages, windows;
};

template <typename T>
__device__ __forceinline__ float bits_to_float(unsigned short u) {
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(u));
  else return __bfloat162float(__ushort_as_bfloat16(u));
}
template <typename T>
__device__ __forceinline__ unsigned pack_pair(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&v);
  } else {
    return pack_bf16(a, b);
  }
}
template <typename T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

__device__ __forceinline__ void cp_async16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(unsigned dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(unsigned a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// rint(x / by) in the low byte, for |x / by| up to 127 and r = 1 / by rounded. The product x r is off by
// some units in its last place; one step of residual correction (Markstein, IBM J. Res. Dev. 34, 1990) gives
// the quotient rounded, exact where it is half an integer, and so the integer that the division would: x has
// at most 18 and by 11 significant bits, so other quotients are 2^-12 and more away from such ties. Adding
// 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the low bits.
__device__ __forceinline__ unsigned round_quotient(float x, float by, float r) {
  const float t = x * r;
  return __float_as_uint(fmaf(fmaf(-t, by, x), r, t) + 12582912.f);
}
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// One block of tokens of one head of k or v: its live tokens and the new ones end under the larger
// of their magnitudes. WARPS warps share it, at most 32 tokens each, whose values wait in shared memory
// between the maximum and the rounding. A row's append starts at starts[b] and ends at lens[b]; tokens
// before position 0 are dropped, and what the cache held from starts[b] on is void. A block with an infinite or NaN input gets the magnitude
// NaN: reading it gives NaN, as the input would have.
// Bound by its chain of loads (lengths, tokens, magnitude) at decode sizes, 2 us for 32 single tokens; 32 x 512
// tokens of 4 heads of 128 take 19 us, 0.4 of the copy rate. A block to a warp needs one pass over the input and no
// atomics; holding the values in registers instead unrolled into code that ran at the rate of instruction fetches.
template <typename T, int D, int BLOCK>
__global__ void __launch_bounds__(128) kv8_append_kernel(const AppendParams p) {
  constexpr int WARPS = BLOCK > 32 ? BLOCK / 32 : 1;  // warps per item
  constexpr int TOK = BLOCK / WARPS;                  // tokens per warp
  constexpr int LPT = D / 8;                          // 16-byte pieces (8 values) per token
  __shared__ __align__(16) unsigned char hold[4][TOK * D * 2];
  __shared__ unsigned most_s[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x * (4 / WARPS) + warp / WARPS;
  const int kv = item & 1;
  const unsigned bwh = (unsigned)item >> 1, bw = bwh / (unsigned)p.Hkv;
  const int h = (int)(bwh - bw * p.Hkv), b = (int)(bw / (unsigned)p.windows), w = (int)(bw - (unsigned)b * p.windows);
  begin_early();
  bool on = b < p.B;
  int first_pos = 0, start = 0, end = 0, base = 0, page = -1, off = 0;  // first_pos: of the row's first token in src
  if (on) {
    first_pos = min(max(p.starts[b], -(1 << 30)), p.max_pages * p.page_size);
    start = max(first_pos, 0);
    end = min(p.lens[b], first_pos + p.S);
    base = (start / BLOCK + w) * BLOCK;
    on = base < end && start < end;
  }
  // this warp's tokens first .. first + n - 1 of the block are new
  const int mine = warp % WARPS * TOK;
  const int first = max(start - base, mine), n = on ? max(0, min(end - base, mine + TOK) - first) : 0;
  const T* src = static_cast<const T*>(p.src[kv]) + (long long)b * p.sb[kv] + (long long)h * p.sh[kv] +
                 (long long)(base + first - first_pos) * p.st[kv];
  const unsigned held = (unsigned)__cvta_generic_to_shared(hold[warp]) + lane * 16;
#pragma unroll 4
  for (int i = lane; i < n * LPT; i += 32)
    cp_async16(held + (i - lane) * 16, src + (i / LPT) * p.st[kv] + i % LPT * 8);
  cp_async_commit();
  if (on) {
    const int lp = base / p.page_size;
    if (lp < p.max_pages) page = p.table[(long long)b * p.max_pages + lp];
    off = base - lp * p.page_size;
    on = page >= 0 && page < p.n_pages;
  }
  const long long row0 = ((long long)page * p.Hkv + h) * p.page_size + off;  // the block's first token
  float* ap = p.absmax[kv] + row0 / BLOCK;
  const float was = on && base < start ? *ap : 0.f;  // live tokens only
  cp_async_wait<0>();
  unsigned most = 0;
#pragma unroll 4
  for (int i = lane; i < n * LPT; i += 32) {  // magnitudes compare as integers, infinities and NaN above all others
    const uint4 v = lds128(held + (i - lane) * 16);
    most = __vmaxu2(most, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                   __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
  }
  most = max(most & 0xffffu, most >> 16);
  most = __reduce_max_sync(0xffffffff, most);
  if (WARPS > 1) {
    if (lane == 0) most_s[warp] = most;
    __syncthreads();  // and every warp has read the old magnitude before one replaces it
    const int w0 = warp / WARPS * WARPS;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) most = max(most, most_s[w0 + i]);
  } else {
    __syncwarp();  // every lane has read the old magnitude before one replaces it
  }
  if (!on) return;
  const float fresh = bits_to_float<T>((unsigned short)most);
  const bool finite = fresh < INFINITY;  // false for NaN, too
  const float now = finite ? (was >= fresh || was != was ? was : fresh) : __int_as_float(0x7fffffff);
  if (lane == 0 && warp % WARPS == 0) *ap = now;
  // scaled by a power of two, which changes no quotient, magnitude and products stay normal numbers
  const float pre = now > 1e30f ? 0x1p-16f : now < 1e-30f ? 0x1p40f : 1.f;
  const bool some = now > 0.f;
  const float by = some ? now * pre : 1.f, r = 1.f / by, mul = some ? 127.f * pre : 0.f;
  signed char* dst = p.cache[kv] + (row0 + first) * D;
#pragma unroll 2
  for (int i = lane; i < n * LPT; i += 32) {
    const uint4 v = lds128(held + (i - lane) * 16);
    const unsigned short* e = reinterpret_cast<const unsigned short*>(&v);
    unsigned q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = round_quotient(some ? bits_to_float<T>(e[j]) * mul : 0.f, by, r);
    *reinterpret_cast<uint2*>(dst + i * 8) =
        make_uint2(low_bytes(q[0], q[1], q[2], q[3]), low_bytes(q[4], q[5], q[6], q[7]));
  }
  if (now > was && base < start) {  // live tokens under a magnitude that grew
    const float old = was * pre;
    uint2* live = reinterpret_cast<uint2*>(p.cache[kv] + (row0 + mine) * D);
#pragma unroll 1
    for (int i = lane; i < min(start - base - mine, TOK) * LPT; i += 32) {
      const uint2 v = live[i];
      const signed char* e = reinterpret_cast<const signed char*>(&v);
      unsigned q[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = round_quotient((float)e[j] * old, by, r);
      live[i] = make_uint2(low_bytes(q[0], q[1], q[2], q[3]), low_bytes(q[4], q[5], q[6], q[7]));
    }
  }
}

// ------------------------------------------------------------------ read-back
struct GatherParams {
  const signed char* cache[2];
  const float* absmax[2];
  const int* table;
  const int* starts;  // null: from token 0
  const int* lens;
  void* out[2];       // [B, total, Hkv, D]
  int B, total, Hkv, page_size, n_pages, max_pages;
  int blocks_per_page, block_bits;  // magnitudes per page and head; log2(block)
};

constexpr float kStep = 1.f / 127.f;

// integers of a word (as q + 128) to four fp32 numbers: under the high bytes of 2^23 a byte is 2^23 + u
__device__ __forceinline__ void word_to_floats(unsigned u, float* v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 | j)) - 8388736.f;
}

constexpr int kGatherTokens = 64;  // of a CTA

// Grid (tokens, heads, rows); a lane 16 values of k and the same 16 of v. Bound by HBM, two thirds of it writes: 32 x
// 4096 tokens of 4 heads of 128 take 81 us, 0.76 of the copy rate.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_gather_kernel(const GatherParams p) {
  constexpr int C = D / 16, PER = 256 / C, N = kGatherTokens / PER;
  const int b = blockIdx.z, h = blockIdx.y, c = threadIdx.x % C;
  begin_early();
  const int start = p.starts ? min(max(p.starts[b], -(1 << 30)), 1 << 30) : 0, len = p.lens[b];
  const int t0 = blockIdx.x * kGatherTokens + threadIdx.x / C;
  uint4 raw[N][2];
  float step[N][2];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t = t0 + i * PER, pos = start + t, lp = pos / p.page_size;
    int page = -1;
    if (t < p.total && pos >= 0 && pos < len && lp < p.max_pages) page = p.table[(long long)b * p.max_pages + lp];
    raw[i][0] = raw[i][1] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);  // zeros, below
    step[i][0] = step[i][1] = 0.f;
    if (page >= 0 && page < p.n_pages) {
      const long long head = (long long)page * p.Hkv + h;
      const int in = pos - lp * p.page_size;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint4 v = *reinterpret_cast<const uint4*>(p.cache[kv] + (head * p.page_size + in) * D + c * 16);
        raw[i][kv] = make_uint4(v.x ^ 0x80808080u, v.y ^ 0x80808080u, v.z ^ 0x80808080u, v.w ^ 0x80808080u);
        step[i][kv] = p.absmax[kv][head * p.blocks_per_page + (in >> p.block_bits)] * kStep;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t = t0 + i * PER;
    if (t >= p.total) break;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const unsigned u[4] = {raw[i][kv].x, raw[i][kv].y, raw[i][kv].z, raw[i][kv].w};
      unsigned o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v[4];
        word_to_floats(u[j], v);
        o[2 * j] = pack_pair<T>(v[0] * step[i][kv], v[1] * step[i][kv]);
        o[2 * j + 1] = pack_pair<T>(v[2] * step[i][kv], v[3] * step[i][kv]);
      }
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out[kv]) +
                                            (((long long)b * p.total + t) * p.Hkv + h) * D + c * 16);
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

// ------------------------------------------------------------------ attention
struct AttendParams {
  const void* q;  // [B, S, Hq, D]
  long long qb, qs, qh;
  const signed char* kc;
  const signed char* vc;
  const float* ka;
  const float* va;
  const int* table;
  const int* lens;
  const int* starts;  // null: lens - S
  void* out;          // [B, S, Hq, D] contiguous
  float* part_o;      // [2 * ctas][R][D]
  float* part_s;      // [2 * ctas][R][3]: running max of scores, of weights, sum
  int B, S, Hq, Hkv, G, groups, page_size, n_pages, max_pages, ctas;
  int tiles_per_page, blocks_per_page, block_shift;  // magnitudes per page and head; log2(block / kTile)
  int unit_tiles;     // tiles of a unit of work
  float scale;        // softmax scale * log2(e) / 127
};

constexpr int kWarps = 8;
constexpr int kTile = 16;                // tokens per warp step
constexpr int kUnit = kWarps * kTile;    // tokens per unit of work: one step of all warps
constexpr int kPad = 4;                  // units that a segment's start weighs when work is dealt out
constexpr int kMaxBatch = 1024;        // rows of a launch
// Running maxima start here: below every score, and finite, so that no difference of maxima is NaN.
constexpr float kNone = -1.7e38f;
// A running maximum follows the scores only when they pass it by this much (powers of two): most tiles then need no
// reduction over lanes and no rescaling.
constexpr float kSlack = 8.f;
// The weights' reference stays this far below their largest, which is then 2^kLift to 2^(kLift + kSlack) as fp16, half
// its range: a weight of 2^-32 of the largest still reaches its last place.
constexpr float kLift = 7.f;

__device__ __forceinline__ float2 lds_float2(unsigned a) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
  return v;
}
// four 8 x 8 matrices of 16-bit elements, each transposed
__device__ __forceinline__ uint4 ldmatrix4_trans(unsigned a) {
  uint4 v;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float* d, const unsigned* a, const unsigned* b) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Integers to fp16 pairs. With u = q + 128 a byte:
//  * under a zero high byte u is the subnormal fp16 number u 2^-24. Sums over the channels then carry
//    128 sum(query), no larger than the sums themselves, which is taken off afterwards (keys);
//  * under the high byte 0x64 it is 1024 + u, and taking 1152 away is exact (values: the weights of a long
//    context all have one sign, so an offset would grow far past the result).
// `sel` picks the two bytes of `u` that make the pair.
__device__ __forceinline__ unsigned bytes_to_subnormal2(unsigned u, unsigned sel) { return __byte_perm(u, 0u, sel); }
__device__ __forceinline__ unsigned bytes_to_half2(unsigned u, unsigned sel) {
  const unsigned m = __byte_perm(u, 0x64646464u, sel);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), __float2half2_rn(1152.f));
  return *reinterpret_cast<const unsigned*>(&r);
}

// Tokens that the queries of row b, of length len, see at most, and the position of its first query.
__device__ __forceinline__ void row_extent(const AttendParams& p, int b, int len, int& first, int& keys) {
  first = p.starts ? min(max(p.starts[b], -(1 << 30)), 1 << 30) : len - p.S;
  keys = max(0, min(min(len, first + p.S), p.max_pages * p.page_size));
}
// Units of row b in the dealing: those of its keys (a row without keys still has its zeros to write), behind
// kPad that stand for what starting and merging a piece costs.
__device__ __forceinline__ int row_units(const AttendParams& p, int b, int len) {
  int first, keys;
  row_extent(p, b, len, first, keys);
  const int tokens = p.unit_tiles * kTile;
  return kPad + max(1, (keys + tokens - 1) / tokens);
}
// CTAs that take part: each has a unit at least, so that the CTAs of a segment's keys are all those from
// its first unit's to its last unit's
__device__ __forceinline__ int live_ctas(const AttendParams& p, long long total) {
  return (int)min((long long)p.ctas, total);
}
// CTA that has unit u when `total` units are dealt out as [c * total / ctas, (c + 1) * total / ctas)
__device__ __forceinline__ int cta_of(long long u, long long total, int ctas) {
  return (int)(((u + 1) * ctas - 1) / total);
}

// A [16][D] tile of bytes in shared memory: the 16-byte chunks of a token are permuted so that the reads
// below (8 tokens, one chunk each, or 2 tokens, 4 chunks each) touch all banks once.
template <int D>
__device__ __forceinline__ int swizzle(int row, int chunk) {
  return D == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}

template <int C>
__device__ __forceinline__ void load_floats(const float* src, float* v) {
  if constexpr (C == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
  else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
}
// D / 32 channels of query row r of KV head h, scaled
template <typename T, int D>
__device__ __forceinline__ void store_out(const AttendParams& p, int b, int h, int r, int ch, const float* a, float by) {
  const int i = r / p.G;
  T* dst = static_cast<T*>(p.out) + (((long long)b * p.S + i) * p.Hq + h * p.G + (r - i * p.G)) * D + ch;
  T v[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) v[j] = from_float<T>(a[j] * by);
  if constexpr (D == 128) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
  else *reinterpret_cast<unsigned*>(dst) = *reinterpret_cast<const unsigned*>(v);
}

struct Piece {       // of a segment, on one CTA
  int b, h, grp;     // row, kv head, group
  int unit0, units;  // its first unit of keys and their number
  int dealt;         // units taken from the dealing, those that stand for the start among them
  int len, first, keys;  // of the row
  bool whole;
};

// Work: every (row b, kv head h, group g of R query rows) is a segment of ceil(keys / 128) units, and kPad
// more at its start; the units of all segments, in order, are dealt out evenly over the CTAs, whatever the
// rows' lengths. A CTA's warps take the 16-token tiles of its piece of a segment in turn, each with its own
// running softmax, and are merged once per piece. A piece that is a whole segment writes the output; others
// leave partials (two per CTA at most: one that it begins inside, one that it does not end) for
// kv8_combine_kernel.
//
// Softmax per query row: a reference m near the maximum of the scores s (within kSlack) and
// l = sum 2^(s - m). The weights of the integers v are 2^s * absmax_v; they have a reference M of their
// own, kLift below the maximum of s + log2 absmax_v (within kSlack), so as fp16 they keep their precision whatever
// the magnitudes of the blocks. out = sum w v / l * 2^(M - m) / 127.
//
// Bound by HBM on long rows (4 x 131072 tokens of 4 heads of 128: 94 us, 0.88 of the copy rate), by its start (1.7 us
// to the first copy), merge (2 us) and join (3 us) on short ones (32 x 4096: 31.9 us, 0.65). Two CTAs of 8 warps per
// SM: with 4 or 16 warps per CTA the long case took 114 or 96 us.
//
// A weight is held as two fp16 numbers, itself and what that leaves, 22 bits in all. Rounded once, the weights put
// errors of up to 3.3e-4 in norm into fp16 outputs, whose own rounding is 2.1e-4, and bfloat16 outputs differed by
// 6e-4 to 8e-4 from those of weights in fp32; as two numbers by less than 2e-4. TWIN: at most four query rows, each
// in two columns, one of which takes what the other's weights leave (32 x 4096 tokens: 32.3 us); otherwise a second
// product does (34.5 us for the same).
template <typename T, int D, int NT, int STAGES, bool TWIN>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 2 : 1) kv8_attend_kernel(const AttendParams p) {
  constexpr int KS = D / 16;     // k-steps of S^T = K Q^T
  constexpr int MT = D / 16;     // channel tiles of O^T = V^T P^T
  constexpr int R = 8 * NT;      // query rows of a group
  constexpr int TB = kTile * D;  // bytes of a tile
  constexpr int SLOT = 2 * TB;   // a ring slot: a tile of keys, then one of values
  constexpr int AHEAD = STAGES - NT;  // tiles that the copies run ahead: the other NT slots are for merges
  extern __shared__ __align__(128) unsigned char smem[];  // [stage][warp][SLOT]
  __shared__ int prefix[kMaxBatch + 1];
  __shared__ int len_s[kMaxBatch];
  __shared__ int scan_s[kWarps];
  __shared__ float stat_s[kWarps][R][3];
  __shared__ float2 mag_s[kWarps][STAGES];  // magnitudes of k and v of the tiles in the ring
  // This grid may have been scheduled before the one before it ended. The combine may be scheduled from
  // here on: what it reads before its own wait is then complete.
  begin_early();

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const unsigned ring = (unsigned)__cvta_generic_to_shared(smem) + warp * SLOT;
  const unsigned mags = (unsigned)__cvta_generic_to_shared(&mag_s[warp][0]);

  // units of the rows before each row
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += kWarps * 32) {
    const int b = b0 + tid;
    int v = 0;
    if (b < p.B) {
      len_s[b] = max(p.lens[b], 0);
      v = row_units(p, b, len_s[b]);
    }
    const int own = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffff, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) scan_s[warp] = v;
    __syncthreads();
    int sum = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      sum += i < warp ? scan_s[i] : 0;
      all += scan_s[i];
    }
    if (b < p.B) prefix[b] = before + sum + v - own;
    before += all;
    __syncthreads();
  }
  if (tid == 0) prefix[p.B] = before;
  __syncthreads();
  const int per = p.Hkv * p.groups;  // segments per row
  const long long total = (long long)before * per;
  const int ctas = live_ctas(p, total);
  if ((int)blockIdx.x >= ctas) return;
  const long long u_begin = total * blockIdx.x / ctas, u_end = total * (blockIdx.x + 1) / ctas;

  // this lane's places in a tile: 16 bytes copied per step of 32 chunks; keys: token g, channels
  // t * D / 4 ..; values: token lane & 15 of the matrices of chunks lane >> 4, ..
  const unsigned put0 = swizzle<D>(lane / (D / 16), lane % (D / 16));
  const unsigned put1 = swizzle<D>(lane / (D / 16) + 512 / D, lane % (D / 16));
  const unsigned key_at = swizzle<D>(g, t * (D / 64)), value_at = TB + swizzle<D>(lane & 15, lane >> 4);

  auto find = [&](long long u) {
    int lo = 0, hi = p.B - 1;  // the row of unit u: last b with prefix[b] * per <= u
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if ((long long)prefix[mid] * per <= u) lo = mid;
      else hi = mid - 1;
    }
    Piece c;
    c.b = lo;
    const int all = prefix[lo + 1] - prefix[lo];
    const int rem = (int)(u - (long long)prefix[lo] * per);
    const int hg = rem / all, at = rem - hg * all;
    c.dealt = (int)min((long long)(all - at), u_end - u);
    c.unit0 = max(0, at - kPad);
    c.units = max(0, at + c.dealt - kPad) - c.unit0;
    c.whole = c.units == all - kPad;
    c.h = hg / p.groups, c.grp = hg - c.h * p.groups;
    c.len = len_s[lo];
    row_extent(p, lo, c.len, c.first, c.keys);
    return c;
  };

  // A warp's tiles of a piece: first0, first0 + 8, ..., `count` of them. Lane i knows the page and the tile
  // in it of the i-th of every 32.
  int first0, count, ahead, my_page, my_tip;
  unsigned have;  // bit i: the i-th tile from the current one has a page
  const int* trow;
  auto look_up = [&]() {
    const int i = ahead + lane, tile = first0 + i * kWarps, lp = tile / p.tiles_per_page;
    my_tip = tile - lp * p.tiles_per_page;
    my_page = i < count ? trow[lp] : -1;
    if (my_page >= p.n_pages) my_page = -1;
  };
  auto issue = [&](int stage, unsigned bit, int h) {  // copies of the next tile
    if ((ahead & 31) == 0 && ahead > 0 && ahead < count) look_up();
    const int page = __shfl_sync(0xffffffff, my_page, ahead & 31), tip = __shfl_sync(0xffffffff, my_tip, ahead & 31);
    if (ahead < count && page >= 0) {
      have |= bit;
      const long long head = (long long)page * p.Hkv + h;
      const long long at = (head * p.page_size + tip * kTile) * D + lane * 16;
      const unsigned dst = ring + stage * kWarps * SLOT;
#pragma unroll
      for (int j = 0; j < TB / 512; ++j) {
        const unsigned to = dst + (j & 1 ? put1 : put0) + (j >> 1) * 1024;
        cp_async16(to, p.kc + at + j * 512);
        cp_async16(to + TB, p.vc + at + j * 512);
      }
      const long long blk = head * p.blocks_per_page + (tip >> p.block_shift);
      if (lane < 2) cp_async4(mags + stage * 8 + lane * 4, (lane ? p.va : p.ka) + blk);
    }
    cp_async_commit();
    ++ahead;
  };
  // lane (g, t): channels t * D / 4 .. of query row g of each 8-row tile
  uint4 q_raw[NT][D / 32];
  auto begin = [&](const Piece& c) {  // loads that the piece starts with
    const int tile_end = min((c.unit0 + c.units) * p.unit_tiles, (c.keys + kTile - 1) / kTile);
    first0 = c.unit0 * p.unit_tiles + warp;
    count = first0 < tile_end ? (tile_end - first0 + kWarps - 1) / kWarps : 0;
    trow = p.table + (long long)c.b * p.max_pages;
    ahead = 0, have = 0;
    look_up();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = TWIN ? g & 3 : c.grp * R + n * 8 + g, i = r / p.G;
      const T* src = static_cast<const T*>(p.q) + (long long)c.b * p.qb + (long long)i * p.qs +
                     (long long)(c.h * p.G + (r - i * p.G)) * p.qh + t * (D / 4);
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
        q_raw[n][j] = r < p.S * p.G ? reinterpret_cast<const uint4*>(src)[j] : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) issue(i, 1u << i, c.h);
  };

  long long u = u_begin;
  Piece c = find(u);
  if (c.units == 0) {  // the range begins with a segment's start alone: the keys after it are another CTA's
    u += c.dealt;
    if (u >= u_end) return;
    c = find(u);
  }
  begin(c);
  for (;;) {
    // query fragments: fp16 scaled by a power of two that brings the row's largest magnitude to [2^14, 2^15)
    unsigned qf[NT][KS][2];
    float qscale[NT][2], qbias[NT][2];  // of the columns 2t, 2t + 1 of S^T
    int vis[NT][2];                     // keys that those columns see
    int seen_by_all = c.keys;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const unsigned short* e = reinterpret_cast<const unsigned short*>(q_raw[n]);
      unsigned bits = 0;  // magnitudes compare as integers
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
        bits = __vmaxu2(bits, __vmaxu2(__vmaxu2(q_raw[n][j].x & 0x7fff7fffu, q_raw[n][j].y & 0x7fff7fffu),
                                       __vmaxu2(q_raw[n][j].z & 0x7fff7fffu, q_raw[n][j].w & 0x7fff7fffu)));
      bits = max(bits & 0xffffu, bits >> 16);
      bits = max(bits, __shfl_xor_sync(0xffffffff, bits, 1));
      bits = max(bits, __shfl_xor_sync(0xffffffff, bits, 2));
      // the magnitude's exponent, as that of an fp32 number; subnormals and what is not finite scale by 2^14
      const int fe = (int)(__float_as_uint(bits_to_float<T>((unsigned short)bits)) >> 23);
      const int ex = fe == 0 || fe == 255 ? 0 : max(fe - 127, -100);
      const float down = __int_as_float((127 + 14 - ex) << 23);
      const float up = p.scale * __int_as_float((127 - 14 + max(ex, -100)) << 23);
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const __half2 v = __floats2half2_rn(bits_to_float<T>(e[4 * s + 2 * k]) * down,
                                              bits_to_float<T>(e[4 * s + 2 * k + 1]) * down);
          qf[n][s][k] = *reinterpret_cast<const unsigned*>(&v);
          sum += __low2float(v) + __high2float(v);
        }
      sum += __shfl_xor_sync(0xffffffff, sum, 1);
      sum += __shfl_xor_sync(0xffffffff, sum, 2);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        qscale[n][k] = __shfl_sync(0xffffffff, up, (2 * t + k) * 4);
        qbias[n][k] = -128.f * qscale[n][k] * __shfl_sync(0xffffffff, sum, (2 * t + k) * 4);
        qscale[n][k] *= 0x1p24f;
        const int rc = TWIN ? (2 * t + k) & 3 : c.grp * R + n * 8 + 2 * t + k, pos = c.first + rc / p.G;
        // columns behind the last query row are computed like the others and never written
        vis[n][k] = rc >= p.S * p.G ? c.keys : pos >= 0 && pos < c.len ? min(pos + 1, c.keys) : 0;
        seen_by_all = min(seen_by_all, vis[n][k]);
      }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) seen_by_all = min(seen_by_all, __shfl_xor_sync(0xffffffff, seen_by_all, d));

    float o[NT][MT][4], m[NT][2], M[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < 2; ++k) m[n][k] = M[n][k] = kNone, l[n][k] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[n][i][k] = 0.f;
    }

    int stage = 0, refill = AHEAD, tok = first0 * kTile;
    for (int it = 0; it < count; ++it, tok += kUnit) {
      cp_async_wait<AHEAD - 1>();
      __syncwarp();  // this tile has landed for all lanes, and all have left the stage that is refilled now
      const bool held = have & 1u;
      have >>= 1;
      issue(refill, 1u << (AHEAD - 1), c.h);
      refill = refill + 1 == STAGES ? 0 : refill + 1;
      const unsigned tile = ring + stage * kWarps * SLOT;
      const float2 mag = lds_float2(mags + stage * 8);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      if (!held) continue;  // the same for the whole warp

      // S^T: tokens g and g + 8, channels t * D / 4 + 4s .. of k-step s on both sides
      float sc[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        const uint4 x = lds128(tile + (key_at ^ (j << 4))), y = lds128(tile + (key_at ^ (j << 4)) + 8 * D);
        const unsigned xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned ux = xs[k] ^ 0x80808080u, uy = ys[k] ^ 0x80808080u;
          const unsigned a[4] = {bytes_to_subnormal2(ux, 0x4140), bytes_to_subnormal2(uy, 0x4140),
                                 bytes_to_subnormal2(ux, 0x4342), bytes_to_subnormal2(uy, 0x4342)};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816(sc[n], a, qf[n][j * 4 + k]);
        }
      }

      const float lv = __log2f(mag.y);
      bool rises = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float a = qscale[n][k] * mag.x, c0 = qbias[n][k] * mag.x;
          sc[n][k] = fmaf(sc[n][k], a, c0);
          sc[n][2 + k] = fmaf(sc[n][2 + k], a, c0);
        }
        if (tok + kTile > seen_by_all) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (tok + g >= vis[n][k]) sc[n][k] = -INFINITY;
            if (tok + g + 8 >= vis[n][k]) sc[n][2 + k] = -INFINITY;
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float top = fmaxf(sc[n][k], sc[n][2 + k]);
          rises = rises || top > m[n][k] + kSlack || top + lv > M[n][k] + (kSlack + kLift);
        }
      }
      if (__any_sync(0xffffffff, rises)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float fall[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float top = fmaxf(sc[n][k], sc[n][2 + k]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffff, top, d));
            const float m1 = fmaxf(m[n][k], top), M1 = fmaxf(M[n][k], top + lv - kLift);
            l[n][k] *= ex2(m[n][k] - m1);
            fall[k] = ex2(M[n][k] - M1);
            m[n][k] = m1;
            M[n][k] = M1;
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[n][i][0] *= fall[0], o[n][i][1] *= fall[1];
            o[n][i][2] *= fall[0], o[n][i][3] *= fall[1];
          }
        }
      }
      // weights as fp16, and what that leaves of them
      unsigned pf[NT][2], pr[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          l[n][k] += ex2(sc[n][k] - m[n][k]) + ex2(sc[n][2 + k] - m[n][k]);
          const float to = lv - M[n][k];
          // a hidden key has weight 0 whatever its block's magnitude is
          w[k] = sc[n][k] == -INFINITY ? 0.f : ex2(sc[n][k] + to);
          w[2 + k] = sc[n][2 + k] == -INFINITY ? 0.f : ex2(sc[n][2 + k] + to);
        }
        __half2 w0 = __floats2half2_rn(w[0], w[1]), w1 = __floats2half2_rn(w[2], w[3]);
        const float2 f0 = __half22float2(w0), f1 = __half22float2(w1);
        const __half2 r0 = __floats2half2_rn(w[0] - f0.x, w[1] - f0.y), r1 = __floats2half2_rn(w[2] - f1.x, w[3] - f1.y);
        if (TWIN) {
          w0 = t < 2 ? w0 : r0, w1 = t < 2 ? w1 : r1;
        } else {
          pr[n][0] = transpose8x8(*reinterpret_cast<const unsigned*>(&r0));
          pr[n][1] = transpose8x8(*reinterpret_cast<const unsigned*>(&r1));
        }
        pf[n][0] = transpose8x8(*reinterpret_cast<const unsigned*>(&w0));
        pf[n][1] = transpose8x8(*reinterpret_cast<const unsigned*>(&w1));
      }

      // O^T: a transposed matrix of 8 tokens and 16 channels, read as 16-bit pairs of channels, gives lane
      // (g, t) channels 2g and 2g + 1 of tokens 2t and 2t + 1; channel tile i has channel 16 i + 2g in its row
      // g and channel 16 i + 2g + 1 in row g + 8
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint4 x = ldmatrix4_trans(tile + (value_at ^ (j << 5)));
        const unsigned xs[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned a[4] = {bytes_to_half2(xs[2 * e], 0x4240), bytes_to_half2(xs[2 * e], 0x4341),
                                 bytes_to_half2(xs[2 * e + 1], 0x4240), bytes_to_half2(xs[2 * e + 1], 0x4341)};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816(o[n][j * 2 + e], a, pf[n]);
            if (!TWIN) mma16816(o[n][j * 2 + e], a, pr[n]);
          }
        }
      }
    }
    cp_async_wait<0>();
    __syncwarp();

    // The next piece's first copies fly while this one is merged: they fill the first AHEAD slots, and the
    // last NT hold what the warps merge.
    const Piece done = c;
    const long long slot = 2LL * blockIdx.x + (done.unit0 > 0 ? 0 : 1);
    u += done.dealt;
    bool more = u < u_end;
    if (more) {
      c = find(u);
      more = c.units > 0;  // else the range ends with a segment's start alone
      if (more) begin(c);
    }

    // [R][D] floats of warp w, 8 rows per ring slot; the channels of a row are permuted by 16 so that the
    // four rows that a warp writes at a time lie on different banks
    auto merge_at = [&](int w, int row, int ch) {
      return reinterpret_cast<float*>(smem + ((STAGES - NT + row / 8) * kWarps + w) * SLOT) + row % 8 * D +
             (ch ^ ((row >> 1 & 3) << 4));
    };
    const int rows = min(R, p.S * p.G - done.grp * R);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float s = l[n][k];  // sums over the tokens of a warp lie on lanes of equal t
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) s += __shfl_xor_sync(0xffffffff, s, d);
        const int row = n * 8 + 2 * t + k;
        if ((TWIN ? row & 3 : row) < rows) {
          if (g == 0) stat_s[warp][row][0] = m[n][k], stat_s[warp][row][1] = M[n][k], stat_s[warp][row][2] = s;
#pragma unroll
          for (int i = 0; i < MT; ++i)
            *reinterpret_cast<float2*>(merge_at(warp, row, 16 * i + 2 * g)) = make_float2(o[n][i][k], o[n][i][2 + k]);
        }
      }
    __syncthreads();
    for (int row = warp; row < rows; row += kWarps) {  // a warp per row, a lane D / 32 channels
      constexpr int C = D / 32;
      const float* st = stat_s[lane & 7][row];
      float mm = st[0], MM = st[1];
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) {
        mm = fmaxf(mm, __shfl_xor_sync(0xffffffff, mm, d));
        MM = fmaxf(MM, __shfl_xor_sync(0xffffffff, MM, d));
      }
      const float f = ex2(st[1] - MM);
      float sum = st[2] * ex2(st[0] - mm);
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) sum += __shfl_xor_sync(0xffffffff, sum, d);
      float a[C];
#pragma unroll
      for (int j = 0; j < C; ++j) a[j] = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        float v[C];
        load_floats<C>(merge_at(i, row, lane * C), v);
        if (TWIN) {
          float rest[C];
          load_floats<C>(merge_at(i, row + 4, lane * C), rest);
#pragma unroll
          for (int j = 0; j < C; ++j) v[j] += rest[j];
        }
        const float fi = __shfl_sync(0xffffffff, f, i);
#pragma unroll
        for (int j = 0; j < C; ++j) a[j] += v[j] * fi;
      }
      if (done.whole) {
        const float to = sum == 0.f ? 0.f : exp2f(MM - mm) * kStep / sum;  // no key seen: zeros
        store_out<T, D>(p, done.b, done.h, done.grp * R + row, lane * C, a, to);
      } else {
        float* to = p.part_o + (slot * R + row) * D + lane * C;
        if constexpr (C == 4) *reinterpret_cast<float4*>(to) = make_float4(a[0], a[1], a[2], a[3]);
        else *reinterpret_cast<float2*>(to) = make_float2(a[0], a[1]);
        if (lane == 0) {
          float* ps = p.part_s + (slot * R + row) * 3;
          ps[0] = mm, ps[1] = MM, ps[2] = sum;
        }
      }
    }
    if (!more) return;
    __syncthreads();  // what was merged may be overwritten
  }
}

// Joins the pieces of a segment that several CTAs worked on: one CTA per (segment, query row). Its warps
// take the pieces in turn, a lane D / 32 channels, and are merged at the end.
template <typename T, int D, int R, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) kv8_combine_kernel(const AttendParams p, int rows) {
  constexpr int C = D / 32, N = 8;  // pieces of a warp whose loads are in flight together
  __shared__ int sums[2][WARPS];
  __shared__ float stat_s[WARPS][3], o_s[WARPS][D];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int seg = blockIdx.x / rows, row = blockIdx.x - seg * rows;
  const int per = p.Hkv * p.groups, b = seg / per, hg = seg - b * per;
  const int h = hg / p.groups, grp = hg - h * p.groups, r = grp * R + row;
  int pre = 0, all = 0;
  for (int i = tid; i < p.B; i += 32 * WARPS) {
    const int v = row_units(p, i, max(p.lens[i], 0));
    all += v;
    pre += i < b ? v : 0;
  }
  all = __reduce_add_sync(0xffffffff, all);
  pre = __reduce_add_sync(0xffffffff, pre);
  if (lane == 0) sums[0][warp] = all, sums[1][warp] = pre;
  const int units = row_units(p, b, max(p.lens[b], 0));
  __syncthreads();
  all = pre = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) all += sums[0][i], pre += sums[1][i];
  const long long total = (long long)all * per;
  const long long u1 = (long long)pre * per + (long long)(hg + 1) * units, u0 = u1 - units + kPad;  // of the keys
  const int ctas = live_ctas(p, total);
  const int c0 = cta_of(u0, total, ctas), c1 = cta_of(u1 - 1, total, ctas);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // up to here only lengths were read
  if (c0 == c1 || r >= p.S * p.G) return;  // one CTA had it all and wrote the output
  float m = kNone, M = kNone, sum = 0.f, a[C];
#pragma unroll
  for (int i = 0; i < C; ++i) a[i] = 0.f;
  for (int c = c0 + warp; c <= c1; c += N * WARPS) {
    float st[N][3], v[N][C];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int ck = c + k * WARPS;
      st[k][0] = st[k][1] = kNone, st[k][2] = 0.f;
#pragma unroll
      for (int i = 0; i < C; ++i) v[k][i] = 0.f;
      if (ck > c1) continue;
      const long long slot = 2LL * ck + (ck == c0);  // the first of the CTAs does not begin inside the keys
      const float* s = p.part_s + (slot * R + row) * 3;
      st[k][0] = s[0], st[k][1] = s[1], st[k][2] = s[2];
      load_floats<C>(p.part_o + (slot * R + row) * D + lane * C, v[k]);
    }
    float m1 = m, M1 = M;
#pragma unroll
    for (int k = 0; k < N; ++k) m1 = fmaxf(m1, st[k][0]), M1 = fmaxf(M1, st[k][1]);
    const float f = ex2(M - M1);
    sum *= ex2(m - m1);
#pragma unroll
    for (int i = 0; i < C; ++i) a[i] *= f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float e = ex2(st[k][1] - M1);
      sum += st[k][2] * ex2(st[k][0] - m1);
#pragma unroll
      for (int i = 0; i < C; ++i) a[i] += v[k][i] * e;
    }
    m = m1, M = M1;
  }
  if (lane == 0) stat_s[warp][0] = m, stat_s[warp][1] = M, stat_s[warp][2] = sum;
#pragma unroll
  for (int i = 0; i < C; ++i) o_s[warp][lane * C + i] = a[i];
  __syncthreads();
  if (tid >= D) return;
  float mm = kNone, MM = kNone, l = 0.f, o = 0.f;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) mm = fmaxf(mm, stat_s[i][0]), MM = fmaxf(MM, stat_s[i][1]);
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    l += stat_s[i][2] * ex2(stat_s[i][0] - mm);
    o += o_s[i][tid] * ex2(stat_s[i][1] - MM);
  }
  const float f = l == 0.f ? 0.f : exp2f(MM - mm) * kStep / l;
  const int i = r / p.G;
  static_cast<T*>(p.out)[(((long long)b * p.S + i) * p.Hq + h * p.G + (r - i * p.G)) * D + tid] = from_float<T>(o * f);
}

constexpr int stages_for(int NT) { return NT == 1 ? 3 : 6; }

template <typename T, int D, int NT, bool TWIN>
void launch_attend(const AttendParams& p, bool combine, cudaStream_t s) {
  constexpr int smem = kWarps * stages_for(NT) * 2 * kTile * D;
  auto kernel = kv8_attend_kernel<T, D, NT, stages_for(NT), TWIN>;
  static bool set[64] = {};  // the attribute belongs to the device that is current
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev]) {
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (dev >= 0 && dev < 64) set[dev] = true;
  }
  launch_early(kernel, dim3(p.ctas), dim3(kWarps * 32), smem, s, p);
  if (!combine) return;
  const int rows = std::min(8 * NT, p.S * p.G), segs = p.B * p.Hkv * p.groups;
  // warps for the pieces that a segment has on average: with 3 pieces 4 warps take 2 us less than 8, with 64
  // pieces 1 us more
  if (p.ctas < 12 * segs) launch_early(kv8_combine_kernel<T, D, 8 * NT, 4>, dim3(segs * rows), dim3(128), 0, s, p, rows);
  else launch_early(kv8_combine_kernel<T, D, 8 * NT, 8>, dim3(segs * rows), dim3(256), 0, s, p, rows);
}

}  // namespace
}  // namespace astrai

namespace astrai_host {

bool kv8_block_supported(int block) { return block == 16 || block == 32 || block == 64 || block == 128; }

void kv8_append(const void* k, const long long* ks, const void* v, const long long* vs, void* kc, void* vc, float* ka,
                float* va, const int* table, const int* starts, const int* lens, int B, int S, int Hkv, int D,
                int page_size, int n_pages, int max_pages, int block, int dtype, cudaStream_t s) {
  using namespace astrai;
  if (B <= 0 || S <= 0) return;
  AppendParams p{};
  p.src[0] = k, p.src[1] = v;
  p.sb[0] = ks[0], p.st[0] = ks[1], p.sh[0] = ks[2];
  p.sb[1] = vs[0], p.st[1] = vs[1], p.sh[1] = vs[2];
  p.cache[0] = static_cast<signed char*>(kc), p.cache[1] = static_cast<signed char*>(vc);
  p.absmax[0] = ka, p.absmax[1] = va;
  p.table = table, p.starts = starts, p.lens = lens;
  p.B = B, p.S = S, p.Hkv = Hkv, p.page_size = page_size, p.n_pages = n_pages, p.max_pages = max_pages;
  p.windows = (S - 1 + block - 1) / block + 1;  // blocks that S tokens from any offset can touch
  const long long items = 2LL * B * Hkv * p.windows;
  const int per_cta = block > 32 ? 4 / (block / 32) : 4;
  const int blocks = (int)((items + per_cta - 1) / per_cta);
#define ASTRAI_APPEND(T, D_)                                                                     \
  switch (block) {                                                                               \
    case 16: launch_early(kv8_append_kernel<T, D_, 16>, dim3(blocks), dim3(128), 0, s, p); break; \
    case 32: launch_early(kv8_append_kernel<T, D_, 32>, dim3(blocks), dim3(128), 0, s, p); break; \
    case 64: launch_early(kv8_append_kernel<T, D_, 64>, dim3(blocks), dim3(128), 0, s, p); break; \
    default: launch_early(kv8_append_kernel<T, D_, 128>, dim3(blocks), dim3(128), 0, s, p); break; \
  }
  if (dtype == 0 && D == 128) { ASTRAI_APPEND(__nv_bfloat16, 128) }
  else if (dtype == 0) { ASTRAI_APPEND(__nv_bfloat16, 64) }
  else if (D == 128) { ASTRAI_APPEND(__half, 128) }
  else { ASTRAI_APPEND(__half, 64) }
#undef ASTRAI_APPEND
}

void kv8_gather(const void* kc, const void* vc, const float* ka, const float* va, const int* table, const int* starts,
                const int* lens, void* ko, void* vo, int B, int total, int Hkv, int D, int page_size, int n_pages,
                int max_pages, int block, int dtype, cudaStream_t s) {
  using namespace astrai;
  GatherParams p{};
  p.cache[0] = static_cast<const signed char*>(kc), p.cache[1] = static_cast<const signed char*>(vc);
  p.absmax[0] = ka, p.absmax[1] = va, p.table = table, p.starts = starts, p.lens = lens;
  p.out[0] = ko, p.out[1] = vo;
  p.B = B, p.total = total, p.Hkv = Hkv, p.page_size = page_size, p.n_pages = n_pages, p.max_pages = max_pages;
  p.blocks_per_page = page_size / block;
  while ((1 << p.block_bits) < block) ++p.block_bits;
  if (B <= 0 || total <= 0) return;
  const dim3 grid((total + kGatherTokens - 1) / kGatherTokens, Hkv, B);
  if (dtype == 0 && D == 128) launch_early(kv8_gather_kernel<__nv_bfloat16, 128>, grid, dim3(256), 0, s, p);
  else if (dtype == 0) launch_early(kv8_gather_kernel<__nv_bfloat16, 64>, grid, dim3(256), 0, s, p);
  else if (D == 128) launch_early(kv8_gather_kernel<__half, 128>, grid, dim3(256), 0, s, p);
  else launch_early(kv8_gather_kernel<__half, 64>, grid, dim3(256), 0, s, p);
}

namespace {

// Launch shape of an attention call, from sizes the host knows: the lengths are on the device, so a row counts
// as the tokens that its pages hold.
struct AttendPlan {
  int R, groups;       // query rows per group, groups
  int ctas, unit;      // CTAs, tokens per unit of work
  bool split;          // whether a segment can be split over CTAs
  long long floats;    // workspace
};

// Splitting rows over CTAs evens the work out but costs the join, a second piece for many CTAs and, with
// that, about kJoinUs; whole rows cost the idle slots of the last wave and, if they are few, the rate that one
// CTA reaches alone. Both sides are estimated from rates measured on B200 (cache bytes: 6 TB/s in all, 36 GB/s
// for one CTA): at 64 rows of 1024 tokens of 4 heads of 128 whole rows take 18.8 us and split ones 24.6, at 4 rows of
// 1000 11.7 and 9.0. The estimate is of full tables: 32 rows of 500 tokens in tables of 4096 are split (13.1 us, whole
// 8.5), and 64 rows of 1 to 8192 tokens, most of them short, in tables of 8192 are whole (69 us, split 25).
constexpr double kAllRate = 6e6, kOneRate = 3.6e4, kJoinUs = 3.3;  // bytes per us

AttendPlan attend_plan(int B, int S, int Hq, int Hkv, int D, int page_size, int max_pages, int sms) {
  using namespace astrai;
  AttendPlan a{};
  const long long cap = (long long)max_pages * page_size;
  const int rows = S * (Hq / Hkv);
  a.R = rows <= 8 ? 8 : 16;
  a.groups = (rows + a.R - 1) / a.R;
  const long long segs = (long long)B * Hkv * a.groups, slots = (long long)sms * (a.R == 8 ? 2 : 1);
  const long long units = (cap + kUnit - 1) / kUnit;
  const double bytes = 2.0 * D * (double)cap;
  const auto rate = [&](double busy) { return std::min(kOneRate, kAllRate / busy); };
  const double at_once = (double)std::min(segs, slots), waves = (double)((segs + slots - 1) / slots);
  const double whole = waves * bytes / rate(at_once);
  const double spread = (double)std::min(segs * units, slots);
  const double parts = (double)segs * bytes / (spread * rate(spread)) + kJoinUs;
  a.split = units > 1 && parts < whole;
  a.unit = (int)(a.split ? kUnit : std::max<long long>(1, units) * kUnit);
  a.ctas = (int)std::min(a.split ? segs * (units + kPad) : segs, slots);
  a.floats = a.split ? 2LL * a.ctas * a.R * (D + 3) : 0;
  return a;
}

}  // namespace

// fp32 elements of workspace that kv8_attend needs (0: none)
long long kv8_attend_workspace(int B, int S, int Hq, int Hkv, int D, int page_size, int max_pages, int device) {
  // rows beyond the batch of one launch come in launches of their own, one after the other
  return attend_plan(std::min(B, astrai::kMaxBatch), S, Hq, Hkv, D, page_size, max_pages, num_sms(device)).floats;
}

void kv8_attend(const void* q, const long long* qs, const void* kc, const void* vc, const float* ka, const float* va,
                const int* table, const int* lens, const int* starts, void* out, float* workspace, int B, int S,
                int Hq, int Hkv, int D, int page_size, int n_pages, int max_pages, int block, float scale, int dtype,
                int device, cudaStream_t s) {
  using namespace astrai;
  if (B <= 0 || S <= 0) return;
  for (int b0 = 0; b0 < B; b0 += kMaxBatch) {
    const int n = std::min(B - b0, kMaxBatch);
    // the workspace was sized for the first launch; a later, smaller one keeps its shape
    const AttendPlan a = attend_plan(std::min(B, kMaxBatch), S, Hq, Hkv, D, page_size, max_pages, num_sms(device));
    AttendParams p{};
    p.q = static_cast<const char*>(q) + 2LL * b0 * qs[0];
    p.qb = qs[0], p.qs = qs[1], p.qh = qs[2];
    p.kc = static_cast<const signed char*>(kc), p.vc = static_cast<const signed char*>(vc), p.ka = ka, p.va = va;
    p.table = table + (long long)b0 * max_pages, p.lens = lens + b0, p.starts = starts ? starts + b0 : nullptr;
    p.out = static_cast<char*>(out) + 2LL * b0 * S * Hq * D;
    p.B = n, p.S = S, p.Hq = Hq, p.Hkv = Hkv, p.G = Hq / Hkv, p.groups = a.groups;
    p.page_size = page_size, p.n_pages = n_pages, p.max_pages = max_pages;
    p.tiles_per_page = page_size / kTile;
    p.blocks_per_page = page_size / block;
    p.unit_tiles = a.unit / kTile;
    while ((kTile << p.block_shift) < block) ++p.block_shift;
    p.ctas = a.ctas, p.scale = scale * 1.4426950408889634f * kStep;
    p.part_o = workspace;
    p.part_s = workspace ? workspace + 2LL * p.ctas * a.R * D : nullptr;
#define ASTRAI_ATTEND(T, D_) \
  if (a.R == 16) launch_attend<T, D_, 2, false>(p, a.split, s); \
  else if (S * p.G > 4) launch_attend<T, D_, 1, false>(p, a.split, s); \
  else launch_attend<T, D_, 1, true>(p, a.split, s);
    if (dtype == 0 && D == 128) { ASTRAI_ATTEND(__nv_bfloat16, 128) }
    else if (dtype == 0) { ASTRAI_ATTEND(__nv_bfloat16, 64) }
    else if (D == 128) { ASTRAI_ATTEND(__half, 128) }
    else { ASTRAI_ATTEND(__half, 64) }
#undef ASTRAI_ATTEND
  }
}

}  // namespace astrai_host
