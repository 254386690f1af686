// Rows of logits as 16-byte vectors: what the kernels over [rows, vocab] share.
//
// A row may start at any element. Its vectors lie on the 16-byte grid of memory: vector i holds the row's elements
// i * E - head .. i * E - head + E - 1 (E elements in 16 bytes, head the elements between the grid and the row's start),
// so that every vector but the first and the last is one aligned access; those two are read and written by element.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace astrai {

template <typename T>
struct LogitType;
template <>
struct LogitType<__nv_bfloat16> {
  static constexpr int E = 8;
  static constexpr uint32_t kNegInf = 0xFF80u;
  __device__ static float one(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
  __device__ static float2 pair(uint32_t u) { return unpack_bf16(u); }
  __device__ static uint32_t pack(float a, float b) { return pack_bf16(a, b); }
};
template <>
struct LogitType<__half> {
  static constexpr int E = 8;
  static constexpr uint32_t kNegInf = 0xFC00u;
  __device__ static float one(__half v) { return __half2float(v); }
  __device__ static __half round(float v) { return __float2half_rn(v); }
  __device__ static float2 pair(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  __device__ static uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct LogitType<float> {
  static constexpr int E = 4;
  static constexpr uint32_t kNegInf = 0xFF800000u;
  __device__ static float one(float v) { return v; }
  __device__ static float round(float v) { return v; }
};

// The E elements of a vector as floats.
template <typename T>
__device__ __forceinline__ void vec_floats(const uint4& u, float (&f)[LogitType<T>::E]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (LogitType<T>::E == 4) {
      f[j] = __uint_as_float(w[j]);
    } else {
      const float2 p = LogitType<T>::pair(w[j]);
      f[2 * j] = p.x;
      f[2 * j + 1] = p.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 vec_round(const float (&f)[LogitType<T>::E]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (LogitType<T>::E == 4)
      w[j] = __float_as_uint(f[j]);
    else
      w[j] = LogitType<T>::pack(f[2 * j], f[2 * j + 1]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
__device__ __forceinline__ uint4 vec_neg_inf() {
  const uint32_t w = LogitType<T>::E == 4 ? LogitType<T>::kNegInf : LogitType<T>::kNegInf * 0x10001u;
  return make_uint4(w, w, w, w);
}

// Largest element, a NaN only if there is nothing else.
template <typename T>
__device__ __forceinline__ float vec_max_number(const uint4& u) {
  if constexpr (LogitType<T>::E == 4) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
  }
}

// The vectors of one row.
template <typename T>
struct RowVecs {
  static constexpr int E = LogitType<T>::E;
  const T* row;
  int V, head, n;  // elements, elements before the row on the 16-byte grid, vectors
  __device__ RowVecs(const T* x, int vocab) : row(x), V(vocab) {
    head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    n = (V + head + E - 1) / E;
  }
  __device__ int first(int vec) const { return vec * E - head; }  // its first element (negative: before the row)
  __device__ bool whole(int vec) const { return first(vec) >= 0 && first(vec) + E <= V; }
  // Elements outside the row read as -inf.
  __device__ uint4 load(int vec) const {
    const int at = first(vec);
    if (at >= 0 && at + E <= V) return __ldg(reinterpret_cast<const uint4*>(row + at));
    return load_edge(at);
  }
  // This lane's vectors at + lane, at + 32 + lane, .., of which the warp has `rows` and this lane `mine` before its part ends
  // (-inf from there). Away from the row's ends they are N loads without a branch.
  template <int N>
  __device__ __forceinline__ void load(int at, int rows, int mine, uint4 (&u)[N]) const {
    const int lane = threadIdx.x & 31;
    if (at > 0 && N <= rows && at + N * 32 < n) {
      const uint4* const from = reinterpret_cast<const uint4*>(row - head) + at + lane;
#pragma unroll
      for (int j = 0; j < N; ++j) u[j] = __ldg(from + j * 32);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) u[j] = j < mine ? load(at + j * 32 + lane) : vec_neg_inf<T>();
    }
  }
  __device__ __noinline__ uint4 load_edge(int at) const {
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = at + e >= 0 && at + e < V ? LogitType<T>::one(row[at + e]) : -INFINITY;
    return vec_round<T>(f);
  }
  // `out` is a row with the same head.
  __device__ void store(T* out, int vec, const uint4& u) const {
    const int at = first(vec);
    if (at >= 0 && at + E <= V) {
      *reinterpret_cast<uint4*>(out + at) = u;
    } else {
      float f[E];
      vec_floats<T>(u, f);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at + e >= 0 && at + e < V) out[at + e] = LogitType<T>::round(f[e]);
    }
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in one register pair: one instruction works on both.
struct Pair {
  unsigned long long v;
  Pair() = default;
  __device__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ explicit Pair(float2 f) : Pair(f.x, f.y) {}
  __device__ float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
  __device__ float sum() const {
    const float2 f = get();
    return f.x + f.y;
  }
};
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair exp2_fast(Pair p) {
  const float2 f = p.get();
  return Pair(exp2_fast(f.x), exp2_fast(f.y));
}

// The E elements of a vector as pairs.
template <typename T>
__device__ __forceinline__ void vec_pairs(const uint4& u, Pair (&p)[LogitType<T>::E / 2]) {
  if constexpr (LogitType<T>::E == 4) {
    p[0] = Pair(__uint_as_float(u.x), __uint_as_float(u.y));
    p[1] = Pair(__uint_as_float(u.z), __uint_as_float(u.w));
  } else {
    p[0] = Pair(LogitType<T>::pair(u.x));
    p[1] = Pair(LogitType<T>::pair(u.y));
    p[2] = Pair(LogitType<T>::pair(u.z));
    p[3] = Pair(LogitType<T>::pair(u.w));
  }
}
template <typename T>
__device__ __forceinline__ uint4 pairs_round(const Pair (&p)[LogitType<T>::E / 2]) {
  float f[LogitType<T>::E];
#pragma unroll
  for (int j = 0; j < LogitType<T>::E / 2; ++j) {
    const float2 g = p[j].get();
    f[2 * j] = g.x;
    f[2 * j + 1] = g.y;
  }
  return vec_round<T>(f);
}

// Greater logits have greater keys; -0 and 0 the same one, a NaN the greatest.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// largest element, NaN if there is one
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& u) {
  if constexpr (LogitType<T>::E == 4) {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)), max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
    const float2 f = __half22float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    return max_nan(f.x, f.y);
  } else {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
    const float2 f = __bfloat1622float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    return max_nan(f.x, f.y);
  }
}

}  // namespace astrai
