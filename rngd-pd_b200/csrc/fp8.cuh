// Rows and weights held in 8 bits (e4m3) with fp32 scales: what the quantisers (fp8.cu) and the products
// (fp8_mm.cu) share.
//
// A row of K values has a scale for each 128 of them from the left (the last group may be shorter), a weight
// [N][K] one for each 128 x 128 block.  With m = max(amax, 2^-100) of a group's magnitudes,
//   scale = m / 448,   q = e4m3(x * (448 / m)),   x stands as q * scale.
// The lower limit keeps 448 / m finite; a group below it (zeros above all) is held in steps of 2^-118, which no
// sum with ordinary values could show.  The quotient is taken once a group and the values are multiplied with it:
// one rounding to 24 bits more than a division each, against half a step of e4m3 of 2^-4.  A NaN makes m, the
// scale and so the whole group NaN; an infinity makes 448 / m zero and the scale infinite, whose products are NaN too.
#pragma once
#include "common.cuh"

#include <cuda_fp16.h>

namespace rngd {

constexpr int kGroup = 128;
constexpr int kMostK = 1 << 30, kMostRows = 0x7FFFFFFF - 255;  // places within a row, and tiles' ends, are 32-bit numbers

enum : int { F8_BF16 = 0, F8_F16 = 1, F8_F32 = 2 };

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// m of a group whose magnitudes reach amax
__device__ __forceinline__ float held_max(float amax) { return max_nan(amax, 7.888609052210118e-31f); }  // 2^-100

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}
__device__ __forceinline__ uint8_t e4m3(float a) { return (uint8_t)e4m3x2(a, 0.f); }

// one value of type DT
template <int DT>
__device__ __forceinline__ float load_as_f32(const void* p, long i) {
  if constexpr (DT == F8_BF16)
    return bf2f(((const uint16_t*)p)[i]);
  else if constexpr (DT == F8_F16)
    return __half2float(((const __half*)p)[i]);
  else
    return ((const float*)p)[i];
}
template <int DT>
__device__ __forceinline__ void store_f32_as(void* p, long i, float v) {
  if constexpr (DT == F8_BF16)
    ((uint16_t*)p)[i] = f2bf_bits(v);
  else if constexpr (DT == F8_F16)
    ((__half*)p)[i] = __float2half_rn(v);
  else
    ((float*)p)[i] = v;
}
template <int DT>
__device__ __forceinline__ float rounded_to(float v) {
  if constexpr (DT == F8_BF16)
    return bf2f(f2bf_bits(v));
  else if constexpr (DT == F8_F16)
    return __half2float(__float2half_rn(v));
  else
    return v;
}
// Eight values from a 16-byte aligned place: the registers that hold them, and their values.
template <int DT>
struct Eight {
  uint4 r[DT == F8_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void* p, long i) {
    if constexpr (DT == F8_F32) {
      const uint4* q = (const uint4*)((const float*)p + i);
      r[0] = ldg_nc_v4(q);
      r[1] = ldg_nc_v4(q + 1);
    } else {
      r[0] = ldg_nc_v4((const uint16_t*)p + i);
    }
  }
  // an aligned eight of memory that this kernel may write
  __device__ __forceinline__ void load_any(const void* p, long i) {
    const uint4* q = (const uint4*)((const char*)p + i * (DT == F8_F32 ? 4 : 2));
#pragma unroll
    for (int j = 0; j < (DT == F8_F32 ? 2 : 1); j++) r[j] = q[j];
  }
  __device__ __forceinline__ void values(float* f) const {
    if constexpr (DT == F8_F32) {
#pragma unroll
      for (int j = 0; j < 2; j++) {
        f[4 * j] = __uint_as_float(r[j].x);
        f[4 * j + 1] = __uint_as_float(r[j].y);
        f[4 * j + 2] = __uint_as_float(r[j].z);
        f[4 * j + 3] = __uint_as_float(r[j].w);
      }
    } else if constexpr (DT == F8_BF16) {
      unpack8(r[0], f);
    } else {
      const uint32_t w[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 v = __half22float2(*(const __half2*)&w[j]);
        f[2 * j] = v.x;
        f[2 * j + 1] = v.y;
      }
    }
  }
};
// The first n of eight values, zeros for the others, from any place of a matrix that ends before `end`.  They come as the
// aligned vectors around them (neighbouring rows' values may come along), fetched first and shifted into place when they
// are needed, so that several are on their way at a time; where the vectors would reach beyond the matrix, value by value.
template <int DT>
struct EightAt {
  static constexpr int SZ = DT == F8_F32 ? 4 : 2, V = 8 * SZ / 16;  // vectors where the place is aligned, else one more
  uint4 v[V + 1];
  __device__ __forceinline__ static bool inside(const void* p, long i, const char* end) {
    const char* at = (const char*)p + i * SZ;
    const int s = (int)((uintptr_t)at & 15);
    return at - s >= (const char*)p && at - s + 16 * (V + (s != 0)) <= end;
  }
  __device__ __forceinline__ void fetch(const void* p, long i, const char* end) {
    const char* at = (const char*)p + i * SZ;
    const int s = (int)((uintptr_t)at & 15);
    if (inside(p, i, end)) {
#pragma unroll
      for (int j = 0; j < V; j++) v[j] = ldg_nc_v4(at - s + 16 * j);
      if (s != 0) v[V] = ldg_nc_v4(at - s + 16 * V);
    }
  }
  __device__ __forceinline__ Eight<DT> get(const void* p, long i, int n, const char* end) const {
    Eight<DT> r;
    const char* at = (const char*)p + i * SZ;
    uint32_t w[4 * V + 4];
    if (inside(p, i, end)) {
      const int s = (int)((uintptr_t)at & 15);
#pragma unroll
      for (int j = 0; j <= V; j++) {
        const uint4 x = v[j];
        w[4 * j] = x.x;
        w[4 * j + 1] = x.y;
        w[4 * j + 2] = x.z;
        w[4 * j + 3] = x.w;
      }
#pragma unroll
      for (int j = 0; j < 4 * V + 2; j++) w[j] = s & 8 ? w[j + 2] : w[j];
#pragma unroll
      for (int j = 0; j < 4 * V + 1; j++) w[j] = s & 4 ? w[j + 1] : w[j];
      if constexpr (SZ == 2) {
#pragma unroll
        for (int j = 0; j < 4 * V; j++) w[j] = __funnelshift_r(w[j], w[j + 1], (s & 2) * 8);
      }
      if (n < 8) {
#pragma unroll
        for (int j = 0; j < 4 * V; j++) {
          if constexpr (SZ == 4)
            w[j] = j < n ? w[j] : 0u;
          else
            w[j] = 2 * j + 1 < n ? w[j] : 2 * j < n ? w[j] & 0xFFFFu : 0u;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4 * V; j++) {
        if constexpr (SZ == 4) {
          w[j] = j < n ? __float_as_uint(((const float*)at)[j]) : 0u;
        } else {
          const uint16_t* half = (const uint16_t*)at;
          const uint32_t l = 2 * j < n ? half[2 * j] : 0u, h = 2 * j + 1 < n ? half[2 * j + 1] : 0u;
          w[j] = l | h << 16;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < V; j++) r.r[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    return r;
  }
};
// one past a matrix of rows ld apart
template <int DT>
__device__ __forceinline__ const char* end_of(const void* p, long rows, long ld, int K) {
  return (const char*)p + ((rows - 1) * ld + K) * (DT == F8_F32 ? 4 : 2);
}

// Eight values rounded to DT.
template <int DT>
__device__ __forceinline__ Eight<DT> eight_of(const float* f) {
  Eight<DT> v;
  if constexpr (DT == F8_F32) {
#pragma unroll
    for (int j = 0; j < 2; j++)
      v.r[j] = make_uint4(__float_as_uint(f[4 * j]), __float_as_uint(f[4 * j + 1]), __float_as_uint(f[4 * j + 2]),
                          __float_as_uint(f[4 * j + 3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if constexpr (DT == F8_BF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(f[2 * j + 1]), "f"(f[2 * j]));
      } else {
        const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
        w[j] = *(const uint32_t*)&h;
      }
    }
    v.r[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
// Eight values to a 16-byte aligned place.
template <int DT>
__device__ __forceinline__ void store_eight(void* p, long i, const Eight<DT>& v) {
  uint4* q = (uint4*)((char*)p + i * (DT == F8_F32 ? 4 : 2));
#pragma unroll
  for (int j = 0; j < (DT == F8_F32 ? 2 : 1); j++) q[j] = v.r[j];
}

// A group lies in 8 neighbouring lanes, 16 values each: lane l has the vectors of eight at 8 l and at 64 + 8 l.  (16 lanes
// with eight each take a third more steps to the group's maximum, and the quotients twice as often a value: rows of
// 8191 x 4096 bf16 then take 17.6 us, not 16.4.)
constexpr int kLanes = 8;
__device__ __forceinline__ float amax_lanes(float m) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
template <int N>
__device__ __forceinline__ float amax_of(const float* f, float m = 0.f) {
#pragma unroll
  for (int e = 0; e < N; e++) m = max_nan(m, fabsf(f[e]));
  return m;
}
// 448 / m of P groups that 8 lanes have in common (m: each group's held_max, known to all of them).  The quotients
// cost as much as all else that is done with eight values, so lane l works out group l % P alone; its scale is
// returned, and the first P lanes store them.
template <int P>
__device__ __forceinline__ float quotients(const float (&m)[P], float (&inv)[P]) {
  static_assert((P & (P - 1)) == 0 && P <= kLanes, "");
  const int l = threadIdx.x & (kLanes - 1), lane = threadIdx.x & 31;
  float mine = m[0];
#pragma unroll
  for (int j = 1; j < P; j++)
    if ((l & (P - 1)) == j) mine = m[j];
  const float iv = 448.0f / mine;
#pragma unroll
  for (int j = 0; j < P; j++) inv[j] = P == 1 ? iv : __shfl_sync(0xffffffffu, iv, (lane & ~(kLanes - 1)) + j);
  return mine / 448.0f;
}
__device__ __forceinline__ uint2 held8(const float* f, float inv) {
  return make_uint2(e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                    e4m3x4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
}
// Eight values rounded to dst, 8-byte aligned; `left` of them exist (whole: all or none).
template <bool WHOLE>
__device__ __forceinline__ void store_held(uint8_t* dst, int left, const float* f, float inv) {
  if (WHOLE ? left > 0 : left >= 8) {
    *(uint2*)dst = held8(f, inv);
  } else if (!WHOLE) {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (e < left) dst[e] = e4m3(f[e] * inv);
  }
}

// SwiGLU in fp32: silu(g) * u, g / (1 + 2^(-g log2 e)) by the machine's power of two and reciprocal (2 and 1 units in the
// last place; the exponent's rounding is |g| / 2 of them).  A power beyond the range gives a reciprocal of 0, the limit.
__device__ __forceinline__ float swiglu(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r * u;
}
// the largest magnitude of three, NaN if any is
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

}  // namespace rngd
