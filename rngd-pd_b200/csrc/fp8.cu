// Quantisers to e4m3: rows, weights, and the RMS norm that adds the residual (fp8.cuh gives the format).
//
// All three read each value once and write it once in 8 bits; the memory bounds them where there are many
// rows, the launch where there are few.  16 lanes hold a group, eight values each, so a group's maximum is four
// shuffles away.  The rows of the result start on 16 bytes whatever their width (the caller's row stride), as the
// products' tile loads want them.
#include "fp8.cuh"
#include "tc.cuh"

namespace rngd {

struct RowsArgs {
  const void* x;
  long ldx;  // elements between rows
  long T;
  int K, G;
  uint8_t* q;
  long ldq;
  float* scale;  // [T][G]
};

constexpr int kRowsThreads = 256, kRowsPer = 4;  // groups of a half warp

// VEC: rows of whole 16-byte vectors.  Else lane l of a group takes its values l, l + 16, ..: loads of
// neighbouring lanes stay together.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kRowsThreads) f8_rows_kernel(RowsArgs a) {
  grid_dep_wait();
  const int l = threadIdx.x & 15;
  const uint32_t total = (uint32_t)(a.T * a.G);
  const uint32_t i0 = (uint32_t)blockIdx.x * (kRowsThreads / 16 * kRowsPer) + (threadIdx.x >> 4);
  Eight<DT> in[kRowsPer];
  uint32_t row[kRowsPer];
  int grp[kRowsPer];
  float v[8];
  bool there[kRowsPer];
#pragma unroll
  for (int j = 0; j < kRowsPer; j++) {
    const uint32_t i = i0 + j * (kRowsThreads / 16);
    row[j] = i / (uint32_t)a.G;
    grp[j] = (int)(i - row[j] * (uint32_t)a.G);
    there[j] = i < total && i >= i0;
    if (VEC && there[j] && grp[j] * kGroup + 8 * l < a.K) in[j].load(a.x, (long)row[j] * a.ldx + grp[j] * kGroup + 8 * l);
  }
  grid_dep_launch();
#pragma unroll
  for (int j = 0; j < kRowsPer; j++) {
    const int k0 = grp[j] * kGroup;
    const bool mine = there[j] && (!VEC || k0 + 8 * l < a.K);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = 0.f;
    if (VEC) {
      if (mine) in[j].values(v);
    } else if (there[j]) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (k0 + l + 16 * e < a.K) v[e] = load_as_f32<DT>(a.x, (long)row[j] * a.ldx + k0 + l + 16 * e);
    }
    const float m = held_max(amax16(amax_of(v)));
    const float inv = 448.0f / m;
    uint8_t* dst = a.q + (long)row[j] * a.ldq + k0;
    if (VEC) {
      if (mine) *(uint2*)(dst + 8 * l) = held8(v, inv);
    } else if (there[j]) {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (k0 + l + 16 * e < a.K) dst[l + 16 * e] = e4m3(v[e] * inv);
    }
    if (there[j] && l == 0) a.scale[(long)row[j] * a.G + grp[j]] = m / 448.0f;
  }
}

// ------------------------------------------------------------------------------------------ weights
// One CTA per block of 128 x 128: 16 rows of 8 warps' half-warps at a time, kept in registers between the maximum
// and the rounding.
struct WeightArgs {
  const void* w;
  long ldw;
  int N, K, G;
  uint8_t* q;
  long ldq;
  float* scale;  // [ceil(N / 128)][G]
};

template <int DT, bool VEC>
__global__ void __launch_bounds__(256) f8_weight_kernel(WeightArgs a) {
  __shared__ float s_max[8];
  grid_dep_wait();
  const int b = blockIdx.x, nb = b / a.G, kb = b - nb * a.G;
  const int l = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int k0 = kb * kGroup;
  Eight<DT> in[8];
  float most = 0.f, v[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int n = nb * kGroup + r0 + 16 * j;
    if (VEC && n < a.N && k0 + 8 * l < a.K) in[j].load(a.w, (long)n * a.ldw + k0 + 8 * l);
  }
  grid_dep_launch();
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int n = nb * kGroup + r0 + 16 * j;
    if (n >= a.N) continue;
    if (VEC) {
      if (k0 + 8 * l < a.K) {
        in[j].values(v);
        most = amax_of(v, most);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (k0 + l + 16 * e < a.K) most = max_nan(most, fabsf(load_as_f32<DT>(a.w, (long)n * a.ldw + k0 + l + 16 * e)));
    }
  }
  most = amax16(most);
  most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, 16));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) most = max_nan(most, s_max[i]);
  const float m = held_max(most), inv = 448.0f / m;
  if (threadIdx.x == 0) a.scale[b] = m / 448.0f;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const int n = nb * kGroup + r0 + 16 * j;
    if (n >= a.N) continue;
    uint8_t* dst = a.q + (long)n * a.ldq + k0;
    if (VEC) {
      if (k0 + 8 * l < a.K) {
        in[j].values(v);
        *(uint2*)(dst + 8 * l) = held8(v, inv);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (k0 + l + 16 * e < a.K)
          dst[l + 16 * e] = e4m3(load_as_f32<DT>(a.w, (long)n * a.ldw + k0 + l + 16 * e) * inv);
    }
  }
}

// --------------------------------------------------------------------------------------------- norm
// h = x + residual rounded to its type (where there is a residual, and written then), y = h * rsqrt(mean h^2 + eps) * w
// in fp32, quantised by groups.  One CTA a row, which stays in its registers (PER vectors of eight a thread)
// between the sum of squares and the rounding; PER = 0: rows too wide for that are read twice.
struct NormArgs {
  const void *x, *res, *w;
  long ldx, ldr;
  int K, G, w32;  // w32: the weights are fp32, else of x's type
  float eps;
  void* total;  // [T][K] of x's type, rows ldt apart
  long ldt;
  uint8_t* q;
  long ldq;
  float* scale;
};

// h of the eight values from k on (VEC), or k, k + 16, ..
template <int DT, bool VEC>
__device__ __forceinline__ void norm_row(const NormArgs& a, long row, int k, bool write, float* h) {
  if (VEC) {
    Eight<DT> x;
    x.load(a.x, row * a.ldx + k);
    if (a.res != nullptr) {
      Eight<DT> r;
      float f[8];
      r.load(a.res, row * a.ldr + k);
      x.values(h);
      r.values(f);
#pragma unroll
      for (int e = 0; e < 8; e++) h[e] = rounded_as<DT>(h[e] + f[e]);
      if (write) store_eight<DT>(a.total, row * a.ldt + k, h);
    } else {
      x.values(h);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int c = k + 16 * e;
      h[e] = 0.f;
      if (c < a.K) {
        h[e] = load_as_f32<DT>(a.x, row * a.ldx + c);
        if (a.res != nullptr) {
          h[e] = rounded_as<DT>(h[e] + load_as_f32<DT>(a.res, row * a.ldr + c));
          if (write) store_f32_as<DT>(a.total, row * a.ldt + c, h[e]);
        }
      }
    }
  }
}

template <int DT, bool VEC>
__device__ __forceinline__ void norm_out(const NormArgs& a, long row, int grp, int l, bool mine, float r, float* h) {
  const int k0 = grp * kGroup;
  if (VEC) {
    if (mine) {
      float w[8];
      if (a.w32 || DT == F8_F32) {
        Eight<F8_F32> g;
        g.load(a.w, k0 + 8 * l);
        g.values(w);
      } else {
        Eight<DT> g;
        g.load(a.w, k0 + 8 * l);
        g.values(w);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) h[e] = h[e] * r * w[e];
    }
  } else if (mine) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int c = k0 + l + 16 * e;
      if (c < a.K) h[e] = h[e] * r * (a.w32 ? ((const float*)a.w)[c] : load_as_f32<DT>(a.w, c));
    }
  }
  const float m = held_max(amax16(mine ? amax_of(h) : 0.f));
  const float inv = 448.0f / m;
  uint8_t* dst = a.q + row * a.ldq + k0;
  if (VEC) {
    if (mine) *(uint2*)(dst + 8 * l) = held8(h, inv);
  } else if (mine) {
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (k0 + l + 16 * e < a.K) dst[l + 16 * e] = e4m3(h[e] * inv);
  }
  if (l == 0 && grp < a.G) a.scale[row * a.G + grp] = m / 448.0f;
}

template <int DT, bool VEC, int PER>
__global__ void __launch_bounds__(1024) f8_norm_kernel(NormArgs a) {
  __shared__ float s_sum[32];
  grid_dep_wait();
  const long row = blockIdx.x;
  const int l = threadIdx.x & 15, g0 = threadIdx.x >> 4, gs = blockDim.x >> 4;
  constexpr int HOLD = PER > 0 ? PER : 1;
  float h[HOLD][8];
  float ss = 0.f;
  const int rounds = PER > 0 ? PER : (a.G + gs - 1) / gs;
  auto first = [&](int j, float* f) {
    const int grp = g0 + j * gs, k = grp * kGroup + (VEC ? 8 * l : l);
    if (grp < a.G && k < a.K) {
      norm_row<DT, VEC>(a, row, k, true, f);
#pragma unroll
      for (int e = 0; e < 8; e++) ss = fmaf(f[e], f[e], ss);
    }
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int j = 0; j < PER; j++) first(j, h[j]);
  } else {
    for (int j = 0; j < rounds; j++) first(j, h[0]);
  }
  grid_dep_launch();
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = ss;
  __syncthreads();
  ss = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 5); i++) ss += s_sum[i];
  const float r = rsqrtf(ss / (float)a.K + a.eps);
  auto second = [&](int j, float* f, bool again) {
    const int grp = g0 + j * gs, k = grp * kGroup + (VEC ? 8 * l : l);
    const bool mine = grp < a.G && k < a.K;
    if (again && mine) norm_row<DT, VEC>(a, row, k, false, f);
    norm_out<DT, VEC>(a, row, grp, l, mine, r, f);
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int j = 0; j < PER; j++) second(j, h[j], false);
  } else {
    for (int j = 0; j < rounds; j++) second(j, h[0], true);
  }
}

// -------------------------------------------------------------------------------------------- host
static int dtype_size(int dtype) { return dtype == F8_F32 ? 4 : 2; }
static bool whole_vectors(const void* p, long ld, int K, int dtype) {
  return K % 8 == 0 && ((uintptr_t)p & 15) == 0 && ld * dtype_size(dtype) % 16 == 0;
}
static int check_held(const char* what, const uint8_t* q, long ldq, long rows, int K, const float* scale) {
  RNGD_REQUIRE(q != nullptr && scale != nullptr, "%s: null pointer", what);
  RNGD_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)scale & 3) == 0 && ldq % 16 == 0 && (ldq >= K || rows <= 1),
               "%s: 8-bit rows must start on 16 bytes and not overlap (%ld bytes apart)", what, ldq);
  return RNGD_OK;
}

template <template <int, bool> class F, typename... A>
static int by_type(int dtype, bool vec, A... args) {
  if (dtype == F8_BF16) return vec ? F<F8_BF16, true>::go(args...) : F<F8_BF16, false>::go(args...);
  if (dtype == F8_F16) return vec ? F<F8_F16, true>::go(args...) : F<F8_F16, false>::go(args...);
  return vec ? F<F8_F32, true>::go(args...) : F<F8_F32, false>::go(args...);
}

template <int DT, bool VEC>
struct RowsLaunch {
  static int go(const RowsArgs& a, cudaStream_t s) {
    constexpr int per = kRowsThreads / 16 * kRowsPer;
    return launch_pdl(f8_rows_kernel<DT, VEC>, dim3((unsigned)((a.T * a.G + per - 1) / per)), dim3(kRowsThreads), 0, s,
                      "f8_rows_kernel", a);
  }
};
template <int DT, bool VEC>
struct WeightLaunch {
  static int go(const WeightArgs& a, cudaStream_t s) {
    return launch_pdl(f8_weight_kernel<DT, VEC>, dim3((unsigned)(((long)a.N + 127) / 128 * a.G)), dim3(256), 0, s,
                      "f8_weight_kernel", a);
  }
};
template <int DT, bool VEC>
struct NormLaunch {
  static int go(const NormArgs& a, long T, cudaStream_t s) {
    const int lanes = a.G * 16;  // lanes that a row fills, eight values each
    auto run = [&](auto kernel, int per) {
      int threads = (lanes + per - 1) / per;
      threads = threads > 1024 ? 1024 : (threads + 31) / 32 * 32;
      return launch_pdl(kernel, dim3((unsigned)T), dim3(threads), 0, s, "f8_norm_kernel", a);
    };
    if (lanes <= 512) return run(f8_norm_kernel<DT, VEC, 1>, 1);
    if (lanes <= 1024) return run(f8_norm_kernel<DT, VEC, 2>, 2);
    if (lanes <= 4096) return run(f8_norm_kernel<DT, VEC, 4>, 4);
    return run(f8_norm_kernel<DT, VEC, 0>, 4);
  }
};

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_f8_rows(const void* x, int dtype, int64_t ldx, int64_t T, int K, void* q, int64_t ldq, float* scale,
                            rngd_stream_t stream) {
  RNGD_REQUIRE(dtype >= F8_BF16 && dtype <= F8_F32, "f8_rows: data type %d", dtype);
  RNGD_REQUIRE(T >= 0 && K >= 0, "f8_rows: %ld rows of %d", (long)T, K);
  if (T == 0 || K == 0) return RNGD_OK;
  const int G = (int)(((long)K + kGroup - 1) / kGroup);
  RNGD_REQUIRE(T <= 0xFFFFFFFFl / G && T <= 0x7FFFFFFFl, "f8_rows: %ld rows of %d", (long)T, K);
  RNGD_REQUIRE(x != nullptr && (uintptr_t)x % dtype_size(dtype) == 0, "f8_rows: x is null or misaligned");
  RNGD_TRY(check_held("f8_rows", (uint8_t*)q, ldq, T, K, scale));
  RowsArgs a = {x, (long)ldx, (long)T, K, G, (uint8_t*)q, (long)ldq, scale};
  return by_type<RowsLaunch>(dtype, whole_vectors(x, ldx, K, dtype), a, (cudaStream_t)stream);
}

extern "C" int rngd_f8_weight(const void* w, int dtype, int64_t ldw, int N, int K, void* q, int64_t ldq, float* scale,
                              rngd_stream_t stream) {
  RNGD_REQUIRE(dtype >= F8_BF16 && dtype <= F8_F32, "f8_weight: data type %d", dtype);
  RNGD_REQUIRE(N >= 0 && K >= 0, "f8_weight: %d x %d", N, K);
  if (N == 0 || K == 0) return RNGD_OK;
  const int G = (int)(((long)K + kGroup - 1) / kGroup);
  RNGD_REQUIRE(((long)N + 127) / 128 * G <= 0x7FFFFFFFl, "f8_weight: %d x %d", N, K);
  RNGD_REQUIRE(w != nullptr && (uintptr_t)w % dtype_size(dtype) == 0, "f8_weight: w is null or misaligned");
  RNGD_TRY(check_held("f8_weight", (uint8_t*)q, ldq, N, K, scale));
  WeightArgs a = {w, (long)ldw, N, K, G, (uint8_t*)q, (long)ldq, scale};
  return by_type<WeightLaunch>(dtype, whole_vectors(w, ldw, K, dtype), a, (cudaStream_t)stream);
}

extern "C" int rngd_f8_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                                int dtype, int weight_dtype, int64_t T, int K, float eps, void* total, int64_t ldt,
                                void* q, int64_t ldq, float* scale, rngd_stream_t stream) {
  RNGD_REQUIRE(dtype >= F8_BF16 && dtype <= F8_F32, "f8_rms_norm: data type %d", dtype);
  RNGD_REQUIRE(weight_dtype == dtype || weight_dtype == F8_F32, "f8_rms_norm: weights of data type %d with rows of %d",
               weight_dtype, dtype);
  RNGD_REQUIRE(T >= 0 && T <= 0x7FFFFFFFl && K >= 0, "f8_rms_norm: %ld rows of %d", (long)T, K);
  if (T == 0 || K == 0) return RNGD_OK;
  const int sz = dtype_size(dtype), G = (int)(((long)K + kGroup - 1) / kGroup);
  RNGD_REQUIRE(x != nullptr && weight != nullptr, "f8_rms_norm: null pointer");
  RNGD_REQUIRE((residual == nullptr) == (total == nullptr), "f8_rms_norm: a residual comes with a place for the sum");
  RNGD_REQUIRE(((uintptr_t)x | (uintptr_t)residual | (uintptr_t)total) % sz == 0 &&
                   (uintptr_t)weight % dtype_size(weight_dtype) == 0,
               "f8_rms_norm: misaligned pointer");
  RNGD_REQUIRE(total == nullptr || (total != x && total != residual), "f8_rms_norm: the sum needs a place of its own");
  RNGD_REQUIRE(total == nullptr || ldt >= K || T <= 1, "f8_rms_norm: rows of the sum lie on one another");
  RNGD_TRY(check_held("f8_rms_norm", (uint8_t*)q, ldq, T, K, scale));
  NormArgs a = {x, residual, weight, (long)ldx, (long)ldr, K, G, weight_dtype == F8_F32, eps,
                total, (long)ldt, (uint8_t*)q, (long)ldq, scale};
  const bool vec = whole_vectors(x, ldx, K, dtype) && whole_vectors(weight, 0, K, weight_dtype) &&
                   (residual == nullptr || (whole_vectors(residual, ldr, K, dtype) && whole_vectors(total, ldt, K, dtype)));
  return by_type<NormLaunch>(dtype, vec, a, (long)T, (cudaStream_t)stream);
}
