// Quantisers to e4m3: rows, weights, and the RMS norm that adds the residual (fp8.cuh gives the format).
//
// All three read each value once and write it once in 8 bits; the memory bounds them where there are many rows, the
// launch where there are few.  The rows of the result start on 16 bytes whatever their width (the caller's row stride),
// as the products' tile loads want them.  Measured, inputs larger than the L2 cache: rows 8191 x 4096 bf16 16.4 us, 6.2
// TB/s; weight 14336 x 4096 bf16 28.6 us, 6.2 TB/s; norm 8192 x 4096 bf16 with a residual 38.3 us, 6.2 TB/s (the copy
// rate is 6.55).  Rows of 4097 values, which start anywhere: 8000 of them in bf16 26 us, the norm with a residual 98:
// eight values come as one aligned vector more than they fill, which the neighbouring lane asks the L2 cache for too, and
// are shifted into place; more instructions a value, and fewer blocks an SM.
#include "fp8.cuh"
#include "tc.cuh"

#include <type_traits>

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

constexpr int kRowsThreads = 256, kRowsPer = 2;  // neighbouring groups of a row that eight lanes take

// VEC: rows of whole 16-byte vectors; else they start anywhere.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kRowsThreads) f8_rows_kernel(RowsArgs a) {
  grid_dep_wait();
  const int l = threadIdx.x & (kLanes - 1);
  const uint32_t runs = (uint32_t)(a.G + kRowsPer - 1) / kRowsPer;
  const uint32_t i = blockIdx.x * (uint32_t)(kRowsThreads / kLanes) + threadIdx.x / kLanes;
  const uint32_t row = i / runs;
  const int g0 = (int)(i - row * runs) * kRowsPer;
  const bool there = row < a.T;
  const long k0 = (long)g0 * kGroup, in0 = row * a.ldx + k0;
  const int left = there ? (int)min((long)a.K - k0, (long)kRowsPer * kGroup) : 0;  // values of this run
  const char* end = end_of<DT>(a.x, a.T, a.ldx, a.K);
  std::conditional_t<VEC, Eight<DT>, EightAt<DT>> in[kRowsPer][2];
  float v[kRowsPer][16], m[kRowsPer], inv[kRowsPer];
#pragma unroll
  for (int j = 0; j < kRowsPer; j++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = j * kGroup + 64 * c + 8 * l;
      if (k < left) {
        if constexpr (VEC)
          in[j][c].load(a.x, in0 + k);
        else
          in[j][c].fetch(a.x, in0 + k, end);
      }
    }
  grid_dep_launch();
#pragma unroll
  for (int j = 0; j < kRowsPer; j++) {
#pragma unroll
    for (int e = 0; e < 16; e++) v[j][e] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = j * kGroup + 64 * c + 8 * l;
      if (k < left) {
        if constexpr (VEC)
          in[j][c].values(v[j] + 8 * c);
        else
          in[j][c].get(a.x, in0 + k, left - k, end).values(v[j] + 8 * c);
      }
    }
    m[j] = held_max(amax_lanes(amax_of<16>(v[j])));
  }
  const float scale = quotients<kRowsPer>(m, inv);
  uint8_t* dst = a.q + (long)row * a.ldq + k0;
#pragma unroll
  for (int j = 0; j < kRowsPer; j++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = j * kGroup + 64 * c + 8 * l;
      store_held<VEC>(dst + k, left - k, v[j] + 8 * c, inv[j]);
    }
  if (l < kRowsPer && l * kGroup < left) a.scale[(long)row * a.G + g0 + l] = scale;
}

// ------------------------------------------------------------------------------------------ weights
// One CTA per block of 128 x 128, 16 rows at a time (16 lanes a row, eight values each), kept in registers between the
// maximum and the rounding.
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
  const int k = k0 + 8 * l;
  const char* end = end_of<DT>(a.w, a.N, a.ldw, a.K);
  std::conditional_t<VEC, Eight<DT>, EightAt<DT>> raw[8];
  Eight<DT> in[8];
  float most = 0.f, v[8];
  auto there = [&](int j) { return nb * kGroup + r0 + 16 * j < a.N && k < a.K; };
  auto at = [&](int j) { return (long)(nb * kGroup + r0 + 16 * j) * a.ldw + k; };
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (there(j)) {
      if constexpr (VEC)
        raw[j].load(a.w, at(j));
      else
        raw[j].fetch(a.w, at(j), end);
    }
  grid_dep_launch();
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (there(j)) {
      if constexpr (VEC)
        in[j] = raw[j];
      else
        in[j] = raw[j].get(a.w, at(j), a.K - k, end);
      in[j].values(v);
      most = amax_of<8>(v, most);
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) most = max_nan(most, s_max[i]);
  const float m = held_max(most), inv = 448.0f / m;
  if (threadIdx.x == 0) a.scale[b] = m / 448.0f;
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (there(j)) {
      in[j].values(v);
      store_held<VEC>(a.q + (long)(nb * kGroup + r0 + 16 * j) * a.ldq + k, a.K - k, v, inv);
    }
}

// --------------------------------------------------------------------------------------------- norm
// h = x + residual rounded to its type (where there is a residual, and written then), y = h * rsqrt(mean h^2 + eps) * w
// in fp32, quantised by groups.  One CTA has a row at a time, which stays in its registers (PER vectors of eight a
// thread) between the sum of squares and the rounding.
struct NormArgs {
  const void *x, *res, *w;
  long ldx, ldr;
  int K, G;
  float eps;
  long T;
  int stage;    // rows of the sum go out through shared memory
  void* total;  // [T][K] of x's type, rows ldt apart
  long ldt;
  uint8_t* q;
  long ldq;
  float* scale;
};

// A lane's 16 values of x and the residual in the group from k0 on, as they are loaded.
template <int DT, bool VEC>
struct NormIn {
  std::conditional_t<VEC, Eight<DT>, EightAt<DT>> x[2], r[2];
  __device__ __forceinline__ void load(const NormArgs& a, long row, int k0, int l) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = k0 + 64 * c + 8 * l;
      if (k >= a.K) continue;
      if constexpr (VEC) {
        x[c].load(a.x, row * a.ldx + k);
        if (a.res != nullptr) r[c].load(a.res, row * a.ldr + k);
      } else {
        x[c].fetch(a.x, row * a.ldx + k, end_of<DT>(a.x, a.T, a.ldx, a.K));
        if (a.res != nullptr) r[c].fetch(a.res, row * a.ldr + k, end_of<DT>(a.res, a.T, a.ldr, a.K));
      }
    }
  }
  // their sum as it is kept (zeros beyond the row), written to total where that is asked for, or to `room` (VEC: null)
  __device__ __forceinline__ void sum(const NormArgs& a, long row, int k0, int l, bool write, float* f, char* room) const {
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = k0 + 64 * c + 8 * l;
      float* fc = f + 8 * c;
      if (k < a.K) {
        if constexpr (VEC)
          x[c].values(fc);
        else
          x[c].get(a.x, row * a.ldx + k, a.K - k, end_of<DT>(a.x, a.T, a.ldx, a.K)).values(fc);
        if (a.res != nullptr) {
          float g[8];
          if constexpr (VEC)
            r[c].values(g);
          else
            r[c].get(a.res, row * a.ldr + k, a.K - k, end_of<DT>(a.res, a.T, a.ldr, a.K)).values(g);
#pragma unroll
          for (int e = 0; e < 8; e++) fc[e] += g[e];
          const Eight<DT> kept = eight_of<DT>(fc);
          kept.values(fc);
          if (write) {
            if constexpr (VEC) {
              store_eight<DT>(a.total, row * a.ldt + k, kept);
            } else if (room != nullptr) {
              store_eight<DT>(room, k, kept);
            } else {
#pragma unroll
              for (int e = 0; e < 8; e++)
                if (k + e < a.K) store_f32_as<DT>(a.total, row * a.ldt + k + e, fc[e]);
            }
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) fc[e] = 0.f;
      }
    }
  }
};
template <int WT, bool VEC>
struct NormWeight {  // the weights of the same 16
  Eight<WT> w[2];
  __device__ __forceinline__ void load(const NormArgs& a, int k0, int l) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = k0 + 64 * c + 8 * l;
      if (k >= a.K) continue;
      if constexpr (VEC) {
        w[c].load(a.w, k);
      } else {
        const char* end = end_of<WT>(a.w, 1, 0, a.K);
        EightAt<WT> raw;
        raw.fetch(a.w, k, end);
        w[c] = raw.get(a.w, k, a.K - k, end);
      }
    }
  }
  __device__ __forceinline__ void scale(const NormArgs& a, int k0, int l, float r, float* f) const {
#pragma unroll
    for (int c = 0; c < 2; c++)
      if (k0 + 64 * c + 8 * l < a.K) {
        float g[8];
        w[c].values(g);
#pragma unroll
        for (int e = 0; e < 8; e++) f[8 * c + e] = f[8 * c + e] * r * g[e];
      }
  }
};

// A row of the sum from shared memory to a place of any alignment, four bytes a thread at a time.
template <int DT>
__device__ __forceinline__ void norm_row_out(const NormArgs& a, long row, const char* room) {
  if constexpr (DT == F8_F32) {
    float* to = (float*)a.total + row * a.ldt;
    for (int i = threadIdx.x; i < a.K; i += blockDim.x) to[i] = ((const float*)room)[i];
  } else {
    uint16_t* to = (uint16_t*)a.total + row * a.ldt;
    const uint16_t* from = (const uint16_t*)room;
    const int head = (int)((uintptr_t)to >> 1) & 1, pairs = (a.K - head) >> 1;
    for (int i = threadIdx.x; i < pairs; i += blockDim.x)
      ((uint32_t*)(to + head))[i] = from[head + 2 * i] | (uint32_t)from[head + 2 * i + 1] << 16;
    if (threadIdx.x == 0 && head) to[0] = from[0];
    if (threadIdx.x == 0 && ((a.K - head) & 1)) to[a.K - 1] = from[a.K - 1];
  }
}

__device__ __forceinline__ float block_sum(float v, float* s_sum) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  v = warp_sum(v);
  if (lane == 0) s_sum[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < warps ? s_sum[lane] : 0.f);
}
// Rows beyond about 2^64, and those below 2^-48 where eps is as small, have squares that fp32 does not hold.
constexpr float kLeastMean = 0x1p-96f, kMostMean = 0x1p127f;
__device__ __forceinline__ bool beyond(float v) { return v < kLeastMean || v > kMostMean; }
// mean + eps of the block's sums of squares
__device__ __forceinline__ float norm_mean(float ss, float* s_sum, const NormArgs& a) {
  return block_sum(ss, s_sum) / (float)a.K + a.eps;
}
// Such rows among this block's, once more after the others: their 8-bit values, of squares of the values times c, which is
// 2^-80 or 2^80.  Values up to 2^128 then have squares up to 2^96, and 2^30 of those a sum below 2^127.  (Apart from the
// rows' own loop, for its registers: with this in its middle 1001 x 4104 fp16 took 6.0 us, not 5.2, and 3000 x 12288 bf16
// 49, not 44.)
template <int DT, int WT>
__device__ __forceinline__ void norm_rows_again(const NormArgs& a, float* s_sum) {
  const int lane = threadIdx.x & 31;
  for (long row = blockIdx.x; row < a.T; row += gridDim.x) {
    auto value = [&](int k) {
      const float h = load_as_f32<DT>(a.x, row * a.ldx + k);
      return a.res == nullptr ? h : rounded_to<DT>(h + load_as_f32<DT>(a.res, row * a.ldr + k));
    };
    auto mean = [&](float c) {
      float ss = 0.f;
#pragma unroll 1
      for (int k = threadIdx.x; k < a.K; k += blockDim.x) {
        const float h = value(k) * c;
        ss = fmaf(h, h, ss);
      }
      __syncthreads();  // everybody has read the sums before
      return block_sum(ss, s_sum) / (float)a.K + a.eps * c * c;
    };
    const float v = mean(1.f);
    if (!(v < 2 * kLeastMean || v > kMostMean / 2)) continue;  // (summed in another order, so that all of them are found)
    const float c = v > 1.f ? 0x1p-80f : 0x1p80f, r = rsqrtf(mean(c));
#pragma unroll 1
    for (int g = threadIdx.x >> 5; g < a.G; g += blockDim.x >> 5) {
      float y[4], m = 0.f;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int k = g * kGroup + 32 * e + lane;
        y[e] = k < a.K ? value(k) * c * r * load_as_f32<WT>(a.w, k) : 0.f;
        m = max_nan(m, fabsf(y[e]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      m = held_max(m);
      const float inv = 448.0f / m;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int k = g * kGroup + 32 * e + lane;
        if (k < a.K) a.q[row * a.ldq + k] = e4m3(y[e] * inv);
      }
      if (lane == 0) a.scale[row * a.G + g] = m / 448.0f;
    }
  }
}
template <int DT, int WT>
__device__ __noinline__ void norm_rows_again_apart(NormArgs a, float* s_sum) {
  norm_rows_again<DT, WT>(a, s_sum);
}

template <int DT, bool VEC, int PER>
__device__ __forceinline__ void norm_store(const NormArgs& a, long row, int g0, int gs, int l, float (*f)[16]) {
  float m[PER], inv[PER];
#pragma unroll
  for (int j = 0; j < PER; j++) m[j] = held_max(amax_lanes(amax_of<16>(f[j])));
  const float scale = quotients<PER>(m, inv);
#pragma unroll
  for (int j = 0; j < PER; j++) {
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = (g0 + j * gs) * kGroup + 64 * c + 8 * l;
      store_held<VEC>(a.q + row * a.ldq + k, a.K - k, f[j] + 8 * c, inv[j]);
    }
  }
  if (l < PER && g0 + l * gs < a.G) a.scale[row * a.G + g0 + l * gs] = scale;
}

template <bool VEC>
constexpr int kNormThreads = VEC ? 512 : 384;  // 384: at 80 registers two blocks' warps fit an SM's quarters
// The next row is on its way while the present one is summed and rounded, and the weights stay in registers.  (Only where
// rows are whole vectors: the others' registers go further as a second block an SM; 8000 x 4097 bf16 with a residual
// takes 98 us, 121 with the next row on its way.)  What two runs of groups a thread (PER = 2) need is more than the
// registers: rows that start anywhere keep some 300 bytes a thread in local memory then, fp32 ones 432 (2000 x 12001 fp16
// with a residual 103 us, 1.6 TB/s), fp32 rows in whole vectors 112 (3000 x 12288 129 us, 3.7 TB/s).
template <int DT, int WT, bool VEC, int PER>
__global__ void __launch_bounds__(kNormThreads<VEC>, VEC ? 0 : 2) f8_norm_kernel(NormArgs a) {
  __shared__ float s_sum[2][32];  // for each of two rows in turn
  __shared__ int s_again;         // rows are beyond() (all threads write it alike, each reads its own)
  int again = 0;                  // the same where a row is held in few registers
  extern __shared__ uint4 s_row[];
  char* room = !VEC && a.stage ? (char*)s_row : nullptr;
  s_again = 0;
  grid_dep_wait();
  const int l = threadIdx.x & (kLanes - 1), g0 = threadIdx.x / kLanes, gs = blockDim.x / kLanes;
  NormIn<DT, VEC> in[PER];
  NormWeight<WT, VEC> w[PER];
  long row = blockIdx.x;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    if (VEC) in[j].load(a, row, (g0 + j * gs) * kGroup, l);
    w[j].load(a, (g0 + j * gs) * kGroup, l);
  }
  grid_dep_launch();
  for (int half = 0; row < a.T; row += gridDim.x, half ^= 1) {
    float f[PER][16], ss = 0.f;
    if (!VEC) {
#pragma unroll
      for (int j = 0; j < PER; j++) in[j].load(a, row, (g0 + j * gs) * kGroup, l);
    }
#pragma unroll
    for (int j = 0; j < PER; j++) {
      in[j].sum(a, row, (g0 + j * gs) * kGroup, l, true, f[j], room);
#pragma unroll
      for (int e = 0; e < 16; e++) ss = fmaf(f[j][e], f[j][e], ss);
    }
    if (VEC && row + gridDim.x < a.T) {
#pragma unroll
      for (int j = 0; j < PER; j++) in[j].load(a, row + gridDim.x, (g0 + j * gs) * kGroup, l);
    }
    const float v = norm_mean(ss, s_sum[half], a), r = rsqrtf(v);
    if (beyond(v)) (PER == 1 ? again : s_again) = 1;
    if (room != nullptr) norm_row_out<DT>(a, row, room);
#pragma unroll
    for (int j = 0; j < PER; j++) w[j].scale(a, (g0 + j * gs) * kGroup, l, r, f[j]);
    norm_store<DT, VEC, PER>(a, row, g0, gs, l, f);
    if (room != nullptr) __syncthreads();  // the next row's sum goes to the same place
  }
  // (1001 x 4104 fp16 5.2 us, 5.7 with the other form; 2000 x 12001 fp16 103 us, 107.)
  if (PER == 1) {
    if (again) norm_rows_again_apart<DT, WT>(a, s_sum[0]);
  } else if (s_again) {
    norm_rows_again<DT, WT>(a, s_sum[0]);
  }
}

// Rows too wide for the registers are read twice.
template <int DT, int WT, bool VEC>
__global__ void __launch_bounds__(512) f8_norm_wide_kernel(NormArgs a) {
  __shared__ float s_sum[32];
  __shared__ int s_again;  // the row is beyond()
  s_again = 0;
  grid_dep_wait();
  const int l = threadIdx.x & (kLanes - 1), gs = blockDim.x / kLanes;
  const long row = blockIdx.x;
  float f[1][16], ss = 0.f;
  NormIn<DT, VEC> in;
  NormWeight<WT, VEC> w;
  const int rounds = (a.G + gs - 1) / gs;
  for (int j = 0, g = threadIdx.x / kLanes; j < rounds; j++, g += gs) {
    in.load(a, row, g * kGroup, l);
    in.sum(a, row, g * kGroup, l, true, f[0], nullptr);
#pragma unroll
    for (int e = 0; e < 16; e++) ss = fmaf(f[0][e], f[0][e], ss);
  }
  const float v = norm_mean(ss, s_sum, a), r = rsqrtf(v);
  if (beyond(v)) s_again = 1;
  grid_dep_launch();
  for (int j = 0, g = threadIdx.x / kLanes; j < rounds; j++, g += gs) {
    in.load(a, row, g * kGroup, l);
    w.load(a, g * kGroup, l);
    in.sum(a, row, g * kGroup, l, false, f[0], nullptr);
    w.scale(a, g * kGroup, l, r, f[0]);
    norm_store<DT, VEC, 1>(a, row, g, gs, l, f);
  }
  if (s_again) norm_rows_again<DT, WT>(a, s_sum);
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
    const long runs = a.T * ((a.G + kRowsPer - 1) / kRowsPer);
    constexpr int per = kRowsThreads / kLanes;
    return launch_pdl(f8_rows_kernel<DT, VEC>, dim3((unsigned)((runs + per - 1) / per)), dim3(kRowsThreads), 0, s,
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
constexpr int kSmSmem = 200 * 1024;  // what the blocks of an SM may have of its shared memory
constexpr int kStageSmem = 47 * 1024;  // what a block may have for its row beside the kernel's own, without asking
template <int DT, bool VEC>
struct NormLaunch {
  static int go(const NormArgs& a, bool w32, cudaStream_t s) {
    return w32 ? with<F8_F32>(a, s) : with<DT>(a, s);
  }
  template <int WT>
  static int with(const NormArgs& a, cudaStream_t s) {
    const int lanes = a.G * kLanes;  // lanes that a row fills, 16 values each
    // One row at a time for as many blocks as the GPU holds at once, no more: 8192 x 4096 bf16 with a residual takes
    // 38.2 us with three blocks of 256 threads an SM, 45.8 with two, 47.8 with four (a third of a wave of them alone).
    auto run = [&](auto kernel, int per) {
      static std::atomic<int> known[3][17];
      const int warps = ((lanes + per - 1) / per + 31) / 32;
      int n = known[per][warps].load(std::memory_order_relaxed);
      if (n == 0) {
        RNGD_TRY(check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, warps * 32, 0),
                            "occupancy(f8_norm_kernel)"));
        if (n < 1) n = 1;
        known[per][warps].store(n, std::memory_order_relaxed);
      }
      const int smem = a.stage ? a.G * kGroup * dtype_size(DT) : 0;
      if (smem > 0 && n > kSmSmem / smem) n = kSmSmem / smem;
      const long most = (long)num_sms() * n;
      return launch_pdl(kernel, dim3((unsigned)(a.T < most ? a.T : most)), dim3(warps * 32), smem, s, "f8_norm_kernel", a);
    };
    if (lanes <= kNormThreads<VEC>) return run(f8_norm_kernel<DT, WT, VEC, 1>, 1);
    if (lanes <= 2 * kNormThreads<VEC>) return run(f8_norm_kernel<DT, WT, VEC, 2>, 2);
    return launch_pdl(f8_norm_wide_kernel<DT, WT, VEC>, dim3((unsigned)a.T), dim3(512), 0, s, "f8_norm_wide_kernel", a);
  }
};

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_f8_rows(const void* x, int dtype, int64_t ldx, int64_t T, int K, void* q, int64_t ldq, float* scale,
                            rngd_stream_t stream) {
  RNGD_REQUIRE(dtype >= F8_BF16 && dtype <= F8_F32, "f8_rows: data type %d", dtype);
  RNGD_REQUIRE(T >= 0 && K >= 0 && K <= kMostK, "f8_rows: %ld rows of %d", (long)T, K);
  if (T == 0 || K == 0) return RNGD_OK;
  const int G = (int)(((long)K + kGroup - 1) / kGroup);
  RNGD_REQUIRE(T <= 0x7FFFFFFFl && T * ((G + kRowsPer - 1) / kRowsPer) <= 0x7FFFFFFFl, "f8_rows: %ld rows of %d", (long)T, K);
  RNGD_REQUIRE(x != nullptr && (uintptr_t)x % dtype_size(dtype) == 0, "f8_rows: x is null or misaligned");
  RNGD_TRY(check_held("f8_rows", (uint8_t*)q, ldq, T, K, scale));
  RowsArgs a = {x, (long)ldx, (long)T, K, G, (uint8_t*)q, (long)ldq, scale};
  return by_type<RowsLaunch>(dtype, whole_vectors(x, ldx, K, dtype), a, (cudaStream_t)stream);
}

extern "C" int rngd_f8_weight(const void* w, int dtype, int64_t ldw, int N, int K, void* q, int64_t ldq, float* scale,
                              rngd_stream_t stream) {
  RNGD_REQUIRE(dtype >= F8_BF16 && dtype <= F8_F32, "f8_weight: data type %d", dtype);
  RNGD_REQUIRE(N >= 0 && N <= kMostRows && K >= 0 && K <= kMostK, "f8_weight: %d x %d", N, K);
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
  RNGD_REQUIRE(T >= 0 && T <= 0x7FFFFFFFl && K >= 0 && K <= kMostK, "f8_rms_norm: %ld rows of %d", (long)T, K);
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
  NormArgs a = {x, residual, weight, (long)ldx, (long)ldr, K, G, eps, (long)T, 0,
                total, (long)ldt, (uint8_t*)q, (long)ldq, scale};
  const bool vec = whole_vectors(x, ldx, K, dtype) && whole_vectors(weight, 0, K, weight_dtype) &&
                   (residual == nullptr || (whole_vectors(residual, ldr, K, dtype) && whole_vectors(total, ldt, K, dtype)));
  a.stage = !vec && total != nullptr && (long)G * kGroup * sz <= kStageSmem;
  return by_type<NormLaunch>(dtype, vec, a, weight_dtype == F8_F32, (cudaStream_t)stream);
}
