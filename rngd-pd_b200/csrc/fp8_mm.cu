// Products of 8-bit operands with fp32 scales (fp8.cuh gives the format), on tcgen05.
//
//   y[m][n] = sum_g sa[m][g] * sb[n / 128][g] * d_g[m][n],   d_g[m][n] = sum_{k in group g} a[m][k] b[n][k]
//
// The tensor cores hold d_g of one group of 128 (four steps of kind::f8f6f4, exact products, fp32 sums) in tensor
// memory; the epilogue's threads multiply it with the two scales and add it to sums in their registers while the
// next group's products run into the other half of the tensor memory.
#include "fp8.cuh"
#include "tc.cuh"

namespace rngd {

__device__ int g_status_f8 = 0;

// Instruction descriptor: kind::f8f6f4, A = B = e4m3, D = fp32, both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

struct MmArgs {
  int M, N, K, G;
  const float* sa;  // [M][G], strides in elements
  long sa_m, sa_g;
  const float* sb;  // [ceil(N / 128)][G]
  long sb_n, sb_g;
  void* y;
  long ldy;
  const void* add;  // of y's type, or null
  long ldadd;
};

constexpr int kMmStages = 4, kMmTile = 128 * 128, kMmThreads = 192;
constexpr size_t kMmSmem = 1024 + kMmStages * 2 * kMmTile + (2 * kMmStages + 5) * 8 + 16;

template <int DT>
__global__ void __launch_bounds__(kMmThreads, 1) f8_mm_kernel(const __grid_constant__ CUtensorMap tmA,
                                                              const __grid_constant__ CUtensorMap tmB, MmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(base + kMmStages * 2 * kMmTile);
  uint64_t* empty = full + kMmStages;
  uint64_t* acc_full = empty + kMmStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;      // [2]
  uint64_t* done = acc_empty + 2;
  uint32_t* slot = (uint32_t*)(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tn = (a.N + 127) / 128, mt = blockIdx.x / tn, nt = blockIdx.x - mt * tn;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMmStages; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 128);
    }
    mbar_init(done, 128);
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  grid_dep_wait();
  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (; i < a.G; i++) {
        const int s = i % kMmStages;
        if (!mbar_wait(&empty[s], ((uint32_t)(i / kMmStages) & 1u) ^ 1u, ST_TMA_WAIT, &g_status_f8)) break;
        uint8_t* st = base + s * 2 * kMmTile;
        mbar_arrive_expect_tx(&full[s], 2 * kMmTile);
        tma_load_2d(st, &tmA, &full[s], i * kGroup, mt * 128);
        tma_load_2d(st + kMmTile, &tmB, &full[s], i * kGroup, nt * 128);
      }
      if (i < a.G)  // a wait ran out: the copies in flight land before the block may end
        for (int j = i < kMmStages ? 0 : i - kMmStages; j < i; j++)
          mbar_wait(&full[j % kMmStages], (uint32_t)(j / kMmStages) & 1u, ST_TMA_WAIT, &g_status_f8);
      grid_dep_launch();
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_e4m3_f32(128, 128);
      for (int i = 0; i < a.G; i++) {
        const int s = i % kMmStages, buf = i & 1;
        if (!mbar_wait(&acc_empty[buf], ((uint32_t)(i >> 1) & 1u) ^ 1u, ST_MMA_WAIT, &g_status_f8)) break;
        if (!mbar_wait(&full[s], (uint32_t)(i / kMmStages) & 1u, ST_MMA_WAIT, &g_status_f8)) break;
        tc_fence_after();
        const uint32_t sa = smem_u32(base + s * 2 * kMmTile), sb = sa + kMmTile;
#pragma unroll
        for (int kk = 0; kk < 4; kk++)
          umma_e4m3(tmem + buf * 128, sw128_kmajor_desc(sa + kk * 32), sw128_kmajor_desc(sb + kk * 32), idesc, kk != 0);
        umma_commit(&empty[s]);
        umma_commit(&acc_full[buf]);
      }
      mbar_wait(done, 0u, ST_EPI_WAIT, &g_status_f8);
      tc_fence_after();
    }
    __syncwarp();
    tmem_dealloc(tmem, 256);
  } else {
    const int r = ((warp & 3) << 5) | lane, m = mt * 128 + r;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    float acc[128];
#pragma unroll
    for (int j = 0; j < 128; j++) acc[j] = 0.f;
    for (int i = 0; i < a.G; i++) {
      const int buf = i & 1;
      const float s = m < a.M ? a.sa[m * a.sa_m + i * a.sa_g] * a.sb[nt * a.sb_n + i * a.sb_g] : 0.f;
      const bool ok = mbar_wait(&acc_full[buf], (uint32_t)(i >> 1) & 1u, ST_EPI_WAIT, &g_status_f8);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 4; c++) {
        float v[32];
        tmem_ld_32x32b_x32(tmem + lane_base + buf * 128 + c * 32, v);
#pragma unroll
        for (int j = 0; j < 32; j++) acc[c * 32 + j] = fmaf(s, v[j], acc[c * 32 + j]);
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[buf]);
    }
    mbar_arrive(done);
    if (m < a.M) {
#pragma unroll
      for (int j = 0; j < 128; j++) {
        const int n = nt * 128 + j;
        if (n < a.N) {
          float v = acc[j];
          if (a.add != nullptr) v += load_as_f32<DT>(a.add, m * a.ldadd + n);
          store_f32_as<DT>(a.y, m * a.ldy + n, v);
        }
      }
    }
  }
}

// silu(gate) * up of fp32 rows, quantised by groups: 16 lanes a group, eight values each.
struct SwigluArgs {
  const float *g, *u;  // [M][N], N a multiple of 4
  int N, NG;
  long total;  // groups
  int cols;
  uint8_t* q;
  long ldq;
  float* scale;
};
__global__ void __launch_bounds__(256) f8_swiglu_kernel(SwigluArgs a) {
  grid_dep_wait();
  const int l = threadIdx.x & 15;
  const long i = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool there = i < a.total;
  const long row = there ? i / a.NG : 0;
  const int grp = (int)(i - row * a.NG);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int n = grp * kGroup + l + 16 * e;
    v[e] = there && n < a.cols ? swiglu(a.g[row * a.N + n], a.u[row * a.N + n]) : 0.f;
  }
  const float m = held_max(amax16(amax_of(v))), inv = 448.0f / m;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const int n = grp * kGroup + l + 16 * e;
    if (there && n < a.cols) a.q[row * a.ldq + n] = e4m3(v[e] * inv);
  }
  if (there && l == 0) a.scale[row * a.NG + grp] = m / 448.0f;
}

// -------------------------------------------------------------------------------------------- host
struct Operand {
  const void* q;
  int64_t ld;
  const float* scale;
  int64_t s0, s1;
};
static int check_operand(const char* what, const Operand& o, long rows, int K) {
  RNGD_REQUIRE(o.q != nullptr && o.scale != nullptr, "%s: null pointer", what);
  RNGD_REQUIRE(((uintptr_t)o.q & 15) == 0 && ((uintptr_t)o.scale & 3) == 0, "%s: misaligned operand", what);
  RNGD_REQUIRE(rows <= 1 || (o.ld % 16 == 0 && o.ld >= K && o.ld < (1l << 40)),
               "%s: rows of %d bytes, %ld apart (a multiple of 16)", what, K, (long)o.ld);
  return RNGD_OK;
}
// rows x K bytes, rows ld apart, read in boxes of 128 bytes x `box` rows; zeros beyond the edges
static int operand_map(const Operand& o, long rows, int K, int box, CUtensorMap* out) {
  const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows};
  const uint64_t strides[1] = {rows <= 1 ? ((uint64_t)K + 15) / 16 * 16 : (uint64_t)o.ld};
  const uint32_t bx[2] = {kGroup, (uint32_t)box};
  return encode_tmap_u8(out, o.q, 2, dims, strides, bx);
}

static int mm_launch(const Operand& a, const Operand& b, int M, int N, int K, const void* add, long ldadd, void* y,
                     long ldy, int dtype, cudaStream_t s) {
  CUtensorMap ta, tb;
  RNGD_TRY(operand_map(a, M, K, 128, &ta));
  RNGD_TRY(operand_map(b, N, K, 128, &tb));
  MmArgs g = {M, N, K, (K + 127) / 128, a.scale, (long)a.s0, (long)a.s1, b.scale, (long)b.s0, (long)b.s1, y, ldy, add, ldadd};
  const long tiles = ((long)M + 127) / 128 * (((long)N + 127) / 128);
  RNGD_REQUIRE(tiles <= 0x7FFFFFFFl, "f8_matmul: %d x %d results", M, N);
  auto kernel = dtype == F8_BF16 ? f8_mm_kernel<F8_BF16> : dtype == F8_F16 ? f8_mm_kernel<F8_F16> : f8_mm_kernel<F8_F32>;
  static std::atomic<unsigned long long> smem_set[3];
  RNGD_TRY(set_smem_limit_once((const void*)kernel, kMmSmem, &smem_set[dtype], "cudaFuncSetAttribute(f8_mm_kernel)"));
  return launch_pdl(kernel, dim3((unsigned)tiles), dim3(kMmThreads), kMmSmem, s, "f8_mm_kernel", ta, tb, g);
}

int read_status_f8(int* st, int reset) {
  RNGD_TRY(check_cuda(cudaMemcpyFromSymbol(st, g_status_f8, sizeof(int)), "read device status"));
  if (reset) {
    const int zero = 0;
    RNGD_TRY(check_cuda(cudaMemcpyToSymbol(g_status_f8, &zero, sizeof(int)), "reset device status"));
  }
  return RNGD_OK;
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_f8_matmul(const void* a, int64_t lda, const float* a_scale, const int64_t* a_strides, const void* b,
                              int64_t ldb, const float* b_scale, const int64_t* b_strides, int M, int N, int K,
                              const void* add, int64_t ldadd, void* y, int64_t ldy, int dtype, rngd_stream_t stream) {
  RNGD_REQUIRE(dtype >= F8_BF16 && dtype <= F8_F32, "f8_matmul: data type %d", dtype);
  RNGD_REQUIRE(M >= 0 && N >= 0 && K >= 1, "f8_matmul: %d x %d x %d", M, N, K);
  RNGD_REQUIRE(K <= 0x7FFFFFFF - 127, "f8_matmul: K=%d", K);
  if (M == 0 || N == 0) return RNGD_OK;
  const uintptr_t mis = dtype == F8_F32 ? 3 : 1;
  RNGD_REQUIRE(y != nullptr && a_strides != nullptr && b_strides != nullptr, "f8_matmul: null pointer");
  RNGD_REQUIRE((((uintptr_t)y | (uintptr_t)add) & mis) == 0, "f8_matmul: misaligned result");
  RNGD_REQUIRE(M <= 1 || ldy >= N, "f8_matmul: rows of the result lie on one another");
  const Operand oa = {a, lda, a_scale, a_strides[0], a_strides[1]}, ob = {b, ldb, b_scale, b_strides[0], b_strides[1]};
  RNGD_TRY(check_operand("f8_matmul", oa, M, K));
  RNGD_TRY(check_operand("f8_matmul", ob, N, K));
  return mm_launch(oa, ob, M, N, K, add, (long)ldadd, y, (long)ldy, dtype, (cudaStream_t)stream);
}

static size_t swiglu_pitch(int N) { return ((size_t)N + 3) / 4 * 4; }

extern "C" int rngd_f8_swiglu_workspace(int M, int N, int K, size_t* bytes) {
  RNGD_REQUIRE(bytes != nullptr, "f8_swiglu_workspace: null output");
  RNGD_REQUIRE(M >= 0 && N >= 0 && K >= 1, "f8_swiglu: %d x %d x %d", M, N, K);
  *bytes = 2 * (size_t)M * swiglu_pitch(N) * 4;
  return RNGD_OK;
}

extern "C" int rngd_f8_swiglu(const void* a, int64_t lda, const float* a_scale, const int64_t* a_strides,
                              const void* gate, int64_t ldg, const float* gate_scale, const int64_t* gate_strides,
                              const void* up, int64_t ldu, const float* up_scale, const int64_t* up_strides, int M, int N,
                              int K, void* q, int64_t ldq, float* scale, void* workspace, size_t workspace_bytes,
                              rngd_stream_t stream) {
  size_t need = 0;
  RNGD_TRY(rngd_f8_swiglu_workspace(M, N, K, &need));
  RNGD_REQUIRE(K <= 0x7FFFFFFF - 127 && N <= 0x7FFFFFFF - 127, "f8_swiglu: %d x %d x %d", M, N, K);
  if (M == 0 || N == 0) return RNGD_OK;
  RNGD_REQUIRE(q && scale && a_strides && gate_strides && up_strides, "f8_swiglu: null pointer");
  RNGD_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)scale & 3) == 0 && (M <= 1 || (ldq >= N && ldq % 16 == 0)),
               "f8_swiglu: 8-bit rows must start on 16 bytes and not overlap");
  RNGD_REQUIRE(workspace != nullptr && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need,
               "f8_swiglu: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
  const Operand oa = {a, lda, a_scale, a_strides[0], a_strides[1]};
  const Operand og = {gate, ldg, gate_scale, gate_strides[0], gate_strides[1]};
  const Operand ou = {up, ldu, up_scale, up_strides[0], up_strides[1]};
  RNGD_TRY(check_operand("f8_swiglu", oa, M, K));
  RNGD_TRY(check_operand("f8_swiglu", og, N, K));
  RNGD_TRY(check_operand("f8_swiglu", ou, N, K));
  const long pitch = (long)swiglu_pitch(N);
  float* g = (float*)workspace;
  float* u = g + M * pitch;
  cudaStream_t s = (cudaStream_t)stream;
  RNGD_TRY(mm_launch(oa, og, M, N, K, nullptr, 0, g, pitch, F8_F32, s));
  RNGD_TRY(mm_launch(oa, ou, M, N, K, nullptr, 0, u, pitch, F8_F32, s));
  const int NG = (N + 127) / 128;
  SwigluArgs w = {g, u, (int)pitch, NG, (long)M * NG, N, (uint8_t*)q, (long)ldq, scale};
  RNGD_REQUIRE((w.total + 15) / 16 <= 0x7FFFFFFFl, "f8_swiglu: %d x %d results", M, N);
  return launch_pdl(f8_swiglu_kernel, dim3((unsigned)((w.total + 15) / 16)), dim3(256), 0, s, "f8_swiglu_kernel", w);
}
