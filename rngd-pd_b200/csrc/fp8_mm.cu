// Products of 8-bit operands with fp32 scales (fp8.cuh gives the format), on tcgen05.
//
//   y[m][n] = sum_g sa[m][g] * sb[n / 128][g] * d_g[m][n],   d_g[m][n] = sum_{k in group g} a[m][k] b[n][k]
//
// The tensor cores hold d_g of one group of 128 (four steps of kind::f8f6f4: exact products, fp32 sums) in tensor
// memory; threads multiply it with the two scales and add it to sums in their registers while the next groups'
// products run into other columns of the tensor memory.  Results in fp32 are within 1.1e-7 of 64 bits
// (16 x 128256 x 4096, 2-norm), a tenth of what sums in plain fp32 are off.
//
// Two kernels: pairs of CTAs with tiles of 256 x 256 where there are many rows, and one whose tiles have the weight's
// rows as lanes and 16 to 128 rows of a where there are few; pairs_pay() below chooses.
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

// ---------------------------------------------------------------------- pieces of the kernels
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ bool elect_one() {  // one lane of the warp, all of which are here
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {  // the same place in another CTA
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Starts a tile's way from this GPU's memory into its L2 cache.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* tm, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(tm)),
               "r"(c0), "r"(c1)
               : "memory");
}
// A tile load of this GPU's memory into this CTA, counted by a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* tm, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {  // a warp of both CTAs
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void umma_e4m3_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this place of both CTAs once every product issued so far has completed.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\t"
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}\n" ::"r"(
          smem_u32(bar))
      : "memory");
}

// 64 columns of this warp's 32 lanes.  The wait is part of the same statement, so nothing reads the registers earlier.
__device__ __forceinline__ void tmem_ld_x64(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 parts_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
// acc[0..31] += s * 64 columns, two an instruction
__device__ __forceinline__ void scale_add(uint64_t* acc, const uint32_t* r, float s) {
  const uint64_t ss = pair_of(s, s);
#pragma unroll
  for (int j = 0; j < 32; j++) {
    const uint64_t v = pair_of(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[j]) : "l"(v), "l"(ss));
  }
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
  int unanswered;   // rngd_f8_unanswered: the sums wait for a barrier that nothing completes
};

// When a wait runs out.  Whoever gave up waits for nothing more, but comes to every barrier that the others wait at, and
// its sums are NaN from there on, so that no result can pass for a good one.  It no longer says that it has read the
// tensor memory: the products then stop (by their own wait), instead of going on into columns that slower warps still read.
__device__ __forceinline__ float lost() { return __int_as_float(0x7FFFFFFF); }

constexpr int kMmTile = 128 * 128;  // bytes of 128 rows of a group

// ------------------------------------------------------------- few rows: the weight's rows as lanes
// One CTA works on 128 rows of the weight (DUAL: of gate and of up) and NT rows of a: the weight is the products'
// first operand, so NT may be as small as 16 and the weight's bytes, which bound this, are read once.  The groups of
// K are cut into `split` runs, one for each CTA of a cluster, whose sums meet in shared memory, in the order of the
// runs: the same bits every time, one launch, no workspace.  A thread holds NT sums of its row of the weight (NT / 2
// from 64 on); the scales of 32 groups at a time, each row's times the block's, lie in shared memory.
//
// 16 x 128256 x 4096 with an fp32 result: 83 us, 6.4 TB/s, 0.98 of the copy rate.  16 x 14336 x 4096 gate and up: 24.5 us,
// 4.8 TB/s; 18 at the copy rate, the rest is the way in (scales, first copies) and out (cluster, code that runs once).
// 1 x 4096 x 4096: 6.7 us, latency.  With 128 rows of a every CTA fetches as much of a as of the weight:
// 128 x 18944 x 4096, one tile an SM, takes 23.8 us, 6.5 TB/s into shared memory; 200 x 4096 x 4096, K cut in two, 14.0 us.
template <int NT, bool DUAL>
struct FewCfg {
  static constexpr int A = (DUAL ? 2 : 1) * kMmTile, STAGE = A + NT * 128;
  static constexpr int COLS = (DUAL ? 2 : 1) * NT;     // columns of one buffer in tensor memory
  static constexpr int GROUPS = NT >= 64 ? 2 : 1;      // warpgroups that share them, by rows of a
  static constexpr int SUMMERS = 128 * GROUPS, THREADS = 64 + SUMMERS, TN = NT / GROUPS;
  static constexpr int STEP = NT == 16 || NT == 64 ? 16 : 32;  // columns read at a time (with NT = 64 reads of 32 would spill)
  static constexpr int BUFS = NT <= 32 ? 4 : 2;
  static constexpr int CHUNK = 32;                     // groups whose scales are in shared memory
  static constexpr int PITCH = COLS + 4;               // floats of a group's; fewer of the stores' banks meet
  static constexpr int SCALES = CHUNK * PITCH * 4;
  static constexpr int FIXED = 1024 + SCALES + 256;
  // two CTAs an SM where three stages of each fit (an SM has 227 KB, a block's own KB taken off), else one
  static constexpr int PER_SM = (113 * 1024 - FIXED) / STAGE >= 3 ? 2 : 1;
  static constexpr int MOST = ((PER_SM == 2 ? 113 : 226) * 1024 - FIXED) / STAGE;
  static constexpr int STAGES = MOST < 8 ? MOST : 8;
  static constexpr size_t SMEM = FIXED + STAGES * STAGE;
  static_assert(STAGES * STAGE >= COLS * 128 * 4, "the sums fit where the stages were");
  static_assert(BUFS * COLS * PER_SM <= 512 && BUFS * COLS >= 32 && ((BUFS * COLS) & (BUFS * COLS - 1)) == 0, "");
  static_assert((2 * STAGES + 3 * BUFS + 2) * 8 + 16 <= 256, "barriers");
};
struct FewArgs {
  MmArgs m;
  const float* sb1;  // of the second weight (DUAL)
  long sb1_n, sb1_g;
  int tn, split;
  int vec;           // rows of y and add are whole 16-byte vectors
  uint8_t* q;        // DUAL: 8-bit rows and their scales [M][ceil(N / 128)]
  long ldq;
  float* scale;
};
// Eight neighbouring sums at this place of each CTA of the cluster, added in the CTAs' order.
// self: -1, or the CTA whose own place stands for all of them.
__device__ __forceinline__ void few_sum(float* y, uint32_t at, int split, int self) {
  float4 v[8][2];
#pragma unroll
  for (int k = 0; k < 8; k++) {
    v[k][0] = v[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (k < split) {
      const uint32_t from = mapa(at, self < 0 ? k : self);
#pragma unroll
      for (int c = 0; c < 2; c++)
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[k][c].x), "=f"(v[k][c].y), "=f"(v[k][c].z), "=f"(v[k][c].w)
                     : "r"(from + 16 * c));
    }
  }
#pragma unroll
  for (int c = 0; c < 2; c++) {
    float* z = y + 4 * c;
    z[0] = z[1] = z[2] = z[3] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      z[0] += v[k][c].x;
      z[1] += v[k][c].y;
      z[2] += v[k][c].z;
      z[3] += v[k][c].w;
    }
  }
}
// Eight sums of row m from column n on: plus add, rounded, stored.
template <int DT>
__device__ __forceinline__ void store_sums(const MmArgs& a, float* v, long m, int n, int vec) {
  const long o = m * a.ldy + n, oa = m * a.ldadd + n;
  if (vec && n + 8 <= a.N) {
    if (a.add != nullptr) {
      Eight<DT> r;
      float w[8];
      r.load_any(a.add, oa);
      r.values(w);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] += w[e];
    }
    store_eight<DT>(a.y, o, eight_of<DT>(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)  // (all loads before the first store, which might be to the same place)
      if (a.add != nullptr && n + e < a.N) v[e] += load_as_f32<DT>(a.add, oa + e);
#pragma unroll
    for (int e = 0; e < 8; e++)
      if (n + e < a.N) store_f32_as<DT>(a.y, o + e, v[e]);
  }
}
template <int THREADS>
__device__ __forceinline__ void few_bar() {
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

// acc[0 .. N / 2) += (N columns from taddr) * s[0 .. N), two columns an instruction
template <int N, int STEP>
__device__ __forceinline__ void scale_add_cols(uint64_t* acc, uint32_t taddr, const float* s) {
#pragma unroll
  for (int c = 0; c < N; c += STEP) {
    uint32_t r[STEP];
    if constexpr (STEP == 16)
      tmem_ld_x16(taddr + c, r);
    else
      tmem_ld_x32(taddr + c, r);
#pragma unroll
    for (int j = 0; j < STEP / 4; j++) {
      const ulonglong2 f = *(const ulonglong2*)(s + c + 4 * j);
      const uint64_t v0 = pair_of(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]));
      const uint64_t v1 = pair_of(__uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
      asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[c / 2 + 2 * j]) : "l"(v0), "l"(f.x));
      asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[c / 2 + 2 * j + 1]) : "l"(v1), "l"(f.y));
    }
  }
}

template <int NT, bool DUAL, int DT>
__global__ void __launch_bounds__(FewCfg<NT, DUAL>::THREADS, FewCfg<NT, DUAL>::PER_SM)
    f8_few_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                  const __grid_constant__ CUtensorMap tmW1, FewArgs p) {
  using C = FewCfg<NT, DUAL>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* s_scale = (float*)(base + ST * C::STAGE);   // [CHUNK][PITCH]
  uint64_t* full = (uint64_t*)(s_scale + C::CHUNK * C::PITCH);
  uint64_t* empty = full + ST;
  uint64_t* acc_full = empty + ST;           // [BUFS]
  uint64_t* acc_empty = acc_full + C::BUFS;  // [BUFS]
  uint64_t* done = acc_empty + C::BUFS;
  uint64_t* quiet = done + 1;                // no copy and no product is on its way any more
  uint64_t* never = quiet + 1;               // [BUFS]
  uint32_t* slot = (uint32_t*)(never + C::BUFS);
  const MmArgs& a = p.m;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % p.split, tile = blockIdx.x / p.split;
  const int mt = tile / p.tn, nt = tile - mt * p.tn;
  const int g0 = (int)((long)a.G * rank / p.split), g1 = (int)((long)a.G * (rank + 1) / p.split);
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < C::BUFS; i++) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], C::SUMMERS / 32);
      mbar_init(&never[i], 1);
    }
    mbar_init(done, C::SUMMERS / 32);
    mbar_init(quiet, 2);
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
    if (DUAL) tma_prefetch_desc(&tmW1);
  }
  if (warp == 1) {
    tmem_alloc(slot, C::BUFS * C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  if (warp == 0) {
    // The weight's first eight groups are on their way into the L2 cache while the launch before this one ends: gate and
    // up 16 x 14336 x 4096 25.3 -> 24.5 us, 16 x 4096 x 14336 14.1 -> 13.2 (with 16 groups 28.7 and 13.9).  Should that
    // launch write them, the cache has what it wrote: only copies into shared memory have to wait.
    if (lane == 0)
      for (int g = g0; g < g1 && g < g0 + 8; g++) {
        tma_prefetch_2d(&tmW, g * kGroup, nt * 128);
        if (DUAL) tma_prefetch_2d(&tmW1, g * kGroup, nt * 128);
      }
    grid_dep_wait();
    grid_dep_launch();
    if (lane == 0) {
      int i = 0;
      bool ok = true;
      for (int g = g0; g < g1; g++, i++) {
        const int s = i % ST;
        ok = mbar_wait(&empty[s], ((uint32_t)(i / ST) & 1u) ^ 1u, ST_TMA_WAIT, &g_status_f8);
        if (!ok) break;
        uint8_t* st = base + s * C::STAGE;
        mbar_arrive_expect_tx(&full[s], C::STAGE);
        tma_load_2d(st, &tmW, &full[s], g * kGroup, nt * 128);
        if (DUAL) tma_load_2d(st + kMmTile, &tmW1, &full[s], g * kGroup, nt * 128);
        tma_load_2d(st + C::A, &tmA, &full[s], g * kGroup, mt * NT);
      }
      if (!ok)  // a wait ran out: the copies in flight land before the block may end
        for (int j = i < ST ? 0 : i - ST; j < i; j++)
          mbar_wait(&full[j % ST], (uint32_t)(j / ST) & 1u, ST_TMA_WAIT, &g_status_f8);
      mbar_arrive(quiet);
    }
    __syncwarp();
  } else if (warp == 1) {
    grid_dep_wait();
    grid_dep_launch();
    const uint32_t idesc = idesc_e4m3_f32(128, NT);
    const uint64_t desc = sw128_kmajor_desc(smem_u32(base));
    int i = 0;
    for (; i < g1 - g0; i++) {
      const int s = i % ST, buf = i % C::BUFS;
      bool ok = mbar_wait(&acc_empty[buf], ((uint32_t)(i / C::BUFS) & 1u) ^ 1u, ST_MMA_WAIT, &g_status_f8) &&
                mbar_wait(&full[s], (uint32_t)(i / ST) & 1u, ST_MMA_WAIT, &g_status_f8);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint64_t dw = desc + (uint64_t)(s * (C::STAGE >> 4)), da = dw + (C::A >> 4);
      const uint32_t d = tmem + (uint32_t)(buf * C::COLS);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {
          umma_e4m3(d, dw + 2 * kk, da + 2 * kk, idesc, kk != 0);
          if (DUAL) umma_e4m3(d + NT, dw + (kMmTile >> 4) + 2 * kk, da + 2 * kk, idesc, kk != 0);
        }
        umma_commit(&empty[s]);
        umma_commit(&acc_full[buf]);
      }
      __syncwarp();
    }
    // The last product has completed before the tensor memory goes, or anything is written where the tiles were.  (Where no
    // wait ran out, the sums have seen it.)
    if (i > 0) mbar_wait(&acc_full[(i - 1) % C::BUFS], (uint32_t)((i - 1) / C::BUFS) & 1u, ST_MMA_WAIT, &g_status_f8);
    __syncwarp();
    if (lane == 0) mbar_arrive(quiet);
    mbar_wait(done, 0u, ST_EPI_WAIT, &g_status_f8);
    tc_fence_after();
    __syncwarp();
    tmem_dealloc(tmem, C::BUFS * C::COLS);
  } else {
    // thread: row r of the weight's 128, rows wt .. wt + TN - 1 of a's NT
    constexpr int TN = C::TN;
    const int r = ((warp & 3) << 5) | lane, et = threadIdx.x - 64, wt = (et >> 7) * TN;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    // The end of the kernel runs once in front without storing anything: its code, which would come from memory at
    // the end while everything waits, comes while the data do.  (Not where a block has the SM for itself, and so starts
    // after the launch before it: nothing is gained there.)
#pragma unroll 1
    for (int work = C::PER_SM == 1; work < 2; work++) {
      if (work) {
        grid_dep_wait();
        grid_dep_launch();
        uint64_t acc[(DUAL ? 2 : 1) * TN / 2];
#pragma unroll
        for (int j = 0; j < (DUAL ? 2 : 1) * TN / 2; j++) acc[j] = 0ull;
        bool ok = true;
        uint64_t* seen = a.unanswered ? never : acc_full;
        for (int c0 = g0; c0 < g1; c0 += C::CHUNK) {
          const int n = min(C::CHUNK, g1 - c0);
          if (c0 != g0) few_bar<C::SUMMERS>();  // every warp is past the previous scales
          // a row's scales by neighbouring threads, eight loads a thread at a time, so that their latencies overlap
          for (int e0 = et; e0 < NT * C::CHUNK; e0 += 8 * C::SUMMERS) {
            const int g = et % C::CHUNK, gg = c0 + min(g, n - 1);
            const float b = __ldg(a.sb + nt * a.sb_n + gg * a.sb_g);
            const float b1 = DUAL ? __ldg(p.sb1 + nt * p.sb1_n + gg * p.sb1_g) : 0.f;
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
              const int t = (e0 + u * C::SUMMERS) / C::CHUNK, m = mt * NT + t;
              x[u] = t < NT && m < a.M ? __ldg(a.sa + m * a.sa_m + gg * a.sa_g) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
              const int t = (e0 + u * C::SUMMERS) / C::CHUNK;
              if (t < NT) {
                s_scale[g * C::PITCH + t] = x[u] * b;
                if (DUAL) s_scale[g * C::PITCH + NT + t] = x[u] * b1;
              }
            }
          }
          few_bar<C::SUMMERS>();
          for (int k = 0; k < n; k++) {
            const int i = c0 - g0 + k, buf = i % C::BUFS;
            if (ok) ok = mbar_wait(&seen[buf], (uint32_t)(i / C::BUFS) & 1u, ST_EPI_WAIT, &g_status_f8);
            __syncwarp();
            tc_fence_after();
            const uint32_t d = tmem + lane_base + (uint32_t)(buf * C::COLS + wt);
            const float* s = s_scale + k * C::PITCH + wt;
            scale_add_cols<TN, C::STEP>(acc, d, s);
            if (DUAL) scale_add_cols<TN, C::STEP>(acc + TN / 2, d + NT, s + NT);
            tc_fence_before();
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive(&acc_empty[buf]);
          }
        }
        if (lane == 0) mbar_arrive(done);
        if (!ok) {
          mbar_wait(quiet, 0u, ST_EPI_WAIT, &g_status_f8);
#pragma unroll
          for (int j = 0; j < (DUAL ? 2 : 1) * TN / 2; j++) acc[j] = pair_of(lost(), lost());
        }
        float* part = (float*)base;  // [COLS][128]: the stages are done with
        few_bar<C::SUMMERS>();       // (every warp has seen the last products)
#pragma unroll
        for (int j = 0; j < (DUAL ? 2 : 1) * TN / 2; j++) {
          const float2 v = parts_of(acc[j]);
          const int c = wt + 2 * j + (DUAL && j >= TN / 2 ? NT - TN : 0);
          part[c * 128 + r] = v.x;
          part[(c + 1) * 128 + r] = v.y;
        }
        if (p.split > 1)
          cluster_sync();
        else
          few_bar<C::SUMMERS>();
      }
      // This CTA's rows of a: their sums over the cluster, in the order of the runs, and the result.  16 threads have a
      // row's 128 columns, eight each.  (A short loop: code that runs once costs its way from memory.)
      const int l = et & 15, n = nt * 128 + 8 * l;
      const int t0 = NT * rank / p.split, t1 = min(NT * (rank + 1) / p.split, a.M - mt * NT);
      const uint32_t at = smem_u32(base) + l * 32;
      for (int tb = t0; tb < (work ? t1 : t0 + 1); tb += C::SUMMERS / 16) {
        const int t = tb + (et >> 4);
        const bool there = work && t < t1;
        const long m = mt * NT + t;
        float y[8], u[8];
        few_sum(y, at + (there ? t : 0) * 512, p.split, there ? -1 : (int)rank);
        if constexpr (DUAL) {
          few_sum(u, at + (NT + (there ? t : 0)) * 512, p.split, there ? -1 : (int)rank);
          float most = 0.f;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            y[e] = swiglu(y[e], u[e]);  // (zeros beyond N: the tile loads filled the weights' rows with them)
            most = max_nan(most, fabsf(y[e]));
          }
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
          const float lim = held_max(most), inv = 448.0f / lim;
          if (there) {
            uint8_t* q = p.q + m * p.ldq + n;
            if (n + 8 <= a.N) {
              *(uint2*)q = held8(y, inv);
            } else {
#pragma unroll
              for (int e = 0; e < 8; e++)
                if (n + e < a.N) q[e] = e4m3(y[e] * inv);
            }
            if (l == 0) p.scale[m * p.tn + nt] = lim / 448.0f;
          }
        } else if (there) {
          store_sums<DT>(a, y, m, n, p.vec);
        }
      }
    }
  }
  if (p.split > 1) {
    if (warp < 2) cluster_sync();
    cluster_sync();  // nobody reads this CTA's sums any more
  }
}

// ------------------------------------------------------------------ many rows: pairs of CTAs
// Two CTAs (a cluster) work on 256 rows x 256 columns: each holds 128 rows of a and 128 of the weight's in shared
// memory (32 KB a group), one thread of the first issues the products of both, and each ends with its own 128
// rows x 256 columns.  A persistent grid, one CTA per SM.
//
// 8192 x 4096 x 14336: 507 to 516 us, 1900 to 1865 TFLOP/s, in runs of a second and more, which the power limit holds to
// 1.37 to 1.53 GHz; 430 us in bursts of 30 ms.  4096 x 14336 x 4096 gate and up with SwiGLU and its rounding: 516 to 527
// us, 1865 to 1825 TFLOP/s, and 440 to 460.  A tile's results take 4000 to 8000 cycles to go out, while the products run
// two groups ahead.  A group's products take 512 cycles, and 780 to 800 pass for each: the way from them through the
// eight warps that add them up (two tensor memory reads of 85 cycles and 128 multiply-adds each, two warps a quarter of
// the SM) and back is longer than the other buffer's products.  Tried: products of 128 columns with barriers of their own
// (they run at half the rate, by shared memory's bandwidth: 472 us in bursts where this took 457), sixteen warps of 64
// columns (518 where eight took 467), multiply-adds of one column (509 where two at a time took 463).  The sums and what
// is read take 192 registers; with 224 a thread instead of 232 the compiler moves them about (484 us where 232 took 427).
struct PairArgs {
  MmArgs m;
  const float* sb1;  // of the second weight (SWIGLU)
  long sb1_n, sb1_g;
  int tm, tn;        // tiles
  int vec;           // rows of y and add are whole 16-byte vectors
  uint8_t* q;        // SWIGLU: 8-bit rows and their scales [M][NG]
  long ldq;
  float* scale;
};
constexpr int kPairStages = 5, kPairStage = 2 * kMmTile, kPairThreads = 128 + 256;
constexpr int kPairPitch = 36;  // floats of a row of 32 on its way out: 16-byte accesses meet in no bank
constexpr size_t kPairSmem =
    1024 + kPairStages * kPairStage + (2 * kPairStages + 6) * 8 + 16 + 2 * 2 * 128 * 4 + 8 * 32 * kPairPitch * 4;

// A warp's 32 rows x 128 sums (row m0 + lane, from column n0 on) go out 32 columns at a time through shared memory, so
// that the stores of a row lie together whatever its alignment.
template <int DT>
__device__ __forceinline__ void pair_store(const PairArgs& p, const uint64_t* acc, long m0, int n0, float* room) {
  const MmArgs& a = p.m;
  const int lane = threadIdx.x & 31;
  // What is added comes while the sums are laid out; in fp32 the registers reach for two rows at a time only.
  constexpr bool AHEAD = DT != F8_F32;
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const int n = n0 + 32 * c, n8 = n + (lane & 3) * 8;
    const bool whole = p.vec && n + 32 <= a.N, plus = whole && a.add != nullptr;
    Eight<DT> add[AHEAD ? 4 : 2];
    auto fetch = [&](Eight<DT>& to, int i) {
      const long m = m0 + 8 * i + (lane >> 2);
      if (plus && m < a.M) to.load_any(a.add, m * a.ldadd + n8);
    };
    if (AHEAD) {
#pragma unroll
      for (int i = 0; i < 4; i++) fetch(add[i], i);
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float2 x = parts_of(acc[16 * c + 2 * j]), y = parts_of(acc[16 * c + 2 * j + 1]);
      *(float4*)(room + lane * kPairPitch + 4 * j) = make_float4(x.x, x.y, y.x, y.y);
    }
    __syncwarp();
    if (whole) {
#pragma unroll(AHEAD ? 4 : 2)
      for (int i = 0; i < 4; i++) {
        const int r = 8 * i + (lane >> 2);
        const float* f = room + r * kPairPitch + (lane & 3) * 8;
        float v[8];
        *(float4*)v = *(const float4*)f;
        *(float4*)(v + 4) = *(const float4*)(f + 4);
        if (plus) {
          float w[8];
          if (!AHEAD && i % 2 == 0) {
            fetch(add[0], i);
            fetch(add[1], i + 1);
          }
          add[AHEAD ? i : i % 2].values(w);
#pragma unroll
          for (int e = 0; e < 8; e++) v[e] += w[e];
        }
        if (m0 + r < a.M) store_eight<DT>(a.y, (m0 + r) * a.ldy + n8, eight_of<DT>(v));
      }
    } else if (n + lane < a.N && a.add == nullptr) {  // a column a lane
#pragma unroll 2
      for (int r = 0; r < 32; r++)
        if (m0 + r < a.M) store_f32_as<DT>(a.y, (m0 + r) * a.ldy + n + lane, room[r * kPairPitch + lane]);
    } else if (n + lane < a.N) {
      // with what is added, eight rows at a time: 6206 x 1423 x 4519 fp32 93 us, 219 two at a time
      for (int r0 = 0; r0 < 32 && m0 + r0 < a.M; r0 += 8) {
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const long m = m0 + r0 + i;
          w[i] = m < a.M ? load_as_f32<DT>(a.add, m * a.ldadd + n + lane) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const long m = m0 + r0 + i;
          if (m < a.M) store_f32_as<DT>(a.y, m * a.ldy + n + lane, room[(r0 + i) * kPairPitch + lane] + w[i]);
        }
      }
    }
    __syncwarp();
  }
}

// 64 gate sums and 64 up sums of row m, columns n0 ..: the other 64 of the group are another warp's, so the maximum
// meets in shared memory.  (Columns beyond N come last in a row, and their sums are zeros: the tile loads filled the
// weights' rows with them.  A row that is not there may hold anything.)
__device__ __forceinline__ void pair_store_swiglu(const PairArgs& p, const uint64_t* acc, int m, bool row, int n0, int grp,
                                                  int h, int r, int quarter, float* s_amax) {
  const int N = p.m.N;
  float v[64], most = 0.f;
#pragma unroll
  for (int j = 0; j < 32; j++) {
    const float2 g = parts_of(acc[j]), u = parts_of(acc[32 + j]);
    v[2 * j] = swiglu(g.x, u.x);
    v[2 * j + 1] = swiglu(g.y, u.y);
    most = max3_abs(most, v[2 * j], v[2 * j + 1]);
  }
  s_amax[h * 128 + r] = most;
  asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
  const float lim = held_max(max_nan(most, s_amax[(1 - h) * 128 + r])), inv = 448.0f / lim;
  if (!row) return;
  if (h == 0) p.scale[(long)m * ((N + 127) / 128) + grp] = lim / 448.0f;
  uint8_t* q = p.q + (long)m * p.ldq + n0;
  if (n0 + 64 <= N) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint2 x = held8(v + 16 * j, inv), y = held8(v + 16 * j + 8, inv);
      *(uint4*)(q + 16 * j) = make_uint4(x.x, x.y, y.x, y.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) store_held<false>(q + 8 * j, N - n0 - 8 * j, v + 8 * j, inv);
  }
}

// Row tiles are taken eight at a time: the pairs at work at one time then share few rows of a and of the weight.
__device__ __forceinline__ void pair_tile(int t, int tm, int tn, int* mt, int* nt) {
  const int band = t / (8 * tn), first = band * 8, rows = tm - first < 8 ? tm - first : 8, in = t - band * 8 * tn;
  *mt = first + in % rows;
  *nt = in / rows;
}

template <int DT, bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    f8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmB1, PairArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = (uint64_t*)(base + kPairStages * kPairStage);  // used in the first CTA
  uint64_t* empty = full + kPairStages;
  uint64_t* acc_full = empty + kPairStages;  // [2]
  uint64_t* acc_empty = acc_full + 2;        // [2], used in the first CTA
  uint64_t* never = acc_empty + 2;           // [2]
  uint32_t* slot = (uint32_t*)(never + 2);
  float* s_amax = (float*)(slot + 4);        // [2][2][128]
  float* s_room = s_amax + 2 * 2 * 128;      // [8 warps][32][kPairPitch]
  const MmArgs& a = p.m;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pairs = gridDim.x >> 1, pair = blockIdx.x >> 1, tiles = p.tm * p.tn;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 16);  // a warp each of both CTAs' eight
      mbar_init(&never[i], 1);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (SWIGLU) tma_prefetch_desc(&tmB1);
  }
  if (warp == 1) tmem_alloc_pair(slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA's barriers are there
  tc_fence_after();
  const uint32_t tmem = *slot;
  grid_dep_wait();
  // The 384 threads start with 168 registers each: 64512.  Four warps give up theirs for the eight that hold the sums:
  // 128 * (40 + 2 * 232) = 64512.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
      if (lane == 0) {
        int it = 0;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += pairs) {
          int mt, nt;
          pair_tile(t, p.tm, p.tn, &mt, &nt);
          const CUtensorMap* tb = SWIGLU && rank ? &tmB1 : &tmB;
          const int n0 = SWIGLU ? nt * 128 : nt * 256 + (int)rank * 128;
          for (int i = 0; i < a.G; i++, it++) {
            const int s = it % kPairStages;
            ok = mbar_wait(&empty[s], ((uint32_t)(it / kPairStages) & 1u) ^ 1u, ST_TMA_WAIT, &g_status_f8);
            if (!ok) break;
            uint8_t* st = base + s * kPairStage;
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kPairStage);  // both CTAs' tiles
            const uint32_t bar = mapa(smem_u32(&full[s]), 0);
            tma_load_2d_pair(st, &tmA, bar, i * kGroup, mt * 256 + (int)rank * 128);
            tma_load_2d_pair(st + kMmTile, tb, bar, i * kGroup, n0);
          }
        }
        // what is in flight lands before the blocks may end: the last products' arrivals, or, where a wait ran out, copies
        if (ok || rank == 0)
          for (int j = it < kPairStages ? 0 : it - kPairStages; j < it; j++)
            mbar_wait(ok ? &empty[j % kPairStages] : &full[j % kPairStages], (uint32_t)(j / kPairStages) & 1u, ST_TMA_WAIT,
                      &g_status_f8);
        grid_dep_launch();
      }
      __syncwarp();
    } else if (warp == 1) {
      // The whole warp runs the loop and one elected lane issues: with operands that the compiler knows to be the
      // warp's own, an issue takes a fraction of the time that it takes under a branch on the lane.
      if (rank == 0) {
        const uint32_t idesc = idesc_e4m3_f32(256, 256);
        const uint64_t desc = sw128_kmajor_desc(smem_u32(base));
        int it = 0;
        bool ok = true;
        for (int t = pair; t < tiles && ok; t += pairs)
          for (int i = 0; i < a.G; i++, it++) {
            const int s = it % kPairStages, buf = it & 1;
            ok = mbar_wait(&full[s], (uint32_t)(it / kPairStages) & 1u, ST_MMA_WAIT, &g_status_f8) &&
                 mbar_wait(&acc_empty[buf], ((uint32_t)(it >> 1) & 1u) ^ 1u, ST_MMA_WAIT, &g_status_f8);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint64_t da = desc + (uint64_t)(s * (kPairStage >> 4)), db = da + (kMmTile >> 4);
            const uint32_t d = tmem + (uint32_t)(buf * 256);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < 4; kk++) umma_e4m3_pair(d, da + 2 * kk, db + 2 * kk, idesc, kk != 0);
              umma_commit_pair(&empty[s]);
              umma_commit_pair(&acc_full[buf]);
            }
            __syncwarp();
          }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // Eight warps: the lane quarter warp & 3 (the rows that a warp may read), half h of the columns.  A thread's
    // 128 sums are two pieces of 64 columns; with SWIGLU the gate's (columns 0..127 of the tile) and the up's.
    const int h = (warp - 4) >> 2, r = ((warp & 3) << 5) | lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int c0 = SWIGLU ? 64 * h : 128 * h, c1 = SWIGLU ? 128 + 64 * h : 128 * h + 64;
    const uint32_t bar_empty = mapa(smem_u32(acc_empty), 0);
    const int nblocks = (a.N + 127) / 128;
    int it = 0, round = 0;
    bool ok = true;
    uint64_t* seen = a.unanswered ? never : acc_full;
    // Scales are fetched a group ahead, a tile's first before the last one's results go out.  A row that is not there
    // takes the first one's, and nothing of it is stored.
    int mt, nt;
    const float *sa, *sb, *sb1;
    float na, nb0, nb1;
    auto begin = [&](int t) {
      pair_tile(t, p.tm, p.tn, &mt, &nt);
      const int m = mt * 256 + (int)rank * 128 + r, nb = SWIGLU ? nt : min(2 * nt + h, nblocks - 1);
      sa = a.sa + (m < a.M ? m : 0) * a.sa_m;
      sb = a.sb + nb * a.sb_n;
      sb1 = SWIGLU ? p.sb1 + nb * p.sb1_n : nullptr;
      na = __ldg(sa);
      nb0 = __ldg(sb);
      nb1 = SWIGLU ? __ldg(sb1) : 0.f;
    };
    begin(pair);
    for (int t = pair; t < tiles; t += pairs, round++) {
      uint64_t acc[64];
#pragma unroll
      for (int j = 0; j < 64; j++) acc[j] = 0ull;
      for (int i = 0; i < a.G; i++, it++) {
        const int buf = it & 1;
        float s0 = na * nb0, s1 = SWIGLU ? na * nb1 : s0;
        if (i + 1 < a.G) {
          na = __ldg(sa += a.sa_g);
          nb0 = __ldg(sb += a.sb_g);
          if (SWIGLU) nb1 = __ldg(sb1 += p.sb1_g);
        }
        if (ok) ok = mbar_wait(&seen[buf], (uint32_t)(it >> 1) & 1u, ST_EPI_WAIT, &g_status_f8);
        if (!ok) s0 = s1 = lost();
        __syncwarp();
        tc_fence_after();
        const uint32_t d = tmem + lane_base + (uint32_t)(buf * 256);
        uint32_t v[64];
        tmem_ld_x64(d + c0, v);
        scale_add(acc, v, s0);
        tmem_ld_x64(d + c1, v);
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive_cluster(bar_empty + 8 * buf);  // before the rest is added: the products wait for it
        scale_add(acc + 32, v, s1);
      }
      const int m = mt * 256 + (int)rank * 128 + r, n = nt;
      if (t + pairs < tiles) begin(t + pairs);
      if (SWIGLU)
        pair_store_swiglu(p, acc, m, m < a.M, n * 128 + 64 * h, n, h, r, warp & 3, s_amax + (round & 1) * 256);
      else
        pair_store<DT>(p, acc, m - lane, n * 256 + 128 * h, s_room + (warp - 4) * 32 * kPairPitch);
    }
  }
  tc_fence_before();
  cluster_sync();  // nothing of this pair's is in flight any more
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
  cluster_sync();
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
static std::atomic<int> g_unanswered{0};  // rngd_f8_unanswered

// rows x K bytes, rows ld apart, read in boxes of 128 bytes x `box` rows; zeros beyond the edges
static int operand_map(const Operand& o, long rows, int K, int box, CUtensorMap* out) {
  const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows};
  const uint64_t strides[1] = {rows <= 1 ? ((uint64_t)K + 15) / 16 * 16 : (uint64_t)o.ld};
  const uint32_t bx[2] = {kGroup, (uint32_t)box};
  return encode_tmap_u8(out, o.q, 2, dims, strides, bx);
}

static int whole_rows(const void* y, long ldy, const void* add, long ldadd, int dtype) {
  const int sz = dtype == F8_F32 ? 4 : 2;
  return (((uintptr_t)y | (uintptr_t)add) & 15) == 0 && ldy * sz % 16 == 0 && ldadd * sz % 16 == 0;
}

// The few-row kernel's tiles: rows of a in each, and the runs that K is cut into, as many as fill the SMs' places, none
// shorter than four groups.  (Runs for up to twice the places: 16 x 6144 x 4096 11.9 us, not 8.6; gate and up
// 16 x 14336 x 4096 29.8, not 23.7.  Without runs, 1 x 4096 x 4096 has 32 blocks for 148 SMs.)
struct FewPlan {
  long tiles, waves;
  int split;
  bool two;  // blocks an SM
};
static int few_rows(int M, bool dual) { return M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 || dual ? 64 : 128; }
static FewPlan few_plan(int M, int N, int G, bool dual) {
  const int rows = few_rows(M, dual);
  const bool two = rows == 16 || (rows <= 64 && !dual);
  const long places = (long)num_sms() * (two ? 2 : 1);
  static_assert(FewCfg<16, true>::PER_SM == 2 && FewCfg<32, true>::PER_SM == 1 && FewCfg<64, true>::PER_SM == 1, "");
  static_assert(FewCfg<16, false>::PER_SM == 2 && FewCfg<32, false>::PER_SM == 2 && FewCfg<64, false>::PER_SM == 2 &&
                    FewCfg<128, false>::PER_SM == 1, "");
  FewPlan f = {((long)N + 127) / 128 * (((long)M + rows - 1) / rows), 0, 1, two};
  while (f.split < 8 && f.tiles * f.split * 2 <= places && f.split * 8 <= G) f.split *= 2;
  f.waves = (f.tiles * f.split + places - 1) / places;
  return f;
}

// The few-row kernel's launch: y, or (b1: the second weight) q and its scales.
template <int NT, bool DUAL, int DT>
static int few_launch_as(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb1, const FewArgs& p,
                         unsigned grid, cudaStream_t s) {
  using C = FewCfg<NT, DUAL>;
  static std::atomic<unsigned long long> smem_set{0};
  auto kernel = f8_few_kernel<NT, DUAL, DT>;
  RNGD_TRY(set_smem_limit_once((const void*)kernel, (int)C::SMEM, &smem_set, "cudaFuncSetAttribute(f8_few_kernel)"));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, ta, tb, tb1, p), "f8_few_kernel");
}
template <int NT, bool DUAL>
static int few_launch_nt(const Operand& a, const Operand& b, const Operand* b1, FewArgs& p, int dtype, cudaStream_t s) {
  CUtensorMap ta, tb, tb1;
  const MmArgs& m = p.m;
  RNGD_TRY(operand_map(a, m.M, m.K, NT, &ta));
  RNGD_TRY(operand_map(b, m.N, m.K, 128, &tb));
  tb1 = tb;
  if (DUAL) RNGD_TRY(operand_map(*b1, m.N, m.K, 128, &tb1));
  const FewPlan plan = few_plan(m.M, m.N, m.G, DUAL);
  p.tn = (m.N + 127) / 128;
  p.split = plan.split;
  const long tiles = plan.tiles;
  RNGD_REQUIRE(tiles * p.split <= 0x7FFFFFFFl, "f8_matmul: %d x %d results", m.M, m.N);
  const unsigned grid = (unsigned)(tiles * p.split);
  if constexpr (DUAL) return few_launch_as<NT, true, F8_F32>(ta, tb, tb1, p, grid, s);
  else {
    if (dtype == F8_BF16) return few_launch_as<NT, false, F8_BF16>(ta, tb, tb1, p, grid, s);
    if (dtype == F8_F16) return few_launch_as<NT, false, F8_F16>(ta, tb, tb1, p, grid, s);
    return few_launch_as<NT, false, F8_F32>(ta, tb, tb1, p, grid, s);
  }
}
static int few_launch(const Operand& a, const Operand& b, const Operand* b1, int M, int N, int K, const void* add,
                      long ldadd, void* y, long ldy, int dtype, uint8_t* q, long ldq, float* scale, cudaStream_t s) {
  FewArgs p = {};
  p.m = {M, N, K, (K + 127) / 128, a.scale, (long)a.s0, (long)a.s1, b.scale, (long)b.s0, (long)b.s1, y, ldy, add, ldadd,
         g_unanswered.load(std::memory_order_relaxed)};
  p.vec = whole_rows(y, ldy, add, ldadd, dtype);
  p.q = q;
  p.ldq = ldq;
  p.scale = scale;
  if (b1 != nullptr) {
    p.sb1 = b1->scale;
    p.sb1_n = (long)b1->s0;
    p.sb1_g = (long)b1->s1;
    switch (few_rows(M, true)) {
      case 16: return few_launch_nt<16, true>(a, b, b1, p, dtype, s);
      case 32: return few_launch_nt<32, true>(a, b, b1, p, dtype, s);
      default: return few_launch_nt<64, true>(a, b, b1, p, dtype, s);
    }
  }
  switch (few_rows(M, false)) {
    case 16: return few_launch_nt<16, false>(a, b, b1, p, dtype, s);
    case 32: return few_launch_nt<32, false>(a, b, b1, p, dtype, s);
    case 64: return few_launch_nt<64, false>(a, b, b1, p, dtype, s);
    default: return few_launch_nt<128, false>(a, b, b1, p, dtype, s);
  }
}

// The pairs' launch: one weight, or gate and up (b1) with the 8-bit result (q, scale).
static int pair_launch(const Operand& a, const Operand& b, const Operand* b1, int M, int N, int K, const void* add,
                       long ldadd, void* y, long ldy, int dtype, uint8_t* q, long ldq, float* scale, cudaStream_t s) {
  CUtensorMap ta, tb, tb1;
  RNGD_TRY(operand_map(a, M, K, 128, &ta));
  RNGD_TRY(operand_map(b, N, K, 128, &tb));
  tb1 = tb;
  if (b1 != nullptr) RNGD_TRY(operand_map(*b1, N, K, 128, &tb1));
  PairArgs p = {};
  p.m = {M, N, K, (K + 127) / 128, a.scale, (long)a.s0, (long)a.s1, b.scale, (long)b.s0, (long)b.s1, y, ldy, add, ldadd,
         g_unanswered.load(std::memory_order_relaxed)};
  if (b1 != nullptr) {
    p.sb1 = b1->scale;
    p.sb1_n = (long)b1->s0;
    p.sb1_g = (long)b1->s1;
  }
  p.tm = (M + 255) / 256;
  p.tn = b1 != nullptr ? (N + 127) / 128 : (N + 255) / 256;
  RNGD_REQUIRE((long)p.tm * p.tn <= 0x7FFFFFFFl / 2, "f8_matmul: %d x %d results", M, N);
  p.vec = whole_rows(y, ldy, add, ldadd, dtype);
  p.q = q;
  p.ldq = ldq;
  p.scale = scale;
  auto kernel = b1 != nullptr       ? f8_pair_kernel<F8_F32, true>
                : dtype == F8_BF16 ? f8_pair_kernel<F8_BF16, false>
                : dtype == F8_F16  ? f8_pair_kernel<F8_F16, false>
                                   : f8_pair_kernel<F8_F32, false>;
  static std::atomic<unsigned long long> smem_set[4];
  RNGD_TRY(set_smem_limit_once((const void*)kernel, kPairSmem, &smem_set[b1 != nullptr ? 3 : dtype],
                               "cudaFuncSetAttribute(f8_pair_kernel)"));
  const int tiles = p.tm * p.tn, most = num_sms() / 2;
  return launch_pdl(kernel, dim3(2 * (tiles < most ? tiles : most)), dim3(kPairThreads), kPairSmem, s, "f8_pair_kernel",
                    ta, tb, tb1, p);
}

// Which of the two kernels: a wave of either takes about 7 us and 0.4 us for each of its groups (256 rows a tile of the
// pairs', 64 or 128 of the other, whose K may be cut).  Measured over 65 to 2000 rows, N from 300 to 28000 and K from 300
// to 8192 this takes the faster one but for ties within a fifth: 200 x 4096 x 4096 20 us by pairs, 14 by the other;
// 1000 x 4096 x 4096 21 and 40.  With so few rows that two blocks fit an SM the other kernel's wave is shorter, and a tie
// is its: 1 x 4864 x 896 8.2 us by pairs, 3.9 by the other; 64 x 896 x 512 6.6 and 5.2; gate and up 16 x 4864 x 896 8.0
// and 5.9 (32 rows, one block an SM, 8.1 and 7.5, but 32 x 128 x 512 5.5 and 5.8).
static bool pairs_pay(int M, int N, int K, bool dual) {
  const int G = (K + 127) / 128;
  const FewPlan f = few_plan(M, N, G, dual);
  const long tiles = ((long)M + 255) / 256 * (((long)N + (dual ? 127 : 255)) / (dual ? 128 : 256));
  const long pairs = num_sms() / 2, waves = (tiles + pairs - 1) / pairs;
  const long by_pairs = waves * (18 + G), by_few = f.waves * (18 + (G + f.split - 1) / f.split);
  return by_pairs < by_few || (by_pairs == by_few && !f.two);
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_f8_tile_rows(int M, int N, int K, int gated, int* rows) {
  RNGD_REQUIRE(rows != nullptr, "f8_tile_rows: null output");
  RNGD_REQUIRE(M >= 1 && N >= 1 && K >= 1 && M <= kMostRows && N <= kMostRows && K <= kMostK, "f8_tile_rows: %d x %d x %d",
               M, N, K);
  *rows = pairs_pay(M, N, K, gated != 0) ? 256 : few_rows(M, gated != 0);
  return RNGD_OK;
}

// A word of its own: whoever uses the engines reads and clears theirs (rngd_device_status).
extern "C" int rngd_f8_status(int* status, int reset) {
  RNGD_REQUIRE(status != nullptr, "f8_status: null output");
  RNGD_TRY(check_cuda(cudaMemcpyFromSymbol(status, g_status_f8, sizeof(int)), "read device status"));
  if (reset) {
    const int zero = 0;
    RNGD_TRY(check_cuda(cudaMemcpyToSymbol(g_status_f8, &zero, sizeof(int)), "reset device status"));
  }
  return RNGD_OK;
}

extern "C" int rngd_f8_unanswered(int on) {
  g_unanswered.store(on != 0, std::memory_order_relaxed);
  return RNGD_OK;
}

extern "C" int rngd_f8_matmul(const void* a, int64_t lda, const float* a_scale, const int64_t* a_strides, const void* b,
                              int64_t ldb, const float* b_scale, const int64_t* b_strides, int M, int N, int K,
                              const void* add, int64_t ldadd, void* y, int64_t ldy, int dtype, rngd_stream_t stream) {
  RNGD_REQUIRE(dtype >= F8_BF16 && dtype <= F8_F32, "f8_matmul: data type %d", dtype);
  RNGD_REQUIRE(M >= 0 && N >= 0 && K >= 1, "f8_matmul: %d x %d x %d", M, N, K);
  RNGD_REQUIRE(M <= kMostRows && N <= kMostRows && K <= kMostK, "f8_matmul: %d x %d x %d is too much", M, N, K);
  if (M == 0 || N == 0) return RNGD_OK;
  const uintptr_t mis = dtype == F8_F32 ? 3 : 1;
  RNGD_REQUIRE(y != nullptr && a_strides != nullptr && b_strides != nullptr, "f8_matmul: null pointer");
  RNGD_REQUIRE((((uintptr_t)y | (uintptr_t)add) & mis) == 0, "f8_matmul: misaligned result");
  RNGD_REQUIRE(M <= 1 || ldy >= N, "f8_matmul: rows of the result lie on one another");
  const Operand oa = {a, lda, a_scale, a_strides[0], a_strides[1]}, ob = {b, ldb, b_scale, b_strides[0], b_strides[1]};
  RNGD_TRY(check_operand("f8_matmul", oa, M, K));
  RNGD_TRY(check_operand("f8_matmul", ob, N, K));
  if (pairs_pay(M, N, K, false))
    return pair_launch(oa, ob, nullptr, M, N, K, add, (long)ldadd, y, (long)ldy, dtype, nullptr, 0, nullptr,
                       (cudaStream_t)stream);
  return few_launch(oa, ob, nullptr, M, N, K, add, (long)ldadd, y, (long)ldy, dtype, nullptr, 0, nullptr,
                    (cudaStream_t)stream);
}

extern "C" int rngd_f8_swiglu(const void* a, int64_t lda, const float* a_scale, const int64_t* a_strides,
                              const void* gate, int64_t ldg, const float* gate_scale, const int64_t* gate_strides,
                              const void* up, int64_t ldu, const float* up_scale, const int64_t* up_strides, int M, int N,
                              int K, void* q, int64_t ldq, float* scale, rngd_stream_t stream) {
  RNGD_REQUIRE(M >= 0 && N >= 0 && K >= 1, "f8_swiglu: %d x %d x %d", M, N, K);
  RNGD_REQUIRE(M <= kMostRows && N <= kMostRows && K <= kMostK, "f8_swiglu: %d x %d x %d is too much", M, N, K);
  if (M == 0 || N == 0) return RNGD_OK;
  RNGD_REQUIRE(q && scale && a_strides && gate_strides && up_strides, "f8_swiglu: null pointer");
  RNGD_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)scale & 3) == 0 && (M <= 1 || (ldq >= N && ldq % 16 == 0)),
               "f8_swiglu: 8-bit rows must start on 16 bytes and not overlap");
  const Operand oa = {a, lda, a_scale, a_strides[0], a_strides[1]};
  const Operand og = {gate, ldg, gate_scale, gate_strides[0], gate_strides[1]};
  const Operand ou = {up, ldu, up_scale, up_strides[0], up_strides[1]};
  RNGD_TRY(check_operand("f8_swiglu", oa, M, K));
  RNGD_TRY(check_operand("f8_swiglu", og, N, K));
  RNGD_TRY(check_operand("f8_swiglu", ou, N, K));
  auto launch = pairs_pay(M, N, K, true) ? pair_launch : few_launch;
  return launch(oa, og, &ou, M, N, K, nullptr, 0, nullptr, 0, F8_F32, (uint8_t*)q, (long)ldq, scale, (cudaStream_t)stream);
}
