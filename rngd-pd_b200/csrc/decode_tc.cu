// Tensor-core decode step: persistent stream-K tcgen05 GEMMs with fused epilogues.
//
// A decode GEMM is Y[b][n] = sum_k W[n][k] * h[b][k] with W bf16 (HBM, read
// once per step) and h fp32.  It runs on tcgen05 as D = A * B^T with
//   A = a 128-row tile of W (TMA, 128-byte swizzle, K-major),
//   B = the activation operand: 32 bf16 rows = 16 streams x {hi, lo}, where
//       hi = bf16(h) and lo = bf16(h - hi), so hi + lo carries ~16 mantissa
//       bits of the fp32 activation and W*hi + W*lo (fp32 accumulation in
//       TMEM) keeps fp32-level accuracy,
//   D = 128 x 32 fp32 accumulators in tensor memory (double-buffered).
//
// Scheduling (stream-K).  One CTA per SM.  The GEMM's tiles x K-blocks are laid
// end to end and cut into one equal contiguous range per CTA, so every SM
// streams the same number of weight bytes and the TMA ring never drains between
// tiles.  A tile cut between CTAs is summed by its first owner (the CTA holding
// the tile's first K blocks, which it reaches at the end of its range, when
// the other owners are finishing too).  Each other owner stores its piece as
// 64-bit words {fp32 value, flag}; a single-copy-atomic word needs no fence,
// so the first owner polls the words of the pieces it misses and adds them in
// K order.  The flag is (shape tag, tile epoch + 1): the epoch is a per-shape,
// per-tile counter that the first owner advances once it has every piece, so
// a word left by an earlier launch (older epoch) or another shape sharing the
// scratch (other tag) never reads as ready and nothing needs clearing.  The cut
// depends only on (N, K, CTA count), never on B, so a stream's result is
// deterministic and independent of what else is batched with it.
//
// Programmatic dependent launch.  The producer issues the first weight tiles
// BEFORE griddepcontrol.wait (weights do not depend on the previous kernel),
// so each GEMM's HBM stream starts while the previous kernel finishes.
//
// RMSNorm is folded in: rms(x) * w @ W^T = (x * w) @ W^T / sqrt(mean(x^2) + eps).
// The producer of x (embedding, residual epilogues) writes the operand of
// x * w_next and per-128-column sums of squares; the consumer's epilogue
// scales each stream's row by 1 / sqrt(sum / H + eps).
//
// Epilogues (run for a tile once all its K pieces are in):
//   QKV     RoPE (rotate-half, fp32 angles) on q and k; q -> fp32 buffer,
//           k and v -> bf16 cache at pos[b]      (kernels/decode_batch.py:76-82)
//   RESID   x[b][n] += y, plus the next GEMM's operand and its sums of squares
//                                                 (zipadd + rms, kernels/decode_batch.py:87-88,91)
//   SWIGLU  silu(gate) * up for the tile's 64 features -> hi/lo operand of the
//           down GEMM                             (kernels/decode_batch.py:88-90)
//   LOGITS  logits[b][n] = y and a first-max argmax key per stream
//                                                 (engines/decode_batch.py:122-171)
#include <mutex>
#include <unordered_map>

#include "tc.cuh"

namespace rngd {

__device__ int g_status_decode = 0;  // this file's bounded-wait status word

constexpr int BM = 128, BK = 64, BNC = 32, MAXB = 16;
constexpr int A_BYTES = BM * BK * 2;   // 16 KB weight tile per stage
constexpr int B_BYTES = BNC * BK * 2;  // 4 KB activation tile per stage
// 8 x 20 KB stages: what a CTA prefetches before the previous kernel's output is readable covers
// most of that kernel's tail (measured best among 5..10 stages; deeper rings slowed the
// short QKV and O GEMMs)
constexpr int STAGES = 8;
constexpr int YS_LD = 17;
constexpr int EPI_THREADS = 256;       // two warpgroups, each 8 of the 16 streams
constexpr int SPG = MAXB / 2;          // streams per epilogue warpgroup
constexpr int THREADS = 64 + EPI_THREADS;  // warp 0 TMA, warp 1 MMA, warps 2-9 epilogue
constexpr int TMEM_COLS = 64;          // two 32-column accumulators
constexpr int kRedBatch = 5;           // split-tile pieces whose partials are loaded together

enum Epi : int { EPI_QKV = 0, EPI_RESID = 1, EPI_SWIGLU = 2, EPI_LOGITS = 3 };

struct GemmArgs {
  int N, K, nkb, tiles, total, maxseg, layer, B;
  float* partial;   // [tiles][maxseg][8 stream pairs][128 rows][2] words {fp32 value, flag}, zeroed once
  int* counters;    // [tiles] epochs of this shape's split tiles, zeroed once
  int tag;          // 1..15, distinct for GEMM shapes sharing `partial`
  // rms scale of the result (QKV, SWIGLU, LOGITS); ss_in == nullptr -> no scaling
  const float* ss_in;  // [ss_tiles][16] per-128-column sums of squares of x
  int ss_tiles;
  float eps, inv_h;
  // QKV
  const int32_t* pos;
  const float* inv;
  float* q;
  int ldq;
  uint16_t* kc;
  uint16_t* vc;
  const int32_t* lanes;  // [B] cache lane of each stream, nullptr = stream b -> lane b
  int NH, NKV, S;
  int kv_rows;  // 1: kc and vc are the new rows alone, [B][NKV][128] (S = 1), whatever their position
  // RESID: x += y; act_next = hi/lo(x * w_next); ss_out = per-tile sums of squares of x
  float* x;
  int ldx;
  const float* w_next;
  uint16_t* act_next;
  int ld_next;
  float* ss_out;
  // SWIGLU
  uint16_t* act_out;
  int ld_act;
  // LOGITS
  float* logits;
  unsigned long long* best;
  int V;
  // optional per-CTA timeline (ns, %globaltimer), 16 entries per CTA: start, operand ready, last
  // TMA issued, last stage arrived, last MMA committed, last accumulator ready, epilogue done,
  // end; then for the last segment: accumulator read, poll rounds of a split tile's first owner
// (a count, not a time), later pieces summed,
  // epilogue stores issued, segment done; nullptr = off
  unsigned long long* trace;
};

// smem: stages | barriers (2*STAGES + 5) + tmem slot/flags (64 B) | scale (64 B) | pos (64 B) | lane (64 B)
//       | ys | s_red
constexpr size_t kBarBytes = (2 * STAGES + 5) * 8;
constexpr size_t kSmemBytes = 1024 /*align*/ + STAGES * (A_BYTES + B_BYTES) + kBarBytes + 64 + 64 + 64 + 64 +
                              BM * YS_LD * 4 + 4 * MAXB * 8;

__device__ __forceinline__ uint32_t orderable(float f) {
  uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// One 16-byte store of two {value, flag} words of a split-tile piece.  Each 64-bit word is
// single-copy atomic, so a reader that sees the flag sees the value stored with it.
__device__ __forceinline__ void st_piece(unsigned long long* p, uint32_t flag, float v0, float v1) {
  const unsigned long long w0 = ((unsigned long long)flag << 32) | __float_as_uint(v0);
  const unsigned long long w1 = ((unsigned long long)flag << 32) | __float_as_uint(v1);
  asm volatile("st.volatile.global.v2.u64 [%0], {%1, %2};" ::"l"(p), "l"(w0), "l"(w1) : "memory");
}
__device__ __forceinline__ void ld_piece(const unsigned long long* p, unsigned long long& w0,
                                         unsigned long long& w1) {
  asm volatile("ld.volatile.global.v2.u64 {%0, %1}, [%2];" : "=l"(w0), "=l"(w1) : "l"(p) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// ------------------------------------------------------------------ the GEMM's three roles
// Shared-memory layout of a GEMM CTA (the same for every phase of a fused launch).
struct Ring {
  uint8_t* sA;
  uint8_t* sB;
  uint64_t* full;
  uint64_t* empty;
  uint64_t* acc_full;   // [2]
  uint64_t* acc_empty;  // [2]
  uint64_t* epi_done;   // the epilogue threads are past their last TMEM read
  uint32_t* tmem_slot;
  float* s_scale;       // [16]
  int* s_pos;           // [16]
  int* s_lane;          // [16] cache lane of each stream
  float* ys;
  unsigned long long* s_red;  // [4][16]
};

__device__ __forceinline__ Ring ring_layout(uint8_t* smem_raw) {
  Ring R;
  uint8_t* base = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  R.sA = base;
  R.sB = base + STAGES * A_BYTES;
  R.full = (uint64_t*)(R.sB + STAGES * B_BYTES);
  R.empty = R.full + STAGES;
  R.acc_full = R.empty + STAGES;
  R.acc_empty = R.acc_full + 2;
  R.epi_done = R.acc_empty + 2;
  uint8_t* tail = (uint8_t*)R.full + kBarBytes;
  R.tmem_slot = (uint32_t*)tail;
  R.s_scale = (float*)(tail + 64);
  R.s_pos = (int*)(tail + 128);
  R.s_lane = (int*)(tail + 192);
  R.ys = (float*)(tail + 256);
  R.s_red = (unsigned long long*)(R.ys + BM * YS_LD);
  return R;
}

// Barrier init (thread 0) and TMEM allocation (warp 1), then a CTA-wide sync.  Returns the
// TMEM base of the two accumulators.
__device__ __forceinline__ uint32_t ring_setup(const Ring& R) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&R.full[s], 1);
      mbar_init(&R.empty[s], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&R.acc_full[i], 1);
      mbar_init(&R.acc_empty[i], EPI_THREADS);
    }
    mbar_init(R.epi_done, EPI_THREADS);
    fence_mbar_init();
  }
  if ((threadIdx.x >> 5) == 1) {
    tmem_alloc(R.tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return *R.tmem_slot;
}

// TMA loads of one GEMM's k-steps [f0, f1) through the ring, from ring position i on (the
// positions continue across the phases of a fused launch).  The weight tiles of the first
// min(f1 - f0, STAGES) steps are requested as soon as their ring slots are free and before
// wait_operand(): weights never depend on earlier work, so they stream while the previous
// kernel or phase finishes.  The operand tiles follow wait_operand().  Returns the ring
// position after the phase, or -1 when a bounded wait gave up (the status word is set).
template <class WaitOperand>
__device__ __forceinline__ long produce_phase(const CUtensorMap* tmW, const CUtensorMap* tmX, const GemmArgs& a,
                                              const Ring& R, long i, long f0, long f1, WaitOperand wait_operand) {
  const long nk = f1 - f0;
  const long pre = nk < STAGES ? nk : STAGES;
  long issued = 0;
  for (; issued < pre; issued++) {
    const long q = i + issued;
    const int s = (int)(q % STAGES);
    if (!mbar_wait(&R.empty[s], ((uint32_t)(q / STAGES) & 1u) ^ 1u, ST_TMA_WAIT, &g_status_decode)) break;
    const long f = f0 + issued;
    const int tile = (int)(f / a.nkb), kb = (int)(f - (long)tile * a.nkb);
    mbar_arrive_expect_tx(&R.full[s], A_BYTES + B_BYTES);
    tma_load_3d(R.sA + s * A_BYTES, tmW, &R.full[s], kb * BK, tile * BM, a.layer);
  }
  wait_operand();
  for (long j = 0; j < issued; j++) {
    const int s = (int)((i + j) % STAGES);
    tma_load_2d(R.sB + s * B_BYTES, tmX, &R.full[s], (int)((f0 + j) % a.nkb) * BK, 0);
  }
  if (issued < pre) return -1;
  for (long j = pre; j < nk; j++) {
    const long q = i + j;
    const int s = (int)(q % STAGES);
    if (!mbar_wait(&R.empty[s], ((uint32_t)(q / STAGES) & 1u) ^ 1u, ST_TMA_WAIT, &g_status_decode)) return -1;
    const long f = f0 + j;
    const int tile = (int)(f / a.nkb), kb = (int)(f - (long)tile * a.nkb);
    mbar_arrive_expect_tx(&R.full[s], A_BYTES + B_BYTES);
    tma_load_3d(R.sA + s * A_BYTES, tmW, &R.full[s], kb * BK, tile * BM, a.layer);
    tma_load_2d(R.sB + s * B_BYTES, tmX, &R.full[s], kb * BK, 0);
  }
  return i + nk;
}

// MMAs of one GEMM's k-steps [f0, f1): 4 x (128x32x16) per K block into the segment's TMEM
// accumulator; the ring position i and the segment count seg continue across phases.
__device__ __forceinline__ bool mma_phase(const GemmArgs& a, const Ring& R, uint32_t tmem, long& i, int& seg,
                                          long f0, long f1, unsigned long long* tr) {
  const uint32_t idesc = idesc_bf16_f32(BM, BNC);
  bool ok = true;
  for (long f = f0; f < f1 && ok; seg++) {
    const int tile = (int)(f / a.nkb);
    const long fend = ((long)tile + 1) * a.nkb < f1 ? ((long)tile + 1) * a.nkb : f1;
    const int buf = seg & 1;
    const uint32_t aph = (uint32_t)(seg >> 1) & 1u;
    ok = mbar_wait(&R.acc_empty[buf], aph ^ 1u, ST_MMA_WAIT, &g_status_decode);
    tc_fence_after();
    const uint32_t d = tmem + (uint32_t)(buf * BNC);
    for (long g = f; g < fend && ok; g++, i++) {
      const int s = (int)(i % STAGES);
      const uint32_t ph = (uint32_t)(i / STAGES) & 1u;
      ok = mbar_wait(&R.full[s], ph, ST_MMA_WAIT, &g_status_decode);
      if (!ok) break;
      if (tr != nullptr && g + 1 == f1) tr[3] = globaltimer();
      tc_fence_after();
      const uint32_t aBase = smem_u32(R.sA + s * A_BYTES), bBase = smem_u32(R.sB + s * B_BYTES);
#pragma unroll
      for (int kk = 0; kk < BK / 16; kk++)
        umma_bf16(d, sw128_kmajor_desc(aBase + kk * 32), sw128_kmajor_desc(bBase + kk * 32), idesc,
                  (g != f || kk != 0) ? 1u : 0u);
      umma_commit(&R.empty[s]);
    }
    umma_commit(&R.acc_full[buf]);
    f = fend;
  }
  return ok;
}

// Epilogue of one GEMM's k-steps [f0, f1) on the 256 epilogue threads: two warpgroups over
// the same 128 TMEM lanes; thread (group g, row r) owns row r of the tile (TMEM lane r) for the
// streams 8g .. 8g+7, which halves each thread's serial work on the GEMM's tail.  The caller
// has already waited for the data the GEMM consumes (the previous kernel or phase).  seg
// continues across phases.  Values other CTAs write earlier in the same launch (x, the sums of
// squares) are read with L1-bypassing loads.
template <int EPI>
__device__ __forceinline__ void epilogue_phase(const GemmArgs& a, const Ring& R, uint32_t tmem, int& seg, long f0,
                                               long f1, unsigned long long* tr) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = gridDim.x, cta = blockIdx.x;
  const int r = ((warp & 3) << 5) | lane;
  const int ep = threadIdx.x - 64;   // 0..255 among the epilogue threads
  const int sb = (ep >> 7) * SPG;    // first stream of this thread's group
  // Per-launch constants, read once with independent loads: a chain of dependent global
  // loads inside each segment's epilogue was most of the GEMM's tail.  The RMS sums are
  // added in the same order as ever (t = 0, 1, ...), so the scale is bit-identical.
  if (EPI != EPI_RESID && a.ss_in != nullptr && ep < MAXB) {
    float ssum = 0.f;
    for (int t0 = 0; t0 < a.ss_tiles; t0 += 16) {
      float v16[16];
#pragma unroll
      for (int j = 0; j < 16; j++) v16[j] = t0 + j < a.ss_tiles ? __ldcg(a.ss_in + (t0 + j) * MAXB + ep) : 0.f;
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (t0 + j < a.ss_tiles) ssum += v16[j];
    }
    R.s_scale[ep] = 1.0f / sqrtf(ssum * a.inv_h + a.eps);
  }
  // RoPE factors of this step for this thread's frequency (r mod 64) and streams, computed
  // while the weights stream rather than on the GEMM's tail
  float rcos[SPG], rsin[SPG];
  if constexpr (EPI == EPI_QKV) {
    if (ep < MAXB) {
      R.s_pos[ep] = ep < a.B ? a.pos[ep] : -1;
      R.s_lane[ep] = ep < a.B ? (a.lanes != nullptr ? a.lanes[ep] : ep) : 0;
    }
    const float invf = a.inv[r & 63];
#pragma unroll
    for (int i = 0; i < SPG; i++) {
      const int p = sb + i < a.B ? a.pos[sb + i] : -1;
      sincosf((float)p * invf, &rsin[i], &rcos[i]);
    }
  }
  epi_sync();
  for (long f = f0; f < f1; seg++) {
    const int tile = (int)(f / a.nkb);
    const long tstart = (long)tile * a.nkb;
    const long fend = tstart + a.nkb < f1 ? tstart + a.nkb : f1;
    const int buf = seg & 1;
    const int n = tile * BM + r;
    // the residual row and norm weight do not depend on this GEMM: fetch them while the
    // accumulator is still being computed (only the tile's reducing CTA writes x[.][n])
    float xo[SPG];
    float wn = 0.f;
    // epoch of the tile's split (read before the accumulator wait; only the tile's first owner
    // advances it, after every piece of this launch was stored under the value read here)
    const int epoch = a.maxseg > 1 ? __ldcg(a.counters + tile) : 0;
    if constexpr (EPI == EPI_RESID) {
#pragma unroll
      for (int i = 0; i < SPG; i++) xo[i] = sb + i < a.B ? __ldcg(a.x + (size_t)(sb + i) * a.ldx + n) : 0.f;
      if (a.act_next != nullptr) wn = a.w_next[n];
    }
    const int first = owner_of(tstart, a.total, G), last = owner_of(tstart + a.nkb - 1, a.total, G);
    const int nseg = last - first + 1;
    const int slot = cta - first;
    // piece layout [stream pair][row][2 words]: the 32 rows of a warp read or write 512
    // contiguous bytes per instruction.  This thread's pairs are sb/2 .. sb/2 + SPG/2 - 1.
    constexpr size_t kPieceWords = (size_t)BM * MAXB;
    constexpr size_t kPairWords = (size_t)BM * 2;
    unsigned long long* pw = reinterpret_cast<unsigned long long*>(a.partial) +
                             (size_t)tile * a.maxseg * kPieceWords + ((size_t)(sb / 2) * BM + r) * 2;
    // a tile's first owner reads the first batch of later pieces while its own accumulator is
    // still being computed: pieces already stored cost no round trip after it
    unsigned long long w[kRedBatch][SPG];
    if (nseg > 1 && slot == 0) {
#pragma unroll
      for (int q = 0; q < kRedBatch; q++) {
        if (1 + q < nseg) {
#pragma unroll
          for (int j = 0; j < SPG / 2; j++)
            ld_piece(pw + (size_t)(1 + q) * kPieceWords + j * kPairWords, w[q][2 * j], w[q][2 * j + 1]);
        }
      }
    }
    mbar_wait(&R.acc_full[buf], (uint32_t)(seg >> 1) & 1u, ST_EPI_WAIT, &g_status_decode);
    if (tr != nullptr && ep == 0 && fend == f1) tr[5] = globaltimer();
    __syncwarp();
    tc_fence_after();
    float vh[SPG], vl[SPG];  // the hi and lo operand columns of this group's streams
    const uint32_t tb = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(buf * BNC);
    tmem_ld_32x32b_2x8(tb + sb, tb + MAXB + sb, vh, vl);
    tc_fence_before();
    mbar_arrive(&R.acc_empty[buf]);
    const bool tlast = tr != nullptr && ep == 0 && fend == f1;
    if (tlast) tr[8] = globaltimer();
    float y[SPG];
#pragma unroll
    for (int i = 0; i < SPG; i++) y[i] = vh[i] + vl[i];

    bool run = true;
    if (nseg > 1) {
      const uint32_t flag = ((uint32_t)a.tag << 28) | ((uint32_t)(epoch + 1) & 0x0FFFFFFFu);
      if (slot > 0) {
        // a later piece of the tile: publish it, no wait
        unsigned long long* dst = pw + (size_t)slot * kPieceWords;
#pragma unroll
        for (int j = 0; j < SPG / 2; j++) st_piece(dst + j * kPairWords, flag, y[2 * j], y[2 * j + 1]);
        run = false;
      } else {
        // the tile's first piece is this CTA's own: wait (bounded) until all of this thread's
        // words of the later pieces carry the flag, re-reading every missing piece together
        // (one L2 round trip per poll, not per piece), then add them in K order
        bool ok = true;
        for (int s0 = 1; s0 < nseg; s0 += kRedBatch) {
          uint32_t pend = 0;
#pragma unroll
          for (int q = 0; q < kRedBatch; q++) {
            if (s0 + q < nseg) {
              pend |= 1u << q;
              if (s0 > 1) {  // the first batch was read before the accumulator wait
#pragma unroll
                for (int j = 0; j < SPG / 2; j++)
                  ld_piece(pw + (size_t)(s0 + q) * kPieceWords + j * kPairWords, w[q][2 * j], w[q][2 * j + 1]);
              }
            }
          }
          uint64_t t0 = 0;
          int polls = 0;
          while (true) {
#pragma unroll
            for (int q = 0; q < kRedBatch; q++) {
              if (pend & (1u << q)) {
                bool ready = true;
#pragma unroll
                for (int i = 0; i < SPG; i++) ready &= (uint32_t)(w[q][i] >> 32) == flag;
                if (ready) pend &= ~(1u << q);
              }
            }
            if (pend == 0 || !ok) break;
            polls++;
            const uint64_t now = globaltimer();
            if (t0 == 0) {
              t0 = now;
            } else if (now - t0 > kWaitTimeoutNs) {
              atomicCAS(&g_status_decode, 0, ST_PIECE_WAIT);
              ok = false;
              break;
            }
#pragma unroll
            for (int q = 0; q < kRedBatch; q++) {
              if (pend & (1u << q)) {
#pragma unroll
                for (int j = 0; j < SPG / 2; j++)
                  ld_piece(pw + (size_t)(s0 + q) * kPieceWords + j * kPairWords, w[q][2 * j], w[q][2 * j + 1]);
              }
            }
          }
          if (tlast) tr[9] = (unsigned long long)polls;
#pragma unroll
          for (int q = 0; q < kRedBatch; q++) {
            if (s0 + q < nseg) {
#pragma unroll
              for (int i = 0; i < SPG; i++) y[i] += __uint_as_float((uint32_t)w[q][i]);
            }
          }
        }
        // every piece of this launch is in: the next launch uses the next epoch
        if (ep == 0) a.counters[tile] = epoch + 1;
        if (tlast) tr[10] = globaltimer();
      }
    }
    if (run) {
      if (EPI != EPI_RESID && a.ss_in != nullptr) {
#pragma unroll
        for (int i = 0; i < SPG; i++) y[i] *= R.s_scale[sb + i];
      }
      if constexpr (EPI == EPI_RESID) {
        // every stream of the group is computed (streams >= B hold zeros) so the per-stream
        // chains interleave; only the stores are predicated on B
        float xs[SPG];
#pragma unroll
        for (int i = 0; i < SPG; i++) {
          xs[i] = xo[i] + y[i];
          if (sb + i < a.B) a.x[(size_t)(sb + i) * a.ldx + n] = xs[i];
        }
        if (tlast) tr[13] = globaltimer();
        if (a.act_next != nullptr) {
#pragma unroll
          for (int i = 0; i < SPG; i++) {
            const float h = xs[i] * wn;
            const uint16_t hi = f2bf_bits(h);
            const uint16_t lo = f2bf_bits(h - bf2f(hi));
            if (sb + i < a.B) {
              a.act_next[(size_t)(sb + i) * a.ld_next + n] = hi;
              a.act_next[(size_t)(MAXB + sb + i) * a.ld_next + n] = lo;
            }
          }
          if (tlast) tr[14] = globaltimer();
          // per-tile sum of squares of the new x: the same xor butterfly for every stream,
          // the group's 8 interleaved
          float sq[SPG];
#pragma unroll
          for (int i = 0; i < SPG; i++) sq[i] = xs[i] * xs[i];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < SPG; i++) sq[i] += __shfl_xor_sync(0xffffffffu, sq[i], o);
          }
          if (lane == 0) {
#pragma unroll
            for (int i = 0; i < SPG; i++) R.ys[(warp & 3) * YS_LD + sb + i] = sq[i];
          }
          if (tlast) tr[15] = globaltimer();
          epi_sync();
          if (ep < a.B) {
            const float t4 = (R.ys[0 * YS_LD + ep] + R.ys[1 * YS_LD + ep]) + (R.ys[2 * YS_LD + ep] + R.ys[3 * YS_LD + ep]);
            a.ss_out[tile * MAXB + ep] = t4;
          }
        }
      } else if constexpr (EPI == EPI_QKV) {
#pragma unroll
        for (int i = 0; i < SPG; i++) R.ys[r * YS_LD + sb + i] = y[i];
        epi_sync();
        const int head = tile;  // one 128-row tile = one head
        const bool lo_half = r < 64;
        const int partner = r ^ 64;
        if (head < a.NH + a.NKV) {
          if (tlast) tr[13] = globaltimer();
          float o[SPG];
#pragma unroll
          for (int i = 0; i < SPG; i++) {  // all streams (pos -1 past B), stores predicated
            const float other = R.ys[partner * YS_LD + sb + i];
            o[i] = lo_half ? y[i] * rcos[i] - other * rsin[i] : y[i] * rcos[i] + other * rsin[i];
          }
          if (tlast) tr[14] = globaltimer();
#pragma unroll
          for (int i = 0; i < SPG; i++) {
            const int b = sb + i, p = R.s_pos[b];
            if (b < a.B) {
              if (head < a.NH) {
                a.q[(size_t)b * a.ldq + n] = o[i];
              } else if (const int at = a.kv_rows ? 0 : p; p >= 0 && at < a.S) {
                a.kc[(((size_t)R.s_lane[b] * a.NKV + (head - a.NH)) * a.S + at) * 128 + r] = f2bf_bits(o[i]);
              }
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < SPG; i++) {
            const int b = sb + i, p = R.s_pos[b], at = a.kv_rows ? 0 : p;
            if (b < a.B && p >= 0 && at < a.S)
              a.vc[(((size_t)R.s_lane[b] * a.NKV + (head - a.NH - a.NKV)) * a.S + at) * 128 + r] = f2bf_bits(y[i]);
          }
        }
      } else if constexpr (EPI == EPI_SWIGLU) {
#pragma unroll
        for (int i = 0; i < SPG; i++) R.ys[r * YS_LD + sb + i] = y[i];
        epi_sync();
        if (r < 64) {
          const int fcol = tile * 64 + r;
#pragma unroll
          for (int i = 0; i < SPG; i++) {
            const float g = y[i], u = R.ys[(r + 64) * YS_LD + sb + i];
            const float act = g / (1.0f + expf(-g)) * u;
            const uint16_t hi = f2bf_bits(act);
            const uint16_t lo = f2bf_bits(act - bf2f(hi));
            if (sb + i < a.B) {
              a.act_out[(size_t)(sb + i) * a.ld_act + fcol] = hi;
              a.act_out[(size_t)(MAXB + sb + i) * a.ld_act + fcol] = lo;
            }
          }
        }
      } else if constexpr (EPI == EPI_LOGITS) {
        unsigned long long key[SPG];
#pragma unroll
        for (int i = 0; i < SPG; i++) {
          key[i] = 0;
          if (n < a.V) {
            if (sb + i < a.B) a.logits[(size_t)(sb + i) * a.V + n] = y[i];
            key[i] = ((unsigned long long)orderable(y[i]) << 32) | (0xFFFFFFFFu - (uint32_t)n);
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
          for (int i = 0; i < SPG; i++) {
            const unsigned long long t = __shfl_xor_sync(0xffffffffu, key[i], o);
            key[i] = t > key[i] ? t : key[i];
          }
        }
        if (lane == 0) {
#pragma unroll
          for (int i = 0; i < SPG; i++) R.s_red[(warp & 3) * MAXB + sb + i] = key[i];
        }
        epi_sync();
        if (ep < a.B) {
          unsigned long long k = R.s_red[ep];
          for (int w = 1; w < 4; w++) k = R.s_red[w * MAXB + ep] > k ? R.s_red[w * MAXB + ep] : k;
          atomicMax(&a.best[ep], k);
        }
      }
      if (tlast) tr[11] = globaltimer();
      epi_sync();  // R.ys / R.s_red are reused by the next segment
      if (tlast) tr[12] = globaltimer();
    }
    f = fend;
  }
}

template <int EPI>
__global__ void __launch_bounds__(THREADS, 1) skgemm_kernel(const __grid_constant__ CUtensorMap tmW,
                                                            const __grid_constant__ CUtensorMap tmX, GemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  const Ring R = ring_layout(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = gridDim.x, cta = blockIdx.x;
  const long f0 = (long)cta * a.total / G, f1 = (long)(cta + 1) * a.total / G;
  // RNGD_TRACE == 0 (the product build): tr is a constant null and every stamp below folds away
  unsigned long long* tr = (RNGD_TRACE && a.trace != nullptr) ? a.trace + (size_t)cta * 16 : nullptr;
  if (tr != nullptr && threadIdx.x == 0) tr[0] = globaltimer();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  const uint32_t tmem = ring_setup(R);

  if (warp == 0) {
    if (lane == 0) {
      // the activation operand is written by the previous kernel
      produce_phase(&tmW, &tmX, a, R, 0, f0, f1, [&] {
        grid_dep_wait();
        if (tr != nullptr) tr[1] = globaltimer();
      });
      if (tr != nullptr) tr[2] = globaltimer();
      grid_dep_launch();  // all weight reads issued: the next kernel may start prefetching
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      long i = 0;
      int seg = 0;
      mma_phase(a, R, tmem, i, seg, f0, f1, tr);
      if (tr != nullptr) tr[4] = globaltimer();
      // TMEM is freed below only after every epilogue thread has read its last accumulator
      mbar_wait(R.epi_done, 0u, ST_EPI_WAIT, &g_status_decode);
      tc_fence_after();
      if (tr != nullptr) tr[7] = globaltimer();
    }
    __syncwarp();
    tmem_dealloc(tmem, TMEM_COLS);
  } else {
    grid_dep_wait();
    int seg = 0;
    epilogue_phase<EPI>(a, R, tmem, seg, f0, f1, tr);
    if (tr != nullptr && threadIdx.x == 64) tr[6] = globaltimer();
    tc_fence_before();
    mbar_arrive(R.epi_done);
  }
}

// -------------------------------------------------------- operand producers
// act[b] = hi(h), act[lo_off+b] = lo(h) with h = x * w (w == nullptr: h = x), and,
// when ss != nullptr, ss[t*ss_ld + b] = sum of x^2 over columns [128t, 128t+128).
// One CTA per row.  Also clears the argmax keys when best != nullptr.
__global__ void __launch_bounds__(256) operand_kernel(const float* __restrict__ x, int ldx, int H,
                                                      const float* __restrict__ w, uint16_t* __restrict__ act,
                                                      int ld_act, int lo_off, float* __restrict__ ss, int ss_ld,
                                                      unsigned long long* best) {
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* xr = x + (size_t)b * ldx;
  for (int k = threadIdx.x; k < H; k += 256) {
    const float h = w != nullptr ? xr[k] * w[k] : xr[k];
    const uint16_t hi = f2bf_bits(h);
    act[(size_t)b * ld_act + k] = hi;
    act[(size_t)(lo_off + b) * ld_act + k] = f2bf_bits(h - bf2f(hi));
  }
  if (ss != nullptr) {
    // tile t: four 32-column quarters, each a warp sum, added pairwise like the residual epilogue
    for (int t = warp; t < H / 128; t += 8) {
      float q[4];
#pragma unroll
      for (int qq = 0; qq < 4; qq++) {
        const float v = xr[t * 128 + qq * 32 + lane];
        q[qq] = warp_sum(v * v);
      }
      if (lane == 0) ss[(size_t)t * ss_ld + b] = (q[0] + q[1]) + (q[2] + q[3]);
    }
  }
  if (best != nullptr && threadIdx.x == 0) best[b] = 0ull;
}

__global__ void finalize_argmax_kernel(const unsigned long long* __restrict__ best, int32_t* __restrict__ next,
                                       int B) {
  grid_dep_wait();
  grid_dep_launch();
  const int b = threadIdx.x;
  if (b < B) next[b] = (int32_t)(0xFFFFFFFFu - (uint32_t)(best[b] & 0xFFFFFFFFull));
}

// ------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn get_encode() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)p;
  });
  return fn;
}

static int encode_tmap(CUtensorMapDataType type, CUtensorMap* out, const void* base, int rank, const uint64_t* dims,
                       const uint64_t* strides_bytes, const uint32_t* box) {
  EncodeTiledFn enc = get_encode();
  RNGD_REQUIRE(enc != nullptr, "cuTensorMapEncodeTiled is unavailable");
  RNGD_REQUIRE(((uintptr_t)base & 15) == 0, "tensor map base must be 16-byte aligned");
  cuuint64_t d[5], st[4];
  cuuint32_t bx[5], es[5];
  for (int i = 0; i < rank; i++) {
    d[i] = dims[i];
    bx[i] = box[i];
    es[i] = 1;
  }
  for (int i = 0; i < rank - 1; i++) {
    RNGD_REQUIRE(strides_bytes[i] % 16 == 0, "tensor map strides must be multiples of 16 bytes");
    st[i] = strides_bytes[i];
  }
  CUresult r = enc(out, type, (cuuint32_t)rank, const_cast<void*>(base), d, st, bx, es,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RNGD_ERR_CUDA;
  }
  return RNGD_OK;
}
int encode_tmap_bf16(CUtensorMap* out, const void* base, int rank, const uint64_t* dims,
                     const uint64_t* strides_bytes, const uint32_t* box) {
  return encode_tmap(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, out, base, rank, dims, strides_bytes, box);
}
int encode_tmap_u8(CUtensorMap* out, const void* base, int rank, const uint64_t* dims,
                   const uint64_t* strides_bytes, const uint32_t* box) {
  return encode_tmap(CU_TENSOR_MAP_DATA_TYPE_UINT8, out, base, rank, dims, strides_bytes, box);
}

// cached tensor maps: weights [L][N][K] (3-D) and activation operands [32][K] (2-D)
struct MapKey {
  const void* p;
  uint64_t a, b, c;
  bool operator==(const MapKey& o) const { return p == o.p && a == o.a && b == o.b && c == o.c; }
};
struct MapKeyHash {
  size_t operator()(const MapKey& k) const {
    return std::hash<const void*>()(k.p) ^ (k.a * 0x9E3779B97F4A7C15ull) ^ (k.b << 21) ^ (k.c << 42);
  }
};
static std::mutex g_map_mu;
static std::unordered_map<MapKey, CUtensorMap, MapKeyHash> g_maps;

int get_weight_map(const void* w, int L, int N, int K, CUtensorMap* out) {
  return get_weight_map_rows(w, L, N, K, BM, out);
}

int get_weight_map_rows(const void* w, int L, int N, int K, int rows, CUtensorMap* out) {
  MapKey key{w, (uint64_t)L | ((uint64_t)rows << 32), (uint64_t)N, (uint64_t)K};
  std::lock_guard<std::mutex> g(g_map_mu);
  auto it = g_maps.find(key);
  if (it != g_maps.end()) {
    *out = it->second;
    return RNGD_OK;
  }
  const uint64_t dims[3] = {(uint64_t)K, (uint64_t)N, (uint64_t)L};
  const uint64_t strides[2] = {(uint64_t)K * 2, (uint64_t)K * 2 * N};
  const uint32_t box[3] = {BK, (uint32_t)rows, 1};
  RNGD_TRY(encode_tmap_bf16(out, w, 3, dims, strides, box));
  g_maps[key] = *out;
  return RNGD_OK;
}

int get_operand_map(const void* act, int K, int ld, int rows, int box_rows, CUtensorMap* out) {
  MapKey key{act, (uint64_t)K, (uint64_t)ld, 0xAC70000ull ^ ((uint64_t)rows << 9) ^ (uint64_t)box_rows};
  std::lock_guard<std::mutex> g(g_map_mu);
  auto it = g_maps.find(key);
  if (it != g_maps.end()) {
    *out = it->second;
    return RNGD_OK;
  }
  const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows};
  const uint64_t strides[1] = {(uint64_t)ld * 2};
  const uint32_t box[2] = {BK, (uint32_t)box_rows};
  RNGD_TRY(encode_tmap_bf16(out, act, 2, dims, strides, box));
  g_maps[key] = *out;
  return RNGD_OK;
}

int get_map3_bf16(const void* base, const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
                  CUtensorMap* out) {
  MapKey key{base, dims[0] | (dims[1] << 32), dims[2] | ((uint64_t)box[0] << 32) | ((uint64_t)box[1] << 48),
             (uint64_t)box[2] | (strides_bytes[0] << 8) | (0x3Dull << 56)};
  std::lock_guard<std::mutex> g(g_map_mu);
  auto it = g_maps.find(key);
  if (it != g_maps.end()) {
    *out = it->second;
    return RNGD_OK;
  }
  RNGD_TRY(encode_tmap_bf16(out, base, 3, dims, strides_bytes, box));
  g_maps[key] = *out;
  return RNGD_OK;
}

int num_sms() {
  static int n = 0;
  if (n == 0) {
    int dev = 0, v = 0;
    cudaGetDevice(&dev);
    n = (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0) ? v : kNumSMs;
  }
  return n;
}

// CTAs of a GEMM: one per SM, fewer when there are fewer K blocks than SMs
static int gemm_grid(int N, int K) {
  const long total = (long)((N + BM - 1) / BM) * (K / BK);
  const int g = num_sms();
  return total < g ? (int)total : g;
}

// pieces a tile can be cut into under the stream-K split (for the partial buffer)
static int max_segments(int N, int K, int grid) {
  const long tiles = (N + BM - 1) / BM, nkb = K / BK, total = tiles * nkb;
  int mx = 1;
  for (long t = 0; t < tiles; t++) {
    const int s = owner_of(t * nkb + nkb - 1, total, grid) - owner_of(t * nkb, total, grid) + 1;
    mx = s > mx ? s : mx;
  }
  return mx;
}

// set by rngd_trace_decode_gemms (diagnostics): later GEMM launches without a trace of their
// own record their CTA timelines into consecutive [1024][8] blocks until g_seq_left runs out
static unsigned long long* g_seq = nullptr;
static int g_seq_left = 0;

// the next block of the launch-sequence trace (null when off or used up)
unsigned long long* next_seq_trace() {
  if (!RNGD_TRACE || g_seq == nullptr || g_seq_left <= 0) return nullptr;
  unsigned long long* t = g_seq;
  g_seq += 1024 * 16;
  g_seq_left--;
  return t;
}

static void seq_trace(GemmArgs* a) {
  if (RNGD_TRACE && a->trace == nullptr) a->trace = next_seq_trace();
}

template <int EPI>
static int launch_skgemm(const void* W, int L, int layer, int N, int K, const void* act, int ld_act_in, GemmArgs a,
                         cudaStream_t s) {
  RNGD_REQUIRE(K % BK == 0 && K >= BK, "decode GEMM: K=%d must be a multiple of 64", K);
  RNGD_REQUIRE(N % BM == 0 || EPI == EPI_LOGITS, "decode GEMM: N=%d must be a multiple of 128", N);
  CUtensorMap tw, tx;
  RNGD_TRY(get_weight_map(W, L, N, K, &tw));
  RNGD_TRY(get_operand_map(act, K, ld_act_in, 2 * MAXB, BNC, &tx));
  const int grid = gemm_grid(N, K);
  a.N = N;
  a.K = K;
  a.nkb = K / BK;
  a.tiles = (N + BM - 1) / BM;
  a.total = a.tiles * a.nkb;
  a.maxseg = max_segments(N, K, grid);
  a.layer = layer;
  RNGD_REQUIRE(a.total >= grid, "decode GEMM: %d K blocks cannot feed %d CTAs", a.total, grid);
  RNGD_REQUIRE(a.maxseg == 1 || (a.partial && a.counters), "decode GEMM: split tiles need partial/counters");
  RNGD_REQUIRE(a.tag >= 1 && a.tag <= 15, "decode GEMM: shape tag %d outside 1..15", a.tag);
  seq_trace(&a);
  static std::atomic<unsigned long long> attr_set{0};  // one per EPI instantiation
  RNGD_TRY(set_smem_limit_once((const void*)skgemm_kernel<EPI>, (int)kSmemBytes, &attr_set,
                               "cudaFuncSetAttribute(skgemm)"));
  return launch_pdl(skgemm_kernel<EPI>, dim3(grid), dim3(THREADS), kSmemBytes, s, "skgemm_kernel", tw, tx, a);
}

int launch_operand_ex(const float* x, int ldx, int rows, int H, const float* w, void* act, int ld_act, int lo_off,
                      float* ss, int ss_ld, unsigned long long* best, cudaStream_t s) {
  return launch_pdl(operand_kernel, dim3(rows), dim3(256), 0, s, "operand_kernel", x, ldx, H, w, (uint16_t*)act,
                    ld_act, lo_off, ss, ss_ld, best);
}

int launch_operand(const float* x, int ldx, int B, int H, const float* w, void* act, int ld_act, float* ss,
                   unsigned long long* best, cudaStream_t s) {
  return launch_operand_ex(x, ldx, B, H, w, act, ld_act, MAXB, ss, MAXB, best, s);
}

int launch_attn_decode_act(const float* q, int ldq, const void* kc, const void* vc, const int32_t* pos,
                           const int32_t* lanes, int B,
                           int NH, int NKV, int HD, int S, float* part, void* act, int ld_act, cudaStream_t s);
int launch_embed(const void* emb, const int32_t* toks, int H, int V, float* x, int B, cudaStream_t s);
int launch_kv4_decode_store(void* pool, int P, int NKV, int HD, const int32_t* table, int ld_table, const int32_t* pos,
                            int B, const void* k, const void* v, cudaStream_t s);
int launch_kv4_decode_attn(const float* q, const void* pool, int P, int NKV, int HD, const int32_t* table, int ld_table,
                           const int32_t* pos, int B, int NH, int window, int sinks, void* act, int ld_act,
                           void* workspace, size_t workspace_bytes, cudaStream_t s);

// scratch sizes of one GEMM shape under the stream-K split
static void shape_workspace(int N, int K, size_t* pf, size_t* ct) {
  const int ms = max_segments(N, K, gemm_grid(N, K));
  const size_t tiles = (size_t)(N + BM - 1) / BM;
  *pf = ms > 1 ? 2 * tiles * ms * BM * MAXB : 0;  // 4-byte units of the 64-bit piece words
  *ct = ms > 1 ? tiles : 0;
}

}  // namespace rngd

using namespace rngd;

static int check_tc_io(const rngd_model_t* m, const rngd_decode_io_t* io) {
  RNGD_REQUIRE(m && io, "null model or io");
  RNGD_REQUIRE(m->HD == 128 && m->NH == 4 * m->NKV, "decode: kernels are built for HD=128, NH=4*NKV");
  RNGD_REQUIRE(m->H % 128 == 0 && (2 * m->M) % 128 == 0 && m->M % 64 == 0,
               "decode: H and 2*M must be multiples of 128");
  RNGD_REQUIRE(io->B >= 1 && io->B <= 16 && (io->lanes != nullptr || io->B <= io->Bcap) && io->Bcap >= 1,
               "decode: B=%d outside 1..16 (and <= Bcap=%d without a lane map)", io->B, io->Bcap);
  RNGD_REQUIRE(io->S % 128 == 0 && io->S > 0 && io->S <= 8192, "decode: S=%d must be a multiple of 128", io->S);
  RNGD_REQUIRE(io->kcache && io->vcache && io->toks && io->pos && io->x && io->q && io->act && io->act_o &&
                   io->act2 && io->ss && io->logits && io->attn_part && io->partial && io->counters && io->best &&
                   io->next,
               "decode: null buffer");
  return RNGD_OK;
}

// The decode step's GEMM shapes: QKV, O, gate/up, down, LM head.  They share one partial
// scratch (their flags carry tag = index + 1) and each has its own run of tile epochs in the
// counters array, starting at off[index].
static void decode_shapes(const rngd_model_t* m, size_t off[5], size_t* pf_max, size_t* ct_sum) {
  const int QN = m->NH * m->HD, KN = m->NKV * m->HD;
  const int shapes[5][2] = {{QN + 2 * KN, m->H}, {m->H, QN}, {2 * m->M, m->H}, {m->H, m->M}, {m->V, m->H}};
  size_t pf = 0, ct = 0;
  for (int i = 0; i < 5; i++) {
    size_t p, c;
    shape_workspace(shapes[i][0], shapes[i][1], &p, &c);
    off[i] = ct;
    pf = pf > p ? pf : p;
    ct += c;
  }
  *pf_max = pf;
  *ct_sum = ct;
}

extern "C" int rngd_decode_workspace(const rngd_model_t* m, int S, size_t* partial_floats, size_t* counters,
                                     size_t* act_cols, size_t* act2_cols) {
  RNGD_REQUIRE(m && partial_floats && counters && act_cols && act2_cols, "workspace: null argument");
  const int QN = m->NH * m->HD;
  size_t off[5], pf, ct;
  decode_shapes(m, off, &pf, &ct);
  *partial_floats = pf;
  *counters = ct;
  *act_cols = (size_t)(m->H > QN ? m->H : QN);
  *act2_cols = (size_t)m->M;
  (void)S;
  return RNGD_OK;
}

extern "C" int rngd_decode_attn_workspace(const rngd_model_t* m, int Bcap, int S, size_t* attn_units) {
  RNGD_REQUIRE(m && attn_units, "attn_workspace: null argument");
  RNGD_REQUIRE(Bcap >= 1 && Bcap <= 16 && S % 128 == 0 && S > 0, "attn_workspace: Bcap=%d S=%d", Bcap, S);
  *attn_units = attn_fused_scratch_units(Bcap, m->NKV, S);
  return RNGD_OK;
}

static unsigned long long* g_trace = nullptr;  // set by rngd_tc_gemv_trace (diagnostics)

unsigned long long* rngd::gemm_trace() { return g_trace; }

extern "C" int rngd_tc_gemv_trace(uint64_t* trace) {
  if (!RNGD_TRACE && trace != nullptr) {
    set_error("tc_gemv_trace: this library was built without tracing (make TRACE=1)");
    return RNGD_ERR_UNSUPPORTED;
  }
  g_trace = (unsigned long long*)trace;
  return RNGD_OK;
}

extern "C" int rngd_trace_decode_gemms(uint64_t* trace, int launches) {
  RNGD_REQUIRE(launches >= 0, "trace_decode_gemms: negative launch count");
  if (!RNGD_TRACE && trace != nullptr) {
    set_error("trace_decode_gemms: this library was built without tracing (make TRACE=1)");
    return RNGD_ERR_UNSUPPORTED;
  }
  g_seq = (unsigned long long*)trace;
  g_seq_left = trace != nullptr ? launches : 0;
  return RNGD_OK;
}


extern "C" int rngd_tc_gemv(const void* W, int N, int K, const float* X, int ldx, int B, float* Y, int ldy,
                            void* act, float* partial, int32_t* counters, int prep, rngd_stream_t stream) {
  RNGD_REQUIRE(W && X && Y && act, "tc_gemv: null pointer");
  RNGD_REQUIRE(B >= 1 && B <= MAXB, "tc_gemv: B=%d outside 1..16", B);
  RNGD_REQUIRE(N % BM == 0 && K % BK == 0, "tc_gemv: need N %% 128 == 0 and K %% 64 == 0 (N=%d K=%d)", N, K);
  cudaStream_t s = (cudaStream_t)stream;
  if (prep) RNGD_TRY(launch_operand(X, ldx, B, K, nullptr, act, K, nullptr, nullptr, s));
  GemmArgs a = {};
  a.B = B;
  a.partial = partial;
  a.counters = counters;
  a.tag = 6;
  a.x = Y;
  a.ldx = ldy;
  a.trace = g_trace;
  return launch_skgemm<EPI_RESID>(W, 1, 0, N, K, act, K, a, s);
}

extern "C" int rngd_tc_gemv_workspace(int N, int K, size_t* partial_floats, size_t* counters) {
  RNGD_REQUIRE(partial_floats && counters, "tc_gemv_workspace: null argument");
  shape_workspace(N, K, partial_floats, counters);
  return RNGD_OK;
}

// Arguments of one of a decode layer's GEMMs (kind 0 QKV, 1 O, 2 gate/up, 3 down) at layer l of
// a call that holds layers [layer0, ..) in io's cache block.
static GemmArgs layer_args(const rngd_model_t* m, const rngd_decode_io_t* io, int layer0, int l, int kind,
                           const size_t off[5]) {
  const int H = m->H, QN = m->NH * m->HD;
  const int ld_act = H > QN ? H : QN;
  const size_t lane_elems = (size_t)m->NKV * io->S * m->HD;
  GemmArgs a = {};
  a.B = io->B;
  a.partial = io->partial;
  a.counters = io->counters + off[kind];
  a.tag = kind + 1;
  a.ss_in = io->ss;
  a.ss_tiles = H / BM;
  a.eps = m->eps;
  a.inv_h = 1.0f / (float)H;
  if (kind == 0) {  // RoPE + KV append at pos; q for the attention
    a.pos = io->pos;
    a.inv = m->inv_freq;
    a.q = io->q;
    a.ldq = QN;
    a.kc = (uint16_t*)io->kcache + (size_t)(l - layer0) * io->Bcap * lane_elems;
    a.vc = (uint16_t*)io->vcache + (size_t)(l - layer0) * io->Bcap * lane_elems;
    a.lanes = io->lanes;
    a.NH = m->NH;
    a.NKV = m->NKV;
    a.S = io->S;
  } else if (kind == 2) {  // SwiGLU into the down projection's operand
    a.act_out = (uint16_t*)io->act2;
    a.ld_act = m->M;
  } else {  // residual; the O GEMM writes x * n2[l], the down GEMM x * n1[l+1] (or the final norm)
    a.x = io->x;
    a.ldx = H;
    a.w_next = kind == 1 ? m->n2 + (size_t)l * H : (l + 1 < m->L ? m->n1 + (size_t)(l + 1) * H : m->norm);
    a.act_next = (uint16_t*)io->act;
    a.ld_next = ld_act;
    a.ss_out = io->ss;
  }
  return a;
}

extern "C" int rngd_decode_layers(const rngd_model_t* m, const rngd_decode_io_t* io, int layer0, int layer1,
                                  rngd_stream_t stream) {
  RNGD_TRY(check_tc_io(m, io));
  RNGD_REQUIRE(0 <= layer0 && layer0 <= layer1 && layer1 <= m->L, "decode: layers [%d, %d) outside [0, %d)",
               layer0, layer1, m->L);
  RNGD_REQUIRE(layer1 - layer0 <= io->kv_layers, "decode: %d layers requested but the cache block holds %d",
               layer1 - layer0, io->kv_layers);
  if (layer0 == layer1) return RNGD_OK;
  cudaStream_t s = (cudaStream_t)stream;
  const int H = m->H, Mi = m->M, QN = m->NH * m->HD, KN = m->NKV * m->HD, NQKV = QN + 2 * KN;
  const int ld_act = H > QN ? H : QN;
  const size_t lane_elems = (size_t)m->NKV * io->S * m->HD;
  size_t off[5], pf, ct;
  decode_shapes(m, off, &pf, &ct);
  auto attention = [&](int l) {
    const uint16_t* kc = (const uint16_t*)io->kcache + (size_t)(l - layer0) * io->Bcap * lane_elems;
    const uint16_t* vc = (const uint16_t*)io->vcache + (size_t)(l - layer0) * io->Bcap * lane_elems;
    return launch_attn_decode_act(io->q, QN, kc, vc, io->pos, io->lanes, io->B, m->NH, m->NKV, m->HD, io->S,
                                  io->attn_part, io->act_o, QN, s);
  };
  // layer0's QKV GEMM reads io->act = x * n1[layer0] (the prologue's or the previous call's)
  RNGD_TRY(launch_skgemm<EPI_QKV>(m->wqkv, m->L, layer0, NQKV, H, io->act, ld_act,
                                  layer_args(m, io, layer0, layer0, 0, off), s));
  for (int l = layer0; l < layer1; l++) {
    RNGD_TRY(attention(l));
    RNGD_TRY(launch_skgemm<EPI_RESID>(m->wo, m->L, l, H, QN, io->act_o, QN, layer_args(m, io, layer0, l, 1, off), s));
    RNGD_TRY(launch_skgemm<EPI_SWIGLU>(m->wgu, m->L, l, 2 * Mi, H, io->act, ld_act,
                                       layer_args(m, io, layer0, l, 2, off), s));
    RNGD_TRY(launch_skgemm<EPI_RESID>(m->wd, m->L, l, H, Mi, io->act2, Mi, layer_args(m, io, layer0, l, 3, off), s));
    if (l + 1 < layer1)
      RNGD_TRY(launch_skgemm<EPI_QKV>(m->wqkv, m->L, l + 1, NQKV, H, io->act, ld_act,
                                      layer_args(m, io, layer0, l + 1, 0, off), s));
  }
  return RNGD_OK;
}

extern "C" int rngd_decode_kv4_workspace(const rngd_model_t* m, int B, int ld_table, int window, int sinks, size_t* bytes) {
  RNGD_REQUIRE(m && bytes, "decode_kv4_workspace: null argument");
  return rngd_kv4_attn_workspace(RNGD_DT_F32, B, 1, m->NH, m->NKV, m->HD, ld_table, window, sinks, bytes);
}

// The layers of rngd_decode_layers over the paged 4-bit cache: the QKV GEMM leaves the new rows in bf16, a
// kernel stores them in the pages, the attention reads the pages and writes the O projection's operand.
extern "C" int rngd_decode_layers_kv4(const rngd_model_t* m, const rngd_decode_io_t* io_in, const rngd_kv4_t* kv,
                                      int layer0, int layer1, rngd_stream_t stream) {
  RNGD_REQUIRE(m && io_in && kv, "decode_layers_kv4: null argument");
  RNGD_REQUIRE(kv->pool && kv->rows && (kv->table || kv->ld_table == 0) && kv->ld_table >= 0,
               "decode_layers_kv4: null buffer");
  rngd_decode_io_t io = *io_in;  // the cache of the checks and of the GEMM's epilogue: the new rows
  const size_t row_elems = (size_t)MAXB * m->NKV * m->HD;
  io.kcache = kv->rows;
  io.vcache = (uint16_t*)kv->rows + row_elems;
  io.Bcap = MAXB;
  io.S = 128;
  io.lanes = nullptr;
  RNGD_TRY(check_tc_io(m, &io));
  RNGD_REQUIRE(0 <= layer0 && layer0 <= layer1 && layer1 <= m->L, "decode_layers_kv4: layers [%d, %d) outside [0, %d)",
               layer0, layer1, m->L);
  if (layer0 == layer1) return RNGD_OK;
  cudaStream_t s = (cudaStream_t)stream;
  const int H = m->H, Mi = m->M, QN = m->NH * m->HD, KN = m->NKV * m->HD, NQKV = QN + 2 * KN;
  const int ld_act = H > QN ? H : QN;
  size_t off[5], pf, ct;
  decode_shapes(m, off, &pf, &ct);
  auto qkv = [&](int l) {
    GemmArgs a = layer_args(m, &io, layer0, l, 0, off);
    a.kc = (uint16_t*)io.kcache;
    a.vc = (uint16_t*)io.vcache;
    a.S = 1;
    a.kv_rows = 1;
    return launch_skgemm<EPI_QKV>(m->wqkv, m->L, l, NQKV, H, io.act, ld_act, a, s);
  };
  for (int l = layer0; l < layer1; l++) {
    uint8_t* pool = (uint8_t*)kv->pool + (size_t)(l - layer0) * kv->layer_bytes;
    RNGD_TRY(qkv(l));
    RNGD_TRY(launch_kv4_decode_store(pool, kv->P, m->NKV, m->HD, kv->table, kv->ld_table, io.pos, io.B, io.kcache,
                                     io.vcache, s));
    RNGD_TRY(launch_kv4_decode_attn(io.q, pool, kv->P, m->NKV, m->HD, kv->table, kv->ld_table, io.pos, io.B, m->NH,
                                    kv->window, kv->sinks, io.act_o, QN, kv->workspace, kv->workspace_bytes, s));
    RNGD_TRY(launch_skgemm<EPI_RESID>(m->wo, m->L, l, H, QN, io.act_o, QN, layer_args(m, &io, layer0, l, 1, off), s));
    RNGD_TRY(launch_skgemm<EPI_SWIGLU>(m->wgu, m->L, l, 2 * Mi, H, io.act, ld_act, layer_args(m, &io, layer0, l, 2, off), s));
    RNGD_TRY(launch_skgemm<EPI_RESID>(m->wd, m->L, l, H, Mi, io.act2, Mi, layer_args(m, &io, layer0, l, 3, off), s));
  }
  return RNGD_OK;
}

extern "C" int rngd_decode_lmhead(const rngd_model_t* m, const rngd_decode_io_t* io, rngd_stream_t stream) {
  RNGD_TRY(check_tc_io(m, io));
  cudaStream_t s = (cudaStream_t)stream;
  const int H = m->H, QN = m->NH * m->HD;
  const int ld_act = H > QN ? H : QN;
  // io->act holds x * norm from the last layer's residual epilogue
  GemmArgs a = {};
  size_t off[5], pf, ct;
  decode_shapes(m, off, &pf, &ct);
  a.B = io->B;
  a.partial = io->partial;
  a.counters = io->counters + off[4];
  a.tag = 5;
  a.ss_in = io->ss;
  a.ss_tiles = H / BM;
  a.eps = m->eps;
  a.inv_h = 1.0f / (float)H;
  a.logits = io->logits;
  a.best = (unsigned long long*)io->best;
  a.V = m->V;
  RNGD_TRY(launch_skgemm<EPI_LOGITS>(m->lm, 1, 0, m->V, H, io->act, ld_act, a, s));
  return launch_pdl(finalize_argmax_kernel, dim3(1), dim3(32), 0, s, "finalize_argmax_kernel",
                    (const unsigned long long*)io->best, io->next, io->B);
}

// x = embed[toks]; act = hi/lo(x * n1[0]); ss = per-tile sums of squares; argmax
// keys cleared for this step's lm_head (engines/decode_batch.py:432).
extern "C" int rngd_decode_embed(const rngd_model_t* m, const rngd_decode_io_t* io, rngd_stream_t stream) {
  RNGD_TRY(check_tc_io(m, io));
  cudaStream_t s = (cudaStream_t)stream;
  RNGD_TRY(launch_embed(m->embed, io->toks, m->H, m->V, io->x, io->B, s));
  const int H = m->H, QN = m->NH * m->HD;
  const int ld_act = H > QN ? H : QN;
  return launch_operand(io->x, H, io->B, H, m->n1, io->act, ld_act, io->ss, (unsigned long long*)io->best, s);
}

// io->x already holds the residual stream (fp32 [B][H], written by the caller): layer0's first
// operand hi/lo(x * n1[layer0]) and the sums of squares, argmax keys cleared.  Starts a run of
// layer groups from a hidden state the caller supplies (kernels/decode_batch.py:100-109:
// DecodeModel.forward receives x rather than token ids).
extern "C" int rngd_decode_begin(const rngd_model_t* m, const rngd_decode_io_t* io, int layer0,
                                 rngd_stream_t stream) {
  RNGD_TRY(check_tc_io(m, io));
  RNGD_REQUIRE(0 <= layer0 && layer0 < m->L, "decode_begin: layer %d outside [0, %d)", layer0, m->L);
  const int H = m->H, QN = m->NH * m->HD;
  const int ld_act = H > QN ? H : QN;
  return launch_operand(io->x, H, io->B, H, m->n1 + (size_t)layer0 * H, io->act, ld_act, io->ss,
                        (unsigned long long*)io->best, (cudaStream_t)stream);
}

// Final norm + lm_head + first-max argmax for `rows` (<= 16) rows of x, e.g. the
// last prompt position of a prefill (engines/prefill_full.py:265-270).
extern "C" int rngd_lmhead_rows(const rngd_model_t* m, const float* x, int ldx, int rows, void* act, float* ss,
                                float* logits, uint64_t* best, int32_t* next, float* partial, int32_t* counters,
                                rngd_stream_t stream) {
  RNGD_REQUIRE(m && x && act && ss && logits && best && next, "lmhead_rows: null argument");
  RNGD_REQUIRE(rows >= 1 && rows <= MAXB, "lmhead_rows: rows=%d outside 1..16", rows);
  cudaStream_t s = (cudaStream_t)stream;
  const int H = m->H;
  RNGD_TRY(launch_operand_ex(x, ldx, rows, H, m->norm, act, H, MAXB, ss, MAXB, (unsigned long long*)best, s));
  GemmArgs a = {};
  a.B = rows;
  a.partial = partial;
  a.counters = counters;
  a.tag = 5;
  a.ss_in = ss;
  a.ss_tiles = H / BM;
  a.eps = m->eps;
  a.inv_h = 1.0f / (float)H;
  a.logits = logits;
  a.best = (unsigned long long*)best;
  a.V = m->V;
  RNGD_TRY(launch_skgemm<EPI_LOGITS>(m->lm, 1, 0, m->V, H, act, H, a, s));
  return launch_pdl(finalize_argmax_kernel, dim3(1), dim3(32), 0, s, "finalize_argmax_kernel",
                    (const unsigned long long*)best, next, rows);
}

extern "C" int rngd_lmhead_workspace(const rngd_model_t* m, size_t* partial_floats, size_t* counters) {
  RNGD_REQUIRE(m && partial_floats && counters, "lmhead_workspace: null argument");
  shape_workspace(m->V, m->H, partial_floats, counters);
  return RNGD_OK;
}

int rngd::read_status_decode(int* st, int reset) {
  RNGD_TRY(check_cuda(cudaMemcpyFromSymbol(st, g_status_decode, sizeof(int)), "read device status"));
  if (reset) {
    const int zero = 0;
    RNGD_TRY(check_cuda(cudaMemcpyToSymbol(g_status_decode, &zero, sizeof(int)), "reset device status"));
  }
  return RNGD_OK;
}

extern "C" int rngd_device_status(int* status, int reset) {
  RNGD_REQUIRE(status != nullptr, "device_status: null output");
  int st = 0, sp = 0, sa = 0, s4 = 0;
  RNGD_TRY(read_status_decode(&st, reset));
  RNGD_TRY(read_status_prefill(&sp, reset));
  RNGD_TRY(read_status_attn(&sa, reset));
  RNGD_TRY(read_status_kv4(&s4, reset));
  *status = st != 0 ? st : (sp != 0 ? sp : (sa != 0 ? sa : s4));
  return RNGD_OK;
}
