// Attention of a few query tokens over the paged 4-bit KV cache (layout in kv4.cuh).
//
// The reference attends over bf16 lanes (src/rngd_pd/kernels/decode_batch.py:73-91); the cache read here
// takes 5 bits a value, and positions may be limited to a window and a few first ones (sinks).
#include "kv4.cuh"

namespace rngd {

// ------------------------------------------------------------------------------------ attention
// o = softmax(scale q K^T) V over the pages of each stream, on the warp-level tensor cores.
//
// Work is cut into units of 32 positions of a (stream, kv head, row tile), laid end to end, and every
// warp (a CTA of its own) takes an equal contiguous run of them, whatever the lengths: a long stream is
// split over many warps, many short streams share one.  A segment (all units of one (stream, kv head,
// row tile)) that one warp holds whole is written at once; a cut one leaves its pieces as records
// (maximum, sum, unnormalised output), which a second kernel joins in the order of the positions.
//
// Units arrive by bulk copy (a unit is one contiguous run of 2 blocks) in a ring of stages.  The lane
// whose turn it is looks its unit up 32 units ahead (stream by search in the prefix sums, page id) and
// issues the copy itself.
//
// A block's codes go straight from shared memory into matrix fragments: or-ing a code into the upper
// mantissa bits of fp16 16.0 gives 16 + u, and one fused multiply-add per pair of values by the group's
// (s, c) gives the value, exactly as it is defined.  S = K q^T has the keys as its 16 rows and 8 columns
// for the query rows that share the kv head; O^T = V^T P has 16 dimensions as its rows.  q enters as
// fp16 scaled by a power of two (exact for 16-bit q), fp32 q as fp16 hi + lo, and P as hi + lo, so that
// the result keeps fp32 accuracy.  With up to 4 rows the lo halves take the columns that would stay
// empty (COLS: hi in columns 0..3, lo in 4..7, one matrix instruction for both); with more they are
// products of their own into the same accumulators.  Probabilities are held as 2^(x - m + 8), x the
// score in units of log 2 and m a running maximum that is only moved when a score exceeds it by 6: the
// output is rescaled rarely, and hi + lo hold a probability to 2^-23 of itself, or to 2^-33 of the row's
// largest where that is more.  What is smaller than that is left out of the output and stays in the sum: n
// such positions take n * 2^-33 off the result at most (65000: 8e-6, where all but one are that small).
constexpr int kUnit = 32;
constexpr int kAttnStreams = 1024;  // streams of one launch
constexpr float kPBias = 8.0f, kPMax = 14.0f;

__device__ int g_status_kv4 = 0;

struct AttnArgs {
  const void* q;
  void* out;
  long qs[3], os[3];  // strides in elements: stream, token, head
  long lo_off;        // 0: out is of q's type; else bf16, hi at its place and lo (out - hi) so far behind
  int len_add;        // positions held beyond lens[b]
  int dt, qvec, B, T, NH, NKV, G, RT, P, ld_table, window, sinks;
  const uint8_t* pool;
  const int32_t* table;
  const int32_t* lens;
  float scale;
  int* pre;     // [B + 1] prefix sums of units, for the joining kernel
  float* rec;   // [warps][2][rows][HD + 4]: output, maximum, sum
};

__device__ __forceinline__ void put_out(const AttnArgs& a, size_t at, float v) {
  if (a.lo_off == 0) {
    store1(a.out, at, a.dt, v);
  } else {
    const uint16_t hi = f2bf_bits(v);
    ((uint16_t*)a.out)[at] = hi;
    ((uint16_t*)a.out)[at + a.lo_off] = f2bf_bits(v - bf2f(hi));
  }
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// What a stream of n positions has to look at: units [0, su) hold sinks before the window, units
// [start, end) the window.
struct Span {
  int su, start, end;
  __device__ __forceinline__ int units() const { return su + end - start; }
  __device__ __forceinline__ int at(int x) const { return x < su ? x : start + x - su; }
};
__device__ __forceinline__ Span span_of(int n, const AttnArgs& a) {
  Span s;
  const int held = min(max(n, 0), a.ld_table * kPage);
  const int low = a.window > 0 ? max(0, max(n - a.T, 0) - a.window + 1) : 0;
  s.end = (held + kUnit - 1) / kUnit;
  s.su = min((min(a.sinks, low) + kUnit - 1) / kUnit, s.end);
  s.start = min(max(low / kUnit, s.su), s.end);
  return s;
}

// Prefix sums over the streams of one launch, by one warp: pre[b] = units before stream b.
__device__ __forceinline__ void prefix_units(const AttnArgs& a, int* lens, int* pre) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < a.B ? a.lens[b] + a.len_add : 0;
    int x = b < a.B ? span_of(n, a).units() * a.NKV * a.RT : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (b < a.B) {
      lens[b] = n;
      pre[b + 1] = base + x;
    }
    base += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) pre[0] = 0;
  __syncwarp();
}

// One unit, as its lane looked it up.
struct Unit {
  int seg;    // (stream * NKV + kv head) * RT + row tile
  int pos;    // first position | blocks to read (0..2) | 4: every row sees every position
  size_t off; // of its first block in the pool
};

template <int HD>
__device__ __forceinline__ Unit unit_at(const AttnArgs& a, int b, int kvh, int at, int n, int held) {
  const int p0 = at * kUnit;
  const int page = a.table[(size_t)b * a.ld_table + p0 / kPage];
  const int blocks = page >= 0 && page < a.P ? min(2, (held - p0 + kBlk - 1) / kBlk) : 0;
  const bool all = p0 + kUnit <= held && p0 + kUnit - 1 <= n - a.T &&
                   (a.window == 0 || p0 > n - 1 - a.window || p0 + kUnit <= a.sinks);
  Unit u;
  u.seg = 0;
  u.pos = p0 | blocks | (all ? 4 : 0);
  u.off = (((size_t)max(page, 0) * a.NKV + kvh) * 4 + ((p0 & (kPage - 1)) >> 4)) * kv4_block_bytes(HD);
  return u;
}

template <int HD>
__device__ __forceinline__ Unit look_up(int x, const AttnArgs& a, const int* lens, const int* pre) {
  int lo = 0, hi = a.B - 1;  // pre[lo] <= x < pre[hi + 1]
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= x) lo = mid; else hi = mid - 1;
  }
  const int n = lens[lo], per = a.NKV * a.RT;
  const Span s = span_of(n, a);
  const int ub = s.units(), rem = x - pre[lo], sg = rem / ub;
  Unit u = unit_at<HD>(a, lo, sg / a.RT, s.at(rem - sg * ub), n, min(n, a.ld_table * kPage));
  u.seg = lo * per + sg;
  return u;
}

// Eight consecutive elements of 16-bit q as fp32.
__device__ __forceinline__ void unpack_q8(const uint4& u, int dt, float* x) {
  if (dt == DT_BF16) {
    unpack8(u, x);
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float2 f = __half22float2(u2h(w[e]));
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
  }
}

// How the halves of q and P are laid out (see above), for 16-bit and for fp32 q.  Matrix instructions cut
// their sums off instead of rounding them; for fp32 q, whose results show it, scores are summed in fp32
// from one short chain per 32 dimensions, and the output is moved every kFlush units from the matrix
// accumulators to fp32 sums in shared memory (65000 positions: 5e-7 off instead of 3e-6; 8x40000: 90 us
// instead of 84).
enum : int { COLS = 0, Q16 = 1, Q32 = 2, COLS32 = 3 };
constexpr int kFlush = 4;

// One warp's state for a segment.  NT tiles of 8 columns; a column is a query row, or with COLS the hi
// (columns 0..3) or lo (4..7) half of one.  Lane = 4 g + t as in the fragments.
template <int HD, int NT, int MODE>
struct Rows {
  static constexpr int NG = HD / 32;
  static constexpr bool SPLIT = MODE == COLS || MODE == COLS32, FLUSH = MODE == Q32 || MODE == COLS32;
  static constexpr int CPT = SPLIT ? 4 : 8;  // rows of a column tile
  static constexpr int QL = MODE == Q32 ? NT : 1;
  uint32_t qf[NT][NG][4], ql[QL][NG][4];
  float o[NT][NG][2][4];
  float f[NT][2], mb[NT][2], l[NT][2];  // of columns 2t, 2t + 1 (rows 2 (t & 1), + 1 with SPLIT)
  int i[NT][2];                         // their positions, -1: none
  float* acc;                           // this lane's sums of o, 32 floats apart (FLUSH)
  int since;                            // units since they were last added to

  template <class F>
  __device__ __forceinline__ void each_sum(F f) {  // f(sum, its part in o, its column e)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int j = 0; j < NG; j++)
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
          for (int k = 0; k < 4; k++) f(acc[(((nt * NG + j) * 2 + q) * 4 + k) * 32], o[nt][j][q][k], nt, k & 1);
  }

  // A segment's q as it lies in memory: this lane's eight elements of each row and 32 dimensions.  All loads
  // are issued before any is used (one after the other they cost a memory latency each: 1x387 took 8.1 us in a graph, 7.3
  // so; 16x1000 with 20 rows of 128 16.3 and 13.8).
  static constexpr int QV = FLUSH ? 2 : 1;  // 16-byte vectors of eight elements
  struct Query {
    uint4 v[NT][NG][QV];
  };
  __device__ __forceinline__ void fetch(const AttnArgs& a, int seg, Query& q) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rt = seg % a.RT, kvh = seg / a.RT % a.NKV, b = seg / a.RT / a.NKV;
    const int R = a.T * a.G;
    size_t at[NT];
    bool there[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = (rt * NT + nt) * CPT + (SPLIT ? g & 3 : g);
      there[nt] = r < R;
      at[nt] = (size_t)(b * a.qs[0] + r / a.G * a.qs[1] + (kvh * a.G + r % a.G) * a.qs[2]) + 8 * t;
    }
    if (a.qvec) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < NG; j++)
#pragma unroll
          for (int h = 0; h < QV; h++) {
            q.v[nt][j][h] = make_uint4(0u, 0u, 0u, 0u);
            if (there[nt]) q.v[nt][j][h] = __ldg((const uint4*)((const uint8_t*)a.q + (at[nt] + 32 * j) * (2 * QV)) + h);
          }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < NG; j++)
#pragma unroll
          for (int h = 0; h < QV; h++) {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
            if (there[nt]) {
              const size_t i0 = at[nt] + 32 * j + 4 * h;
#pragma unroll
              for (int e = 0; e < 4; e++) {
                if constexpr (FLUSH)
                  w[e] = ((const uint32_t*)a.q)[i0 + e];
                else
                  w[e] = (uint32_t)((const uint16_t*)a.q)[i0 + 2 * e] | (uint32_t)((const uint16_t*)a.q)[i0 + 2 * e + 1] << 16;
              }
            }
            q.v[nt][j][h] = make_uint4(w[0], w[1], w[2], w[3]);
          }
    }
  }

  __device__ __forceinline__ void begin(const AttnArgs& a, int seg, int n, const Query& q) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rt = seg % a.RT, R = a.T * a.G;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float x[NG][8];
      float mx = 0.0f;
#pragma unroll
      for (int j = 0; j < NG; j++) {
        if constexpr (FLUSH) {
          const uint4 u = q.v[nt][j][0], v = q.v[nt][j][QV - 1];
          const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 8; e++) x[j][e] = __uint_as_float(w[e]);
        } else {
          unpack_q8(q.v[nt][j][0], a.dt, x[j]);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[j][e]));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // scale by the power of two that brings the largest into [2^10, 2^11)
      const int ex = min(max((int)(__float_as_uint(mx) >> 23), 40), 254);
      const float up = __uint_as_float((uint32_t)(264 - ex) << 23);
      const float fc = a.scale * 1.4426950408889634f * (1.0f / up);
#pragma unroll
      for (int j = 0; j < NG; j++) {
#pragma unroll
        for (int p = 0; p < 4; p++) {
          const float x0 = x[j][p] * up, x1 = x[j][p + 4] * up;
          const uint32_t hi = pack_h2(x0, x1);
          qf[nt][j][p] = hi;
          if constexpr (MODE != Q16) {  // 16-bit q has a lo half of zeros
            const float2 hf = __half22float2(u2h(hi));
            const uint32_t lo = pack_h2(x0 - hf.x, x1 - hf.y);
            if constexpr (SPLIT) {
              if (g >= 4) qf[nt][j][p] = lo;
            } else {
              ql[nt][j][p] = lo;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
          for (int k = 0; k < 4; k++) o[nt][j][e][k] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int col = (SPLIT ? 2 * (t & 1) : 2 * t) + e;
        f[nt][e] = __shfl_sync(0xffffffffu, fc, 4 * col);
        const int rr = (rt * NT + nt) * CPT + col;
        i[nt][e] = rr < R ? n - a.T + rr / a.G : -1;
        mb[nt][e] = 1e30f;
        l[nt][e] = 0.0f;
      }
    }
    if constexpr (FLUSH) {
      since = 0;
      each_sum([](float& sum, float&, int, int) { sum = 0.0f; });
    }
  }

  // S += K q^T of one block.
  __device__ __forceinline__ void scores(const uint8_t* blk, float (&c)[NT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t w0[NG], w1[NG], s0[NG], s1[NG];
    if constexpr (NG == 4) {
      const uint4 x = *(const uint4*)(blk + g * 64 + t * 16), y = *(const uint4*)(blk + (g + 8) * 64 + t * 16);
      w0[0] = x.x; w0[1] = x.y; w0[2] = x.z; w0[3] = x.w;
      w1[0] = y.x; w1[1] = y.y; w1[2] = y.z; w1[3] = y.w;
      const uint4 u = *(const uint4*)(blk + 16 * HD + g * 16), v = *(const uint4*)(blk + 16 * HD + (g + 8) * 16);
      s0[0] = u.x; s0[1] = u.y; s0[2] = u.z; s0[3] = u.w;
      s1[0] = v.x; s1[1] = v.y; s1[2] = v.z; s1[3] = v.w;
    } else {
      const uint2 x = *(const uint2*)(blk + g * 32 + t * 8), y = *(const uint2*)(blk + (g + 8) * 32 + t * 8);
      w0[0] = x.x; w0[1] = x.y;
      w1[0] = y.x; w1[1] = y.y;
      const uint2 u = *(const uint2*)(blk + 16 * HD + g * 8), v = *(const uint2*)(blk + 16 * HD + (g + 8) * 8);
      s0[0] = u.x; s0[1] = u.y;
      s1[0] = v.x; s1[1] = v.y;
    }
#pragma unroll
    for (int j = 0; j < NG; j++) {
      uint32_t x[4], y[4];
      decode_word(w0[j], __low2half2(u2h(s0[j])), __high2half2(u2h(s0[j])), x);
      decode_word(w1[j], __low2half2(u2h(s1[j])), __high2half2(u2h(s1[j])), y);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        float t[4] = {};
        float(&d)[4] = FLUSH ? t : c[nt];
        if constexpr (MODE == Q32) {  // the small products first
          mma_f16(d, x[0], y[0], x[1], y[1], ql[nt][j][0], ql[nt][j][1]);
          mma_f16(d, x[2], y[2], x[3], y[3], ql[nt][j][2], ql[nt][j][3]);
        }
        mma_f16(d, x[0], y[0], x[1], y[1], qf[nt][j][0], qf[nt][j][1]);
        mma_f16(d, x[2], y[2], x[3], y[3], qf[nt][j][2], qf[nt][j][3]);
        if constexpr (FLUSH) {
#pragma unroll
          for (int k = 0; k < 4; k++) c[nt][k] += t[k];
        }
      }
    }
  }

  // The pairs of keys (2t, 2t + 1) and (2t + 8, 2t + 9) of a block, as bits of four, whose V is NaN.
  __device__ __forceinline__ uint32_t nan_values(const uint8_t* blk) {
    const int t = threadIdx.x & 3;
    uint32_t bad = 0;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int j = 0; j < NG; j++) {
        const uint32_t s = *(const uint32_t*)(blk + 18 * HD + ((h * 4 + t) * NG + j) * 8);
        bad |= ((s & 0x7FFFu) > 0x7C00u ? 1u : 0u) << (2 * h);
        bad |= ((s >> 16 & 0x7FFFu) > 0x7C00u ? 2u : 0u) << (2 * h);
      }
    return bad;
  }

  // O^T += V^T P of one block; the keys of `drop` (bits as above) are left out.
  template <bool EDGE>
  __device__ __forceinline__ void output(const uint8_t* blk, const uint32_t (&pb)[NT][2],
                                         const uint32_t (&pl)[SPLIT ? 1 : NT][2], uint32_t drop) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint32_t wa[2][NG / 2], wb[2][NG / 2], vs[2][NG], vc[2][NG];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      if constexpr (NG == 4) {
        const uint4 x = *(const uint4*)(blk + 8 * HD + h * 512 + g * 64 + t * 16);
        wa[h][0] = x.x; wa[h][1] = x.y; wb[h][0] = x.z; wb[h][1] = x.w;
      } else {
        const uint2 x = *(const uint2*)(blk + 8 * HD + h * 256 + g * 32 + t * 8);
        wa[h][0] = x.x; wb[h][0] = x.y;
      }
      const uint8_t* sp = blk + 18 * HD + (h * 4 + t) * NG * 8;
#pragma unroll
      for (int j = 0; j < NG; j += 2) {
        const uint4 x = *(const uint4*)(sp + j * 8);
        vs[h][j] = x.x; vc[h][j] = x.y; vs[h][j + 1] = x.z; vc[h][j + 1] = x.w;
      }
      if constexpr (EDGE) {
        const uint32_t d = drop >> (2 * h), keep = (d & 1u ? 0u : 0xFFFFu) | (d & 2u ? 0u : 0xFFFF0000u);
#pragma unroll
        for (int j = 0; j < NG; j++) {
          vs[h][j] &= keep;
          vc[h][j] &= keep;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NG; j++) {
      uint32_t x[4], y[4];
      const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
      decode_word(__byte_perm(wa[0][j / 2], wb[0][j / 2], sel), u2h(vs[0][j]), u2h(vc[0][j]), x);
      decode_word(__byte_perm(wa[1][j / 2], wb[1][j / 2], sel), u2h(vs[1][j]), u2h(vc[1][j]), y);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        mma_f16(o[nt][j][0], x[0], x[1], y[0], y[1], pb[nt][0], pb[nt][1]);
        mma_f16(o[nt][j][1], x[2], x[3], y[2], y[3], pb[nt][0], pb[nt][1]);
        if constexpr (!SPLIT) {
          mma_f16(o[nt][j][0], x[0], x[1], y[0], y[1], pl[nt][0], pl[nt][1]);
          mma_f16(o[nt][j][1], x[2], x[3], y[2], y[3], pl[nt][0], pl[nt][1]);
        }
      }
    }
  }

  // A unit: the two blocks at blk, positions from p0 on.  EDGE: some rows do not see some of them, and
  // what lies past the stream's end (position held) may be anything.
  template <bool EDGE>
  __device__ __forceinline__ void unit(const uint8_t* blk, int p0, int held, const AttnArgs& a) {
    constexpr int BLK = kv4_block_bytes(HD);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float c[2][NT][4] = {};
    scores(blk, c[0]);
    scores(blk + BLK, c[1]);
    uint32_t drop[2] = {0u, 0u}, bad = 0;  // bad: a bit for each of the 32 keys
    if constexpr (EDGE) {
#pragma unroll
      for (int b = 0; b < 2; b++) {
        uint32_t nan = nan_values(blk + b * BLK);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int key = 16 * b + 8 * (k >> 1) + 2 * t + (k & 1);
          if (p0 + key >= held) {
            drop[b] |= 1u << k;
            nan &= ~(1u << k);
          }
          const uint32_t v = __ballot_sync(0xffffffffu, nan >> k & 1u) & 15u;
#pragma unroll
          for (int tt = 0; tt < 4; tt++) bad |= (v >> tt & 1u) << (16 * b + 8 * (k >> 1) + 2 * tt + (k & 1));
        }
        drop[b] |= nan;
      }
    }
    uint32_t pb[2][NT][2], pl[2][SPLIT ? 1 : NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      // this lane's scores: of key key0 + 8 k (+ 16 b) in columns e; COLS: block t / 2 alone
      constexpr int NB = SPLIT ? 1 : 2;
      float x[NB][2][2];
      if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float r = __shfl_xor_sync(0xffffffffu, t < 2 ? c[1][nt][i] : c[0][nt][i], 2);
          x[0][i >> 1][i & 1] = (t < 2 ? c[0][nt][i] : c[1][nt][i]) + r;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i >> 2][i >> 1 & 1][i & 1] = c[i >> 2][nt][i & 3];
      }
      float y[NB][2][2];
      bool over = false;
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float& v = y[b][k][e];
            if constexpr (EDGE) {
              const int key = (SPLIT ? 16 * (t >> 1) : 16 * b) + g + 8 * k, j = p0 + key, i_ = i[nt][e];
              const bool seen = j <= i_ && j < held && (a.window == 0 || j > i_ - a.window || j < a.sinks);
              x[b][k][e] = !seen ? -INFINITY : (bad >> key & 1u) ? __uint_as_float(0x7FFFFFFFu) : x[b][k][e] * f[nt][e];
              v = x[b][k][e] + mb[nt][e];
            } else {
              v = fmaf(x[b][k][e], f[nt][e], mb[nt][e]);
            }
            over |= v > kPMax;
          }
      if (__any_sync(0xffffffffu, over)) {  // move the maxima
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float fe = EDGE ? 1.0f : f[nt][e];
          float m = fmaxf(x[0][0][e] * fe, x[0][1][e] * fe);
          if constexpr (NB == 2) m = fmaxf(m, fmaxf(x[NB - 1][0][e] * fe, x[NB - 1][1][e] * fe));
#pragma unroll
          for (int w = SPLIT ? 2 : 4; w < 32; w <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
          const float nb = fminf(mb[nt][e], kPBias - m);
          const float al = ex2(nb - mb[nt][e]);
          mb[nt][e] = nb;
          l[nt][e] *= al;
#pragma unroll
          for (int j = 0; j < NG; j++)
#pragma unroll
            for (int q = 0; q < 2; q++) {
              o[nt][j][q][e] *= al;
              o[nt][j][q][e + 2] *= al;
            }
          if constexpr (FLUSH)
            each_sum([&](float& sum, float&, int t_, int e_) {
              if (t_ == nt && e_ == e) sum *= al;
            });
#pragma unroll
          for (int b = 0; b < NB; b++)
#pragma unroll
            for (int k = 0; k < 2; k++) y[b][k][e] = fmaf(x[b][k][e], fe, nb);
        }
      }
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const float p0_ = ex2(y[b][k][0]), p1_ = ex2(y[b][k][1]);
          l[nt][0] += p0_;
          l[nt][1] += p1_;
          const uint32_t hi = pack_h2(p0_, p1_);
          const float2 hf = __half22float2(u2h(hi));
          const uint32_t lo = pack_h2(p0_ - hf.x, p1_ - hf.y);
          if constexpr (SPLIT) {  // lanes t < 2 hold block 0 and give hi (columns 0..3), the others block 1 and lo
            const uint32_t other = __shfl_xor_sync(0xffffffffu, t < 2 ? lo : hi, 2);
            pb[0][nt][k] = movmatrix(t < 2 ? hi : other);
            pb[1][nt][k] = movmatrix(t < 2 ? other : lo);
          } else {
            pb[b][nt][k] = movmatrix(hi);
            pl[b][nt][k] = movmatrix(lo);
          }
        }
    }
    output<EDGE>(blk, pb[0], pl[0], drop[0]);
    output<EDGE>(blk + BLK, pb[1], pl[1], drop[1]);
    if constexpr (FLUSH) {
      if (++since == kFlush) {
        since = 0;
        each_sum([](float& sum, float& part, int, int) {
          sum += part;
          part = 0.0f;
        });
      }
    }
  }

  // The segment's piece is done: to `out` (whole) or to a record.
  __device__ __forceinline__ void end(const AttnArgs& a, int seg, bool whole, float* rec) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rt = seg % a.RT, kvh = seg / a.RT % a.NKV, b = seg / a.RT / a.NKV;
    const int R = a.T * a.G;
    if constexpr (FLUSH) each_sum([](float& sum, float& part, int, int) { part += sum; });
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float ls = l[nt][e];
#pragma unroll
        for (int w = SPLIT ? 2 : 4; w < 32; w <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, w);
        const int col = (SPLIT ? 2 * (t & 1) : 2 * t) + e;
        const int rl = nt * CPT + col, r = rt * NT * CPT + rl;
        const float inv = ls > 0.0f ? 1.0f / ls : (ls == 0.0f ? 0.0f : ls);
#pragma unroll
        for (int j = 0; j < NG; j++) {
          float v[4] = {o[nt][j][0][e], o[nt][j][0][e + 2], o[nt][j][1][e], o[nt][j][1][e + 2]};
          if constexpr (SPLIT) {
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] += __shfl_xor_sync(0xffffffffu, v[k], 2);
          }
          if (SPLIT && (j & 1) != (t >> 1)) continue;
          if (whole) {
            if (r < R) {
              const size_t at = (size_t)(b * a.os[0] + r / a.G * a.os[1] + (kvh * a.G + r % a.G) * a.os[2]) + 32 * j + 4 * g;
#pragma unroll
              for (int k = 0; k < 4; k++) put_out(a, at + k, v[k] * inv);
            }
          } else {
            *(float4*)(rec + (size_t)rl * (HD + 4) + 32 * j + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
          }
        }
        if (!whole && g == 0 && (!SPLIT || t < 2)) {
          rec[(size_t)rl * (HD + 4) + HD] = mb[nt][e];
          rec[(size_t)rl * (HD + 4) + HD + 1] = ls;
        }
      }
  }
};

template <int HD>
__host__ __device__ constexpr int attn_stages() { return HD == 128 ? 2 : 4; }
// Bytes of a warp's fp32 sums.
__host__ __device__ constexpr int sum_bytes(int HD, int NT, int mode) { return mode == Q32 || mode == COLS32 ? NT * HD * 8 * 4 : 0; }
template <int HD>
__host__ __device__ constexpr int attn_smem(int B, int NT, int mode) {
  return attn_stages<HD>() * 2 * kv4_block_bytes(HD) + sum_bytes(HD, NT, mode) + 64 + (2 * B + 1) * 4;
}

// 8 streams of 65001 positions, 32 query and 8 kv heads of 128, bf16: 126 us in a graph with the joining
// (5.3 TB/s); from 20480 positions (49 us) on, more of them arrive at 5.9 TB/s, 0.92 of the copy bandwidth, so
// that about 15 us are fixed: the launches, the first copies of a ring and the joining (4 us).  The decoding of
// the codes is what comes after memory: 0.60 instructions a cycle and scheduler, the integer pipe at 57%, the
// tensor pipe at 17% (8x20480).  16 warps an SM is what 128 registers allow.
template <int HD, int NT, int MODE>
__global__ void __launch_bounds__(32, HD == 128 ? (NT == 1 ? (MODE == COLS ? 16 : 12) : 8) : (NT == 1 ? 16 : 12)) kv4_attn_kernel(AttnArgs a) {
  constexpr int ST = attn_stages<HD>(), BLK = kv4_block_bytes(HD);
  extern __shared__ __align__(128) uint8_t sm[];
  uint64_t* bar = (uint64_t*)(sm + ST * 2 * BLK + sum_bytes(HD, NT, MODE));
  int* s_len = (int*)(bar + 8);
  int* s_pre = s_len + a.B;
  const int lane = threadIdx.x;
  if (lane == 0) {
    for (int s = 0; s < ST; s++) mbar_init(bar + s, 1);
    fence_mbar_init();
  }
  grid_dep_wait();
  prefix_units(a, s_len, s_pre);
  if (blockIdx.x == 0)
    for (int b = lane; b <= a.B; b += 32) a.pre[b] = s_pre[b];
  const int N = s_pre[a.B];
  const int W = min((int)gridDim.x, N);  // warps with work: every one of them has a unit
  grid_dep_launch();
  if ((int)blockIdx.x >= W) return;
  const int x0 = (int)((long)N * blockIdx.x / W), x1 = (int)((long)N * (blockIdx.x + 1) / W);
  Unit mine, next;  // of units (u & ~31) + lane, for the reader and for the issuer
  mine = next = look_up<HD>(min(x0 + lane, x1 - 1), a, s_len, s_pre);
  auto issue = [&](int k) {  // the k-th unit of this warp
    if (lane == (k & 31)) {
      uint64_t* b = bar + k % ST;
      const uint32_t bytes = (next.pos & 3) * BLK;
      mbar_arrive_expect_tx(b, bytes);
      if (bytes) bulk_load(sm + k % ST * 2 * BLK, a.pool + next.off, bytes, b);
    }
  };
  const int n = x1 - x0;
  for (int k = 0; k < ST - 1 && k < n; k++) issue(k);
  constexpr int RPT = Rows<HD, NT, MODE>::CPT * NT;
  Rows<HD, NT, MODE> rows;
  rows.acc = (float*)(sm + ST * 2 * BLK) + lane;
  int seg = -1, held = 0;
  bool ok = true;
  float* rec = a.rec + (size_t)blockIdx.x * 2 * RPT * (HD + 4);
  int seg0 = 0, seg1 = 0;  // the segment's units
  auto finish = [&]() {
    const bool whole = seg0 >= x0 && seg1 <= x1;
    rows.end(a, seg, whole, rec + (seg0 < x0 ? 0 : (size_t)RPT * (HD + 4)));
  };
  int k = 0;
  for (; k < n; k++) {
    if ((k & 31) == 0 && k > 0) mine = next;
    const int ahead = k + ST - 1;
    if (ahead < n) {
      if ((ahead & 31) == 0) next = look_up<HD>(min(x0 + ahead + lane, x1 - 1), a, s_len, s_pre);
      issue(ahead);
    }
    const int sg = __shfl_sync(0xffffffffu, mine.seg, k & 31), pos = __shfl_sync(0xffffffffu, mine.pos, k & 31);
    if (sg != seg) {
      if (seg >= 0) finish();
      seg = sg;
      const int per = a.NKV * a.RT, b = seg / per, ub = (s_pre[b + 1] - s_pre[b]) / per;
      seg0 = s_pre[b] + seg % per * ub;
      seg1 = seg0 + ub;
      held = min(s_len[b], a.ld_table * kPage);
      typename Rows<HD, NT, MODE>::Query q;
      rows.fetch(a, seg, q);
      rows.begin(a, seg, s_len[b], q);
    }
    if (ok) ok = mbar_wait(bar + k % ST, (k / ST) & 1, ST_TMA_WAIT, &g_status_kv4);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    const int p0 = pos & ~7, blocks = pos & 3;
    const uint8_t* st = sm + k % ST * 2 * BLK;
    if (blocks) {
      if (pos & 4)
        rows.template unit<false>(st, p0, held, a);
      else
        rows.template unit<true>(st, p0, held, a);
    }
    __syncwarp();
  }
  if (!ok) {  // give up, once the copies in flight are in (waited for with a limit too)
    for (int i = k; i < min(k + ST, n); i++) mbar_wait(bar + i % ST, (i / ST) & 1, ST_TMA_WAIT, &g_status_kv4);
    return;
  }
  finish();
}

// Weighted sum of records: 2^(m - M) of each, as mb = 8 - m.
template <int D>
struct Joined {
  float mb, l, v[D];
  __device__ __forceinline__ void clear() {
    mb = 1e30f;
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < D; d++) v[d] = 0.0f;
  }
  __device__ __forceinline__ void add(float mb2, float l2, const float* v2) {
    const float nb = fminf(mb, mb2), f = ex2(nb - mb), f2 = ex2(nb - mb2);
    mb = nb;
    l = fmaf(l2, f2, l * f);
#pragma unroll
    for (int d = 0; d < D; d++) v[d] = fmaf(v2[d], f2, v[d] * f);
  }
  __device__ __forceinline__ float inverse() const { return l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l); }
};

// Joins the pieces of cut segments.  A CTA takes rows blockIdx.y * rows_cta .. of a segment, `parts`
// warps to a row, each every parts-th record; a lane holds HD / 32 consecutive dimensions.
constexpr int kJoinWarps = 16, kJoinBatch = 6;
template <int HD>
__global__ void __launch_bounds__(32 * kJoinWarps) kv4_join_kernel(AttnArgs a, int grid, int rows_per_tile, int parts) {
  constexpr int D = HD / 32;
  __shared__ float s_m[kJoinWarps], s_l[kJoinWarps];
  __shared__ float s_o[kJoinWarps][HD];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, part = w % parts;
  const int seg = blockIdx.x, rl = blockIdx.y * (blockDim.x / 32 / parts) + w / parts;
  const int rt = seg % a.RT, kvh = seg / a.RT % a.NKV, b = seg / a.RT / a.NKV, per = a.NKV * a.RT;
  const int r = rt * rows_per_tile + rl;
  const bool row = rl < rows_per_tile && r < a.T * a.G;
  grid_dep_wait();
  const int p0 = a.pre[b], p1 = a.pre[b + 1], N = a.pre[a.B];
  const int ub = (p1 - p0) / per;
  Joined<D> x;
  x.clear();
  if (ub > 0) {
    const int seg0 = p0 + seg % per * ub, W = min(grid, N);
    const int w0 = owner_of(seg0, N, W), n = owner_of(seg0 + ub - 1, N, W) - w0 + 1;
    if (n == 1) return;  // written whole
    const size_t step = (size_t)2 * rows_per_tile * (HD + 4);
    const float* rec = a.rec + (size_t)w0 * step + (size_t)(row ? rl : 0) * (HD + 4);
    for (int i = part; i < n; i += kJoinBatch * parts) {
      float mb[kJoinBatch], l[kJoinBatch], v[kJoinBatch][D];
#pragma unroll
      for (int k = 0; k < kJoinBatch; k++) {
        const int ii = i + k * parts;
        if (ii >= n) break;
        const float* rc = rec + ii * step + (ii == 0 ? (size_t)rows_per_tile * (HD + 4) : 0);
        const float2 ml = __ldcg((const float2*)(rc + HD));
        mb[k] = ml.x;
        l[k] = ml.y;
        if constexpr (D == 4) {
          const float4 u = __ldcg((const float4*)rc + lane);
          v[k][0] = u.x; v[k][1] = u.y; v[k][2] = u.z; v[k][3] = u.w;
        } else {
          const float2 u = __ldcg((const float2*)rc + lane);
          v[k][0] = u.x; v[k][1] = u.y;
        }
      }
#pragma unroll
      for (int k = 0; k < kJoinBatch; k++)
        if (i + k * parts < n) x.add(mb[k], l[k], v[k]);
    }
    if (parts > 1) {
      if (lane == 0) {
        s_m[w] = x.mb;
        s_l[w] = x.l;
      }
#pragma unroll
      for (int d = 0; d < D; d++) s_o[w][lane * D + d] = x.v[d];
      __syncthreads();
      if (part != 0) return;
      for (int k = 1; k < min(n, parts); k++) {
        float v[D];
#pragma unroll
        for (int d = 0; d < D; d++) v[d] = s_o[w + k][lane * D + d];
        x.add(s_m[w + k], s_l[w + k], v);
      }
    }
  }
  if (part != 0 || !row) return;
  const float inv = x.inverse();
  const size_t at = (size_t)(b * a.os[0] + r / a.G * a.os[1] + (kvh * a.G + r % a.G) * a.os[2]) + lane * D;
#pragma unroll
  for (int d = 0; d < D; d++) put_out(a, at + d, x.v[d] * inv);
}

// The same for sequences that are known to be short: one CTA holds a segment, its warps take the units
// in turn and join through shared memory, so that one launch is all there is.  Latency bounds it: one stream of
// 387 positions takes 7.3 us in a graph, 16 of 384 with fp32 q 6.8, 64 of 300 10.9 (2.3 TB/s).
template <int HD, int NT, int MODE>
__host__ __device__ constexpr int whole_warps() {  // as many as the registers allow
  return HD == 128 && NT > 1 ? 8 : (NT > 1 || (HD == 128 && (MODE == Q32 || MODE == COLS32)) ? 12 : 16);
}
template <int HD, int NT, int MODE>
__host__ __device__ constexpr int whole_smem(int warps) {
  const int ring = warps * 2 * 2 * kv4_block_bytes(HD), rec = warps * NT * Rows<HD, NT, MODE>::CPT * (HD + 4) * 4;
  return (ring > rec ? ring : rec) + warps * (16 + sum_bytes(HD, NT, MODE));
}
template <int HD, int NT, int MODE>
__global__ void __launch_bounds__(32 * whole_warps<HD, NT, MODE>()) kv4_attn_whole_kernel(AttnArgs a) {
  constexpr int BLK = kv4_block_bytes(HD), ST = 2, RPT = NT * Rows<HD, NT, MODE>::CPT;
  extern __shared__ __align__(128) uint8_t sm[];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint8_t* ring = sm + w * ST * 2 * BLK;
  uint8_t* tail = sm + whole_smem<HD, NT, MODE>(warps) - warps * (16 + sum_bytes(HD, NT, MODE));
  uint64_t* bar = (uint64_t*)(tail + warps * sum_bytes(HD, NT, MODE)) + w * 2;
  if (lane < ST) mbar_init(bar + lane, 1);
  fence_mbar_init();
  __syncwarp();
  grid_dep_wait();
  grid_dep_launch();
  const int seg = blockIdx.x;
  const int rt = seg % a.RT, kvh = seg / a.RT % a.NKV, b = seg / a.RT / a.NKV;
  Rows<HD, NT, MODE> rows;
  typename Rows<HD, NT, MODE>::Query q;
  rows.fetch(a, seg, q);  // ahead of the length, the table and the copies, which come one after the other
  const int n = a.lens[b] + a.len_add, held = min(max(n, 0), a.ld_table * kPage);
  const Span sp = span_of(n, a);
  const int U = sp.units(), mine = U > w ? (U - w + warps - 1) / warps : 0;
  rows.acc = (float*)(tail + w * sum_bytes(HD, NT, MODE)) + lane;
  Unit next = {}, cur;  // of this warp's units (k & ~31) + lane, for the issuer and for the reader
  auto issue = [&](int k) {
    if ((k & 31) == 0) next = unit_at<HD>(a, b, kvh, sp.at(w + min(k + lane, mine - 1) * warps), n, held);
    if (lane == (k & 31)) {
      const uint32_t bytes = (next.pos & 3) * BLK;
      mbar_arrive_expect_tx(bar + (k & 1), bytes);
      if (bytes) bulk_load(ring + (k & 1) * 2 * BLK, a.pool + next.off, bytes, bar + (k & 1));
    }
  };
  for (int k = 0; k < min(mine, 2); k++) issue(k);
  cur = next;
  rows.begin(a, seg, n, q);
  bool ok = true;
  int k = 0;
  for (; k < mine; k++) {
    if ((k & 31) == 0 && k > 0) cur = next;
    const int ps = __shfl_sync(0xffffffffu, cur.pos, k & 31);
    ok = __all_sync(0xffffffffu, mbar_wait(bar + (k & 1), (k >> 1) & 1, ST_TMA_WAIT, &g_status_kv4));
    if (!ok) break;
    const uint8_t* st = ring + (k & 1) * 2 * BLK;
    if (ps & 3) {
      if (ps & 4)
        rows.template unit<false>(st, ps & ~7, held, a);
      else
        rows.template unit<true>(st, ps & ~7, held, a);
    }
    __syncwarp();
    if (k + 2 < mine) issue(k + 2);
  }
  if (!ok)  // give up, once the copies in flight are in (waited for with a limit too)
    for (int i = k; i < min(k + 2, mine); i++) mbar_wait(bar + (i & 1), (i >> 1) & 1, ST_TMA_WAIT, &g_status_kv4);
  float* rec = (float*)sm;
  __syncthreads();
  const int parts = min(U, warps);
  if (w < parts) rows.end(a, seg, false, rec + (size_t)w * RPT * (HD + 4));
  __syncthreads();
  // four dimensions of a row per thread
  for (int i = threadIdx.x; i < RPT * (HD / 4); i += blockDim.x) {
    const int rl = i / (HD / 4), d = i % (HD / 4) * 4, r = rt * RPT + rl;
    if (r >= a.T * a.G) break;
    Joined<4> x;
    x.clear();
#pragma unroll 4
    for (int k = 0; k < parts; k++) {
      const float* rc = rec + ((size_t)k * RPT + rl) * (HD + 4);
      const float4 u = *(const float4*)(rc + d);
      const float v[4] = {u.x, u.y, u.z, u.w};
      x.add(rc[HD], rc[HD + 1], v);
    }
    const float inv = x.inverse();
    const size_t at = (size_t)(b * a.os[0] + r / a.G * a.os[1] + (kvh * a.G + r % a.G) * a.os[2]) + d;
#pragma unroll
    for (int e = 0; e < 4; e++) put_out(a, at + e, x.v[e] * inv);
  }
}

// How a call is laid out over the GPU.
struct AttnPlan {
  int NT, mode, RT, rows, warps, whole;  // whole: warps of a CTA per segment, 0: equal runs of units
  size_t pre_bytes, bytes;
};

typedef void (*AttnKernel)(AttnArgs);
template <int HD>
static AttnKernel attn_kernel(int NT, int mode) {
  if (mode == COLS) return kv4_attn_kernel<HD, 1, COLS>;
  if (mode == COLS32) return kv4_attn_kernel<HD, 1, COLS32>;
  if (mode == Q16) return NT == 1 ? kv4_attn_kernel<HD, 1, Q16> : kv4_attn_kernel<HD, 2, Q16>;
  return NT == 1 ? kv4_attn_kernel<HD, 1, Q32> : kv4_attn_kernel<HD, 2, Q32>;
}

template <int HD, int NT, int MODE>
static int launch_whole(const AttnArgs& a, int warps, cudaStream_t s) {
  static std::atomic<unsigned long long> smem_set{0};
  RNGD_TRY(set_smem_limit_once((const void*)kv4_attn_whole_kernel<HD, NT, MODE>, whole_smem<HD, NT, MODE>(whole_warps<HD, NT, MODE>()),
                               &smem_set, "cudaFuncSetAttribute(kv4_attn_whole_kernel)"));
  return launch_pdl(kv4_attn_whole_kernel<HD, NT, MODE>, dim3(a.B * a.NKV * a.RT), dim3(32 * warps),
                    whole_smem<HD, NT, MODE>(warps), s, "kv4_attn_whole_kernel", a);
}
template <int HD>
static int launch_whole(const AttnArgs& a, const AttnPlan& p, cudaStream_t s) {
  if (p.mode == COLS) return launch_whole<HD, 1, COLS>(a, p.whole, s);
  if (p.mode == COLS32) return launch_whole<HD, 1, COLS32>(a, p.whole, s);
  if (p.mode == Q16)
    return p.NT == 1 ? launch_whole<HD, 1, Q16>(a, p.whole, s)
                     : (p.NT == 2 ? launch_whole<HD, 2, Q16>(a, p.whole, s) : launch_whole<HD, 3, Q16>(a, p.whole, s));
  if constexpr (HD == 64)
    if (p.NT == 3) return launch_whole<HD, 3, Q32>(a, p.whole, s);
  return p.NT == 1 ? launch_whole<HD, 1, Q32>(a, p.whole, s) : launch_whole<HD, 2, Q32>(a, p.whole, s);
}

// Warps that fit one SM at a time (registers, shared memory), remembered per kernel and size class of
// the shared memory.
static int attn_per_sm(int HD, int NT, int mode, int B, int* out) {
  static std::atomic<int> known[2][2][4][kAttnStreams / 32 + 1];
  const int cls = (B + 31) / 32;
  std::atomic<int>& slot = known[HD == 128][NT - 1][mode][cls];
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    const AttnKernel k = HD == 128 ? attn_kernel<128>(NT, mode) : attn_kernel<64>(NT, mode);
    const int smem = HD == 128 ? attn_smem<128>(32 * cls, NT, mode) : attn_smem<64>(32 * cls, NT, mode);
    RNGD_TRY(check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, 32, smem), "occupancy(kv4_attn_kernel)"));
    if (n < 1) n = 1;
    slot.store(n, std::memory_order_relaxed);
  }
  *out = n;
  return RNGD_OK;
}

static int attn_plan(int dtype, int B, int T, int NH, int NKV, int HD, int ld_table, int window, int sinks,
                     AttnPlan* p) {
  RNGD_REQUIRE(HD == 64 || HD == 128, "kv4_attn: built for HD 64 and 128, not %d", HD);
  RNGD_REQUIRE(dtype >= DT_BF16 && dtype <= DT_F32, "kv4_attn: data type %d", dtype);
  RNGD_REQUIRE(B >= 0 && T >= 0 && NKV >= 1 && NH >= 1 && NH % NKV == 0 && ld_table >= 0,
               "kv4_attn: B=%d T=%d NH=%d must be a multiple of NKV=%d, table width %d", B, T, NH, NKV, ld_table);
  RNGD_REQUIRE(window >= 0 && sinks >= 0, "kv4_attn: window=%d sinks=%d", window, sinks);
  // positions are 32-bit numbers, up to the end of the table and of the unit that holds it
  RNGD_REQUIRE(ld_table <= 0x7FFFFFFF / kPage, "kv4_attn: table of %d pages, at most %d", ld_table, 0x7FFFFFFF / kPage);
  const int Bl = B < kAttnStreams ? B : kAttnStreams;  // streams of one launch
  const long R = (long)T * (NH / NKV);
  p->mode = R <= 4 ? (dtype == DT_F32 ? COLS32 : COLS) : (dtype == DT_F32 ? Q32 : Q16);
  const long cpt = R <= 4 ? 4 : 8, tiles = (R + cpt - 1) / cpt;
  RNGD_REQUIRE(R < (1l << 24), "kv4_attn: %ld query rows of a kv head", R);
  p->NT = tiles > 1 ? 2 : 1;
  p->RT = (int)((tiles + p->NT - 1) / p->NT);
  p->rows = p->NT * (int)cpt;
  // units of the longest segment there can be
  long most_u = (long)ld_table * (kPage / kUnit);
  if (window > 0) {
    const long w = ((long)window + T - 2) / kUnit + 2 + ((long)sinks + kUnit - 1) / kUnit;
    most_u = most_u < w ? most_u : w;
  }
  // One CTA per segment saves the joining kernel (and its launch) but leaves a long stream to one SM.  Streams
  // of one length, 32/8 heads of 128, bf16, us in a graph, whole against runs: 1x387 7.4 and 9.0, 1x1000 9.5
  // and 9.5, 1x1536 11.0 and 9.2, 1x2000 13.3 and 9.5; 4x1500 11.6 and 11.7; 16x300 6.9 and 14.6, 16x4000 21.4
  // and 30.1; 64x1000 22.1 and 31.3, 64x4000 70.0 and 71.1, 64x5000 87.1 and 87.8 (fp32 q 97.1 and 93.5).  The
  // limit of 48 units is put to the table's width, which lengths often stay far below.  A CTA has no more warps
  // than let all CTAs run at once (64x300: 10.8 us, 28.7 without).
  long segs = (long)Bl * NKV * p->RT;
  p->whole = 0;
  if (most_u <= 48 || (most_u <= 128 && segs >= 64)) {
    // Three column tiles a warp decode a unit once for 24 rows instead of 16, but halve the CTAs: worth it where
    // those still fill the GPU and no tile stays empty.  us in a graph, 2 kv heads, bf16, two tiles against three:
    // 24 rows of 64, 16x1000 (32 segments) 9.6 and 11.9, 64x1500 (128) 17.4 and 14.4; 24 rows of 128, 64x1500 26.1
    // and 21.9; 52 rows of 128 (seven tiles), 64x1500 47.8 and 83.2.  fp32 q of 128 has no registers for it.
    if (tiles % 3 == 0 && (p->mode == Q16 || HD == 64) && (long)Bl * NKV * (tiles / 3) * 4 >= 3l * num_sms()) {
      p->NT = 3;
      p->RT = (int)(tiles / 3);
      segs = (long)Bl * NKV * p->RT;
    }
    const int cap = HD == 128 && p->NT > 1 ? 8 : (p->NT > 1 || (HD == 128 && (p->mode == Q32 || p->mode == COLS32)) ? 12 : 16);
    long w = segs < 1 ? 1 : (long)num_sms() * cap / segs;  // cap warps fill an SM
    w = w < 2 ? 2 : (w < cap ? w : cap);
    p->whole = (int)(most_u < 1 ? 1 : (most_u < w ? most_u : w));
    p->warps = 0;
    p->pre_bytes = p->bytes = 0;
    RNGD_REQUIRE(segs < (1l << 31), "kv4_attn: %ld segments", segs);
    return RNGD_OK;
  }
  const long units = (long)Bl * NKV * p->RT * most_u;
  RNGD_REQUIRE(units < (1l << 31) && (long)Bl * NKV * p->RT < (1l << 31), "kv4_attn: %ld units of work", units);
  int per = 1;
  RNGD_TRY(attn_per_sm(HD, p->NT, p->mode, Bl, &per));
  const long most = (long)num_sms() * per;
  p->warps = (int)(units < 1 ? 1 : (units < most ? units : most));
  p->pre_bytes = ((size_t)(Bl + 1) * 4 + 15) / 16 * 16;
  p->bytes = p->pre_bytes + (size_t)p->warps * 2 * p->rows * (HD + 4) * 4;
  return RNGD_OK;
}

// The attention of one launch's arguments, streams in groups of kAttnStreams.
static int launch_kv4_attn(AttnArgs a, const AttnPlan& p, int B, int HD, void* workspace, cudaStream_t s) {
  const int esz = a.dt == DT_F32 ? 4 : 2, osz = a.lo_off != 0 ? 2 : esz;
  bool vec = ((uintptr_t)a.q & 15) == 0;
  for (int i = 0; i < 3; i++) vec = vec && a.qs[i] * esz % 16 == 0;
  a.qvec = vec;
  a.G = a.NH / a.NKV;
  a.RT = p.RT;
  a.pre = (int*)workspace;
  a.rec = (float*)((uint8_t*)workspace + p.pre_bytes);
  const AttnArgs all = a;
  for (int b0 = 0; b0 < B; b0 += kAttnStreams) {
    a.B = B - b0 < kAttnStreams ? B - b0 : kAttnStreams;
    a.q = (const uint8_t*)all.q + (long)b0 * a.qs[0] * esz;
    a.out = (uint8_t*)all.out + (long)b0 * a.os[0] * osz;
    a.table = all.table + (size_t)b0 * a.ld_table;
    a.lens = all.lens + b0;
    if (p.whole) {
      RNGD_TRY(HD == 128 ? launch_whole<128>(a, p, s) : launch_whole<64>(a, p, s));
      continue;
    }
    const AttnKernel k = HD == 128 ? attn_kernel<128>(p.NT, p.mode) : attn_kernel<64>(p.NT, p.mode);
    RNGD_TRY(launch_pdl(k, dim3(p.warps), dim3(32), HD == 128 ? attn_smem<128>(a.B, p.NT, p.mode) : attn_smem<64>(a.B, p.NT, p.mode), s,
                        "kv4_attn_kernel", a));
    // few segments have many records each: a CTA per row, its records shared by 16 warps; many segments: a CTA
    // for all rows of one (64x5000: 105 us with 16 warps a row, 91 us so)
    const int segs = a.B * a.NKV * p.RT;
    const bool few = segs * p.rows <= 4 * num_sms();
    const int parts = few ? kJoinWarps : (p.rows <= 8 ? 2 : 1);
    RNGD_TRY(launch_pdl(HD == 128 ? kv4_join_kernel<128> : kv4_join_kernel<64>, dim3(segs, few ? p.rows : 1),
                        dim3(32 * (few ? kJoinWarps : p.rows * parts)), 0, s, "kv4_join_kernel", a, p.warps, p.rows, parts));
  }
  return RNGD_OK;
}

// One layer's attention of the decode step: q fp32 [B][NH * HD], the new tokens at pos[b] (stored already),
// out as the hi / lo rows of the O projection's operand (16 streams apart).
int launch_kv4_decode_attn(const float* q, const void* pool, int P, int NKV, int HD, const int32_t* table, int ld_table,
                           const int32_t* pos, int B, int NH, int window, int sinks, void* act, int ld_act,
                           void* workspace, size_t workspace_bytes, cudaStream_t s) {
  RNGD_TRY(check_pool("decode_layers_kv4", pool, 0, P, NKV, HD));
  AttnPlan p;
  RNGD_TRY(attn_plan(DT_F32, B, 1, NH, NKV, HD, ld_table, window, sinks, &p));
  RNGD_REQUIRE(p.bytes == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= p.bytes),
               "decode_layers_kv4: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, p.bytes);
  AttnArgs a = {};
  a.q = q;
  a.out = act;
  a.qs[0] = a.qs[1] = (long)NH * HD;
  a.os[0] = a.os[1] = ld_act;
  a.qs[2] = a.os[2] = HD;
  a.lo_off = 16l * ld_act;
  a.len_add = 1;
  a.dt = DT_F32;
  a.T = 1;
  a.NH = NH;
  a.NKV = NKV;
  a.P = P;
  a.ld_table = ld_table;
  a.window = window;
  a.sinks = sinks;
  a.pool = (const uint8_t*)pool;
  a.table = table;
  a.lens = pos;
  a.scale = 1.0f / sqrtf((float)HD);
  return launch_kv4_attn(a, p, B, HD, workspace, s);
}

int read_status_kv4(int* st, int reset) {
  RNGD_TRY(check_cuda(cudaMemcpyFromSymbol(st, g_status_kv4, sizeof(int)), "read device status"));
  if (reset) {
    const int zero = 0;
    RNGD_TRY(check_cuda(cudaMemcpyToSymbol(g_status_kv4, &zero, sizeof(int)), "reset device status"));
  }
  return RNGD_OK;
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_kv4_attn_workspace(int dtype, int B, int T, int NH, int NKV, int HD, int ld_table, int window,
                                       int sinks, size_t* bytes) {
  RNGD_REQUIRE(bytes != nullptr, "kv4_attn_workspace: null output");
  AttnPlan p;
  RNGD_TRY(attn_plan(dtype, B, T, NH, NKV, HD, ld_table, window, sinks, &p));
  *bytes = p.bytes;
  return RNGD_OK;
}

extern "C" int rngd_kv4_attn(const void* q, const int64_t* q_strides, void* out, const int64_t* out_strides, int dtype,
                             const void* pool, int P, int NKV, int HD, const int32_t* table, int ld_table,
                             const int32_t* lens, int B, int T, int NH, int window, int sinks, float scale,
                             void* workspace, size_t workspace_bytes, rngd_stream_t stream) {
  RNGD_TRY(check_pool("kv4_attn", pool, 0, P, NKV, HD));
  AttnPlan p;
  RNGD_TRY(attn_plan(dtype, B, T, NH, NKV, HD, ld_table, window, sinks, &p));
  if (B == 0 || T == 0) return RNGD_OK;
  RNGD_REQUIRE(q && out && q_strides && out_strides && lens && (table || ld_table == 0), "kv4_attn: null pointer");
  RNGD_REQUIRE(p.bytes == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= p.bytes),
               "kv4_attn: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, p.bytes);
  AttnArgs a = {};
  a.q = q;
  a.out = out;
  for (int i = 0; i < 3; i++) {
    a.qs[i] = (long)q_strides[i];
    a.os[i] = (long)out_strides[i];
  }
  a.dt = dtype;
  a.T = T;
  a.NH = NH;
  a.NKV = NKV;
  a.P = P;
  a.ld_table = ld_table;
  a.window = window;
  a.sinks = sinks;
  a.pool = (const uint8_t*)pool;
  a.table = table;
  a.lens = lens;
  a.scale = scale;
  return launch_kv4_attn(a, p, B, HD, workspace, (cudaStream_t)stream);
}
