// Paged 4-bit KV cache (layout in kv4.cuh): storing rows into pages and reading them back.
//
// The reference keeps its cache in bf16 lanes of a fixed width (src/rngd_pd/engines/decode_batch.py:
// 300-420); this cache holds the same rows in pages, at 5 bits a value.
#include "kv4.cuh"

namespace rngd {

// min and max that keep a NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float held_to(float x) { return min_nan(max_nan(x, -kKvMax), kKvMax); }

// s and c of a group, in fp32 and each rounded to fp16; NaN for a group with a NaN, s = 0 for a constant
// one.
__device__ __forceinline__ __half2 group_scale(float lo, float hi) {
  const __half s = __float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  return __halves2half2(s, __float2half_rn(__fsub_rn(lo, 16.0f * __half2float(s))));
}

// (x - c) / s rounded to the nearest, ties to even, in fp32, held to a code.
__device__ __noinline__ uint32_t codes4_slow(float x0, float x1, float x2, float x3, float s, float c) {
  const float x[4] = {x0, x1, x2, x3};
  uint32_t unit = 0;
  for (int e = 0; e < 4; e++) {
    const float n = rintf(__fdiv_rn(__fsub_rn(x[e], c), s)) - 16.0f;
    unit |= (uint32_t)fminf(fmaxf(n, 0.0f), 15.0f) << (4 * e);
  }
  return unit;
}

// Codes of four values as 16 bits.  inv ~ 1 / s and k ~ -c / s - 16 give the quotient to 2^-14 of a step
// as long as |k| <= 512, and c and s lie near enough to the group's ends then (s >= 2^-17) that no code
// leaves 0..15; whatever comes within 2^-12 of a tie, and other groups, take the true quotient.
__device__ __forceinline__ uint32_t codes4(const float* x, float s, float c, float inv, float k) {
  if (!(s > 0.0f)) return 0;  // a constant group, or one with a NaN
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number, in the low bits
  uint32_t m[4];
  float off = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float q = fmaf(x[e], inv, k), n = __fadd_rn(q, kMagic);
    m[e] = __float_as_uint(n);
    off = fmaxf(off, fabsf(__fsub_rn(q, __fsub_rn(n, kMagic))));
  }
  if (!(off < 0.5f - 0x1p-12f && s >= 0x1p-17f && fabsf(k) <= 512.0f)) return codes4_slow(x[0], x[1], x[2], x[3], s, c);
  return (m[0] + m[1] * 16u + m[2] * 256u + m[3] * 4096u) & 0xFFFFu;
}

struct StoreArgs {
  uint8_t* pool;
  size_t layer_bytes;
  int P, NKV, L, B, T, ld_table;
  const int32_t* table;
  const int32_t* start;
  const int32_t* count;  // null: T
  const void* k;
  const void* v;
  long ks[4], vs[4];  // strides in elements: layer, stream, token, head
  int dt;
};

// Storing is done in groups of 8 positions that lie in one half of a block, HD / 4 lanes to a group (a
// warp, or half of one with HD = 64), four dimensions a lane: K's and V's codes of such a group are
// 4 * HD contiguous bytes each, its scales HD each.  The eight lanes of a scale group reduce the minima
// and maxima of the eight rows together (each ends up with one row), so that s and c are worked out once
// per row instead of in every lane.
template <int HD>
struct Group {
  uint8_t* blk;  // null: nowhere
  int half;      // which half of the block
  int t0;        // token of the group's first position (may be negative)
  int n;         // tokens of the stream
  int layer, b, h;
  __device__ __forceinline__ bool has(int r) const { return blk != nullptr && t0 + r >= 0 && t0 + r < n; }
};
template <int HD>
__device__ __forceinline__ Group<HD> group_of(const StoreArgs& a, int groups, long i) {
  Group<HD> g;
  g.h = (int)(i % a.NKV);
  i /= a.NKV;
  const int k = (int)(i % groups);
  i /= groups;
  g.b = (int)(i % a.B);
  g.layer = (int)(i / a.B);
  g.blk = nullptr;
  g.n = g.t0 = g.half = 0;
  if (g.layer >= a.L) return g;
  g.n = a.count != nullptr ? min(a.count[g.b], a.T) : a.T;
  const int start = a.start[g.b], pos = (start & ~7) + 8 * k;  // of the group; start may be negative
  g.t0 = pos - start;
  g.half = (pos & 8) >> 3;
  if (pos < 0 || g.t0 >= g.n || pos / kPage >= a.ld_table) return g;
  const int page = a.table[(size_t)g.b * a.ld_table + pos / kPage];
  if (page < 0 || page >= a.P) return g;
  g.blk = a.pool + g.layer * a.layer_bytes +
          (((size_t)page * a.NKV + g.h) * 4 + ((pos & (kPage - 1)) >> 4)) * kv4_block_bytes(HD);
  return g;
}

template <int DT, bool VEC>
struct Raw4 {  // four elements as loaded
  uint32_t w[DT == DT_F32 ? 4 : 2];
  __device__ __forceinline__ void load(const void* p, size_t at) {
    if constexpr (DT == DT_F32) {
      const uint32_t* q = (const uint32_t*)p + at;
      if constexpr (VEC) {
        const uint4 u = *(const uint4*)q;
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = q[e];
      }
    } else {
      const uint16_t* q = (const uint16_t*)p + at;
      if constexpr (VEC) {
        const uint2 u = *(const uint2*)q;
        w[0] = u.x; w[1] = u.y;
      } else {
        w[0] = (uint32_t)q[0] | (uint32_t)q[1] << 16;
        w[1] = (uint32_t)q[2] | (uint32_t)q[3] << 16;
      }
    }
  }
  __device__ __forceinline__ void get(float* x) const {
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = __uint_as_float(w[e]);
    } else if constexpr (DT == DT_BF16) {
      x[0] = bf_lo(w[0]); x[1] = bf_hi(w[0]); x[2] = bf_lo(w[1]); x[3] = bf_hi(w[1]);
    } else {
      const float2 u = __half22float2(*(const __half2*)&w[0]), v = __half22float2(*(const __half2*)&w[1]);
      x[0] = u.x; x[1] = u.y; x[2] = v.x; x[3] = v.y;
    }
  }
};

// The least of some values and of their negatives, as the bits that shuffles move: two 16-bit numbers in
// a word, or two floats.  A NaN stays.
template <int DT>
struct Ends {
  uint32_t w[DT == DT_F32 ? 2 : 1];
  __device__ __forceinline__ void least(const Ends& o) {
    if constexpr (DT == DT_F32) {
#pragma unroll
      for (int i = 0; i < 2; i++) w[i] = __float_as_uint(min_nan(__uint_as_float(w[i]), __uint_as_float(o.w[i])));
    } else {
      w[0] = min2(w[0], o.w[0]);
    }
  }
  static __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (DT == DT_BF16)
      asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  template <bool VEC>
  __device__ __forceinline__ void of(const Raw4<DT, VEC>& x) {
    if constexpr (DT == DT_F32) {
      float v[4];
      x.get(v);
      w[0] = __float_as_uint(min_nan(min_nan(v[0], v[1]), min_nan(v[2], v[3])));
      w[1] = __float_as_uint(-max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])));
    } else {
      const uint32_t a = min2(x.w[0], x.w[1]), b = min2(x.w[0] ^ 0x80008000u, x.w[1] ^ 0x80008000u);
      w[0] = min2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
    }
  }
  __device__ __forceinline__ float2 get() const {  // lo, hi
    if constexpr (DT == DT_F32) return make_float2(__uint_as_float(w[0]), -__uint_as_float(w[1]));
    if constexpr (DT == DT_BF16) return make_float2(bf_lo(w[0]), -bf_hi(w[0]));
    const float2 f = __half22float2(*(const __half2*)&w[0]);
    return make_float2(f.x, -f.y);
  }
};

// Eight rows of one tensor -> this lane's units of the rows, and (s, c) of row l & 7.  there: the rows
// that any lane of the warp holds (one of them, when a decode step appends).
template <int DT, bool VEC>
__device__ __forceinline__ __half2 quantise8(const Raw4<DT, VEC> (&raw)[8], int l, uint32_t there,
                                             uint32_t (&unit)[8]) {
  Ends<DT> e[8];
#pragma unroll
  for (int r = 0; r < 8; r++) e[r].of(raw[r]);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    const bool up = (l & o) != 0;
#pragma unroll
    for (int r = 0; r < o; r++) {
      Ends<DT> other;
#pragma unroll
      for (int i = 0; i < (DT == DT_F32 ? 2 : 1); i++) {
        other.w[i] = __shfl_xor_sync(0xffffffffu, up ? e[r].w[i] : e[r + o].w[i], o);
        e[r].w[i] = up ? e[r + o].w[i] : e[r].w[i];
      }
      e[r].least(other);
    }
  }
  const float2 ends = e[0].get();
  const bool wild = __any_sync(0xffffffffu, !(ends.x >= -kKvMax && ends.y <= kKvMax));
  const __half2 sc = wild ? group_scale(held_to(ends.x), held_to(ends.y)) : group_scale(ends.x, ends.y);
  const uint32_t bits = *(const uint32_t*)&sc;
#pragma unroll
  for (int r = 0; r < 8; r++) {
    unit[r] = 0;
    if (!(there >> r & 1u)) continue;
    const uint32_t u = __shfl_sync(0xffffffffu, bits, r, 8);
    const float2 f = __half22float2(*(const __half2*)&u);
    float x[4];
    raw[r].get(x);
    if (wild) {
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = held_to(x[i]);
    }
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(f.x));
    unit[r] = codes4(x, f.x, f.y, inv, fmaf(-f.y, inv, -16.0f));
  }
  return sc;
}

// Instruction issue bounds it (0.74 a cycle and scheduler): 448 positions of 32 layers, 8 heads of 128, bf16,
// take 27.8 us in a graph (2.8 TB/s read and written, most of it in L2, which these 77 MB fit; 12 us at the
// copy bandwidth); fp32 and 896 positions (271 MB) 70.7 us, 3.8 TB/s.  16 streams of one token and one layer
// take 3.6 us, a launch's latency.
template <int HD, int DT, bool VEC>
__global__ void __launch_bounds__(128) kv4_store_kernel(StoreArgs a, int groups) {
  constexpr int LPG = HD / 4, NG = HD / 32;
  const long i = ((long)blockIdx.x * 128 + threadIdx.x) / LPG;
  const int l = threadIdx.x % LPG;
  grid_dep_wait();
  grid_dep_launch();
  const Group<HD> g = group_of<HD>(a, groups, i);
  if (__all_sync(0xffffffffu, g.blk == nullptr)) return;
  Raw4<DT, VEC> k[8], v[8];
  const size_t ka = (size_t)(g.layer * a.ks[0] + g.b * a.ks[1] + g.t0 * a.ks[2] + g.h * a.ks[3]) + 4 * l;
  const size_t va = (size_t)(g.layer * a.vs[0] + g.b * a.vs[1] + g.t0 * a.vs[2] + g.h * a.vs[3]) + 4 * l;
#pragma unroll
  for (int r = 0; r < 8; r++) {
#pragma unroll
    for (uint32_t& w : k[r].w) w = 0;
#pragma unroll
    for (uint32_t& w : v[r].w) w = 0;
    if (g.has(r)) {
      k[r].load(a.k, ka + (size_t)(r * a.ks[2]));
      v[r].load(a.v, va + (size_t)(r * a.vs[2]));
    }
  }
  uint32_t unit[8], there = 0;
#pragma unroll
  for (int r = 0; r < 8; r++) there |= g.has(r) ? 1u << r : 0u;
  there = __reduce_or_sync(0xffffffffu, there);
  const int r0 = l & 7, j = l >> 3;
  {
    const __half2 sc = quantise8<DT, VEC>(k, l, there, unit);
    uint8_t* rows = g.blk + g.half * 4 * HD;  // of the group's first position
    if (g.has(r0)) *(__half2*)(g.blk + k_scale<HD>(g.half * 8 + r0, j)) = sc;
    // a word is two lanes' units: even lanes put together the even rows', odd lanes the odd rows'
#pragma unroll
    for (int r = 0; r < 8; r += 2) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, l & 1 ? unit[r] : unit[r + 1], 1);
      const int mine = r + (l & 1);
      if (g.has(mine))
        *(uint32_t*)(rows + mine * (HD / 2) + (((l & 7) >> 1) * NG + j) * 4) = l & 1 ? o | unit[r + 1] << 16 : unit[r] | o << 16;
    }
  }
  {
    const __half2 sc = quantise8<DT, VEC>(v, l, there, unit);
    {
      const uint32_t s = __half_as_ushort(__low2half(sc)), c = __half_as_ushort(__high2half(sc));
      const uint32_t o = __shfl_xor_sync(0xffffffffu, l & 1 ? s : c, 1);
      uint8_t* p = g.blk + v_scale<HD>(g.half * 8 + (r0 & 6), j);
      if (g.has(r0) && g.has(r0 ^ 1)) {
        *(uint32_t*)(p + (l & 1) * 4) = l & 1 ? o | c << 16 : s | o << 16;
      } else if (g.has(r0)) {
        *(uint16_t*)(p + (l & 1) * 2) = (uint16_t)s;
        *(uint16_t*)(p + 4 + (l & 1) * 2) = (uint16_t)c;
      }
    }
    // pairs of keys, exchanged among the NG lanes that hold the groups of one g: lane j gets the pairs
    // j (HD 128), or j and j + 2 (HD 64), of all groups
    uint32_t pr[4];
#pragma unroll
    for (int q = 0; q < 4; q++) pr[q] = unit[2 * q] | unit[2 * q + 1] << 16;
    uint8_t* p = g.blk + 8 * HD + (g.half * 8 + (l & 7)) * 8 * (2 * NG);
    if constexpr (NG == 4) {
      // after both exchanges pr[x] is group x's units of pair j
#pragma unroll
      for (int q = 0; q < 2; q++) {  // with lane j ^ 2: keep pairs of own half
        const uint32_t o = __shfl_xor_sync(0xffffffffu, j & 2 ? pr[q] : pr[q + 2], 16);
        const uint32_t m = j & 2 ? pr[q + 2] : pr[q];
        pr[q] = j & 2 ? o : m;      // from groups 0/1
        pr[q + 2] = j & 2 ? m : o;  // from groups 2/3
      }
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 2; q++) {  // with lane j ^ 1
        const uint32_t o = __shfl_xor_sync(0xffffffffu, j & 1 ? pr[2 * q] : pr[2 * q + 1], 8);
        const uint32_t m = j & 1 ? pr[2 * q + 1] : pr[2 * q];
        w[2 * q] = j & 1 ? o : m;
        w[2 * q + 1] = j & 1 ? m : o;
      }
      const uint2 a0 = make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
      const uint2 a1 = make_uint2(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
      const bool h0 = g.has(2 * j), h1 = g.has(2 * j + 1);
      if (h0 && h1) {
        *(uint4*)(p + j * 16) = make_uint4(a0.x, a0.y, a1.x, a1.y);
      } else if (h0) {
        *(uint2*)(p + j * 16) = a0;
      } else if (h1) {
        *(uint2*)(p + j * 16 + 8) = a1;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; q++) {  // lane j = 0 takes pairs 0 and 2, lane 1 pairs 1 and 3
        const uint32_t o = __shfl_xor_sync(0xffffffffu, j ? pr[2 * q] : pr[2 * q + 1], 8);
        const uint32_t m = j ? pr[2 * q + 1] : pr[2 * q];
        const uint32_t u0 = j ? o : m, u1 = j ? m : o;  // of groups 0 and 1
        const uint32_t a0 = __byte_perm(u0, u1, 0x5410), a1 = __byte_perm(u0, u1, 0x7632);
        const int pair = 2 * q + j;
        const bool h0 = g.has(2 * pair), h1 = g.has(2 * pair + 1);
        if (h0 && h1) {
          *(uint2*)(p + pair * 8) = make_uint2(a0, a1);
        } else if (h0) {
          *(uint32_t*)(p + pair * 8) = a0;
        } else if (h1) {
          *(uint32_t*)(p + pair * 8 + 4) = a1;
        }
      }
    }
  }
}

// Eight fp16 values, or their half of four, to the output type; VEC: 16-byte aligned rows.
template <int DT, int N>
__device__ __forceinline__ void put(void* p, size_t at, const uint32_t (&w)[N]) {  // 2 N values
  if constexpr (DT == DT_F16) {
    __half* q = (__half*)p + at;
    if constexpr (N == 4) *(uint4*)q = make_uint4(w[0], w[1], w[2], w[3]);
    else *(uint2*)q = make_uint2(w[0], w[1]);
  } else {
    float x[2 * N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float2 f = __half22float2(*(const __half2*)&w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
    if constexpr (DT == DT_F32) {
      float* q = (float*)p + at;
#pragma unroll
      for (int i = 0; i < N / 2; i++) ((float4*)q)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else {
      uint16_t* q = (uint16_t*)p + at;
      uint32_t b[N];
#pragma unroll
      for (int i = 0; i < N; i++) b[i] = (uint32_t)f2bf_bits(x[2 * i]) | (uint32_t)f2bf_bits(x[2 * i + 1]) << 16;
      if constexpr (N == 4) *(uint4*)q = make_uint4(b[0], b[1], b[2], b[3]);
      else *(uint2*)q = make_uint2(b[0], b[1]);
    }
  }
}

// The inverse, by the same groups of 8 positions; rows outside the cache become zeros.  448 positions of 32
// layers, 8 heads of 128, take 11.5 us in a graph (6.7 TB/s read and written; the 77 MB fit L2), 896 of them
// 26.4 us (154 MB, 5.8 TB/s): memory's latency and bandwidth bound it.
template <int HD, int DT>
__global__ void __launch_bounds__(128) kv4_load_kernel(StoreArgs a, int groups, void* ko, void* vo) {
  constexpr int LPG = HD / 4, NG = HD / 32;
  const long i = ((long)blockIdx.x * 128 + threadIdx.x) / LPG;
  const int l = threadIdx.x % LPG;
  grid_dep_wait();
  const Group<HD> g = group_of<HD>(a, groups, i);
  if (g.layer >= a.L) return;
  // row of token t0 + r
  auto row = [&](int r) { return ((((size_t)g.layer * a.B + g.b) * a.T + (g.t0 + r)) * a.NKV + g.h) * HD; };
  auto want = [&](int r) { return g.t0 + r >= 0 && g.t0 + r < a.T; };
  if constexpr (NG == 4) {
    {
      const int r = l >> 2, t = l & 3, key = g.half * 8 + r;
      uint4 w = make_uint4(0, 0, 0, 0), sc = w;
      if (g.has(r)) {
        w = *(const uint4*)(g.blk + key * 64 + t * 16);
        sc = *(const uint4*)(g.blk + 16 * HD + key * 16);
      }
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w}, ss[4] = {sc.x, sc.y, sc.z, sc.w};
      if (want(r)) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          uint32_t v[4];
          decode_word(ww[j], __low2half2(*(const __half2*)&ss[j]), __high2half2(*(const __half2*)&ss[j]), v);
          const uint32_t o[4] = {__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                                 __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632)};
          put<DT>(ko, row(r) + 32 * j + 8 * t, o);
        }
      }
    }
    {
      const int gg = l >> 2, t = l & 3;
      const bool h0 = g.has(2 * t), h1 = g.has(2 * t + 1);
      uint4 w = make_uint4(0, 0, 0, 0), s0 = w, s1 = w;
      if (h0 || h1) {
        w = *(const uint4*)(g.blk + 8 * HD + g.half * 512 + gg * 64 + t * 16);
        const uint8_t* sp = g.blk + 18 * HD + (g.half * 4 + t) * 32;
        s0 = *(const uint4*)sp;
        s1 = *(const uint4*)(sp + 16);
      }
      const uint32_t keep = (h0 ? 0xFFFFu : 0u) | (h1 ? 0xFFFF0000u : 0u);
      const uint32_t vs[4] = {s0.x & keep, s0.z & keep, s1.x & keep, s1.z & keep};
      const uint32_t vc[4] = {s0.y & keep, s0.w & keep, s1.y & keep, s1.w & keep};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        uint32_t v[4];
        decode_word(j < 2 ? __byte_perm(w.x, w.z, j & 1 ? 0x7632 : 0x5410) : __byte_perm(w.y, w.w, j & 1 ? 0x7632 : 0x5410),
                    *(const __half2*)&vs[j], *(const __half2*)&vc[j], v);
        const uint32_t o0[2] = {__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410)};
        const uint32_t o1[2] = {__byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632)};
        if (want(2 * t)) put<DT>(vo, row(2 * t) + 32 * j + 4 * gg, o0);
        if (want(2 * t + 1)) put<DT>(vo, row(2 * t + 1) + 32 * j + 4 * gg, o1);
      }
    }
  } else {
    {
      const int r = l >> 1, t2 = (l & 1) * 2, key = g.half * 8 + r;  // words of t2 and t2 + 1
      uint4 w = make_uint4(0, 0, 0, 0);
      uint2 sc = make_uint2(0, 0);
      if (g.has(r)) {
        w = *(const uint4*)(g.blk + key * 32 + t2 * 8);
        sc = *(const uint2*)(g.blk + 16 * HD + key * 8);
      }
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w}, ss[2] = {sc.x, sc.y};
      if (want(r)) {
#pragma unroll
        for (int x = 0; x < 4; x++) {  // t = t2 + x / 2, j = x & 1
          uint32_t v[4];
          decode_word(ww[x], __low2half2(*(const __half2*)&ss[x & 1]), __high2half2(*(const __half2*)&ss[x & 1]), v);
          const uint32_t o[4] = {__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410),
                                 __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632)};
          put<DT>(ko, row(r) + 32 * (x & 1) + 8 * (t2 + x / 2), o);
        }
      }
    }
    {
      const int gg = l >> 1;
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const int t = (l & 1) + 2 * y;
        const bool h0 = g.has(2 * t), h1 = g.has(2 * t + 1);
        uint2 w = make_uint2(0, 0);
        uint4 s0 = make_uint4(0, 0, 0, 0);
        if (h0 || h1) {
          w = *(const uint2*)(g.blk + 8 * HD + g.half * 256 + gg * 32 + t * 8);
          s0 = *(const uint4*)(g.blk + 18 * HD + (g.half * 4 + t) * 16);
        }
        const uint32_t keep = (h0 ? 0xFFFFu : 0u) | (h1 ? 0xFFFF0000u : 0u);
        const uint32_t vs[2] = {s0.x & keep, s0.z & keep}, vc[2] = {s0.y & keep, s0.w & keep};
#pragma unroll
        for (int j = 0; j < 2; j++) {
          uint32_t v[4];
          decode_word(__byte_perm(w.x, w.y, j ? 0x7632 : 0x5410), *(const __half2*)&vs[j], *(const __half2*)&vc[j], v);
          const uint32_t o0[2] = {__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410)};
          const uint32_t o1[2] = {__byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632)};
          if (want(2 * t)) put<DT>(vo, row(2 * t) + 32 * j + 4 * gg, o0);
          if (want(2 * t + 1)) put<DT>(vo, row(2 * t + 1) + 32 * j + 4 * gg, o1);
        }
      }
    }
  }
}

static int store_args(const char* what, StoreArgs* a, void* pool, size_t layer_bytes, int P, int NKV, int HD, int L,
                      const int32_t* table, int ld_table, const int32_t* start, const int32_t* count, int B, int T,
                      const void* k, const void* v, int dtype) {
  RNGD_TRY(check_pool(what, pool, layer_bytes, P, NKV, HD));
  RNGD_REQUIRE(L >= 1 && B >= 0 && T >= 0 && ld_table >= 0, "%s: L=%d B=%d T=%d table width %d", what, L, B, T, ld_table);
  RNGD_REQUIRE(dtype >= DT_BF16 && dtype <= DT_F32, "%s: data type %d", what, dtype);
  RNGD_REQUIRE(B == 0 || T == 0 || (k && v && start && (table || ld_table == 0)), "%s: null pointer", what);
  *a = {};
  a->pool = (uint8_t*)pool;
  a->layer_bytes = layer_bytes;
  a->P = P;
  a->NKV = NKV;
  a->L = L;
  a->B = B;
  a->T = T;
  a->ld_table = ld_table;
  a->table = table;
  a->start = start;
  a->count = count;
  a->k = k;
  a->v = v;
  a->dt = dtype;
  return RNGD_OK;
}

static int launch_store(const StoreArgs& a, int HD, cudaStream_t s) {
  if (a.B == 0 || a.T == 0) return RNGD_OK;
  const int groups = (a.T + 14) / 8;  // groups of 8 aligned positions that T positions can touch
  const long blocks = ((long)a.L * a.B * groups * a.NKV * (HD / 4) + 127) / 128;
  RNGD_REQUIRE(blocks < (1l << 31), "kv4_store: %ld groups of rows in one call", blocks);
  const int lane_bytes = a.dt == DT_F32 ? 16 : 8, esz = lane_bytes / 4;
  bool vec = ((uintptr_t)a.k | (uintptr_t)a.v) % lane_bytes == 0;
  for (int i = 0; i < 4; i++) vec = vec && a.ks[i] * esz % lane_bytes == 0 && a.vs[i] * esz % lane_bytes == 0;
  typedef void (*Kernel)(StoreArgs, int);
  static const Kernel kernels[2][3][2] = {
      {{kv4_store_kernel<64, DT_BF16, false>, kv4_store_kernel<64, DT_BF16, true>},
       {kv4_store_kernel<64, DT_F16, false>, kv4_store_kernel<64, DT_F16, true>},
       {kv4_store_kernel<64, DT_F32, false>, kv4_store_kernel<64, DT_F32, true>}},
      {{kv4_store_kernel<128, DT_BF16, false>, kv4_store_kernel<128, DT_BF16, true>},
       {kv4_store_kernel<128, DT_F16, false>, kv4_store_kernel<128, DT_F16, true>},
       {kv4_store_kernel<128, DT_F32, false>, kv4_store_kernel<128, DT_F32, true>}}};
  return launch_pdl(kernels[HD == 128][a.dt][vec], dim3((unsigned)blocks), dim3(128), 0, s, "kv4_store_kernel", a, groups);
}

// One layer's new tokens of the decode step: rows [B][NKV][HD] bf16 to position pos[b].
int launch_kv4_decode_store(void* pool, int P, int NKV, int HD, const int32_t* table, int ld_table, const int32_t* pos,
                            int B, const void* k, const void* v, cudaStream_t s) {
  StoreArgs a;
  RNGD_TRY(store_args("decode_layers_kv4", &a, pool, 0, P, NKV, HD, 1, table, ld_table, pos, nullptr, B, 1, k, v, DT_BF16));
  a.ks[1] = a.vs[1] = (long)NKV * HD;
  a.ks[3] = a.vs[3] = HD;
  return launch_store(a, HD, s);
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_kv4_store(void* pool, size_t layer_bytes, int P, int NKV, int HD, int L, const int32_t* table,
                              int ld_table, const int32_t* start, const int32_t* count, int B, int T, const void* k,
                              const int64_t* k_strides, const void* v, const int64_t* v_strides, int dtype,
                              rngd_stream_t stream) {
  StoreArgs a;
  RNGD_TRY(store_args("kv4_store", &a, pool, layer_bytes, P, NKV, HD, L, table, ld_table, start, count, B, T, k, v,
                      dtype));
  RNGD_REQUIRE(k_strides && v_strides, "kv4_store: null strides");
  for (int i = 0; i < 4; i++) {
    a.ks[i] = (long)k_strides[i];
    a.vs[i] = (long)v_strides[i];
  }
  return launch_store(a, HD, (cudaStream_t)stream);
}

extern "C" int rngd_kv4_load(const void* pool, size_t layer_bytes, int P, int NKV, int HD, int L,
                             const int32_t* table, int ld_table, const int32_t* start, const int32_t* count, int B,
                             int T, void* k, void* v, int dtype, rngd_stream_t stream) {
  StoreArgs a;
  RNGD_TRY(store_args("kv4_load", &a, (void*)pool, layer_bytes, P, NKV, HD, L, table, ld_table, start, count, B, T, k,
                      v, dtype));
  if (B == 0 || T == 0) return RNGD_OK;
  RNGD_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "kv4_load: k and v must be 16-byte aligned");
  const int groups = (T + 14) / 8;
  const long blocks = ((long)L * B * groups * NKV * (HD / 4) + 127) / 128;
  RNGD_REQUIRE(blocks < (1l << 31), "kv4_load: %ld groups of rows in one call", blocks);
  typedef void (*Kernel)(StoreArgs, int, void*, void*);
  static const Kernel kernels[2][3] = {
      {kv4_load_kernel<64, DT_BF16>, kv4_load_kernel<64, DT_F16>, kv4_load_kernel<64, DT_F32>},
      {kv4_load_kernel<128, DT_BF16>, kv4_load_kernel<128, DT_F16>, kv4_load_kernel<128, DT_F32>}};
  return launch_pdl(kernels[HD == 128][dtype], dim3((unsigned)blocks), dim3(128), 0, (cudaStream_t)stream, "kv4_load_kernel", a,
                    groups, k, v);
}
