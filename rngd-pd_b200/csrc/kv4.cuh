// Paged 4-bit KV cache: the layout of a block and what a code stands for.
//
// A page holds 64 positions of one layer: [NKV][4 blocks][20 * HD bytes], a block being 16
// positions of one kv head.  Along the head dimension every 32 values share two fp16 numbers
// (s, c); a 4-bit code u stands for fp16(s * (16 + u) + c).  Storing takes s = fp16((max - min) * (1 / 15)),
// c = fp16(min - 16 s) and u = rint((x - c) / s) - 16 held to 0..15, each step in fp32.  With NG = HD / 32 a block is
//   K codes   [16 keys][t 0..3][j 0..NG-1][4 B]        nibble e of the word: dimension 32 j + 8 t + e
//   V codes   [2][g 0..7][8 keys][j 0..NG-1][2 B]      nibble e of the half word: dimension 32 j + 4 g + e
//   K scales  [16 keys][NG][s, c]
//   V scales  [2][4 key pairs][NG][s of both keys, c of both keys]
// K words sit where lane t of a matrix fragment row reads its NG words with one load, V half words
// where lane (g, t) reads keys 2t and 2t + 1 with one load and all rows of a fragment share a group.
// The 16 in the value comes from the decoding: a code or-ed into the upper mantissa bits of fp16 16.0
// is 16 + u exactly, so one fused multiply-add per pair of values finishes it.  c is held to 2^-11 of itself:
// to s / 64 for groups around zero, to more the farther their mean lies (a step at 2048 of them).  5 bits a
// value in all.
#pragma once
#include <cuda_fp16.h>

#include "tc.cuh"

namespace rngd {

constexpr int kPage = 64;    // positions of a page
constexpr int kBlk = 16;     // positions of a block
constexpr float kKvMax = 16384.0f;  // magnitudes are held to this, so that c stays finite in fp16

enum : int { DT_BF16 = 0, DT_F16 = 1, DT_F32 = 2 };

__host__ __device__ constexpr int kv4_block_bytes(int HD) { return 20 * HD; }

// Byte offsets of a scale inside a block.
template <int HD>
__device__ __forceinline__ int k_scale(int key, int j) {  // s, c: 4 bytes
  return 16 * HD + (key * (HD / 32) + j) * 4;
}
template <int HD>
__device__ __forceinline__ int v_scale(int key, int j) {  // s at +0, c at +4
  return 18 * HD + (((key >> 3) * 4 + ((key & 7) >> 1)) * (HD / 32) + j) * 8 + (key & 1) * 2;
}

// Two fp32 numbers in one register pair: one instruction works on both and rounds each as by itself.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ f32x2 add_pair(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul_pair(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// (a & m) | o by one lop3.  Attention over 8 x (9001..65001) positions takes 79.8 us in a graph so, 93.1 with the
// expression written in C; a window of 1000 in 32 x (901..15001) 13.1 and 13.4.
__device__ __forceinline__ uint32_t lop_ao(uint32_t a, uint32_t m, uint32_t o) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(m), "r"(o));
  return r;
}
// The four pairs (nibble i of the low half, nibble i of the high half) of w -> values.
__device__ __forceinline__ void decode_word(uint32_t w, __half2 s, __half2 c, uint32_t (&v)[4]) {
  v[0] = h2u(__hfma2(u2h(lop_ao(w << 6, 0x03C003C0u, 0x4C004C00u)), s, c));
  v[1] = h2u(__hfma2(u2h(lop_ao(w << 2, 0x03C003C0u, 0x4C004C00u)), s, c));
  v[2] = h2u(__hfma2(u2h(lop_ao(w >> 2, 0x03C003C0u, 0x4C004C00u)), s, c));
  v[3] = h2u(__hfma2(u2h(lop_ao(w >> 6, 0x03C003C0u, 0x4C004C00u)), s, c));
}

__device__ __forceinline__ void store1(void* p, size_t i, int dt, float v) {
  if (dt == DT_F32) {
    ((float*)p)[i] = v;
  } else if (dt == DT_BF16) {
    ((uint16_t*)p)[i] = f2bf_bits(v);
  } else {
    ((__half*)p)[i] = __float2half_rn(v);
  }
}

static inline int check_pool(const char* what, const void* pool, size_t layer_bytes, int P, int NKV, int HD) {
  RNGD_REQUIRE(pool != nullptr && ((uintptr_t)pool & 15) == 0 && (layer_bytes & 15) == 0,
               "%s: the pool must be 16-byte aligned", what);
  RNGD_REQUIRE(HD == 64 || HD == 128, "%s: built for HD 64 and 128, not %d", what, HD);
  RNGD_REQUIRE(P >= 1 && NKV >= 1 && NKV <= 1024, "%s: P=%d NKV=%d", what, P, NKV);
  return RNGD_OK;
}

}  // namespace rngd
