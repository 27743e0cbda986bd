// Paged 4-bit KV cache (layout in kv4.cuh): storing rows into pages, reading them back, and the
// attention of a few query tokens over the pages of each stream.
//
// The reference keeps its cache in bf16 lanes of a fixed width (src/rngd_pd/engines/decode_batch.py:
// 300-420); this cache holds the same rows in pages, at 5 bits a value.
#include "kv4.cuh"

namespace rngd {

__device__ __forceinline__ float load1(const void* p, size_t i, int dt) {
  if (dt == DT_F32) return ((const float*)p)[i];
  if (dt == DT_BF16) return bf2f(((const uint16_t*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}

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

// fp16 of the exact number whose fp32 rounding is x and whose remainder has the sign of `rest`: rounding
// twice would be off by one in the last place where x falls between two fp16 numbers, so a number that
// is not x exactly is first cut to fp32 with its last bit set (a sticky bit, 13 bits below fp16's last).
__device__ __forceinline__ __half half_once(float x, float rest) {
  uint32_t b = __float_as_uint(x);
  if (rest != 0.0f && (b & 0x7FFFFFFFu) != 0u) b = (b - ((rest < 0.0f) != (x < 0.0f) ? 1u : 0u)) | 1u;
  return __float2half_rn(__uint_as_float(b));
}
// a - b = d + e exactly (two-sum)
__device__ __forceinline__ float sub_exact(float a, float b, float* e) {
  const float d = __fsub_rn(a, b), bb = __fsub_rn(a, d);
  *e = __fadd_rn(__fsub_rn(a, __fadd_rn(d, bb)), __fsub_rn(bb, b));
  return d;
}

// Four values of a lane, eight lanes to a group of 32 -> codes, s, c.  s and c are rounded once, the
// quotients in fp32; a group with a NaN gets s = c = NaN, a constant group s = 0.
__device__ __forceinline__ uint32_t quantise4(const float* xin, __half* s, __half* c) {
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; e++) x[e] = min_nan(max_nan(xin[e], -kKvMax), kKvMax);
  float lo = min_nan(min_nan(x[0], x[1]), min_nan(x[2], x[3]));
  float hi = max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  float e;
  const float d = sub_exact(hi, lo, &e);
  const float q = __fdiv_rn(d, 15.0f);
  *s = half_once(q, __fadd_rn(fmaf(-q, 15.0f, d), e));
  const float sf = __half2float(*s);
  const float b = sub_exact(lo, 16.0f * sf, &e);
  *c = half_once(b, e);
  const float cf = __half2float(*c);
  uint32_t unit = 0;
  if (sf > 0.0f) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float t = rintf(__fdiv_rn(__fsub_rn(x[e], cf), sf)) - 16.0f;
      unit |= (uint32_t)fminf(fmaxf(t, 0.0f), 15.0f) << (4 * e);
    }
  }
  return unit;
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

// The block of (layer, stream, token, head) and the position in it; null where there is none.
template <int HD>
__device__ __forceinline__ uint8_t* locate(const StoreArgs& a, int l, int b, int t, int h, int* key) {
  const int n = a.count != nullptr ? min(a.count[b], a.T) : a.T;
  if (t >= n) return nullptr;
  const int pos = a.start[b] + t;
  if (pos < 0 || pos / kPage >= a.ld_table) return nullptr;
  const int page = a.table[(size_t)b * a.ld_table + pos / kPage];
  if (page < 0 || page >= a.P) return nullptr;
  *key = pos & (kBlk - 1);
  return a.pool + l * a.layer_bytes +
         (((size_t)page * a.NKV + h) * 4 + ((pos & (kPage - 1)) >> 4)) * kv4_block_bytes(HD);
}

// One row (a position of a kv head) per HD / 4 lanes, four dimensions a lane.
template <int HD>
__global__ void __launch_bounds__(256) kv4_store_kernel(StoreArgs a) {
  constexpr int LPR = HD / 4;
  const long rows = (long)a.L * a.B * a.T * a.NKV;
  const long r = ((long)blockIdx.x * 256 + threadIdx.x) / LPR;
  const int l = threadIdx.x % LPR;
  const bool in = r < rows;
  const long rr = in ? r : 0;
  const int h = (int)(rr % a.NKV), t = (int)(rr / a.NKV % a.T), b = (int)(rr / a.NKV / a.T % a.B);
  const int layer = (int)(rr / a.NKV / a.T / a.B);
  int key = 0;
  uint8_t* blk = in ? locate<HD>(a, layer, b, t, h, &key) : nullptr;
#pragma unroll
  for (int w = 0; w < 2; w++) {
    const long* st = w ? a.vs : a.ks;
    const size_t at = (size_t)(layer * st[0] + b * st[1] + t * st[2] + h * st[3]) + 4 * l;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = blk ? load1(w ? a.v : a.k, at + e, a.dt) : 0.0f;
    __half s, c;
    const uint32_t unit = quantise4(x, &s, &c);
    if (blk != nullptr) {
      *(uint16_t*)(blk + (w ? v_unit<HD>(key, l) : k_unit<HD>(key, l))) = (uint16_t)unit;
      if ((l & 7) == 0) {
        if (w) {
          __half* d = (__half*)(blk + v_scale<HD>(key, l >> 3));
          d[0] = s;
          d[2] = c;
        } else {
          __half* d = (__half*)(blk + k_scale<HD>(key, l >> 3));
          d[0] = s;
          d[1] = c;
        }
      }
    }
  }
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

// The inverse: rows of positions -> values [L][B][T][NKV][HD], zeros where nothing is stored.
template <int HD>
__global__ void __launch_bounds__(256) kv4_load_kernel(StoreArgs a, void* ko, void* vo) {
  constexpr int LPR = HD / 4;
  const long rows = (long)a.L * a.B * a.T * a.NKV;
  const long r = ((long)blockIdx.x * 256 + threadIdx.x) / LPR;
  const int l = threadIdx.x % LPR;
  if (r >= rows) return;
  const int h = (int)(r % a.NKV), t = (int)(r / a.NKV % a.T), b = (int)(r / a.NKV / a.T % a.B);
  const int layer = (int)(r / a.NKV / a.T / a.B);
  int key = 0;
  const uint8_t* blk = locate<HD>(a, layer, b, t, h, &key);
#pragma unroll
  for (int w = 0; w < 2; w++) {
    __half o[4] = {};
    if (blk != nullptr) {
      const __half* d = (const __half*)(blk + (w ? v_scale<HD>(key, l >> 3) : k_scale<HD>(key, l >> 3)));
      kv4_values(*(const uint16_t*)(blk + (w ? v_unit<HD>(key, l) : k_unit<HD>(key, l))), d[0], d[w ? 2 : 1], o);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) store1(w ? vo : ko, (size_t)r * HD + 4 * l + e, a.dt, __half2float(o[e]));
  }
}

struct AttnArgs {
  const void* q;
  void* out;
  long qs[3], os[3];  // strides in elements: stream, token, head
  int dt, B, T, NH, NKV, P, ld_table, window, sinks;
  const uint8_t* pool;
  const int32_t* table;
  const int32_t* lens;
  float scale;
};

// One CTA per (stream, token, query head): the warps take positions in turn, each with its own
// running maximum and sum, joined at the end.
template <int HD>
__global__ void __launch_bounds__(128) kv4_attn_kernel(AttnArgs a) {
  constexpr int LPR = HD / 4, SUB = 32 / LPR, NW = 4;
  __shared__ float sm[NW * SUB][2];
  __shared__ float so[NW * SUB][HD];
  const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
  const int w = threadIdx.x / 32, l = threadIdx.x % LPR, sub = threadIdx.x % 32 / LPR;
  const int kvh = h / (a.NH / a.NKV);
  const int i = a.lens[b] - a.T + t;
  float q[4];
#pragma unroll
  for (int e = 0; e < 4; e++)
    q[e] = load1(a.q, (size_t)(b * a.qs[0] + t * a.qs[1] + h * a.qs[2]) + 4 * l + e, a.dt) * a.scale;
  float m = -INFINITY, z = 0.0f, o[4] = {};
  for (int j0 = 0; j0 <= i; j0 += NW * SUB) {
    const int j = j0 + w * SUB + sub;
    bool seen = j <= i && (a.window == 0 || j > i - a.window || j < a.sinks) && j / kPage < a.ld_table;
    int page = -1;
    if (seen) page = a.table[(size_t)b * a.ld_table + j / kPage];
    seen = seen && page >= 0 && page < a.P;
    const uint8_t* blk = a.pool + (((size_t)max(page, 0) * a.NKV + kvh) * 4 + ((j & 63) >> 4)) * kv4_block_bytes(HD);
    const int key = j & 15;
    __half x[4] = {};
    float s = 0.0f;
    if (seen) {
      const __half* d = (const __half*)(blk + k_scale<HD>(key, l >> 3));
      kv4_values(*(const uint16_t*)(blk + k_unit<HD>(key, l)), d[0], d[1], x);
#pragma unroll
      for (int e = 0; e < 4; e++) s = fmaf(q[e], __half2float(x[e]), s);
    }
#pragma unroll
    for (int k = 1; k < LPR; k <<= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    if (seen) {
      const __half* d = (const __half*)(blk + v_scale<HD>(key, l >> 3));
      kv4_values(*(const uint16_t*)(blk + v_unit<HD>(key, l)), d[0], d[2], x);
      const float mn = fmaxf(m, s);
      const float f = m == mn ? 1.0f : expf(m - mn), p = s == mn ? 1.0f : expf(s - mn);
      z = fmaf(z, f, p);
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = fmaf(o[e], f, p * __half2float(x[e]));
      m = mn;
    }
  }
  if (l == 0) {
    sm[w * SUB + sub][0] = m;
    sm[w * SUB + sub][1] = z;
  }
#pragma unroll
  for (int e = 0; e < 4; e++) so[w * SUB + sub][4 * l + e] = o[e];
  __syncthreads();
  if (threadIdx.x < HD) {
    float M = -INFINITY, Z = 0.0f, O = 0.0f;
    for (int k = 0; k < NW * SUB; k++) M = fmaxf(M, sm[k][0]);
    for (int k = 0; k < NW * SUB; k++) {
      if (sm[k][1] == 0.0f) continue;
      const float f = sm[k][0] == M ? 1.0f : expf(sm[k][0] - M);
      Z = fmaf(sm[k][1], f, Z);
      O = fmaf(so[k][threadIdx.x], f, O);
    }
    store1(a.out, (size_t)(b * a.os[0] + t * a.os[1] + h * a.os[2]) + threadIdx.x, a.dt, Z == 0.0f ? 0.0f : O / Z);
  }
}

static int check_pool(const char* what, const void* pool, size_t layer_bytes, int P, int NKV, int HD) {
  RNGD_REQUIRE(pool != nullptr && ((uintptr_t)pool & 15) == 0 && (layer_bytes & 15) == 0,
               "%s: the pool must be 16-byte aligned", what);
  RNGD_REQUIRE(HD == 64 || HD == 128, "%s: built for HD 64 and 128, not %d", what, HD);
  RNGD_REQUIRE(P >= 1 && NKV >= 1 && NKV <= 1024, "%s: P=%d NKV=%d", what, P, NKV);
  return RNGD_OK;
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
  const long rows = (long)L * B * T * NKV;
  if (rows == 0) return RNGD_OK;
  const long blocks = (rows * (HD / 4) + 255) / 256;
  RNGD_REQUIRE(blocks < (1l << 31), "kv4_store: %ld rows in one call", rows);
  if (HD == 128)
    kv4_store_kernel<128><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(a);
  else
    kv4_store_kernel<64><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(a);
  return check_launch("kv4_store_kernel");
}

extern "C" int rngd_kv4_load(const void* pool, size_t layer_bytes, int P, int NKV, int HD, int L,
                             const int32_t* table, int ld_table, const int32_t* start, const int32_t* count, int B,
                             int T, void* k, void* v, int dtype, rngd_stream_t stream) {
  StoreArgs a;
  RNGD_TRY(store_args("kv4_load", &a, (void*)pool, layer_bytes, P, NKV, HD, L, table, ld_table, start, count, B, T, k,
                      v, dtype));
  const long rows = (long)L * B * T * NKV;
  if (rows == 0) return RNGD_OK;
  const long blocks = (rows * (HD / 4) + 255) / 256;
  RNGD_REQUIRE(blocks < (1l << 31), "kv4_load: %ld rows in one call", rows);
  if (HD == 128)
    kv4_load_kernel<128><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(a, k, v);
  else
    kv4_load_kernel<64><<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(a, k, v);
  return check_launch("kv4_load_kernel");
}

extern "C" int rngd_kv4_attn_workspace(int B, int T, int NH, int NKV, int HD, int ld_table, size_t* bytes) {
  RNGD_REQUIRE(bytes && B >= 0 && T >= 0 && NH >= 1 && NKV >= 1 && ld_table >= 0, "kv4_attn_workspace: bad argument");
  *bytes = 0;
  (void)HD;
  return RNGD_OK;
}

extern "C" int rngd_kv4_attn(const void* q, const int64_t* q_strides, void* out, const int64_t* out_strides, int dtype,
                             const void* pool, int P, int NKV, int HD, const int32_t* table, int ld_table,
                             const int32_t* lens, int B, int T, int NH, int window, int sinks, float scale,
                             void* workspace, size_t workspace_bytes, rngd_stream_t stream) {
  RNGD_TRY(check_pool("kv4_attn", pool, 0, P, NKV, HD));
  RNGD_REQUIRE(dtype >= DT_BF16 && dtype <= DT_F32, "kv4_attn: data type %d", dtype);
  RNGD_REQUIRE(B >= 0 && T >= 0 && NH >= 1 && NH % NKV == 0 && ld_table >= 0,
               "kv4_attn: B=%d T=%d NH=%d must be a multiple of NKV=%d, table width %d", B, T, NH, NKV, ld_table);
  RNGD_REQUIRE(window >= 0 && sinks >= 0, "kv4_attn: window=%d sinks=%d", window, sinks);
  if (B == 0 || T == 0) return RNGD_OK;
  RNGD_REQUIRE(q && out && q_strides && out_strides && lens && (table || ld_table == 0), "kv4_attn: null pointer");
  AttnArgs a = {};
  a.q = q;
  a.out = out;
  for (int i = 0; i < 3; i++) {
    a.qs[i] = (long)q_strides[i];
    a.os[i] = (long)out_strides[i];
  }
  a.dt = dtype;
  a.B = B;
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
  (void)workspace;
  (void)workspace_bytes;
  if (HD == 128)
    kv4_attn_kernel<128><<<dim3(NH, T, B), 128, 0, (cudaStream_t)stream>>>(a);
  else
    kv4_attn_kernel<64><<<dim3(NH, T, B), 128, 0, (cudaStream_t)stream>>>(a);
  return check_launch("kv4_attn_kernel");
}
