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
