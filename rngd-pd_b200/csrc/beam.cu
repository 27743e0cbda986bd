// Beam search's selection: of each group's W beams x V tokens the W best continuations by
// score + log_softmax(logits), with the beams they continue.
//
// The reference decodes greedily (greedy_tokens, src/rngd_pd/engines/decode_batch.py:162-171); this is
// the same step for a search over several beams of one prompt.
//
// Within a row the order of scores is the order of logits, so one pass over the logits finds both what
// the log-sum-exp needs and the row's W best.  A CTA reads one chunk of a row into registers, 16 bytes
// at a time, and keeps it there.  The threads form 64 sets; the W-th largest of the sets' largest logits
// is a bound that at least W logits reach, and few others do.  What reaches it goes to a list in shared
// memory, whose W largest are found by counting, for each, those above it.  Equal logits are told apart
// by their places, as keys (logit, place) in one 64-bit number, so neither ties nor the order in which
// threads run can show; the bound is taken of plain values first and of keys only where the W-th largest
// is one of several that are equal.  A second kernel, one CTA per group, joins the chunks' sums into
// log-sum-exps and selects among the rows' candidates in the same way, by (score, place).
#include "kv4.cuh"

namespace rngd {

constexpr int kMaxBeams = 32;
constexpr int kRowThreads = 256;

typedef unsigned long long u64;

// Ascending unsigned order of floats; NaN becomes -inf, -0 becomes 0.
__device__ __forceinline__ uint32_t order_bits(float f) {
  if (f != f) f = -INFINITY;
  f += 0.0f;
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
// Larger keys are better: the value first, then the lower place.
__device__ __forceinline__ u64 order_key(float f, uint32_t at) {
  return ((u64)order_bits(f) << 32) | (0xFFFFFFFFu - at);
}

struct BeamArgs {
  const void* logits;
  long ld;
  int R, V, W, eos, chunks;  // chunks per row
  const float* scores;
  const uint8_t* done;
  float* out_scores;
  int32_t* parents;
  int32_t* tokens;
  uint8_t* out_done;
  u64* cand;    // [R][chunks][W] by (logit, token)
  float2* sums; // [R][chunks] (largest logit, sum of exp(logit - largest))
};

constexpr int kSets = 64;

// The W-th largest of the sets' keys (each unique, or 0), 0 if there are fewer: every key counts those
// above it.  s_keys holds the sets' keys; all threads call.
__device__ __forceinline__ u64 nth_key(int W, const u64* s_keys, u64* s_nth) {
  if (threadIdx.x == 0) *s_nth = 0;
  __syncthreads();
  if (threadIdx.x < kSets) {
    const u64 mine = s_keys[threadIdx.x];
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kSets; i += 2) {
      const ulonglong2 k = *(const ulonglong2*)(s_keys + i);
      above += (k.x > mine) + (k.y > mine);
    }
    if (above == W - 1 && mine != 0) *s_nth = mine;
  }
  __syncthreads();
  return *s_nth;
}

// The largest of a thread's keys to its set's place; per: threads of a set.
__device__ __forceinline__ void set_key(u64 k, int per, u64* s_keys) {
  for (int o = 1; o < per; o <<= 1) {
    const u64 y = __shfl_xor_sync(0xffffffffu, k, o);
    k = y > k ? y : k;
  }
  if (threadIdx.x % per == 0) s_keys[threadIdx.x / per] = k;
}

// Writes the W largest of list[0 .. n) (unique keys) to out, largest first, zeros where there are fewer.
__device__ __forceinline__ void take_best(const u64* list, int n, int W, u64* out) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const u64 k = list[i];
    int above = 0;
    for (int j = 0; j < n; j++) above += list[j] > k;
    if (above < W) out[above] = k;
  }
  for (int i = n + threadIdx.x; i < W; i += blockDim.x) out[i] = 0;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int DT>
__host__ __device__ constexpr int vec_len() { return DT == DT_F32 ? 4 : 8; }

// VL elements from an aligned 16 bytes.
template <int DT>
__device__ __forceinline__ void load_vec(const void* p, float* x) {
  const uint4 u = __ldcs((const uint4*)p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; k++) {
    if constexpr (DT == DT_F32) {
      x[k] = __uint_as_float(w[k]);
    } else if constexpr (DT == DT_BF16) {
      x[2 * k] = bf_lo(w[k]);
      x[2 * k + 1] = bf_hi(w[k]);
    } else {
      const float2 f = __half22float2(*(const __half2*)&w[k]);
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
  }
}
template <int DT>
__device__ __forceinline__ float load_one(const void* p, size_t i) {
  if constexpr (DT == DT_F32) return ((const float*)p)[i];
  if constexpr (DT == DT_BF16) return bf2f(((const uint16_t*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}

// EPT logits a thread.
template <int DT, int EPT>
__global__ void __launch_bounds__(kRowThreads) beam_row_kernel(BeamArgs a) {
  constexpr int VL = vec_len<DT>(), ESZ = 16 / VL, PER = kRowThreads / kSets;
  __shared__ __align__(16) float s_set[kSets];
  __shared__ __align__(16) u64 s_keys[kSets];
  __shared__ u64 s_nth;
  __shared__ float s_bound, s_m[kRowThreads / 32], s_z[kRowThreads / 32];
  __shared__ int s_n, s_tie;
  extern __shared__ u64 s_list[];  // [W * PER * EPT]: only W sets reach the bound
  const int tid = threadIdx.x, r = blockIdx.x / a.chunks, c = blockIdx.x % a.chunks;
  if (tid == 0) {
    s_n = 0;
    s_tie = 1;  // until a bound is found
    s_bound = -INFINITY;
  }
  grid_dep_wait();
  grid_dep_launch();
  if (a.done[r]) return;  // its one continuation is known
  // the row as aligned vectors: `lead` elements before it share its first one
  const uint8_t* row = (const uint8_t*)a.logits + (size_t)r * a.ld * ESZ;
  const int lead = (int)((uintptr_t)row & 15) / ESZ;
  const int v0 = c * (kRowThreads * EPT) - lead;
  auto place = [&](int i) { return v0 + (i / VL * kRowThreads + tid) * VL + i % VL; };
  float x[EPT];
#pragma unroll
  for (int i = 0; i < EPT; i += VL) {
    const int v = place(i);
    if (v >= 0 && v + VL <= a.V) {
      load_vec<DT>(row + (ptrdiff_t)v * ESZ, x + i);
    } else {
#pragma unroll
      for (int k = 0; k < VL; k++) x[i + k] = v + k >= 0 && v + k < a.V ? load_one<DT>(row, v + k) : -INFINITY;
    }
  }
  // the thread's largest (a NaN counts as -inf here and spoils the sum below), its sum of exponentials
  float best = x[0];
#pragma unroll
  for (int i = 1; i < EPT; i++) best = fmaxf(best, x[i]);
  if (best != best) best = -INFINITY;
  const float ref = best == -INFINITY ? 0.0f : best;
  float z = 0.0f;
#pragma unroll
  for (int i = 0; i < EPT; i++) z += exp2_fast((x[i] - ref) * 1.4426950408889634f);
  float m = best;
#pragma unroll
  for (int o = 1; o < PER; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (tid % PER == 0) s_set[tid / PER] = m;
  m = warp_max(m);
  if ((tid & 31) == 0) s_m[tid >> 5] = m;
  __syncthreads();
  float M = s_m[0];
#pragma unroll
  for (int k = 1; k < kRowThreads / 32; k++) M = fmaxf(M, s_m[k]);
  z = warp_sum(best == -INFINITY ? z : z * expf(best - M));
  if ((tid & 31) == 0) s_z[tid >> 5] = z;
  if (tid < kSets) {
    const float mine = s_set[tid];
    int above = 0, same = 0;
#pragma unroll
    for (int i = 0; i < kSets; i += 4) {
      const float4 u = *(const float4*)(s_set + i);
      above += (u.x > mine) + (u.y > mine) + (u.z > mine) + (u.w > mine);
      same += (u.x == mine) + (u.y == mine) + (u.z == mine) + (u.w == mine);
    }
    if (above < a.W && above + same == a.W && mine > -INFINITY) {
      s_bound = mine;
      s_tie = 0;
    }
  }
  __syncthreads();
  if (!s_tie) {
    const float bound = s_bound;
    if (best >= bound) {
#pragma unroll
      for (int i = 0; i < EPT; i++)
        if (x[i] >= bound) s_list[atomicAdd(&s_n, 1)] = order_key(x[i], (uint32_t)place(i));
    }
  } else {
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < EPT; i++) {
      const int v = place(i);
      const u64 k = v >= 0 && v < a.V ? order_key(x[i], (uint32_t)v) : 0;
      mine = k > mine ? k : mine;
    }
    set_key(mine, PER, s_keys);
    const u64 bound = nth_key(a.W, s_keys, &s_nth);
    if (mine != 0 && mine >= bound) {
#pragma unroll
      for (int i = 0; i < EPT; i++) {
        const int v = place(i);
        const u64 k = v >= 0 && v < a.V ? order_key(x[i], (uint32_t)v) : 0;
        if (k != 0 && k >= bound) s_list[atomicAdd(&s_n, 1)] = k;
      }
    }
  }
  __syncthreads();
  const size_t o = (size_t)r * a.chunks + c;
  take_best(s_list, s_n, a.W, a.cand + o * a.W);
  if (tid == 0) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < kRowThreads / 32; k++) s += s_z[k];
    a.sums[o] = make_float2(M, s);
  }
}

// One CTA per group.  per: candidates of a thread; with `rounds` the best are taken one after the other
// instead (where the list of a very large vocabulary would not fit shared memory).
constexpr int kGroupThreads = 512;
__global__ void __launch_bounds__(kGroupThreads) beam_group_kernel(BeamArgs a, int rounds) {
  constexpr int PER = kGroupThreads / kSets;
  __shared__ __align__(16) u64 s_keys[kSets];
  __shared__ u64 s_nth;
  __shared__ float s_lse[kMaxBeams];
  __shared__ u64 s_out[kMaxBeams];
  extern __shared__ u64 s_list[];  // [W * PER * candidates of a thread]
  __shared__ int s_n;
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  grid_dep_wait();
  // log-sum-exp of each row, a warp to a row
  for (int w = tid >> 5; w < a.W; w += kGroupThreads / 32) {
    const int r = g * a.W + w;
    if (a.done[r]) continue;
    const float2* s = a.sums + (size_t)r * a.chunks;
    float m = -INFINITY, z = 0.0f;
    for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, s[c].x);
    m = warp_max(m);
    for (int c = lane; c < a.chunks; c += 32) {
      const float2 u = s[c];
      z += u.x == -INFINITY ? u.y : u.y * expf(u.x - m);  // without a logit the sum is 0, or NaN
    }
    z = warp_sum(z);
    if (lane == 0) s_lse[w] = m + logf(z);
  }
  if (tid == 0) s_n = 0;
  __syncthreads();
  const int per_row = a.chunks * a.W, total = a.W * per_row;
  const u64* cand = a.cand + (size_t)g * total;
  auto key_of = [&](int i) -> u64 {
    const int w = i / per_row, r = g * a.W + w;
    const float cum = a.scores[r];
    if (a.done[r]) {
      // eos carries the score, all else is -inf, the lowest places first
      const int k = i - w * per_row;
      if (k >= a.W) return 0;
      const bool carry = a.eos >= 0 && a.eos < a.V && order_bits(cum) > order_bits(-INFINITY);
      const int v = !carry ? k : k == 0 ? a.eos : (k - 1 < a.eos ? k - 1 : k);
      return order_key(carry && k == 0 ? cum : -INFINITY, (uint32_t)w * (uint32_t)a.V + (uint32_t)v);
    }
    const u64 k = cand[i];
    if (k == 0) return 0;
    const float x = order_value((uint32_t)(k >> 32));
    return order_key(cum + (x - s_lse[w]), (uint32_t)w * (uint32_t)a.V + (0xFFFFFFFFu - (uint32_t)k));
  };
  if (!rounds) {
    u64 mine = 0;
    for (int i = tid; i < total; i += kGroupThreads) {
      const u64 k = key_of(i);
      mine = k > mine ? k : mine;
    }
    set_key(mine, PER, s_keys);
    const u64 bound = nth_key(a.W, s_keys, &s_nth);
    if (mine != 0 && mine >= bound)
      for (int i = tid; i < total; i += kGroupThreads) {
        const u64 k = key_of(i);
        if (k != 0 && k >= bound) s_list[atomicAdd(&s_n, 1)] = k;
      }
    __syncthreads();
    take_best(s_list, s_n, a.W, s_out);
  } else {
    u64 last = ~0ull;
    for (int n = 0; n < a.W; n++) {
      u64 mine = 0;
      for (int i = tid; i < total; i += kGroupThreads) {
        const u64 k = key_of(i);
        if (k < last && k > mine) mine = k;
      }
      set_key(mine, PER, s_keys);
      last = nth_key(1, s_keys, &s_nth);
      if (tid == 0) s_out[n] = last;
      __syncthreads();
    }
  }
  __syncthreads();
  if (tid < a.W) {
    const u64 best = s_out[tid];
    const uint32_t at = 0xFFFFFFFFu - (uint32_t)best;
    const int par = g * a.W + (int)(at / (uint32_t)a.V), tok = (int)(at % (uint32_t)a.V);
    const size_t o = (size_t)g * a.W + tid;
    a.out_scores[o] = order_value((uint32_t)(best >> 32));
    a.parents[o] = par;
    a.tokens[o] = tok;
    a.out_done[o] = a.done[par] || tok == a.eos;
  }
}

// Logits a thread holds: with enough rows and tokens 32; fewer give each CTA less to do, so that the one
// pass ends sooner.
static int beam_ept(int R, int V) {
  for (int e = 8; e < 32; e *= 2)
    if ((long)R * ((V + 7 + kRowThreads * e - 1) / (kRowThreads * e)) <= 2 * 148) return e;
  return 32;
}
static int beam_chunks(int R, int V) {  // 7: elements a row may start after an aligned place
  const int per = kRowThreads * beam_ept(R, V);
  return (V + 7 + per - 1) / per;
}

template <int DT>
static int launch_rows(const BeamArgs& a, int ept, cudaStream_t s) {
  const dim3 grid((unsigned)((long)a.R * a.chunks)), block(kRowThreads);
  const size_t smem = (size_t)a.W * (kRowThreads / kSets) * ept * 8;
  if (ept == 8) return launch_pdl(beam_row_kernel<DT, 8>, grid, block, smem, s, "beam_row_kernel", a);
  if (ept == 16) return launch_pdl(beam_row_kernel<DT, 16>, grid, block, smem, s, "beam_row_kernel", a);
  return launch_pdl(beam_row_kernel<DT, 32>, grid, block, smem, s, "beam_row_kernel", a);
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_beam_workspace(int R, int V, int W, size_t* bytes) {
  RNGD_REQUIRE(bytes && R >= 0 && V >= 1 && W >= 1, "beam_workspace: bad argument");
  *bytes = (size_t)R * beam_chunks(R, V) * ((size_t)W + 1) * 8;
  return RNGD_OK;
}

extern "C" int rngd_beam_select(const void* logits, int dtype, int64_t ld, int R, int V, int W, const float* scores,
                                const uint8_t* done, int eos, float* out_scores, int32_t* parents, int32_t* tokens,
                                uint8_t* out_done, void* workspace, size_t workspace_bytes, rngd_stream_t stream) {
  RNGD_REQUIRE(dtype >= DT_BF16 && dtype <= DT_F32, "beam_select: data type %d", dtype);
  RNGD_REQUIRE(W >= 1 && W <= kMaxBeams, "beam_select: %d beams, at most %d", W, kMaxBeams);
  RNGD_REQUIRE(R >= 0 && R % W == 0, "beam_select: %d rows are not whole groups of %d beams", R, W);
  RNGD_REQUIRE(V >= W && (long)V * W < (1l << 31), "beam_select: vocabulary of %d", V);
  RNGD_REQUIRE(ld >= V || R <= 1, "beam_select: rows of %d logits %ld apart", V, (long)ld);
  if (R == 0) return RNGD_OK;
  RNGD_REQUIRE(logits && scores && done && out_scores && parents && tokens && out_done && workspace,
               "beam_select: null pointer");
  size_t need;
  RNGD_TRY(rngd_beam_workspace(R, V, W, &need));
  RNGD_REQUIRE(((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need,
               "beam_select: workspace of %zu bytes, %zu needed (8-byte aligned)", workspace_bytes, need);
  const int ept = beam_ept(R, V), chunks = beam_chunks(R, V);
  RNGD_REQUIRE((long)R * chunks < (1l << 31), "beam_select: %d rows of %d logits", R, V);
  BeamArgs a = {logits, (long)ld, R, V, W, eos, chunks, scores, done, out_scores, parents, tokens, out_done};
  a.cand = (u64*)workspace;
  a.sums = (float2*)(a.cand + (size_t)R * chunks * W);
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == DT_F32)
    RNGD_TRY(launch_rows<DT_F32>(a, ept, s));
  else if (dtype == DT_BF16)
    RNGD_TRY(launch_rows<DT_BF16>(a, ept, s));
  else
    RNGD_TRY(launch_rows<DT_F16>(a, ept, s));
  const long per = ((long)W * W * chunks + kGroupThreads - 1) / kGroupThreads;
  size_t smem = (size_t)W * (kGroupThreads / kSets) * per * 8;
  const bool rounds = smem > 128 * 1024;
  if (rounds) smem = 0;
  static std::atomic<unsigned long long> smem_set{0};
  if (smem > 32 * 1024)
    RNGD_TRY(set_smem_limit_once((const void*)beam_group_kernel, 128 * 1024, &smem_set,
                                 "cudaFuncSetAttribute(beam_group_kernel)"));
  return launch_pdl(beam_group_kernel, dim3(R / W), dim3(kGroupThreads), smem, s, "beam_group_kernel", a, rounds ? 1 : 0);
}
