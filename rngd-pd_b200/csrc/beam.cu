// Beam search's selection: of each group's W beams x V tokens the W best continuations by
// score + log_softmax(logits), with the beams they continue.
//
// The reference decodes greedily (greedy_tokens, src/rngd_pd/engines/decode_batch.py:162-171); this is
// the same step for a search over several beams of one prompt.
#include "kv4.cuh"

namespace rngd {

constexpr int kMaxBeams = 32;

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
__device__ __forceinline__ unsigned long long order_key(float f, uint32_t at) {
  return ((unsigned long long)order_bits(f) << 32) | (0xFFFFFFFFu - at);
}

__device__ __forceinline__ float logit1(const void* p, size_t i, int dt) {
  if (dt == DT_F32) return ((const float*)p)[i];
  if (dt == DT_BF16) return bf2f(((const uint16_t*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}

struct BeamArgs {
  const void* logits;
  long ld;
  int dt, R, V, W, eos;
  const float* scores;
  const uint8_t* done;
  float* out_scores;
  int32_t* parents;
  int32_t* tokens;
  uint8_t* out_done;
  unsigned long long* cand;  // [R][W]
};

__device__ __forceinline__ unsigned long long max_key(unsigned long long v, unsigned long long* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long y = __shfl_xor_sync(0xffffffffu, v, o);
    v = y > v ? y : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[threadIdx.x & 31 & 7];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    const unsigned long long y = __shfl_xor_sync(0xffffffffu, v, o);
    v = y > v ? y : v;
  }
  return v;
}

// One CTA per row: the row's log-sum-exp, then its W best one after the other.
__global__ void __launch_bounds__(256) beam_row_kernel(BeamArgs a) {
  __shared__ unsigned long long s[8];
  __shared__ float sf[8];
  const int r = blockIdx.x, tid = threadIdx.x, w = r % a.W;
  const size_t row = (size_t)r * a.ld;
  const float cum = a.scores[r];
  if (a.done[r]) {
    // eos carries the score, all else is -inf, the lowest places first
    const bool carry = a.eos >= 0 && a.eos < a.V && order_bits(cum) > order_bits(-INFINITY);
    for (int k = tid; k < a.W; k += 256) {
      const int v = !carry ? k : k == 0 ? a.eos : (k - 1 < a.eos ? k - 1 : k);
      a.cand[(size_t)r * a.W + k] = order_key(carry && k == 0 ? cum : -INFINITY, (uint32_t)((long)w * a.V + v));
    }
    return;
  }
  float m = -INFINITY;
  for (int v = tid; v < a.V; v += 256) m = fmaxf(m, logit1(a.logits, row + v, a.dt));
  m = order_value((uint32_t)(max_key(order_key(m, 0), s) >> 32));
  float z = 0.0f;
  for (int v = tid; v < a.V; v += 256) z += expf(logit1(a.logits, row + v, a.dt) - m);
  z = warp_sum(z);
  if ((tid & 31) == 0) sf[tid >> 5] = z;
  __syncthreads();
  z = 0.0f;
  for (int k = 0; k < 8; k++) z += sf[k];
  const float lse = m + logf(z);
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.W; k++) {
    unsigned long long best = 0;
    for (int v = tid; v < a.V; v += 256) {
      const float sc = cum + (logit1(a.logits, row + v, a.dt) - lse);
      const unsigned long long key = order_key(sc, (uint32_t)((long)w * a.V + v));
      if (key < last && key > best) best = key;
    }
    best = max_key(best, s);
    if (tid == 0) a.cand[(size_t)r * a.W + k] = best;
    last = best;
  }
}

// One CTA per group: the W best of its rows' candidates.
__global__ void __launch_bounds__(256) beam_group_kernel(BeamArgs a) {
  __shared__ unsigned long long s[8];
  const int g = blockIdx.x, tid = threadIdx.x;
  const unsigned long long* c = a.cand + (size_t)g * a.W * a.W;
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.W; k++) {
    unsigned long long best = 0;
    for (int i = tid; i < a.W * a.W; i += 256) {
      const unsigned long long key = c[i];
      if (key < last && key > best) best = key;
    }
    best = max_key(best, s);
    if (tid == 0) {
      const uint32_t at = 0xFFFFFFFFu - (uint32_t)best;
      const int par = g * a.W + (int)(at / (uint32_t)a.V), tok = (int)(at % (uint32_t)a.V);
      const size_t o = (size_t)g * a.W + k;
      a.out_scores[o] = order_value((uint32_t)(best >> 32));
      a.parents[o] = par;
      a.tokens[o] = tok;
      a.out_done[o] = a.done[par] || tok == a.eos;
    }
    last = best;
  }
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_beam_workspace(int R, int V, int W, size_t* bytes) {
  RNGD_REQUIRE(bytes && R >= 0 && V >= 1 && W >= 1, "beam_workspace: bad argument");
  *bytes = (size_t)R * W * 8;
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
  RNGD_REQUIRE(workspace_bytes >= need, "beam_select: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  BeamArgs a = {logits, (long)ld, dtype, R, V, W, eos, scores, done, out_scores, parents, tokens, out_done,
                (unsigned long long*)workspace};
  beam_row_kernel<<<R, 256, 0, (cudaStream_t)stream>>>(a);
  RNGD_TRY(check_launch("beam_row_kernel"));
  beam_group_kernel<<<R / W, 256, 0, (cudaStream_t)stream>>>(a);
  return check_launch("beam_group_kernel");
}
