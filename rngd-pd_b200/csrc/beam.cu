// Beam search's selection: of each group's W beams x V tokens the W best continuations by
// score + log_softmax(logits), with the beams they continue.
//
// The reference decodes greedily (greedy_tokens, src/rngd_pd/engines/decode_batch.py:162-171); this is
// the same step for a search over several beams of one prompt.
//
// Within a row the order of scores is the order of logits (but for logits that differ and round to one
// score: of those the largest W take part), so one pass over the logits finds both what the log-sum-exp
// needs and the row's W best.  The rows' chunks lie end to end and every CTA takes an equal run of them
// through a ring in shared memory, every thread copying (asynchronously, ahead) and reading its own vectors
// of 16 bytes, so that nothing makes the warps wait for one another.  In the first chunk of a row (or of
// its part of one) the threads form 64 sets; the W-th largest of the sets' largest logits is a bound that
// at least W logits reach, and few others do.  A bit per vector notes those that hold a logit which reaches
// it.  At the row's end the noted vectors are read again and the W best of their logits kept, once more by
// way of 64 sets and then by counting, for each that is left, those above it.  Equal logits are told apart
// by their places, as keys (logit, place) in one 64-bit number, so neither ties nor the order in which
// threads run can show.  A second kernel, one CTA per group, joins the parts' sums into log-sum-exps and
// selects among the rows' candidates in the same way, by (score, place).
//
// Bytes would allow 20 us for 64 groups of 8 beams by 128256 bf16 logits; the two kernels take 47 (in a
// graph, logits from memory, 2.8 TB/s; 49 with the exponentials' sums one by one instead of in pairs).
// Instruction issue (0.65 a cycle and scheduler) and the barriers where a row ends bound the row kernel; the
// group kernel's 8 us are latency.  1 x 5 x 32003 fp32: 7.7 us, two launches' latency; 16 x 32 x 128256
// fp32: 81 us (3.3 TB/s).
// Four threads rank each set's key: with one, 50.1, 8.1 and 81.5 us.
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
  int R, V, W, eos, n, grid, slots;  // chunks of a row; CTAs; CTAs that may share a row
  const float* scores;
  const uint8_t* done;
  float* out_scores;
  int32_t* parents;
  int32_t* tokens;
  uint8_t* out_done;
  u64* cand;     // [R][slots][W] by (logit, token)
  float2* sums;  // [R][slots] (largest logit, sum of exp(logit - largest))
};

constexpr int kSets = 64;

// The W-th largest of the sets' keys (each unique, or 0), 0 if there are fewer: every key counts those
// above it, four threads to a key.  s_keys holds the sets' keys; all threads call.
__device__ __forceinline__ u64 nth_key(int W, const u64* s_keys, u64* s_nth) {
  if (threadIdx.x == 0) *s_nth = 0;
  __syncthreads();
  if (threadIdx.x < 4 * kSets) {
    const u64 mine = s_keys[threadIdx.x >> 2];
    int above = 0;
#pragma unroll
    for (int i = 0; i < kSets / 4; i += 2) {
      const ulonglong2 k = *(const ulonglong2*)(s_keys + 2 * (threadIdx.x & 3) + 4 * i);
      above += (k.x > mine) + (k.y > mine);
    }
    above += __shfl_xor_sync(0xffffffffu, above, 1);
    above += __shfl_xor_sync(0xffffffffu, above, 2);
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

// The elements of 16 bytes as they come.
template <int DT>
__device__ __forceinline__ void unpack_vec(const uint4& u, float* x) {
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
// The larger of two words' elements (of one, or of two by two), NaN only where both are.
template <int DT>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (DT == DT_F32)
    asm("max.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else if constexpr (DT == DT_BF16)
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int DT>
__device__ __forceinline__ uint32_t max_vec(const uint4& u) {
  return max_word<DT>(max_word<DT>(u.x, u.y), max_word<DT>(u.z, u.w));
}
template <int DT>
__device__ __forceinline__ float word_max(uint32_t w) {  // of its elements
  if constexpr (DT == DT_F32) return __uint_as_float(w);
  if constexpr (DT == DT_BF16) return fmaxf(bf_lo(w), bf_hi(w));
  const float2 f = __half22float2(*(const __half2*)&w);
  return fmaxf(f.x, f.y);
}
// The vector of elements v .. of a row (aligned; v may be negative), -inf for those outside [0, V).
template <int DT>
__device__ __forceinline__ uint4 load_vec(const uint8_t* row, int v, int V) {
  constexpr int VL = vec_len<DT>(), ESZ = 16 / VL;
  if (v >= 0 && v + VL <= V) return __ldcs((const uint4*)(row + (ptrdiff_t)v * ESZ));
  constexpr uint32_t kNone = DT == DT_F32 ? 0xFF800000u : (DT == DT_BF16 ? 0xFF80u : 0xFC00u);
  uint32_t w[4] = {};
#pragma unroll
  for (int k = 0; k < VL; k++) {
    uint32_t e = kNone;
    if (v + k >= 0 && v + k < V) {
      if constexpr (DT == DT_F32)
        e = ((const uint32_t*)row)[v + k];
      else
        e = ((const uint16_t*)row)[v + k];
    }
    if constexpr (DT == DT_F32)
      w[k] = e;
    else
      w[k / 2] |= e << (16 * (k & 1));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int kNoteChunks = 16;  // chunks whose notes are held

template <int NV>
__host__ __device__ constexpr int ring_stages() { return NV == 8 ? 2 : 3; }

// NV vectors a thread and chunk.
template <int DT, int NV>
__global__ void __launch_bounds__(kRowThreads, 3) beam_row_kernel(BeamArgs a) {
  constexpr int VL = vec_len<DT>(), ESZ = 16 / VL, PER = kRowThreads / kSets, NW = kRowThreads / 32;
  constexpr int kChunk = kRowThreads * NV * VL, kWords = kRowThreads * NV / 32, ST = ring_stages<NV>();
  __shared__ __align__(16) float s_set[kSets];
  __shared__ __align__(16) u64 s_keys[kSets];
  __shared__ u64 s_nth, s_best[kMaxBeams];
  __shared__ uint32_t s_bits[kNoteChunks * kWords];  // [chunk][k][warp]
  __shared__ int s_note[kRowThreads], s_n, s_k;
  __shared__ float s_bound, s_m[NW], s_z[NW];
  __shared__ int s_over;  // more than W sets reach the bound
  extern __shared__ __align__(16) uint4 s_ring[];  // [ST][NV][kRowThreads], then s_list [W * (1 + PER * VL)]
  u64* s_list = (u64*)(s_ring + ST * NV * kRowThreads);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kMaxBeams) s_best[tid] = 0;
  grid_dep_wait();
  grid_dep_launch();
  const long total = (long)a.R * a.n, f0 = total * blockIdx.x / a.grid;
  const int runs = (int)(total * (blockIdx.x + 1) / a.grid - f0);  // chunks of this CTA
  // where the thread's first vector of a chunk lies in its row: a row is taken as aligned vectors, `lead`
  // elements before it share its first one; nothing of a row that is done is looked at (its one
  // continuation is known)
  struct At {
    const uint8_t* row;
    int r, c, v, V;
  };
  auto enter = [&](At& p) {
    p.row = (const uint8_t*)a.logits + (size_t)p.r * a.ld * ESZ;
    p.V = a.done[p.r] ? 0 : a.V;
    p.v = p.c * kChunk - (int)((uintptr_t)p.row & 15) / ESZ + tid * VL;
  };
  auto step = [&](At& p) {
    p.c++;
    p.v += kChunk;
    if (p.c == a.n) {
      p.c = 0;
      p.r++;
      if (p.r < a.R) enter(p);
    }
  };
  At now = {nullptr, (int)(f0 / a.n), (int)(f0 % a.n), 0, 0};
  enter(now);
  At ahead = now;
  int to_stage = 0, stage = 0;
  auto fetch = [&](int f) {  // the vectors that lie inside the row; those at its ends are read when it is their turn
    if (f < runs) {
      const uint32_t d = smem_u32(s_ring + to_stage * NV * kRowThreads + tid);
      to_stage = to_stage + 1 == ST ? 0 : to_stage + 1;
      const uint8_t* src = ahead.row + (ptrdiff_t)ahead.v * ESZ;
#pragma unroll
      for (int k = 0; k < NV; k++) {
        const int v = ahead.v + k * kRowThreads * VL;
        if (v >= 0 && v + VL <= ahead.V)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + k * kRowThreads * 16),
                       "l"(src + k * kRowThreads * 16)
                       : "memory");
      }
      step(ahead);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int k = 0; k < ST - 1; k++) fetch(k);
  float top = -INFINITY, ref = 0.0f, z = 0.0f;  // the thread's largest; z: sum of exp(x - ref)
  float bound = -INFINITY;
  int noted = 0;      // chunks of the row that have bits
  bool first = true;  // the first chunk of the row, or of this CTA's part of it
  // the W best of s_best and of the noted vectors -> s_best; no notes are left
  auto settle = [&]() {
    const int first = now.v - tid * VL - (noted - 1) * kChunk;  // of the first chunk that has bits
    int w = tid;                                                // this thread's words: w, w + kRowThreads, ..
    uint32_t bits = w < noted * kWords ? s_bits[w] : 0;
    for (;;) {
      if (tid == 0) s_n = s_k = 0;
      __syncthreads();
      for (;;) {  // notes, as many as there are threads
        while (bits == 0 && w < noted * kWords) {
          w += kRowThreads;
          bits = w < noted * kWords ? s_bits[w] : 0;
        }
        if (bits == 0) break;
        const int at = atomicAdd(&s_n, 1);
        if (at >= kRowThreads) break;
        const int b = __ffs(bits) - 1, k = w / NW % NV;
        bits &= bits - 1;
        s_note[at] = first + w / kWords * kChunk + (k * kRowThreads + w % NW * 32 + b) * VL;
      }
      const bool more = __syncthreads_or(bits != 0);
      const int n = min(s_n, kRowThreads);
      u64 key[VL], mine = 0;
      const int at = tid / PER + tid % PER * kSets;  // neighbours in the notes to different sets
      const int v = at < n ? s_note[at] : now.V;
      const u64 least = s_best[a.W - 1];
      float x[VL];
      unpack_vec<DT>(load_vec<DT>(now.row, v, now.V), x);
#pragma unroll
      for (int i = 0; i < VL; i++) {
        key[i] = v + i >= 0 && v + i < now.V && !(x[i] < bound) ? order_key(x[i], (uint32_t)(v + i)) : 0;
        if (key[i] <= least) key[i] = 0;
        mine = key[i] > mine ? key[i] : mine;
      }
      set_key(mine, PER, s_keys);
      const u64 nth = nth_key(a.W, s_keys, &s_nth);
      if (mine != 0 && mine >= nth) {
#pragma unroll
        for (int i = 0; i < VL; i++)
          if (key[i] != 0 && key[i] >= nth) s_list[atomicAdd(&s_k, 1)] = key[i];  // of W sets at most
      }
      if (tid < a.W && s_best[tid] != 0) s_list[atomicAdd(&s_k, 1)] = s_best[tid];
      __syncthreads();
      take_best(s_list, s_k, a.W, s_best);
      __syncthreads();
      if (!more) break;
    }
    const u64 best = s_best[a.W - 1];
    if (best != 0) bound = order_value((uint32_t)(best >> 32));
    noted = 0;
    __syncthreads();
  };
  for (int f = 0; f < runs; f++) {
    fetch(f + ST - 1);
    if (now.V == 0) {  // a beam that is done: nothing to read, and nothing of it is asked for
      stage = stage + 1 == ST ? 0 : stage + 1;
      step(now);
      continue;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
    uint4 u[NV];
    {
      const uint4* in = s_ring + stage * NV * kRowThreads + tid;
      const int start = now.v - tid * VL;  // of the chunk
      if (start >= 0 && start + kChunk <= now.V) {
#pragma unroll
        for (int k = 0; k < NV; k++) u[k] = in[k * kRowThreads];
      } else {  // at an end of the row
#pragma unroll 1
        for (int k = 0; k < NV; k++) {
          const int v = now.v + k * kRowThreads * VL;
          uint4* p = s_ring + stage * NV * kRowThreads + tid + k * kRowThreads;
          if (!(v >= 0 && v + VL <= now.V)) *p = load_vec<DT>(now.row, v, now.V);
        }
#pragma unroll
        for (int k = 0; k < NV; k++) u[k] = in[k * kRowThreads];
      }
    }
    stage = stage + 1 == ST ? 0 : stage + 1;
    uint32_t vm[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) vm[k] = max_vec<DT>(u[k]);
    uint32_t mw = vm[0];
#pragma unroll
    for (int k = 1; k < NV; k++) mw = max_word<DT>(mw, vm[k]);
    float best = word_max<DT>(mw);
    if (best != best) best = -INFINITY;  // a NaN counts as -inf here and spoils the sum
    if (bound == -INFINITY) {  // none yet: from the sets' largest
      float m = best;
#pragma unroll
      for (int o = 1; o < PER; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (tid % PER == 0) s_set[tid / PER] = m;
      __syncthreads();
      if (tid < 4 * kSets) {  // four threads to a set
        const float mine = s_set[tid >> 2];
        int above = 0, same = 0;
#pragma unroll
        for (int i = 0; i < kSets / 16; i++) {
          const float4 q = *(const float4*)(s_set + 4 * (tid & 3) + 16 * i);
          above += (q.x > mine) + (q.y > mine) + (q.z > mine) + (q.w > mine);
          same += (q.x == mine) + (q.y == mine) + (q.z == mine) + (q.w == mine);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          above += __shfl_xor_sync(0xffffffffu, above, o);
          same += __shfl_xor_sync(0xffffffffu, same, o);
        }
        if (above < a.W && above + same >= a.W) {  // one value, however many say so
          s_bound = mine;
          s_over = above + same > a.W;
          s_k = 0;
        }
      }
      __syncthreads();
      bound = s_bound;
    }
    const bool last = now.c + 1 == a.n || f + 1 == runs;  // of the row, or of this CTA's part of it
    // a row or part of one chunk needs no notes: what reaches the bound is listed from the registers
    const bool direct = first && last && bound > -INFINITY && !s_over;
    if (direct && best >= bound) {
#pragma unroll
      for (int k = 0; k < NV; k++) {
        if (word_max<DT>(vm[k]) >= bound) {
          float x[VL];
          unpack_vec<DT>(u[k], x);
#pragma unroll
          for (int i = 0; i < VL; i++)
            if (x[i] >= bound) {
              const int at = atomicAdd(&s_k, 1);
              if (at < a.W * (1 + PER * VL)) s_list[at] = order_key(x[i], (uint32_t)(now.v + k * kRowThreads * VL + i));
            }
        }
      }
    }
    if (best > top) {
      if (top == -INFINITY || best > ref + 40.0f) {  // a new point of reference for the sum
        z *= top == -INFINITY ? 1.0f : expf(ref - best);
        ref = best;
      }
      top = best;
    }
    f32x2 zz[2] = {};
    const f32x2 off = pair(-ref, -ref), log2e = pair(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
    for (int k = 0; k < NV; k++) {
      float x[VL];
      unpack_vec<DT>(u[k], x);
#pragma unroll
      for (int i = 0; i < VL; i += 2) {
        float y0, y1;
        unpair(mul_pair(add_pair(pair(x[i], x[i + 1]), off), log2e), y0, y1);
        zz[i >> 1 & 1] = add_pair(zz[i >> 1 & 1], pair(exp2_fast(y0), exp2_fast(y1)));
      }
    }
    {
      float z0, z1, z2, z3;
      unpair(zz[0], z0, z1);
      unpair(zz[1], z2, z3);
      z += (z0 + z1) + (z2 + z3);
    }
    // noted are the vectors that reach the bound; of -inf (and NaN) only the lowest places can be wanted,
    // after fewer than W others: they lie in the first vectors
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const float m = word_max<DT>(vm[k]);
      const uint32_t b =
          __ballot_sync(0xffffffffu, (m >= bound && m > -INFINITY) || (k == 0 && first && tid < 2 * kMaxBeams / VL + 2));
      if (lane == k) word = b;
    }
    first = false;
    if (lane < NV) s_bits[(noted * NV + lane) * NW + warp] = word;
    noted++;
    if (!last) {
      if (noted == kNoteChunks) {
        __syncthreads();
        settle();
      }
    } else {  // the row, or this CTA's part of it, is done
      const float wm = warp_max(top);
      if (lane == 0) s_m[warp] = wm;
      __syncthreads();
      float M = s_m[0];
#pragma unroll
      for (int k = 1; k < NW; k++) M = fmaxf(M, s_m[k]);
      z = warp_sum(top == -INFINITY ? z : z * expf(ref - M));
      if (lane == 0) s_z[warp] = z;
      if (direct && s_k <= a.W * (1 + PER * VL)) {
        take_best(s_list, s_k, a.W, s_best);
        noted = 0;
        __syncthreads();
      } else {
        if (direct) __syncthreads();  // settle() clears s_k, by which the others still decide
        settle();
      }
      const int slot = (int)blockIdx.x - owner_of((long)now.r * a.n, total, a.grid);
      const size_t o = (size_t)now.r * a.slots + slot;
      if (tid < a.W) {
        a.cand[o * a.W + tid] = s_best[tid];
        s_best[tid] = 0;
      }
      if (tid == 0) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; k++) s += s_z[k];
        a.sums[o] = make_float2(M, s);
      }
      __syncthreads();
      top = bound = -INFINITY;
      ref = z = 0.0f;
      first = true;
    }
    step(now);
  }
}

// One CTA per group.  per: candidates of a thread; with `rounds` the best are taken one after the other
// instead (where the list of a very large vocabulary would not fit shared memory).
constexpr int kGroupThreads = 512;
static_assert(kRowThreads >= 4 * kSets && kGroupThreads >= 4 * kSets, "sets are ranked by four threads each");
__global__ void __launch_bounds__(kGroupThreads) beam_group_kernel(BeamArgs a, int rounds) {
  constexpr int PER = kGroupThreads / kSets;
  __shared__ __align__(16) u64 s_keys[kSets];
  __shared__ u64 s_nth;
  __shared__ float s_lse[kMaxBeams];
  __shared__ u64 s_out[kMaxBeams];
  extern __shared__ u64 s_list[];  // [W * PER * candidates of a thread]
  __shared__ int s_n;
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  const long chunks = (long)a.R * a.n;
  auto parts_of = [&](int r) {
    return owner_of((long)(r + 1) * a.n - 1, chunks, a.grid) - owner_of((long)r * a.n, chunks, a.grid) + 1;
  };
  __shared__ int s_parts[kMaxBeams];
  if (tid < a.W) s_parts[tid] = parts_of(g * a.W + tid);
  grid_dep_wait();
  __syncthreads();
  // log-sum-exp of each row, a warp to a row
  for (int w = tid >> 5; w < a.W; w += kGroupThreads / 32) {
    const int r = g * a.W + w;
    if (a.done[r]) continue;
    const float2* s = a.sums + (size_t)r * a.slots;
    const int parts = s_parts[w];
    float m = -INFINITY, z = 0.0f;
    for (int c = lane; c < parts; c += 32) m = fmaxf(m, s[c].x);
    m = warp_max(m);
    for (int c = lane; c < parts; c += 32) {
      const float2 u = s[c];
      z += u.x == -INFINITY ? u.y : u.y * expf(u.x - m);  // without a logit the sum is 0, or NaN
    }
    z = warp_sum(z);
    if (lane == 0) s_lse[w] = m + logf(z);
  }
  if (tid == 0) s_n = 0;
  __syncthreads();
  const int per_row = a.slots * a.W, total = a.W * per_row;
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
    if (!(cum > -INFINITY) || !(fabsf(s_lse[w]) < INFINITY)) {  // a row that is lost: all -inf, whatever its logits
      const int k = i - w * per_row;
      return k < a.W ? order_key(-INFINITY, (uint32_t)w * (uint32_t)a.V + (uint32_t)k) : 0;
    }
    if (i - w * per_row >= s_parts[w] * a.W) return 0;
    const u64 k = cand[i];
    if (k == 0) return 0;
    const float x = order_value((uint32_t)(k >> 32));
    return order_key(cum + (x - s_lse[w]), (uint32_t)w * (uint32_t)a.V + (0xFFFFFFFFu - (uint32_t)k));
  };
  constexpr int kHeld = 4;  // candidates a thread holds; more are worked out again
  if (!rounds) {
    u64 held[kHeld], mine = 0;
#pragma unroll
    for (int k = 0; k < kHeld; k++) {
      const int i = tid + k * kGroupThreads;
      held[k] = i < total ? key_of(i) : 0;
      mine = held[k] > mine ? held[k] : mine;
    }
    for (int i = tid + kHeld * kGroupThreads; i < total; i += kGroupThreads) {
      const u64 k = key_of(i);
      mine = k > mine ? k : mine;
    }
    set_key(mine, PER, s_keys);
    const u64 bound = nth_key(a.W, s_keys, &s_nth);
    if (mine != 0 && mine >= bound) {
#pragma unroll
      for (int k = 0; k < kHeld; k++)
        if (held[k] != 0 && held[k] >= bound) s_list[atomicAdd(&s_n, 1)] = held[k];
      for (int i = tid + kHeld * kGroupThreads; i < total; i += kGroupThreads) {
        const u64 k = key_of(i);
        if (k != 0 && k >= bound) s_list[atomicAdd(&s_n, 1)] = k;
      }
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

typedef void (*RowKernel)(BeamArgs);
template <int DT>
static RowKernel row_kernel(int nv) {
  return nv == 1 ? beam_row_kernel<DT, 1> : nv == 2 ? beam_row_kernel<DT, 2> : nv == 4 ? beam_row_kernel<DT, 4> : beam_row_kernel<DT, 8>;
}
static RowKernel row_kernel(int dtype, int nv) {
  return dtype == DT_F32 ? row_kernel<DT_F32>(nv) : (dtype == DT_BF16 ? row_kernel<DT_BF16>(nv) : row_kernel<DT_F16>(nv));
}
static int row_smem(int dtype, int nv, int W) {
  const int vl = dtype == DT_F32 ? 4 : 8;
  return (nv == 8 ? ring_stages<8>() : ring_stages<4>()) * nv * kRowThreads * 16 + W * (1 + kRowThreads / kSets * vl) * 8;
}

// CTAs of the kernel that one SM holds, remembered; also makes the shared memory available to it.
static int rows_per_sm(int dtype, int nv, int W, int* out) {
  static std::atomic<unsigned long long> smem_set[3][9];
  static std::atomic<int> known[3][9][kMaxBeams + 1];
  RNGD_TRY(set_smem_limit_once((const void*)row_kernel(dtype, nv), row_smem(dtype, nv, kMaxBeams), &smem_set[dtype][nv],
                               "cudaFuncSetAttribute(beam_row_kernel)"));
  int n = known[dtype][nv][W].load(std::memory_order_relaxed);
  if (n == 0) {
    RNGD_TRY(check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, row_kernel(dtype, nv), kRowThreads,
                                                                      row_smem(dtype, nv, W)),
                        "occupancy(beam_row_kernel)"));
    if (n < 1) n = 1;
    known[dtype][nv][W].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return RNGD_OK;
}

// How the rows are cut: vectors of a thread and chunk (fewer where there is little to do, so that the one
// pass ends sooner), chunks of a row, CTAs (as many as run at once), CTAs that may share a row.
struct BeamPlan {
  int nv, n, grid, slots;
};
static int beam_plan(int dtype, int R, int V, int W, BeamPlan* p) {
  RNGD_REQUIRE(dtype >= DT_BF16 && dtype <= DT_F32, "beam_select: data type %d", dtype);
  RNGD_REQUIRE(W >= 1 && W <= kMaxBeams, "beam_select: %d beams, at most %d", W, kMaxBeams);
  RNGD_REQUIRE(R >= 0 && V >= 1, "beam_select: %d rows of %d logits", R, V);
  const int vl = dtype == DT_F32 ? 4 : 8;
  auto chunks = [&](int nv) { return ((long)V + vl - 1 + kRowThreads * vl * nv - 1) / (kRowThreads * vl * nv); };
  p->nv = 8;
  for (int nv = 1; nv < 8; nv *= 2)
    if ((long)R * chunks(nv) <= 2 * num_sms()) {
      p->nv = nv;
      break;
    }
  p->n = (int)chunks(p->nv);
  int per = 1;
  RNGD_TRY(rows_per_sm(dtype, p->nv, W, &per));
  const long all = (long)R * p->n, most = (long)num_sms() * per;
  p->grid = (int)(all < most ? all : most);
  const long len = p->grid > 0 ? all / p->grid : 1;  // chunks of a CTA at least
  const long slots = (p->n + len - 2) / len + 1;
  p->slots = (int)(slots < p->n ? slots : p->n);
  return RNGD_OK;
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_beam_workspace(int dtype, int R, int V, int W, size_t* bytes) {
  RNGD_REQUIRE(bytes != nullptr, "beam_workspace: null output");
  BeamPlan p;
  RNGD_TRY(beam_plan(dtype, R, V, W, &p));
  *bytes = (size_t)R * p.slots * ((size_t)W + 1) * 8;
  return RNGD_OK;
}

extern "C" int rngd_beam_select(const void* logits, int dtype, int64_t ld, int R, int V, int W, const float* scores,
                                const uint8_t* done, int eos, float* out_scores, int32_t* parents, int32_t* tokens,
                                uint8_t* out_done, void* workspace, size_t workspace_bytes, rngd_stream_t stream) {
  BeamPlan p;
  RNGD_TRY(beam_plan(dtype, R, V, W, &p));
  RNGD_REQUIRE(R % W == 0, "beam_select: %d rows are not whole groups of %d beams", R, W);
  RNGD_REQUIRE(V >= W && V < (1 << 30) && (long)V * W < (1l << 31), "beam_select: vocabulary of %d", V);
  RNGD_REQUIRE(ld >= V || R <= 1, "beam_select: rows of %d logits %ld apart", V, (long)ld);
  if (R == 0) return RNGD_OK;
  RNGD_REQUIRE(logits && scores && done && out_scores && parents && tokens && out_done && workspace,
               "beam_select: null pointer");
  const size_t need = (size_t)R * p.slots * ((size_t)W + 1) * 8;
  RNGD_REQUIRE(((uintptr_t)workspace & 7) == 0 && workspace_bytes >= need,
               "beam_select: workspace of %zu bytes, %zu needed (8-byte aligned)", workspace_bytes, need);
  BeamArgs a = {logits, (long)ld, R, V, W, eos, p.n, p.grid, p.slots, scores, done, out_scores, parents, tokens, out_done};
  a.cand = (u64*)workspace;
  a.sums = (float2*)(a.cand + (size_t)R * p.slots * W);
  cudaStream_t s = (cudaStream_t)stream;
  RNGD_TRY(launch_pdl(row_kernel(dtype, p.nv), dim3(p.grid), dim3(kRowThreads), row_smem(dtype, p.nv, W), s,
                      "beam_row_kernel", a));
  const long per = ((long)W * W * p.slots + kGroupThreads - 1) / kGroupThreads;
  size_t smem = (size_t)W * (kGroupThreads / kSets) * per * 8;
  const bool rounds = smem > 128 * 1024;
  if (rounds) smem = 0;
  static std::atomic<unsigned long long> smem_set{0};
  if (smem > 32 * 1024)
    RNGD_TRY(set_smem_limit_once((const void*)beam_group_kernel, 128 * 1024, &smem_set,
                                 "cudaFuncSetAttribute(beam_group_kernel)"));
  return launch_pdl(beam_group_kernel, dim3(R / W), dim3(kGroupThreads), smem, s, "beam_group_kernel", a, rounds ? 1 : 0);
}
