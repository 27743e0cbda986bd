// Pages of the 4-bit KV cache: forking, extending, ending and compacting the sequences that hold them.
//
// A pool keeps a count of holders per page (`ref`, 0 = free); a sequence is a row of page ids (-1 = none)
// and a length.  All of it lives on the device and is read and written there, so that a decode loop
// needs no host round trip.  Results do not depend on the order in which threads run: counts are whole
// numbers, and free pages are handed out lowest first, in the order of rows.  New counts, tables and
// lengths go to other buffers than the old; the pool is changed in free pages only.
#include "kv4.cuh"

namespace rngd {

struct Move {  // one page's copy: its first `blocks` blocks
  int src, dst, blocks;
};

struct ForkArgs {
  const int32_t* ref;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* parents;  // null: every row goes on as itself
  int32_t* new_ref;
  int32_t* new_table;
  int32_t* new_lens;
  int32_t* short_out;
  Move* moves;  // [R], blocks = 0: none
  int P, R, ld, room;
};

constexpr int kMetaThreads = 1024;

// Exclusive prefix sum over the CTA; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // s_warp may still be read from an earlier call
  if (lane == 31) s_warp[w] = x;
  __syncthreads();
  if (w == 0) {
    int y = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    s_warp[lane] = y;
  }
  __syncthreads();
  *total = s_warp[31];
  return x - v + (w > 0 ? s_warp[w - 1] : 0);
}

// One CTA of 1024 threads, one thread per row for what is decided row by row.
__global__ void __launch_bounds__(kMetaThreads) kv4_fork_kernel(ForkArgs a) {
  __shared__ int s_warp[32];
  __shared__ int s_tail[kMetaThreads];
  const int tid = threadIdx.x;
  for (int p = tid; p < a.P; p += kMetaThreads) a.new_ref[p] = a.ref[p];
  if (tid == 0) *a.short_out = 0;
  __syncthreads();
  const long cells = (long)a.R * a.ld;
  for (long i = tid; i < cells; i += kMetaThreads) {
    const int r = (int)(i / a.ld), col = (int)(i % a.ld);
    const int old = a.table[i];
    if (old >= 0 && old < a.P) atomicAdd(a.new_ref + old, -1);
    const int par = a.parents != nullptr ? a.parents[r] : r;
    int now = -1;
    if (par >= 0 && par < a.R && col < (a.lens[par] + kPage - 1) / kPage) now = a.table[(size_t)par * a.ld + col];
    if (now >= a.P) now = -1;
    a.new_table[i] = now;
    if (now >= 0) atomicAdd(a.new_ref + now, 1);
  }
  __threadfence();
  __syncthreads();
  // rows
  const int r = tid;
  int len = 0, n = 0, last = 0, tail = -1, over = 0;
  if (r < a.R) {
    const int par = a.parents != nullptr ? a.parents[r] : r;
    const bool on = par >= 0 && par < a.R;
    len = on ? max(a.lens[par], 0) : 0;
    a.new_lens[r] = len;
    n = min((len + kPage - 1) / kPage, a.ld);
    const int want = on ? (len + a.room + kPage - 1) / kPage : 0;
    last = max(n, min(want, a.ld));
    over = max(want - last, 0);
    if (on && len % kPage != 0 && n > 0 && (len + kPage - 1) / kPage <= a.ld) tail = a.new_table[(size_t)r * a.ld + n - 1];
  }
  s_tail[tid] = tail;
  __syncthreads();
  bool copy = false;
  if (tail >= 0) {
    int same = 0;
    bool lower = false;
    for (int k = 0; k < a.R; k++)
      if (s_tail[k] == tail) {
        same++;
        lower |= k < r;
      }
    copy = lower || __ldcg(a.new_ref + tail) > same;
  }
  int need;
  const int base = block_scan((copy ? 1 : 0) + last - n, s_warp, &need);
  // the `need` lowest free pages, in order: the page with rank k answers request k, so each row
  // finds its own by reading the list back
  __shared__ int s_have;
  if (tid == 0) s_have = 0;
  __syncthreads();
  int* list = (int*)(a.moves + a.R);  // [need] at most R * (1 + ld)
  for (int p0 = 0; p0 < a.P; p0 += kMetaThreads) {
    const int have = s_have;
    if (have >= need) break;
    const int p = p0 + tid;
    const bool free = p < a.P && __ldcg(a.new_ref + p) == 0;
    int got;
    const int at = have + block_scan(free ? 1 : 0, s_warp, &got);
    if (free && at < need) list[at] = p;
    if (tid == 0) s_have = have + got;
    __syncthreads();
  }
  __threadfence();
  __syncthreads();
  const int have = min(s_have, need);
  if (r < a.R) {
    int k = base;
    Move mv = {0, 0, 0};
    if (copy) {
      const int p = k < have ? __ldcg(list + k) : -1;
      k++;
      a.new_table[(size_t)r * a.ld + n - 1] = p;
      atomicAdd(a.new_ref + tail, -1);
      if (p >= 0) {
        atomicAdd(a.new_ref + p, 1);
        mv = {tail, p, (len % kPage + kBlk - 1) / kBlk};
      } else {
        over++;
      }
    }
    for (int c = n; c < last; c++, k++) {
      const int p = k < have ? __ldcg(list + k) : -1;
      a.new_table[(size_t)r * a.ld + c] = p;
      if (p >= 0)
        atomicAdd(a.new_ref + p, 1);
      else
        over++;
    }
    a.moves[r] = mv;
    if (over) atomicAdd(a.short_out, over);
  }
}

struct CompactArgs {
  const int32_t* ref;
  const int32_t* table;
  int32_t* new_ref;
  int32_t* new_table;
  int32_t* live_out;
  Move* moves;    // [P]
  int32_t* n_moves;
  int32_t* map;   // [P]
  int P;
  long cells;
};

// One CTA: counts the live pages (n), pairs the k-th live page from n on with the k-th free place
// below n, and rewrites counts and tables.
__global__ void __launch_bounds__(kMetaThreads) kv4_compact_kernel(CompactArgs a) {
  __shared__ int s_warp[32];
  const int tid = threadIdx.x;
  int c = 0, n;
  for (int p = tid; p < a.P; p += kMetaThreads) c += a.ref[p] > 0;
  block_scan(c, s_warp, &n);
  int srcs = 0, dsts = 0;
  for (int p0 = 0; p0 < a.P; p0 += kMetaThreads) {
    const int p = p0 + tid;
    const int rf = p < a.P ? a.ref[p] : 0;
    const bool src = p < a.P && p >= n && rf > 0, dst = p < min(n, a.P) && rf <= 0;
    int got;
    int at = block_scan(src, s_warp, &got);
    if (src) a.moves[srcs + at].src = p;
    srcs += got;
    at = block_scan(dst, s_warp, &got);
    if (dst) a.moves[dsts + at].dst = p;
    dsts += got;
    if (p < a.P) {
      a.map[p] = p;
      a.new_ref[p] = rf;
    }
  }
  __threadfence();
  __syncthreads();
  for (int k = tid; k < srcs; k += kMetaThreads) {
    const int s = __ldcg(&a.moves[k].src), d = __ldcg(&a.moves[k].dst);
    a.moves[k].blocks = kPage / kBlk;
    a.map[s] = d;
    a.new_ref[d] = a.ref[s];
    a.new_ref[s] = 0;
  }
  if (tid == 0) {
    *a.n_moves = srcs;
    *a.live_out = n;
  }
  __threadfence();
  __syncthreads();
  for (long i = tid; i < a.cells; i += kMetaThreads) {
    const int p = a.table[i];
    a.new_table[i] = p >= 0 && p < a.P ? __ldcg(a.map + p) : -1;
  }
}

// Copies pages, one (move, layer, head) per warp and turn.  `n` (device) or `fixed` gives the number
// of moves.
__global__ void __launch_bounds__(256) kv4_copy_kernel(uint8_t* pool, size_t layer_bytes, int L, int NKV, int blk_bytes,
                                                       const Move* moves, const int32_t* n, int fixed) {
  const int lane = threadIdx.x & 31;
  const long warp = ((long)blockIdx.x * 256 + threadIdx.x) >> 5, warps = (long)gridDim.x * 8;
  const long units = (long)(n != nullptr ? *n : fixed) * L * NKV;
  for (long u = warp; u < units; u += warps) {
    const Move mv = moves[u / NKV / L];
    const int h = (int)(u % NKV), l = (int)(u / NKV % L);
    uint8_t* base = pool + l * layer_bytes;
    const uint4* s = (const uint4*)(base + ((size_t)mv.src * NKV + h) * 4 * blk_bytes);
    uint4* d = (uint4*)(base + ((size_t)mv.dst * NKV + h) * 4 * blk_bytes);
    const int words = mv.blocks * blk_bytes / 16;
    for (int i = lane; i < words; i += 32) d[i] = s[i];
  }
}

static int check_pages(const char* what, const void* pool, size_t layer_bytes, int L, int P, int NKV, int HD, int R,
                       int ld) {
  RNGD_REQUIRE(pool != nullptr && ((uintptr_t)pool & 15) == 0 && (layer_bytes & 15) == 0,
               "%s: the pool must be 16-byte aligned", what);
  RNGD_REQUIRE(HD == 64 || HD == 128, "%s: built for HD 64 and 128, not %d", what, HD);
  RNGD_REQUIRE(L >= 1 && P >= 1 && NKV >= 1 && NKV <= 1024, "%s: L=%d P=%d NKV=%d", what, L, P, NKV);
  RNGD_REQUIRE(R >= 0 && ld >= 0 && (long)R * ld < (1l << 30), "%s: table of %d rows of %d pages", what, R, ld);
  return RNGD_OK;
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_kv4_fork_workspace(int R, int ld_table, size_t* bytes) {
  RNGD_REQUIRE(bytes && R >= 0 && ld_table >= 0, "kv4_fork_workspace: bad argument");
  *bytes = (size_t)R * sizeof(Move) + (size_t)R * (1 + ld_table) * 4;
  return RNGD_OK;
}

extern "C" int rngd_kv4_fork(void* pool, size_t layer_bytes, int L, int P, int NKV, int HD, const int32_t* ref,
                             const int32_t* table, int ld_table, const int32_t* lens, int R, const int32_t* parents,
                             int room, int32_t* new_ref, int32_t* new_table, int32_t* new_lens, int32_t* short_out,
                             void* workspace, size_t workspace_bytes, rngd_stream_t stream) {
  RNGD_TRY(check_pages("kv4_fork", pool, layer_bytes, L, P, NKV, HD, R, ld_table));
  RNGD_REQUIRE(R <= kMetaThreads, "kv4_fork: %d rows, at most %d", R, kMetaThreads);
  RNGD_REQUIRE(room >= 0 && room <= (1 << 30), "kv4_fork: room=%d", room);
  RNGD_REQUIRE(ref && new_ref && short_out && ref != new_ref && (R == 0 || (lens && new_lens && workspace)) &&
                   (R == 0 || ld_table == 0 || (table && new_table)) && (table != new_table || table == nullptr),
               "kv4_fork: null pointer, or new state in place of the old");
  size_t need;
  RNGD_TRY(rngd_kv4_fork_workspace(R, ld_table, &need));
  RNGD_REQUIRE(workspace_bytes >= need, "kv4_fork: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  ForkArgs a = {ref, table, lens, parents, new_ref, new_table, new_lens, short_out, (Move*)workspace, P, R, ld_table,
                room};
  cudaStream_t s = (cudaStream_t)stream;
  kv4_fork_kernel<<<1, kMetaThreads, 0, s>>>(a);
  RNGD_TRY(check_launch("kv4_fork_kernel"));
  if (R == 0) return RNGD_OK;
  const long units = (long)R * L * NKV;
  const long blocks = (units + 7) / 8;
  kv4_copy_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, s>>>(
      (uint8_t*)pool, layer_bytes, L, NKV, kv4_block_bytes(HD), a.moves, nullptr, R);
  return check_launch("kv4_copy_kernel");
}

extern "C" int rngd_kv4_compact_workspace(int P, size_t* bytes) {
  RNGD_REQUIRE(bytes && P >= 1, "kv4_compact_workspace: bad argument");
  *bytes = (size_t)P * (sizeof(Move) + 4) + 16;
  return RNGD_OK;
}

extern "C" int rngd_kv4_compact(void* pool, size_t layer_bytes, int L, int P, int NKV, int HD, const int32_t* ref,
                                const int32_t* table, int ld_table, int R, int32_t* new_ref, int32_t* new_table,
                                int32_t* live, void* workspace, size_t workspace_bytes, rngd_stream_t stream) {
  RNGD_TRY(check_pages("kv4_compact", pool, layer_bytes, L, P, NKV, HD, R, ld_table));
  const long cells = (long)R * ld_table;
  RNGD_REQUIRE(ref && new_ref && live && workspace && ref != new_ref && (cells == 0 || (table && new_table)) &&
                   (table != new_table || table == nullptr),
               "kv4_compact: null pointer, or new state in place of the old");
  size_t need;
  RNGD_TRY(rngd_kv4_compact_workspace(P, &need));
  RNGD_REQUIRE(workspace_bytes >= need, "kv4_compact: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  int32_t* n_moves = (int32_t*)workspace;
  Move* moves = (Move*)((uint8_t*)workspace + 16);
  int32_t* map = (int32_t*)(moves + P);
  CompactArgs a = {ref, table, new_ref, new_table, live, moves, n_moves, map, P, cells};
  cudaStream_t s = (cudaStream_t)stream;
  kv4_compact_kernel<<<1, kMetaThreads, 0, s>>>(a);
  RNGD_TRY(check_launch("kv4_compact_kernel"));
  kv4_copy_kernel<<<148 * 8, 256, 0, s>>>((uint8_t*)pool, layer_bytes, L, NKV, kv4_block_bytes(HD), moves, n_moves, 0);
  return check_launch("kv4_copy_kernel");
}
