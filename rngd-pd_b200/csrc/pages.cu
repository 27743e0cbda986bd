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
  int* n_moves;
  Move* moves;  // [R]
  int* list;    // [R * (1 + ld)] free pages
  int P, R, ld, room;
};

// Pages that n positions take, for any n (a sum with kPage - 1 would pass 32 bits).
__device__ __forceinline__ int pages_of(int n) { return n > 0 ? (n - 1) / kPage + 1 : 0; }

constexpr int kMetaThreads = 1024;
constexpr int kForkCtas = 8;  // one cluster

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

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One cluster: its CTAs share the tables (counts go up and down by whole-number atomics), the first one
// then decides row by row, a thread to each.  Latency is what it takes: two rounds of dependent loads over
// the tables and a walk through the free pages.  With the copies it takes 10.9 us in a graph for 16 rows (14 MB
// moved, 2.2 us of it by the bytes) and 16.8 us for 256 rows, most of it at barriers.  The barriers order what the
// CTAs write for one another; fences before them took 0.7 and 0.9 us more.
__global__ void __cluster_dims__(kForkCtas, 1, 1) __launch_bounds__(kMetaThreads) kv4_fork_kernel(ForkArgs a) {
  __shared__ int s_warp[32];
  __shared__ __align__(16) int s_tail[kMetaThreads];
  __shared__ unsigned long long s_over;  // pages that could not be given
  const int tid = threadIdx.x, all = kForkCtas * kMetaThreads, me = blockIdx.x * kMetaThreads + tid;
  grid_dep_wait();
  for (int p = me; p < a.P; p += all) a.new_ref[p] = a.ref[p];
  cluster_sync();
  const int cells = a.R * a.ld;
  for (int i0 = me; i0 < cells; i0 += 4 * all) {
    int old[4], now[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int i = i0 + k * all;
      old[k] = now[k] = -1;
      if (i < cells) {
        const int r = i / a.ld, col = i - r * a.ld;
        old[k] = a.table[i];
        const int par = a.parents != nullptr ? a.parents[r] : r;
        if (par >= 0 && par < a.R && col < pages_of(a.lens[par])) now[k] = a.table[par * a.ld + col];
      }
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int i = i0 + k * all;
      if (i < cells) {
        if (now[k] < 0 || now[k] >= a.P) now[k] = -1;
        if (old[k] < 0 || old[k] >= a.P) old[k] = -1;
        a.new_table[i] = now[k];
        if (old[k] != now[k]) {  // a page that stays needs no counting
          if (old[k] >= 0) atomicAdd(a.new_ref + old[k], -1);
          if (now[k] >= 0) atomicAdd(a.new_ref + now[k], 1);
        }
      }
    }
  }
  cluster_sync();
  if (blockIdx.x != 0) return;
  const int r = tid;
  int len = 0, n = 0, last = 0, tail = -1, over = 0;
  if (r < a.R) {
    const int par = a.parents != nullptr ? a.parents[r] : r;
    const bool on = par >= 0 && par < a.R;
    len = on ? max(a.lens[par], 0) : 0;
    a.new_lens[r] = len;
    n = min(pages_of(len), a.ld);
    const int want = on ? (int)(((long)len + a.room + kPage - 1) / kPage) : 0;
    last = max(n, min(want, a.ld));
    over = max(want - last, 0);
    if (on && len % kPage != 0 && n > 0 && pages_of(len) <= a.ld) tail = __ldcg(a.new_table + r * a.ld + n - 1);
  }
  s_tail[tid] = tail;
  if (tid == 0) s_over = 0;
  __syncthreads();
  bool copy = false;
  if (tail >= 0) {
    const int held = __ldcg(a.new_ref + tail);
    if (held > 1) {
      int same = 0, lower = 0;
      for (int k = 0; k < a.R; k += 4) {
        const int4 t = *(const int4*)(s_tail + k);
        const int h0 = t.x == tail, h1 = t.y == tail, h2 = t.z == tail, h3 = t.w == tail;
        same += h0 + h1 + h2 + h3;
        lower |= (h0 & (k < r)) | (h1 & (k + 1 < r)) | (h2 & (k + 2 < r)) | (h3 & (k + 3 < r));
      }
      copy = lower || held > same;
    }
  }
  int need, got;
  const int base = block_scan((copy ? 1 : 0) + last - n, s_warp, &need);
  // the `need` lowest free pages: the one of rank k answers request k
  int have = 0;
  for (int p0 = 0; p0 < a.P && have < need; p0 += 4 * kMetaThreads) {
    int free = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int p = p0 + 4 * tid + k;
      free |= p < a.P && __ldcg(a.new_ref + p) == 0 ? 1 << k : 0;
    }
    int at = have + block_scan(__popc(free), s_warp, &got);
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (free >> k & 1) {
        if (at < need) a.list[at] = p0 + 4 * tid + k;
        at++;
      }
    have += got;
  }
  __syncthreads();
  have = min(have, need);
  Move mv = {0, 0, 0};
  if (r < a.R) {
    int k = base;
    if (copy) {
      const int p = k < have ? __ldcg(a.list + k) : -1;
      k++;
      a.new_table[r * a.ld + n - 1] = p;
      atomicAdd(a.new_ref + tail, -1);
      if (p >= 0) {
        a.new_ref[p] = 1;
        mv = {tail, p, (len % kPage + kBlk - 1) / kBlk};
      } else {
        over++;
      }
    }
    for (int c = n; c < last; c++, k++) {
      const int p = k < have ? __ldcg(a.list + k) : -1;
      a.new_table[r * a.ld + c] = p;
      if (p >= 0)
        a.new_ref[p] = 1;
      else
        over++;
    }
  }
  const int m = block_scan(mv.blocks > 0, s_warp, &got);
  if (mv.blocks > 0) a.moves[m] = mv;
  if (over > 0) atomicAdd(&s_over, (unsigned long long)over);  // up to 2^36 of 1024 rows
  __syncthreads();
  if (tid == 0) {
    *a.n_moves = got;
    *a.short_out = (int)min(s_over, 0x7FFFFFFFull);
  }
}

struct CompactArgs {
  const int32_t* ref;
  int32_t* new_ref;
  int32_t* live_out;
  int* n_moves;
  Move* moves;    // [P]
  int32_t* map;   // [P]
  int P;
};

// One CTA: counts the live pages (n), pairs the k-th live page from n on with the k-th free place below n,
// and rewrites the counts; the tables are rewritten by the copying kernel's many threads.  A thread has a run of pages of its own, so that one prefix sum counts
// them all.  Latency again: with
// the copies 6.2 us in a graph for 12 pages moved of 300 (7.7 with fences, and the tables rewritten here).
__global__ void __launch_bounds__(kMetaThreads) kv4_compact_kernel(CompactArgs a) {
  __shared__ int s_warp[32];
  const int tid = threadIdx.x, run = (a.P + kMetaThreads - 1) / kMetaThreads;
  const int q0 = min(tid * run, a.P), q1 = min(q0 + run, a.P);
  grid_dep_wait();
  int c = 0, n;
  for (int p = tid; p < a.P; p += kMetaThreads) c += a.ref[p] > 0;
  block_scan(c, s_warp, &n);
  int src = 0, dst = 0, srcs, dsts;
  for (int p = q0; p < q1; p++) {
    const bool live = a.ref[p] > 0;
    src += live && p >= n;
    dst += !live && p < n;
  }
  src = block_scan(src, s_warp, &srcs);
  dst = block_scan(dst, s_warp, &dsts);
  for (int p = q0; p < q1; p++) {
    const int rf = a.ref[p];
    if (rf > 0 && p >= n) a.moves[src++].src = p;
    if (rf <= 0 && p < n) a.moves[dst++].dst = p;
    a.map[p] = p;
    a.new_ref[p] = rf;
  }
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
}

// Copies pages: a warp takes 2560 bytes of a (move, layer, head) at a time, five loads in flight a lane.
// 600 pages of 4 layers, 8 heads of 128 (393 MB read and written): 60 us, 6.5 TB/s, the copy bandwidth; with the
// kernel above 71 us in a graph.
constexpr int kCopyVecs = 160;
struct Tables {  // to rewrite beside the copies: page p becomes map[p]
  const int32_t* table;
  int32_t* new_table;
  const int32_t* map;
  int cells, P;
};
__global__ void __launch_bounds__(256) kv4_copy_kernel(uint8_t* pool, size_t layer_bytes, int L, int NKV, int blk_bytes,
                                                       const Move* moves, const int* n_moves, Tables t) {
  const int lane = threadIdx.x & 31;
  const long warp = ((long)blockIdx.x * 256 + threadIdx.x) >> 5, warps = (long)gridDim.x * 8;
  const int blk_vecs = blk_bytes / 16, subs = 4 * blk_vecs / kCopyVecs;
  grid_dep_wait();
  for (int i = blockIdx.x * 256 + threadIdx.x; i < t.cells; i += gridDim.x * 256) {
    const int p = t.table[i];
    t.new_table[i] = p >= 0 && p < t.P ? t.map[p] : -1;
  }
  const long units = (long)*n_moves * L * NKV * subs;
  for (long u = warp; u < units; u += warps) {
    uint32_t x = (uint32_t)(u % ((long)L * NKV * subs));
    const Move mv = moves[u / ((long)L * NKV * subs)];
    const int sub = (int)(x % subs);
    x /= subs;
    const int h = (int)(x % NKV), l = (int)(x / NKV);
    const int vecs = mv.blocks * blk_vecs - sub * kCopyVecs;  // from this part's start on
    uint8_t* base = pool + l * layer_bytes + (size_t)sub * kCopyVecs * 16;
    const uint4* s = (const uint4*)(base + ((size_t)mv.src * NKV + h) * 4 * blk_bytes);
    uint4* d = (uint4*)(base + ((size_t)mv.dst * NKV + h) * 4 * blk_bytes);
    uint4 v[5];
#pragma unroll
    for (int k = 0; k < 5; k++)
      if (lane + 32 * k < vecs) v[k] = __ldcs(s + lane + 32 * k);
#pragma unroll
    for (int k = 0; k < 5; k++)
      if (lane + 32 * k < vecs) __stcs(d + lane + 32 * k, v[k]);
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

// The copies of up to `most` moves; how many there are is known on the device alone.
static int launch_copy(uint8_t* pool, size_t layer_bytes, int L, int NKV, int HD, const Move* moves, const int* n_moves,
                       int most, const Tables& t, cudaStream_t s) {
  const long units = (long)most * L * NKV * (4 * kv4_block_bytes(HD) / 16 / kCopyVecs), blocks = (units + 7) / 8;
  const long cap = (long)num_sms() * 8;
  return launch_pdl(kv4_copy_kernel, dim3((unsigned)(blocks < cap ? blocks : cap)), dim3(256), 0, s, "kv4_copy_kernel", pool,
                    layer_bytes, L, NKV, kv4_block_bytes(HD), moves, n_moves, t);
}

}  // namespace rngd

using namespace rngd;

extern "C" int rngd_kv4_fork_workspace(int R, int ld_table, size_t* bytes) {
  RNGD_REQUIRE(bytes && R >= 0 && ld_table >= 0, "kv4_fork_workspace: bad argument");
  *bytes = 16 + (size_t)R * sizeof(Move) + (size_t)R * (1 + ld_table) * 4;
  return RNGD_OK;
}

extern "C" int rngd_kv4_fork(void* pool, size_t layer_bytes, int L, int P, int NKV, int HD, const int32_t* ref,
                             const int32_t* table, int ld_table, const int32_t* lens, int R, const int32_t* parents,
                             int room, int32_t* new_ref, int32_t* new_table, int32_t* new_lens, int32_t* short_out,
                             void* workspace, size_t workspace_bytes, rngd_stream_t stream) {
  RNGD_TRY(check_pages("kv4_fork", pool, layer_bytes, L, P, NKV, HD, R, ld_table));
  RNGD_REQUIRE(R <= kMetaThreads, "kv4_fork: %d rows, at most %d", R, kMetaThreads);
  RNGD_REQUIRE(room >= 0 && room <= (1 << 30), "kv4_fork: room=%d", room);
  RNGD_REQUIRE(ref && new_ref && short_out && workspace && ref != new_ref && (R == 0 || (lens && new_lens)) &&
                   (R == 0 || ld_table == 0 || (table && new_table)) && (table != new_table || table == nullptr),
               "kv4_fork: null pointer, or new state in place of the old");
  size_t need;
  RNGD_TRY(rngd_kv4_fork_workspace(R, ld_table, &need));
  RNGD_REQUIRE(((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need,
               "kv4_fork: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
  int* n_moves = (int*)workspace;
  Move* moves = (Move*)((uint8_t*)workspace + 16);
  ForkArgs a = {ref, table, lens, parents, new_ref, new_table, new_lens, short_out, n_moves, moves, (int*)(moves + R),
                P, R, ld_table, room};
  cudaStream_t s = (cudaStream_t)stream;
  RNGD_TRY(launch_pdl(kv4_fork_kernel, dim3(kForkCtas), dim3(kMetaThreads), 0, s, "kv4_fork_kernel", a));
  if (R == 0) return RNGD_OK;
  return launch_copy((uint8_t*)pool, layer_bytes, L, NKV, HD, moves, n_moves, R, Tables{}, s);
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
  RNGD_REQUIRE(((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need,
               "kv4_compact: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
  int* n_moves = (int*)workspace;
  Move* moves = (Move*)((uint8_t*)workspace + 16);
  int32_t* map = (int32_t*)(moves + P);
  CompactArgs a = {ref, new_ref, live, n_moves, moves, map, P};
  cudaStream_t s = (cudaStream_t)stream;
  RNGD_TRY(launch_pdl(kv4_compact_kernel, dim3(1), dim3(kMetaThreads), 0, s, "kv4_compact_kernel", a));
  return launch_copy((uint8_t*)pool, layer_bytes, L, NKV, HD, moves, n_moves, P, Tables{table, new_table, map, (int)cells, P}, s);
}
