// The beams' paged states after a selection: tables, reference counts, free blocks and K/V.
//
// Row i = g K + k takes the state of row s = g K + parent(i), c = lens[s] positions:
//   its whole blocks, c / bs of them, are shared: table'[i][j] = table[s][j];
//   a block that is not full (c mod bs positions of it) is kept by the first child of s if s alone
//   holds it, and copied into a fresh block for every other child: its positions of K and V, in all layers;
//   parent -1, or a parent without positions, empties the row.
// refs[b] counts the rows (and whoever else holds it) of block b: every row lets go of its old table
// and takes hold of its new one. A block that nobody holds any more is free.
//
// Launches: 1. one workgroup: who copies, the fresh blocks (running sum over the rows), the new lengths;
// 2. a workgroup per request and 128 columns of its tables: the new tables, what the reference counts change by,
// the blocks that were let go of; beside them the copies; the last of the former puts those of these blocks that nobody
// holds, each once, in the order (request, column, row) of the old tables, behind the free blocks. Every order is
// fixed: the same state gives the same tables. Fresh blocks are taken before any is freed, so that a copy's source
// is never its own destination. Where something does not fit nothing is changed.
//
// What bounds it: the way of the counts. Tables, counts, lists, the last workgroup's look at all of them and the free blocks are
// five accesses to memory one behind the other, 1 to 2 us each across XCDs, beside which the copies run: a request of 4 beams
// 4 + 7 us, 32 requests of 8 beams (14.6 MB of tables and K/V read and written) 5 + 12, 16 of 4 at 32 layers of 8 heads of 128
// (42.7 MB) 5 + 14. Counts that were waited for one by one and a third launch for the free blocks took 25 us at 32 of 8, freed blocks
// searched for one behind the other 19, now 16.4.
#include "tb_common.h"

namespace tb {

constexpr int REORDER_COLUMNS = 128;
constexpr int32_t MARK = 1 << 30;

struct reorder_args {
  char* storage;               // [layers][NB][2][Hkv][bs][D]
  int64_t layer_bytes;
  int32_t layers, num_blocks, pairs;   // pairs = 2 Hkv
  int32_t row_bytes;           // of a position of a head
  int32_t unit_pairs, parts;   // pairs of a copy's unit, units of a block
  int32_t log2_bs;
  int32_t* tables;             // [rows][max_nb]
  int32_t max_nb, rows, beams;
  const int32_t* lens_in;      // [rows]
  int32_t* lens_out;           // [rows]
  int32_t* refs;               // [NB]
  int32_t* free_blocks;        // [NB]
  const int32_t* num_free_in;
  int32_t* num_free_out;
  int32_t* shared;             // [rows / beams]
  const int32_t* parents;      // [rows]
  uint32_t* status;
  // workspace
  int32_t* head;               // {0 or 1: nothing is done, copies, workgroups that have listed their blocks}
  int4* plan;                  // [rows]: {source row or -1, new length, fresh block or -1, old length}
  int4* copies;                // [rows]: {source block, fresh block, positions, 0}
  int32_t* least;              // [requests]: whole blocks of every live row
  int32_t* gone_count;         // [requests * chunks]
  int32_t* gone;               // [requests * chunks][128 beams]
  int32_t chunks;
};

__device__ __forceinline__ int wave_scan(int x, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}
// Exclusive running sum over a workgroup; `total` gets the whole. One barrier before the result, and the
// next call's writes go to the other half of `waves` [2][THREADS / 64].
template <int THREADS>
__device__ __forceinline__ int group_scan(int x, int (*waves)[THREADS / 64], int turn, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int up = wave_scan(x, lane);
  if (lane == 63) waves[turn & 1][wave] = up;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    const int y = waves[turn & 1][w];
    if (w < wave) before += y;
    total += y;
  }
  return before + up - x;
}

__global__ __launch_bounds__(1024) void reorder_plan_kernel(const reorder_args a) {
  __shared__ int waves[2][16];
  __shared__ int lens[1024], parents[1024], fresh[1024];
  __shared__ uint32_t faults;
  const int bs = 1 << a.log2_bs, K = a.beams, tid = threadIdx.x, each = 1024 / K * K;   // rows of whole requests
  const int room = a.max_nb << a.log2_bs;          // positions of a table
  const int have = a.num_free_in[0];
  if (tid == 0) faults = 0, a.head[2] = 0;
  int base = 0, turn = 0;
  for (int i0 = 0; i0 < a.rows; i0 += each, ++turn) {
    const int i = i0 + tid;
    const bool mine = tid < each && i < a.rows;
    const int p = mine ? a.parents[i] : -1, old = mine ? a.lens_in[i] : 0;
    __syncthreads();                               // (the round before has been read)
    lens[tid] = old;
    parents[tid] = p;
    {                                              // free block number base + tid of the step
      const int at = have - 1 - base - tid, id = a.free_blocks[min(max(at, 0), a.num_blocks - 1)];
      fresh[tid] = id < 0 || id >= a.num_blocks ? 0 : id;
    }
    __syncthreads();
    uint32_t bad = old < 0 || old > room ? TB_TABLES_BAD_LENGTH : 0;
    bool copy = false;
    int src = -1, ctx = 0, open = -1;
    if (mine && (p < -1 || p >= K)) bad |= TB_TABLES_BAD_PARENT;
    else if (p >= 0) {
      const int g0 = tid / K * K;
      ctx = lens[g0 + p];
      if (ctx < 0 || ctx > room) ctx = 0;   // (its own row says so)
      if (ctx > 0) src = i0 + g0 + p;
      if (ctx & (bs - 1)) {
        open = a.tables[(int64_t)src * a.max_nb + (ctx >> a.log2_bs)];
        if (open < 0 || open >= a.num_blocks) {
          bad |= TB_TABLES_BAD_LENGTH;
        } else {
          const int held = a.refs[open];
          bool first = true;
          for (int k = g0; k < tid; ++k) first &= parents[k] != p;
          copy = !(first && held == 1);
        }
      }
    }
    if (bad) atomicOr(&faults, bad);
    int total;
    const int at = group_scan<1024>(copy, waves, turn, total);
    if (mine) {
      a.plan[i] = make_int4(src, ctx, copy ? fresh[at] : -1, old);
      if (copy) a.copies[base + at] = make_int4(open, fresh[at], ctx & (bs - 1), i);
    }
    // the whole blocks that every live row of a request has: an upper bound of those they share
    __syncthreads();
    lens[tid] = ctx;
    __syncthreads();
    if (tid < each / K && i0 + tid * K < a.rows) {
      int least = INT32_MAX;
      for (int k = 0; k < K; ++k) {
        const int len = lens[tid * K + k];
        if (len > 0) least = min(least, len >> a.log2_bs);
      }
      a.least[i0 / K + tid] = least == INT32_MAX ? 0 : least;
    }
    base += total;
  }
  __syncthreads();
  const uint32_t bad = faults | (base > have ? TB_TABLES_OUT_OF_BLOCKS : 0);
  if (tid == 0) {
    a.head[0] = bad != 0;
    a.head[1] = base;
    if (bad) atomicOr(a.status, bad);
  }
  if (bad) return;
  for (int i = tid; i < base; i += 1024) a.refs[a.copies[i].y] = 1;
  for (int g = tid; g < a.rows / K; g += 1024) a.shared[g] = a.least[g];
}

// The positions of an open block, all layers, K and V of every head: runs of n * row_bytes bytes, `unit_pairs` of
// them a unit. Every thread has its loads under way before its first store.
__device__ __forceinline__ void reorder_copy(const reorder_args& a, int unit, int copies) {
  constexpr int AHEAD = 4;
  const int part = unit % a.parts, at = unit / a.parts, layer = at / copies, c = at - layer * copies;
  const int4 rec = a.copies[c];
  const int bs_bytes = a.row_bytes << a.log2_bs, first = part * a.unit_pairs;
  const int64_t block_bytes = (int64_t)a.pairs * bs_bytes, in = (int64_t)first * bs_bytes;
  const char* const from = a.storage + layer * a.layer_bytes + rec.x * block_bytes + in;
  char* const to = a.storage + layer * a.layer_bytes + rec.y * block_bytes + in;
  const int run = rec.z * a.row_bytes / 16, all = run * min(a.unit_pairs, a.pairs - first);
  for (int v0 = threadIdx.x; v0 < all; v0 += AHEAD * REORDER_COLUMNS) {
    vec16 x[AHEAD];
    int off[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int v = min(v0 + u * REORDER_COLUMNS, all - 1), pair = v / run;   // (past the end: the last vector again)
      off[u] = pair * bs_bytes + (v - pair * run) * 16;
      x[u] = ld16(from + off[u]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (v0 + u * REORDER_COLUMNS < all) st16_through(to + off[u], x[u]);
  }
}

// The blocks of the lists that nobody holds, each once, behind the free blocks: by the workgroup whose counts and list
// were the last. A block may have several entries (rows that are not neighbours, requests that shared it); the first one
// counts: up to 512 entries by a hash table in LDS, more by marks in the counts, in two passes.
struct free_lds {
  static constexpr int N = REORDER_COLUMNS, MOST = 4 * N, SLOTS = 1024, NONE = -1;
  int waves[2][N / 64], starts[MOST], seen[SLOTS], first[SLOTS];   // blocks by hash, the first entry of each
};
__device__ __forceinline__ int32_t free_load(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
struct free_lists {
  static constexpr int N = free_lds::N;
  const reorder_args& a;
  free_lds& s;
  int turn, span;                                  // span: of `starts`
  // the running sums of EACH * N lists from l0 on into starts, and the whole
  template <int EACH>
  __device__ __forceinline__ int count(int l0, int lists) {
    const int tid = threadIdx.x;
    int mine[EACH], sum = 0, total;
#pragma unroll
    for (int u = 0; u < EACH; ++u) mine[u] = l0 + EACH * tid + u < lists ? free_load(&a.gone_count[l0 + EACH * tid + u]) : 0;
#pragma unroll
    for (int u = 0; u < EACH; ++u) sum += mine[u];
    __syncthreads();                               // starts has been read
    int at = group_scan<N>(sum, s.waves, turn++, total);
#pragma unroll
    for (int u = 0; u < EACH; ++u) s.starts[EACH * tid + u] = at, at += mine[u];
    span = EACH * N;
    __syncthreads();
    return total;
  }
  // entries x of the lists, several searches side by side
  template <int EACH>
  __device__ __forceinline__ void entries(int l0, const int (&x)[EACH], int total, int32_t (&id)[EACH]) const {
    int lo[EACH] = {};
    for (int step = span / 2; step; step /= 2)
#pragma unroll
      for (int u = 0; u < EACH; ++u) lo[u] += s.starts[lo[u] + step] <= x[u] ? step : 0;
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      id[u] = free_lds::NONE;
      if (x[u] < total) id[u] = free_load(&a.gone[(int64_t)(l0 + lo[u]) * N * a.beams + x[u] - s.starts[lo[u]]]);
    }
  }
  template <int EACH>
  __device__ __forceinline__ void counts(const int32_t (&id)[EACH], int32_t (&refs)[EACH]) const {
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      refs[u] = 1;
      if (id[u] != free_lds::NONE) refs[u] = free_load(&a.refs[id[u]]);
    }
  }
  // this thread's blocks that are free behind the free ones; how many all have
  template <int EACH>
  __device__ __forceinline__ int push(int from, const bool (&free)[EACH], const int32_t (&id)[EACH]) {
    int n = 0, won;
#pragma unroll
    for (int u = 0; u < EACH; ++u) n += free[u];
    int at = from + group_scan<N>(n, s.waves, turn++, won);
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      if (free[u] && at < a.num_blocks) a.free_blocks[at] = id[u];
      at += free[u];
    }
    return won;
  }
  // up to EACH * N entries at once: how many are free
  template <int EACH>
  __device__ __forceinline__ int few(int from, int total) {
    const int tid = threadIdx.x;
    for (int i = tid; i < free_lds::SLOTS; i += N) s.seen[i] = free_lds::NONE, s.first[i] = INT32_MAX;
    int x[EACH], slot[EACH];
    int32_t id[EACH], refs[EACH];
    bool free[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) x[u] = EACH * tid + u;
    entries(0, x, total, id);
    counts(id, refs);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      slot[u] = (uint32_t)id[u] * 2654435761u >> 22;
      if (refs[u] != 0) continue;
      for (;; slot[u] = (slot[u] + 1) % free_lds::SLOTS) {   // (half of them at most)
        const int was = atomicCAS(&s.seen[slot[u]], free_lds::NONE, id[u]);
        if (was == free_lds::NONE || was == id[u]) break;
      }
      atomicMin(&s.first[slot[u]], x[u]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < EACH; ++u) free[u] = refs[u] == 0 && s.first[slot[u]] == x[u];
    return push(from, free, id);
  }
};
__device__ void reorder_free(const reorder_args& a, int lists) {
  constexpr int N = free_lds::N;
  __shared__ free_lds s;
  const int tid = threadIdx.x, left = a.num_free_in[0] - a.head[1];
  free_lists all{a, s, 0, N};
  int total = 4 * N + 1, freed = 0;
  if (lists <= N) total = all.count<1>(0, lists);
  else if (lists <= 4 * N) total = all.count<4>(0, lists);
  if (total <= N) {
    freed = all.few<1>(left, total);
  } else if (total <= 4 * N) {
    freed = all.few<4>(left, total);
  } else {
    for (int pass = 0; pass < 2; ++pass) {         // the first entry of a block marks it; the marks are read
      int before = 0;
      for (int l0 = 0; l0 < lists; l0 += N) {
        total = all.count<1>(l0, lists);
        for (int x0 = 0; x0 < total; x0 += N) {
          const int x[1] = {x0 + tid}, mark = before + x[0] - MARK;
          int32_t id[1], refs[1];
          all.entries(l0, x, total, id);
          all.counts(id, refs);
          const bool free[1] = {refs[0] == mark};
          if (pass == 0) {
            if (refs[0] <= 0) atomicMin(&a.refs[id[0]], mark);
          } else {
            freed += all.push(left + freed, free, id);
            if (free[0]) __hip_atomic_store(&a.refs[id[0]], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
        }
        before += total;
      }
      __threadfence();
      __syncthreads();
    }
  }
  if (tid == 0) a.num_free_out[0] = left + freed;
}

__global__ __launch_bounds__(REORDER_COLUMNS) void reorder_tables_kernel(const reorder_args a, int table_groups) {
  // (aligned: the plan and the holds are read 16 bytes at a time, and 512 K bytes of entries keep them there)
  extern __shared__ __align__(16) int32_t lds[];   // old entries [beams][128], the plan [beams], what rows hold [beams]
  if (a.head[0]) return;
  if ((int)blockIdx.x >= table_groups) {
    const int copies = a.head[1], stride = gridDim.x - table_groups;
    for (int u = blockIdx.x - table_groups; u < copies * a.layers * a.parts; u += stride) reorder_copy(a, u, copies);
    return;
  }
  __shared__ int waves[2][REORDER_COLUMNS / 64];
  __shared__ int differ, arrived;
  const int K = a.beams, g = blockIdx.x / a.chunks, chunk = blockIdx.x - g * a.chunks, row0 = g * K;
  const int tid = threadIdx.x, j = REORDER_COLUMNS * chunk + tid, bs = 1 << a.log2_bs;
  int32_t* const old = lds + tid;                  // [k * 128]
  int4* const plan = (int4*)(lds + REORDER_COLUMNS * K);
  int4* const holds = plan + K;                    // {whole blocks, blocks, children - 1, -1 unless a child keeps the open block}
  if (tid < K) {
    const int4 p = a.plan[row0 + tid];
    plan[tid] = p;
    holds[tid] = make_int4(p.w >> a.log2_bs, (p.w + bs - 1) >> a.log2_bs, -1, -1);
  }
  if (tid == 0) differ = INT32_MAX;
  // (columns are loaded before the request's width is known; the tables have them all)
  for (int k0 = 0; k0 < K; k0 += 8) {
    int32_t e[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) e[u] = a.tables[(int64_t)(row0 + min(k0 + u, K - 1)) * a.max_nb + min(j, a.max_nb - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (k0 + u < K) old[REORDER_COLUMNS * (k0 + u)] = e[u];
  }
  __syncthreads();
  if (tid < K) {
    const int4 p = plan[tid];
    if (chunk == 0) a.lens_out[row0 + tid] = p.y;
    if (p.x >= 0) {
      atomicAdd(&holds[p.x - row0].z, 1);
      if (p.z < 0) atomicMax(&holds[p.x - row0].w, 0);
    }
  }
  __syncthreads();
  // what every old row's hold on its block of this column becomes, rows of one block behind each other at once
  int width = 0;                                   // columns that the request's old tables hold
  uint64_t lost = 0;                               // rows that begin a run that lets go
  {
    int id = -1, from = 0, sum = 0;
    auto end = [&] {
      if (sum != 0 && id >= 0 && id < a.num_blocks) {
        atomicAdd(&a.refs[id], sum);
        if (sum < 0) lost |= (uint64_t)1 << from;
      }
    };
#pragma unroll 4
    for (int k = 0; k < K; ++k) {
      const int4 h = holds[k];
      const int next = j < h.y ? old[REORDER_COLUMNS * k] : -1;
      width = max(width, h.y);
      if (next != id) {
        end();
        id = next, from = k, sum = 0;
      }
      sum += j < h.x ? h.z : j < h.y ? h.w : 0;
    }
    end();
  }
  int total;
  int at = group_scan<REORDER_COLUMNS>(__popcll(lost), waves, 0, total);
  int32_t* const list = a.gone + (int64_t)blockIdx.x * REORDER_COLUMNS * K;
  for (uint64_t left = lost; left; left &= left - 1) {
    const int k = __ffsll((unsigned long long)left) - 1;
    __hip_atomic_store(&list[at++], old[REORDER_COLUMNS * k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (tid == 0) __hip_atomic_store(&a.gone_count[blockIdx.x], total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wave's list and counts are in memory
  __syncthreads();
  int place = 0;
  if (tid == 0) place = __hip_atomic_fetch_add(&a.head[2], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // the new tables, and whether the live rows agree in this column
  if (j < width) {
    int one = -1;
    bool same = true, all = true;                  // all: a whole block of every live row
#pragma unroll 4
    for (int k = 0; k < K; ++k) {
      const int4 p = plan[k];
      int id = old[REORDER_COLUMNS * max(p.x - row0, 0)];
      if (p.z >= 0 && j == p.y >> a.log2_bs) id = p.z;
      if (j >= (p.y + bs - 1) >> a.log2_bs) id = -1;
      a.tables[(int64_t)(row0 + k) * a.max_nb + j] = id;
      if (p.y > 0) {
        all &= j < p.y >> a.log2_bs;
        same &= one < 0 || one == id;
        one = id;
      }
    }
    if (all && !same) atomicMin(&differ, j);
  }
  if (tid == 0) arrived = place;
  __syncthreads();
  if (tid == 0 && differ != INT32_MAX) atomicMin(&a.shared[g], differ);
  if (arrived == table_groups - 1) reorder_free(a, table_groups);
}

struct reorder_sizes {
  int64_t plan, copies, least, count, gone, all, chunks;
  reorder_sizes(int64_t rows, int64_t beams, int64_t max_nb) {
    chunks = (max_nb + REORDER_COLUMNS - 1) / REORDER_COLUMNS;
    const int64_t lists = rows / beams * chunks;
    plan = 64;
    copies = plan + 16 * rows;
    least = copies + 16 * rows;
    count = least + 4 * (rows / beams);
    gone = count + 4 * lists;
    all = gone + 4 * lists * REORDER_COLUMNS * beams;
  }
};

}  // namespace tb

extern "C" size_t tb_beam_reorder_workspace_bytes(int32_t num_rows, int32_t beams, int32_t max_blocks_per_row) {
  if (num_rows <= 0 || beams <= 0 || max_blocks_per_row <= 0) return 64;
  return (size_t)tb::reorder_sizes(num_rows, beams, max_blocks_per_row).all;
}

extern "C" int32_t tb_beam_reorder(void* storage, int32_t num_layers, int64_t layer_stride_bytes, int32_t num_blocks,
                                   int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t dtype,
                                   int32_t* block_tables, int32_t max_blocks_per_row, int32_t num_rows, int32_t beams,
                                   const int32_t* lens_in, int32_t* lens_out, int32_t* ref_counts,
                                   int32_t* free_blocks, const int32_t* num_free_in, int32_t* num_free_out,
                                   int32_t* shared_blocks, const int32_t* parents, uint32_t* status, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_rows >= 0 && beams > 0 && beams <= TB_BEAMS_MAX && num_rows % beams == 0);
  TB_CHECK_ARG(max_blocks_per_row > 0 && num_blocks > 0 && num_layers >= 0 && num_layers <= 65535);
  TB_CHECK_ARG(block_size > 0 && (block_size & (block_size - 1)) == 0);
  TB_CHECK_ARG((int64_t)num_blocks * block_size < ((int64_t)1 << 31));
  TB_CHECK_ARG((int64_t)max_blocks_per_row * block_size < ((int64_t)1 << 31));
  if (num_rows == 0) return TB_OK;
  const reorder_sizes z(num_rows, beams, max_blocks_per_row);
  TB_CHECK_ARG((int64_t)num_rows * z.chunks * REORDER_COLUMNS < MARK);
  TB_CHECK_ARG(block_tables && lens_in && lens_out && ref_counts && free_blocks && num_free_in && num_free_out &&
               shared_blocks && parents && status && workspace);
  TB_CHECK_ARG(workspace_bytes >= (size_t)z.all && ((uintptr_t)workspace & 15u) == 0);
  reorder_args a = {};
  if (num_layers > 0) {
    TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16 && num_kv_heads > 0 && head_dim > 0);
    const int64_t row = (int64_t)head_dim * (dtype == TB_DTYPE_F32 ? 4 : 2);
    if (row % 16) return TB_ERR_UNSUPPORTED;
    const int64_t block = 2 * (int64_t)num_kv_heads * block_size * row;
    TB_CHECK_ARG(block < ((int64_t)1 << 31));
    TB_CHECK_ARG(storage && ((uintptr_t)storage & 15u) == 0 && layer_stride_bytes % 16 == 0);
    TB_CHECK_ARG(num_layers == 1 || layer_stride_bytes >= num_blocks * block);
    a.pairs = 2 * num_kv_heads, a.row_bytes = (int32_t)row;
    // units of some 512 vectors: half a block's positions on average
    const int64_t vectors = block_size * row / 32;
    a.unit_pairs = (int32_t)(vectors >= 512 ? 1 : vectors < 1 ? a.pairs : 512 / vectors);
    if (a.unit_pairs > a.pairs) a.unit_pairs = a.pairs;
    a.parts = (a.pairs + a.unit_pairs - 1) / a.unit_pairs;
    TB_CHECK_ARG((int64_t)num_layers * num_rows * a.parts < ((int64_t)1 << 31));
  }
  a.storage = (char*)storage, a.layer_bytes = layer_stride_bytes, a.layers = num_layers, a.num_blocks = num_blocks;
  a.log2_bs = __builtin_ctz((unsigned)block_size);
  a.tables = block_tables, a.max_nb = max_blocks_per_row, a.rows = num_rows, a.beams = beams;
  a.lens_in = lens_in, a.lens_out = lens_out, a.refs = ref_counts, a.free_blocks = free_blocks;
  a.num_free_in = num_free_in, a.num_free_out = num_free_out, a.shared = shared_blocks, a.parents = parents;
  a.status = status;
  char* const ws = (char*)workspace;
  a.head = (int32_t*)ws, a.plan = (int4*)(ws + z.plan), a.copies = (int4*)(ws + z.copies);
  a.least = (int32_t*)(ws + z.least), a.gone_count = (int32_t*)(ws + z.count), a.gone = (int32_t*)(ws + z.gone), a.chunks = (int32_t)z.chunks;
  const int lists = (int)(num_rows / beams * z.chunks);
  const int64_t units = (int64_t)num_rows * num_layers * a.parts;
  const int movers = (int)(units < 1024 ? units : 1024);
  const size_t lds = sizeof(int32_t) * (REORDER_COLUMNS + 8) * (size_t)beams;
  hipLaunchKernelGGL(reorder_plan_kernel, dim3(1), dim3(1024), 0, stream, a);
  hipLaunchKernelGGL(reorder_tables_kernel, dim3(lists + movers), dim3(REORDER_COLUMNS), lds, stream, a, lists);
  TB_RETURN_LAUNCH_STATUS();
}
