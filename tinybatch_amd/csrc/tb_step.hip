// A step's arrays built on the GPU from the rows' lengths: blocks taken from the free blocks,
// block tables, positions, slots, and the work items of tb_paged_attention.
//
// Row b has c = cached[b] positions and n = new_lens[b] new tokens, so that (bs the block size)
//   have = ceil(c / bs), need = ceil((c + n) / bs) blocks; the need - have new ones are the next of the
//   free blocks, taken from the end, rows in order: number x of the step is free[num_free - 1 - x];
//   token i of row b lies at position p = c + i, in slot table[p / bs] bs + p mod bs, and sees p + 1 positions.
// Work items (partitions of P positions, up to `group` rows of one partition count an item): with
//   F(m) = sum_{k=1..m} ceil(k / P) = P a (a + 1) / 2 + r (a + 1), a = m / P, r = m mod P,
// the partitions of a row's first i tokens are F(c + i) - F(c), and its items and rows of several partitions have
// closed forms too. Five running sums over the rows are therefore all that the step's parts need of each
// other: every workgroup makes them itself (rows in LDS, 256 at a time), and then writes its own tokens. Nothing that is
// read here is written here (new blocks are read from the free blocks, not from the tables),
// so that one launch does, and a step that is built again gives the same arrays.
// A row without positions that gets tokens has no block in common with the other rows of its request, which shared theirs
// without it: shared[b / beams] = 0.
//
// What bounds it: the launch and a chain of dependent loads (lengths, the sums, a free block): 256 rows of one token 8.1 us a call,
// 300 rows of up to 100 tokens each with their work items 10.0, where the smallest of launches takes 4.
// More than STEP_LDS_ROWS rows: the sums by a launch of one workgroup before it, through the workspace, whose passes over the rows come
// one behind the other (from a graph, one token a row, without and with work items: 1024 rows 8.3 and 14.0 us, 1025 16.5 and 23.8,
// 2600 21.9 and 33.7, 8000 48 and 80; its sums take more registers than 1024 threads have, 41 of them lie in memory).
#include "tb_common.h"

namespace tb {

constexpr int STEP_THREADS = 256;
constexpr int STEP_LDS_ROWS = 1024;
constexpr int64_t STEP_MOST = 1 << 24;             // of every capacity: a wave's sums stay within 32 bits
constexpr int STEP_SUMS = 5;                       // tokens, blocks, partitions, items, rows of several partitions
enum { S_TOK, S_BLK, S_PART, S_ITEM, S_SPLIT };

struct step_args {
  int32_t* block_tables;       // [rows][max_nb]
  int32_t max_nb;
  const int32_t* cached;       // [rows]
  const int32_t* new_lens;     // [rows]
  int32_t rows;
  int32_t* shared;             // [rows / beams] or null
  int32_t beams;
  int32_t* refs;               // [num_blocks]
  const int32_t* free_blocks;  // [num_blocks]
  const int32_t* num_free;     // [1]
  int32_t num_blocks, log2_bs;
  int32_t pad;                 // > 0: row b's tokens from flat row b * pad on
  int32_t max_tokens;          // flat rows
  int32_t P, group, max_items, max_parts, max_split;   // P = 0: no work items
  int32_t* lens;               // [rows]
  int32_t* num_free_out;       // [1]
  int32_t* starts;             // [rows + 1]
  int64_t* positions;          // [max_tokens]
  int32_t* slots;              // [max_tokens]
  int32_t* row_ctx;            // [max_tokens]
  int32_t* offsets;            // [max_tokens + 1]
  int4* items;                 // [max_items]
  int4* split;                 // [max_split]
  int32_t* counts;             // [4]
  uint32_t* status;
  int32_t* sums;               // [STEP_SUMS][rows + 1] and the faults, where a launch made them before
};

// (lengths are below 2^31: divisions in 32 bits)
__device__ __forceinline__ int64_t step_parts(uint32_t m, uint32_t P) {   // F(m)
  const uint32_t a = m / P, r = m - a * P;
  return (int64_t)P * ((int64_t)a * (a + 1) / 2) + (int64_t)r * (a + 1);
}
// Items of a row's first n tokens behind c positions, n at the end of an item.
__device__ __forceinline__ int64_t step_items(uint32_t c, uint32_t n, uint32_t P, uint32_t group) {
  if (n == 0) return 0;
  auto some = [&](uint32_t rows) { return (int64_t)((rows + group - 1) / group); };
  const uint32_t n0 = c / P + 1, n1 = (c + n - 1) / P + 1;    // partitions of the first and the last token
  if (n0 == n1) return n0 * some(n);
  const int64_t between = (int64_t)(n0 + n1) * (n1 - n0 - 1) / 2;   // n0 + 1 + .. + n1 - 1
  return n0 * some(n0 * P - c) + between * some(P) + n1 * some(c + n - (n1 - 1) * P);
}

struct step_row {
  int32_t v[STEP_SUMS];
  uint32_t bad;
};
__device__ __forceinline__ step_row step_look(const step_args& a, int b) {
  step_row r;
#pragma unroll
  for (int k = 0; k < STEP_SUMS; ++k) r.v[k] = 0;
  r.bad = 0;
  const int64_t c = a.cached[b], n = a.new_lens[b], bs = (int64_t)1 << a.log2_bs;
  if (c < 0 || n < 0) {
    r.bad = TB_TABLES_BAD_LENGTH;
    return r;
  }
  const int64_t have = (c + bs - 1) >> a.log2_bs, need = (c + n + bs - 1) >> a.log2_bs;
  if (need > a.max_nb) r.bad |= TB_TABLES_ROW_FULL;
  if (n > (a.pad ? a.pad : a.max_tokens)) r.bad |= TB_TABLES_TOO_MANY_TOKENS;
  if (r.bad) return r;
  r.v[S_TOK] = (int32_t)n;
  r.v[S_BLK] = (int32_t)(need - have);
  if (a.P) {
    const int64_t parts = step_parts(c + n, a.P) - step_parts(c, a.P), items = step_items(c, n, a.P, a.group);
    if (parts > a.max_parts || items > a.max_items) {
      r.bad = TB_TABLES_TOO_MUCH_WORK;
      return r;
    }
    r.v[S_PART] = (int32_t)parts;
    r.v[S_ITEM] = (int32_t)items;
    const int64_t split = c + n - max(c, (int64_t)a.P);
    r.v[S_SPLIT] = (int32_t)max(split, (int64_t)0);           // at most n
  }
  return r;
}

// The running sums of the rows into sums[STEP_SUMS][rows + 1]; the step's faults.
template <int THREADS>
__device__ uint32_t step_scan(const step_args& a, int32_t* sums) {
  constexpr int WAVES = THREADS / 64;
  __shared__ int32_t waves[2][WAVES][STEP_SUMS];
  __shared__ uint32_t faults;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) faults = 0;
  int64_t base[STEP_SUMS] = {0, 0, 0, 0, 0};
  const int K = a.P ? STEP_SUMS : 2, stride = a.rows + 1;
  __syncthreads();
  for (int b0 = 0, turn = 0; b0 < a.rows; b0 += THREADS, turn ^= 1) {
    const int b = b0 + threadIdx.x;
    step_row r = {};
    if (b < a.rows) r = step_look(a, b);
    if (r.bad) atomicOr(&faults, r.bad);
    int32_t up[STEP_SUMS];
#pragma unroll
    for (int k = 0; k < STEP_SUMS; ++k) {
      up[k] = r.v[k];
      if (k < K) {
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
          const int32_t y = __shfl_up(up[k], o);
          if (lane >= o) up[k] += y;
        }
        if (lane == 63) waves[turn][wave][k] = up[k];
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < STEP_SUMS; ++k) {
      if (k >= K) continue;
      int64_t before = base[k];
      for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += waves[turn][w][k];
        base[k] += waves[turn][w][k];
      }
      // (past what the host allows the sums stop counting: the step is refused)
      if (b < a.rows) sums[k * stride + b] = (int32_t)min(before + up[k] - r.v[k], (int64_t)INT32_MAX);
    }
  }
  uint32_t bad = 0;
  if (base[S_BLK] > a.num_free[0]) bad |= TB_TABLES_OUT_OF_BLOCKS;
  if (!a.pad && base[S_TOK] > a.max_tokens) bad |= TB_TABLES_TOO_MANY_TOKENS;
  if (base[S_PART] > a.max_parts || base[S_ITEM] > a.max_items || base[S_SPLIT] > a.max_split)
    bad |= a.P ? TB_TABLES_TOO_MUCH_WORK : 0;
  if (threadIdx.x < (unsigned)K) {
    int64_t total = base[0];
#pragma unroll
    for (int k = 1; k < STEP_SUMS; ++k)
      if ((int)threadIdx.x == k) total = base[k];
    sums[threadIdx.x * stride + a.rows] = (int32_t)min(total, (int64_t)INT32_MAX);
  }
  __syncthreads();
  return bad | faults;
}

// The row that number x of a running sum belongs to: the last one that starts at or before x.
__device__ __forceinline__ int step_find(const int32_t* starts, int rows, int x) {
  int lo = 0, hi = rows;                           // starts[lo] <= x < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(1024) void step_sums_kernel(const step_args a) {
  const uint32_t bad = step_scan<1024>(a, a.sums);
  if (threadIdx.x == 0) a.sums[STEP_SUMS * (a.rows + 1)] = (int32_t)bad;
}

template <bool LARGE>
__global__ __launch_bounds__(STEP_THREADS) void step_fill_kernel(const step_args a) {
  __shared__ int32_t lds[LARGE ? 1 : STEP_SUMS * (STEP_LDS_ROWS + 1)];
  uint32_t bad;
  const int32_t* sums;
  if constexpr (LARGE) {
    sums = a.sums;
    bad = (uint32_t)a.sums[STEP_SUMS * (a.rows + 1)];
  } else {
    bad = step_scan<STEP_THREADS>(a, lds);
    sums = lds;
  }
  const int stride = a.rows + 1, first = blockIdx.x * STEP_THREADS + threadIdx.x, all = gridDim.x * STEP_THREADS;
  const int32_t* const tok = sums + S_TOK * stride;
  const int32_t* const blk = sums + S_BLK * stride;
  const int32_t* const part = sums + S_PART * stride;
  const int free_end = a.num_free[0] - 1, bs = 1 << a.log2_bs;
  auto taken = [&](int x) {                        // block number x of the step
    const int at = free_end - x, id = a.free_blocks[at < 0 ? 0 : min(at, a.num_blocks - 1)];
    return id < 0 || id >= a.num_blocks ? 0 : id;  // stay inside the pool, whatever the caller's list holds
  };
  if (first == 0) {
    if (bad) atomicOr(a.status, bad);
    a.num_free_out[0] = a.num_free[0] - (bad ? 0 : blk[a.rows]);
    if (a.counts) {
      a.counts[0] = bad ? 0 : sums[S_ITEM * stride + a.rows];
      a.counts[1] = bad ? 0 : sums[S_SPLIT * stride + a.rows];
      a.counts[2] = 0;
      a.counts[3] = bad ? 0 : part[a.rows];
    }
  }
  for (int b = first; b <= a.rows; b += all) {
    a.starts[b] = a.pad ? b * a.pad : bad ? 0 : tok[b];
    if (b < a.rows) {
      const int c = a.cached[b], n = bad ? 0 : a.new_lens[b];
      a.lens[b] = c + n;
      if (a.shared && c == 0 && n > 0) a.shared[b / a.beams] = 0;
    }
  }
  if (!bad)
    for (int x = first; x < blk[a.rows]; x += all) {
      const int b = step_find(blk, a.rows, x), id = taken(x);
      const int have = (a.cached[b] + bs - 1) >> a.log2_bs;
      a.block_tables[(int64_t)b * a.max_nb + have + x - blk[b]] = id;
      a.refs[id] = 1;
    }
  for (int t = first; t < a.max_tokens + (a.P ? 1 : 0); t += all) {
    int b = 0, i = 0;
    bool inside = !bad && t < a.max_tokens;
    if (inside && a.pad) {
      b = t / a.pad;
      i = t - b * a.pad;
      inside = i < a.new_lens[b];
    } else if (inside) {
      inside = t < tok[a.rows];
      b = inside ? step_find(tok, a.rows, t) : 0;
      i = t - tok[b];
    }
    const int c = inside ? a.cached[b] : 0, pos = c + i;
    if (t < a.max_tokens) {
      int slot = -1;
      if (inside) {
        const int j = pos >> a.log2_bs, have = (c + bs - 1) >> a.log2_bs;
        const int id = j >= have ? taken(blk[b] + j - have) : a.block_tables[(int64_t)b * a.max_nb + j];
        slot = (id << a.log2_bs) + (pos & (bs - 1));
      }
      a.slots[t] = slot;
      a.positions[t] = inside ? pos : 0;
      a.row_ctx[t] = inside ? pos + 1 : 0;
    }
    if (!a.P) continue;
    // partitions before this flat row; a row outside counts none
    int64_t before = bad ? 0 : part[a.rows];
    if (!bad && a.pad && t < a.max_tokens && !inside) before = part[b + 1];
    if (inside) before = part[b] + (step_parts(c + i, a.P) - step_parts(c, a.P));
    a.offsets[t] = (int32_t)before;
    if (!inside) continue;
    const int n = a.new_lens[b], np = pos / a.P + 1;
    if (np > 1)
      a.split[sums[S_SPLIT * stride + b] + pos - max(c, a.P)] = make_int4(t, (int)before, np, 0);
    const int since = max(0, (np - 1) * a.P - c);  // the row's first token of this many partitions
    if ((i - since) % a.group == 0) {
      const int size = min(min(a.group, n - i), np * a.P - pos);
      const int64_t at = sums[S_ITEM * stride + b] + step_items(c, i, a.P, a.group);
      for (int p = 0; p < np; ++p) a.items[at + p] = make_int4(t, b, p | (size - 1) << 24, pos + 1);
    }
  }
}

}  // namespace tb

extern "C" size_t tb_device_step_workspace_bytes(int32_t num_rows) {
  return num_rows > tb::STEP_LDS_ROWS ? ((size_t)tb::STEP_SUMS * ((size_t)num_rows + 1) + 1) * 4 : 0;
}

static int32_t device_step(int32_t* block_tables, int32_t max_blocks_per_row, const int32_t* cached_lens,
                           const int32_t* new_lens, int32_t num_rows, int32_t* shared_blocks, int32_t beams,
                           int32_t* ref_counts, const int32_t* free_blocks, const int32_t* num_free, int32_t num_blocks,
                           int32_t block_size, int32_t pad_tokens, int32_t max_tokens,
                           int32_t* context_lens, int32_t* num_free_out, int32_t* query_start_loc,
                           int64_t* positions, int32_t* slot_mapping, int32_t* row_ctx,
                           int32_t partition_tokens, int32_t rows_per_item, int32_t* row_part_offsets,
                           int32_t* work_items, int32_t max_items, int32_t max_partitions,
                           int32_t* split_rows, int32_t max_split_rows, int32_t* counts, uint32_t* status,
                           void* workspace, size_t workspace_bytes, hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_rows >= 0 && num_rows < STEP_MOST && max_blocks_per_row > 0 && num_blocks > 0);
  TB_CHECK_ARG(block_size > 0 && (block_size & (block_size - 1)) == 0);
  TB_CHECK_ARG((int64_t)num_blocks * block_size < ((int64_t)1 << 31));
  TB_CHECK_ARG((int64_t)max_blocks_per_row * block_size < ((int64_t)1 << 31) && max_blocks_per_row <= STEP_MOST);
  TB_CHECK_ARG(max_tokens >= 0 && max_tokens < STEP_MOST && pad_tokens >= 0);
  TB_CHECK_ARG(pad_tokens == 0 || (int64_t)pad_tokens * num_rows == max_tokens);
  TB_CHECK_ARG(num_free && num_free_out && query_start_loc && status && num_free != num_free_out);
  TB_CHECK_ARG(num_rows == 0 || (block_tables && cached_lens && new_lens && ref_counts && free_blocks && context_lens));
  TB_CHECK_ARG(cached_lens == nullptr || cached_lens != context_lens);
  TB_CHECK_ARG(max_tokens == 0 || (positions && slot_mapping && row_ctx));
  if (partition_tokens) {
    TB_CHECK_ARG(partition_tokens > 0 && rows_per_item >= 1 && rows_per_item <= 16);
    TB_CHECK_ARG(max_items >= 0 && max_items < STEP_MOST && max_partitions >= 0 && max_partitions < STEP_MOST);
    TB_CHECK_ARG(max_split_rows >= 0 && max_split_rows < STEP_MOST);
    TB_CHECK_ARG(row_part_offsets && counts && (max_items == 0 || work_items) && (max_split_rows == 0 || split_rows));
    TB_CHECK_ARG((((uintptr_t)work_items | (uintptr_t)split_rows) & 15u) == 0);
  }
  const size_t need = tb_device_step_workspace_bytes(num_rows);
  TB_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 3u) == 0));
  step_args a;
  a.block_tables = block_tables, a.max_nb = max_blocks_per_row, a.cached = cached_lens, a.new_lens = new_lens;
  a.rows = num_rows, a.shared = shared_blocks, a.beams = beams, a.refs = ref_counts, a.free_blocks = free_blocks, a.num_free = num_free;
  a.num_blocks = num_blocks, a.log2_bs = __builtin_ctz((unsigned)block_size);
  a.pad = pad_tokens, a.max_tokens = max_tokens;
  a.P = partition_tokens, a.group = rows_per_item, a.max_items = max_items, a.max_parts = max_partitions;
  a.max_split = max_split_rows;
  a.lens = context_lens, a.num_free_out = num_free_out, a.starts = query_start_loc, a.positions = positions;
  a.slots = slot_mapping, a.row_ctx = row_ctx, a.offsets = row_part_offsets;
  a.items = (int4*)work_items, a.split = (int4*)split_rows, a.counts = partition_tokens ? counts : nullptr;
  a.status = status, a.sums = (int32_t*)workspace;
  const int most = max_tokens > num_rows ? max_tokens : num_rows;
  const int grid = (most + STEP_THREADS) / STEP_THREADS;   // (one more than the tokens: the last offset)
  if (need) {
    hipLaunchKernelGGL(step_sums_kernel, dim3(1), dim3(1024), 0, stream, a);
    hipLaunchKernelGGL(step_fill_kernel<true>, dim3(grid < 2048 ? grid : 2048), dim3(STEP_THREADS), 0, stream, a);
  } else {
    hipLaunchKernelGGL(step_fill_kernel<false>, dim3(grid < 2048 ? grid : 2048), dim3(STEP_THREADS), 0, stream, a);
  }
  TB_RETURN_LAUNCH_STATUS();
}

extern "C" int32_t tb_device_step(int32_t* block_tables, int32_t max_blocks_per_row, const int32_t* cached_lens,
                                  const int32_t* new_lens, int32_t num_rows, int32_t* ref_counts,
                                  const int32_t* free_blocks, const int32_t* num_free, int32_t num_blocks,
                                  int32_t block_size, int32_t pad_tokens, int32_t max_tokens,
                                  int32_t* context_lens, int32_t* num_free_out, int32_t* query_start_loc,
                                  int64_t* positions, int32_t* slot_mapping, int32_t* row_ctx,
                                  int32_t partition_tokens, int32_t rows_per_item, int32_t* row_part_offsets,
                                  int32_t* work_items, int32_t max_items, int32_t max_partitions,
                                  int32_t* split_rows, int32_t max_split_rows, int32_t* counts, uint32_t* status,
                                  void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return device_step(block_tables, max_blocks_per_row, cached_lens, new_lens, num_rows, nullptr, 1, ref_counts, free_blocks,
                     num_free, num_blocks, block_size, pad_tokens, max_tokens, context_lens, num_free_out, query_start_loc,
                     positions, slot_mapping, row_ctx, partition_tokens, rows_per_item, row_part_offsets, work_items,
                     max_items, max_partitions, split_rows, max_split_rows, counts, status, workspace, workspace_bytes, stream);
}

extern "C" int32_t tb_beam_step(int32_t* block_tables, int32_t max_blocks_per_row, const int32_t* cached_lens,
                                const int32_t* new_lens, int32_t num_rows, int32_t* shared_blocks, int32_t beams,
                                int32_t* ref_counts, const int32_t* free_blocks, const int32_t* num_free,
                                int32_t num_blocks, int32_t block_size, int32_t pad_tokens, int32_t max_tokens,
                                int32_t* context_lens, int32_t* num_free_out, int32_t* query_start_loc,
                                int64_t* positions, int32_t* slot_mapping, int32_t* row_ctx,
                                int32_t partition_tokens, int32_t rows_per_item, int32_t* row_part_offsets,
                                int32_t* work_items, int32_t max_items, int32_t max_partitions,
                                int32_t* split_rows, int32_t max_split_rows, int32_t* counts, uint32_t* status,
                                void* workspace, size_t workspace_bytes, hipStream_t stream) {
  TB_CHECK_ARG(beams > 0 && beams <= TB_BEAMS_MAX && num_rows >= 0 && num_rows % beams == 0);
  TB_CHECK_ARG(num_rows == 0 || shared_blocks);
  return device_step(block_tables, max_blocks_per_row, cached_lens, new_lens, num_rows, shared_blocks, beams, ref_counts,
                     free_blocks, num_free, num_blocks, block_size, pad_tokens, max_tokens, context_lens, num_free_out,
                     query_start_loc, positions, slot_mapping, row_ctx, partition_tokens, rows_per_item, row_part_offsets,
                     work_items, max_items, max_partitions, split_rows, max_split_rows, counts, status, workspace,
                     workspace_bytes, stream);
}
