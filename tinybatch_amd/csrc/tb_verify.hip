// Verification of drafted trees and the move of what it keeps.
//
// verify: from a sequence's root on, a reached node's children are tried in the order of
// their rows; the first one kept becomes the reached node. Row r of `probs` is the target's
// distribution after node r, u[r] node r's random number in [0, 1) (the root's serves the
// token drawn at the end). With p the reached node's row and x a child's token:
//   drafts that were not drawn (no draft rows): left = 1 - sum of p over the tokens refused
//     here; x is kept where p(x) > 0 and u left < p(x), a token refused before holding 0;
//   drafts drawn from q, independently: a = 0, s = 1; x is kept where
//     u q(x) s < p(x) - a q(x); a refusal makes a += s, s = sum_i max(p_i - a q_i, 0).
//     The distribution after m refusals is norm(max(p' - q, 0)) of the one before; with
//     p' = max(p - a q, 0) / s that is max(p - (a + s) q, 0) / (its sum), since what the
//     smaller a had cut to zero the larger one cuts too.
// Then one token is drawn from what is left of the last reached node's row: the first i
// with w_0 + .. + w_i > u sum(w), w = p without the refused tokens, or max(p - a q, 0).
// Where w holds nothing, p itself is taken, and -1 where that holds nothing either; NaN entries
// and those below 0 count as 0.
// Everything is decided in 64 bits: products and differences of 32-bit inputs are then as
// good as exact, and a sum of 150000 terms does not move the border between two tokens.
#include "tb_common.h"

namespace tb {

constexpr int VERIFY_THREADS = 1024;

struct verify_args {
  const void* probs;           // [T][V]
  int64_t probs_stride;        // elements
  const void* draft;           // [T][V] or null
  int64_t draft_stride;
  int32_t vocab;
  const int64_t* tokens;       // [T]
  const float* uniforms;       // [T]
  const int32_t* parents;      // [T], inside the tree; the root's is -1
  const int32_t* row_starts;   // [B + 1]
  int32_t* accepted;           // [B][width]
  int32_t* num_accepted;       // [B]
  int64_t* out_tokens;         // [B][width]
  int32_t width;
};

__device__ __forceinline__ double sum64(double x) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x += __shfl_xor(x, o);
  return x;
}

// One workgroup per sequence: the tree in LDS, every thread walks it the same way; sums over
// the vocabulary by all threads, thread t the tokens t, t + 1024, ...
template <typename T>
__global__ __launch_bounds__(VERIFY_THREADS) void verify_kernel(const verify_args a) {
  __shared__ int32_t tok[TB_TREE_MAX_NODES], par[TB_TREE_MAX_NODES], path[TB_TREE_MAX_NODES];
  __shared__ int32_t refused[TB_TREE_MAX_NODES];
  __shared__ double part[VERIFY_THREADS / 64];
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row0 = a.row_starts[seq], n = min(a.row_starts[seq + 1] - row0, TB_TREE_MAX_NODES);
  int32_t* const acc = a.accepted + (int64_t)seq * a.width;
  int64_t* const out = a.out_tokens + (int64_t)seq * a.width;
  for (int i = tid; i < a.width; i += VERIFY_THREADS) acc[i] = -1, out[i] = -1;
  if (n <= 0) {
    if (tid == 0) a.num_accepted[seq] = 0;
    return;
  }
  for (int i = tid; i < n; i += VERIFY_THREADS) {
    const int64_t t = a.tokens[row0 + i];
    tok[i] = t >= 0 && t < a.vocab ? (int32_t)t : -1;
    par[i] = a.parents[row0 + i];
  }
  __syncthreads();

  const T *p = nullptr, *q = nullptr;
  auto at_row = [&](int node) {
    p = (const T*)a.probs + (int64_t)(row0 + node) * a.probs_stride;
    q = a.draft ? (const T*)a.draft + (int64_t)(row0 + node) * a.draft_stride : nullptr;
  };
  // what is left of token i after the refusals so far (`nref` refused tokens, or a)
  int nref = 0;
  double s = 1., ra = 0.;
  bool whole = false;
  auto weight = [&](int i) -> double {
    double w = (double)(float)p[i];
    if (whole) return w > 0. ? w : 0.;
    if (q) w -= ra * (double)(float)q[i];
    else
      for (int k = 0; k < nref; ++k)
        if (refused[k] == i) w = 0.;
    return w > 0. ? w : 0.;
  };
  auto reduce = [&](double x) -> double {          // over the workgroup
    x = sum64(x);
    __syncthreads();
    if (lane == 0) part[wave] = x;
    __syncthreads();
    double t = 0.;
    for (int w = 0; w < VERIFY_THREADS / 64; ++w) t += part[w];
    return t;
  };
  auto total = [&]() -> double {
    double x = 0.;
    for (int i = tid; i < a.vocab; i += VERIFY_THREADS) x += weight(i);
    return reduce(x);
  };

  int cur = 0, len = 1;
  at_row(0);
  if (tid == 0) path[0] = 0;
  for (int i = 1; i < n; ++i) {
    if (par[i] != cur) continue;
    const int x = tok[i];
    const double u = (double)a.uniforms[row0 + i];
    double px = x < 0 ? 0. : (double)(float)p[x];
    bool keep;
    if (q) {
      const double qx = x < 0 ? 0. : (double)(float)q[x];
      keep = u * qx * s < px - ra * qx;
    } else {
      bool again = false;
      for (int k = 0; k < nref; ++k) again |= refused[k] == x;
      if (again) px = 0.;
      keep = px > 0. && u * s < px;
      if (!keep) s -= px > 0. ? px : 0.;
    }
    if (keep) {
      cur = i;
      nref = 0, s = 1., ra = 0.;
      at_row(i);
      if (tid == 0) path[len] = i;
      ++len;
    } else if (q) {
      ra += s;
      s = total();
    } else {
      __syncthreads();
      if (tid == 0) refused[nref] = x;
      ++nref;
      __syncthreads();
    }
  }
  __syncthreads();

  // the next token: the border's place by sums of contiguous stretches
  double w = total();
  if (!(w > 0.)) {
    whole = true;
    w = total();
  }
  int next = -1;
  if (w > 0.) {
    const double border = (double)a.uniforms[row0] * w;
    int lo = 0, hi = a.vocab;
    double before = 0.;
    while (hi - lo > 1) {
      const int step = (hi - lo + VERIFY_THREADS - 1) / VERIFY_THREADS;
      const int b = min(hi, lo + tid * step), e = min(hi, b + step);
      double x = 0.;
      for (int i = b; i < e; ++i) x += weight(i);
      // sums of the threads before this one
      double run = x;
      for (int o = 1; o < 64; o *= 2) {
        const double y = __shfl_up(run, o);
        if (lane >= o) run += y;
      }
      __syncthreads();
      if (lane == 63) part[wave] = run;
      __syncthreads();
      double base = before;
      for (int v = 0; v < wave; ++v) base += part[v];
      // the first stretch whose end passes the border; the last with any weight if none does
      const bool past = x > 0. && base + run > border;
      const bool some = x > 0.;
      __shared__ int32_t first, last;
      if (tid == 0) first = VERIFY_THREADS, last = -1;
      __syncthreads();
      if (past) atomicMin(&first, tid);
      if (some) atomicMax(&last, tid);
      __syncthreads();
      const int pick = first < VERIFY_THREADS ? first : last;
      __shared__ double start;
      if (tid == pick) start = base + run - x;
      __syncthreads();
      before = start;
      lo = lo + pick * step;
      hi = min(hi, lo + step);
      __syncthreads();
    }
    next = lo;
  }
  for (int i = tid; i < min(len, a.width); i += VERIFY_THREADS) {
    acc[i] = path[i];
    out[i] = i + 1 < len ? a.tokens[row0 + path[i + 1]] : (int64_t)next;
  }
  if (tid == 0) a.num_accepted[seq] = len;
}

// The same walk for greedy targets: a child is kept where its token is the target's choice
// after its parent. One wave per sequence.
__global__ __launch_bounds__(64) void verify_greedy_kernel(const int64_t* target_ids, const int64_t* tokens,
                                                           const int32_t* parents, const int32_t* row_starts,
                                                           int32_t* accepted, int32_t* num_accepted,
                                                           int64_t* out_tokens, int32_t width) {
  const int seq = blockIdx.x, lane = threadIdx.x;
  const int row0 = row_starts[seq], n = row_starts[seq + 1] - row0;
  int32_t* const acc = accepted + (int64_t)seq * width;
  int64_t* const out = out_tokens + (int64_t)seq * width;
  int len = 0, cur = 0;
  if (n > 0) {
    int64_t want = target_ids[row0];
    if (lane == 0) acc[0] = 0;
    len = 1;
    // 64 rows at a time: the first child of the reached node that holds the wanted token
    for (int i0 = 1; i0 < n; i0 += 64) {
      const int i = i0 + lane;
      const int par = i < n ? parents[row0 + i] : -2;
      const int64_t t = i < n ? tokens[row0 + i] : 0;
      for (;;) {
        const uint64_t hit = __ballot(par == cur && t == want);
        if (!hit) break;
        cur = i0 + __ffsll((unsigned long long)hit) - 1;
        if (lane == 0) {
          if (len < width) acc[len] = cur;
          if (len <= width) out[len - 1] = want;
        }
        ++len;
        want = target_ids[row0 + cur];
      }
    }
    if (lane == 0 && len <= width) out[len - 1] = want;
  }
  for (int i = len + lane; i < width; i += 64) acc[i] = -1, out[i] = -1;
  if (lane == 0) num_accepted[seq] = len;
}

// commit: node path[j] of a sequence lies at position cached + path[j] and belongs at cached + j.
// path rises, so path[j] >= j: a thread that moves one 16-byte column of the rows in order never
// reads a row it has written, and no other thread touches its column.
__global__ __launch_bounds__(256) void commit_kernel(char* storage, int64_t layer_bytes, int64_t num_blocks,
                                                     const int32_t* block_tables, int32_t max_nb,
                                                     const int32_t* cached, const int32_t* accepted, int32_t width,
                                                     const int32_t* num_accepted, int32_t num_kv_heads,
                                                     int32_t log2_bs, int32_t row_vecs) {
  const int seq = blockIdx.y, layer = blockIdx.z;
  const int v = blockIdx.x * 256 + threadIdx.x;    // (K or V, head, 16-byte piece)
  if (v >= 2 * num_kv_heads * row_vecs) return;
  const int kvh = v / row_vecs, piece = v - kvh * row_vecs;
  const int len = min(num_accepted[seq], width), c = cached[seq], bs = 1 << log2_bs;
  const int32_t* const table = block_tables + (int64_t)seq * max_nb;
  const int32_t* const path = accepted + (int64_t)seq * width;
  const int64_t head_bytes = (int64_t)bs * row_vecs * 16;
  char* const base = storage + layer * layer_bytes + kvh * head_bytes + 16 * piece;
  auto slot = [&](int pos) -> char* {
    const int blk = pos >> log2_bs;
    const int64_t b = blk < max_nb ? table[blk] : -1;
    if (b < 0 || b >= num_blocks) return nullptr;
    return base + b * (2 * num_kv_heads) * head_bytes + (int64_t)(pos & (bs - 1)) * row_vecs * 16;
  };
  for (int j = 0; j < len; ++j) {
    const int i = path[j];
    if (i <= j) continue;                          // in its place already (or no node)
    const char* const from = slot(c + i);
    char* const to = slot(c + j);
    if (from && to) st16(to, ld16(from));
  }
}

}  // namespace tb

extern "C" int32_t tb_tree_verify(const void* probs, int64_t probs_row_stride, const void* draft_probs,
                                  int64_t draft_row_stride, int32_t vocab, int32_t dtype, const int64_t* tokens,
                                  const float* uniforms, const int32_t* parents, const int32_t* row_starts,
                                  int32_t num_seqs, int32_t* accepted, int32_t* num_accepted, int64_t* out_tokens,
                                  int32_t width, hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_seqs >= 0 && vocab > 0 && width > 0);
  TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16);
  if (width > TB_TREE_MAX_NODES) return TB_ERR_UNSUPPORTED;
  if (num_seqs == 0) return TB_OK;
  TB_CHECK_ARG(probs && tokens && uniforms && parents && row_starts && accepted && num_accepted && out_tokens);
  TB_CHECK_ARG(probs_row_stride >= vocab && (!draft_probs || draft_row_stride >= vocab));
  const verify_args a{probs, probs_row_stride, draft_probs, draft_row_stride, vocab, tokens, uniforms, parents,
                      row_starts, accepted, num_accepted, out_tokens, width};
  const dim3 grid(num_seqs), block(VERIFY_THREADS);
  if (dtype == TB_DTYPE_F32) hipLaunchKernelGGL((verify_kernel<float>), grid, block, 0, stream, a);
  else if (dtype == TB_DTYPE_F16) hipLaunchKernelGGL((verify_kernel<_Float16>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((verify_kernel<__bf16>), grid, block, 0, stream, a);
  TB_RETURN_LAUNCH_STATUS();
}

extern "C" int32_t tb_tree_verify_greedy(const int64_t* target_ids, const int64_t* tokens, const int32_t* parents,
                                         const int32_t* row_starts, int32_t num_seqs, int32_t* accepted,
                                         int32_t* num_accepted, int64_t* out_tokens, int32_t width,
                                         hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_seqs >= 0 && width > 0);
  if (num_seqs == 0) return TB_OK;
  TB_CHECK_ARG(target_ids && tokens && parents && row_starts && accepted && num_accepted && out_tokens);
  hipLaunchKernelGGL(verify_greedy_kernel, dim3(num_seqs), dim3(64), 0, stream, target_ids, tokens, parents,
                     row_starts, accepted, num_accepted, out_tokens, width);
  TB_RETURN_LAUNCH_STATUS();
}

extern "C" int32_t tb_tree_commit(void* storage, int32_t num_layers, int64_t layer_stride_bytes, int64_t num_blocks,
                                  const int32_t* block_tables, int32_t max_blocks_per_seq, const int32_t* cached,
                                  int32_t num_seqs, const int32_t* accepted, int32_t width,
                                  const int32_t* num_accepted, int32_t num_kv_heads, int32_t head_dim,
                                  int32_t block_size, int32_t dtype, hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_layers >= 0 && num_seqs >= 0 && num_blocks > 0 && max_blocks_per_seq >= 0 && width > 0);
  TB_CHECK_ARG(num_kv_heads > 0 && head_dim > 0 && block_size > 0 && (block_size & (block_size - 1)) == 0);
  TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16);
  const int64_t row_bytes = (int64_t)head_dim * (dtype == TB_DTYPE_F32 ? 4 : 2);
  if (row_bytes % 16) return TB_ERR_UNSUPPORTED;
  TB_CHECK_ARG(num_layers <= 65535 && num_seqs <= 65535);
  if (num_layers == 0 || num_seqs == 0) return TB_OK;
  TB_CHECK_ARG(storage && block_tables && cached && accepted && num_accepted && ((uintptr_t)storage & 15u) == 0);
  TB_CHECK_ARG(layer_stride_bytes >= num_blocks * 2 * num_kv_heads * block_size * row_bytes &&
               layer_stride_bytes % 16 == 0);
  const int vecs = (int)(row_bytes / 16);
  const int64_t all = 2 * (int64_t)num_kv_heads * vecs;
  TB_CHECK_ARG(all < (int64_t)1 << 30);
  hipLaunchKernelGGL(commit_kernel, dim3((unsigned)((all + 255) / 256), num_seqs, num_layers), dim3(256), 0, stream,
                     (char*)storage, layer_stride_bytes, num_blocks, block_tables, max_blocks_per_seq, cached,
                     accepted, width, num_accepted, num_kv_heads, __builtin_ctz(block_size), vecs);
  TB_RETURN_LAUNCH_STATUS();
}
