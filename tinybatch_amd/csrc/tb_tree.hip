// Attention for a tree of drafted tokens over the paged cache.
//
// Sequence b has c = cached[b] positions in its cache and n nodes (its rows of q), node j's
// K/V stored at position c + j of its block table. Node i sees the cached positions and the
// nodes of its mask (itself and its ancestors, or any set):
//   S_i = {0 .. c-1} + {c + j : bit j of mask[i]},
//   out[i][h] = sum_{t in S_i} e^(s_t - m) v_t / sum_{t in S_i} e^(s_t - m),  s_t = scale q[i][h] . k_t,
// with m the running maximum of the scores seen so far. A node that sees nothing gives 0.
// What a node does not see has no effect on it, also where it is infinite or NaN.
#include "tb_common.h"

namespace tb {

struct tree_args {
  const char* q;               // [T][Hq][D]
  int64_t q_row_bytes;
  const char* pool;            // [NB][2][Hkv][BS][D]
  int64_t num_blocks;
  char* out;                   // [T][Hq*D]
  int64_t out_row_bytes;
  const int32_t* block_tables; // [B][max_nb]
  int32_t max_nb;
  const int32_t* row_starts;   // [B + 1]
  const int32_t* cached;       // [B]
  const int32_t* row_seq;      // [T]
  const uint32_t* mask;        // [T][mask_words]
  int32_t mask_words;          // 32-bit words
  int32_t num_heads, num_kv_heads, rep;
  int32_t log2_bs;
  float scale;
  const int64_t* positions;    // [T], for the rotation of q
  rope_tables rope;
};

// One wave per (row, head), lane l the positions l, l + 64, ...: each lane holds a softmax
// state of its own, merged across the wave at the end. Any block size.
template <typename Tag, int D>
__global__ __launch_bounds__(64) void tree_rows_kernel(const tree_args a) {
  using T = typename elem<Tag>::type;
  constexpr int N = 16 / sizeof(T), CH = D / N;    // elements of a 16-byte chunk, chunks of a row
  constexpr int RB = D * sizeof(T);
  const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const int seq = a.row_seq[row];
  if (seq < 0) return;
  const int row0 = a.row_starts[seq], n = a.row_starts[seq + 1] - row0, c = a.cached[seq];
  const int kvh = head / a.rep;

  vec16 qc[CH];
  const char* const qrow = a.q + (int64_t)row * a.q_row_bytes + (int64_t)head * RB;
#pragma unroll
  for (int i = 0; i < CH; ++i) qc[i] = ld16(qrow + 16 * i);
  if (a.rope.cos) {
    const int64_t r = a.rope.row(a.positions[row], D / 2);
#pragma unroll
    for (int i = 0; i < CH / 2; ++i)
      rope_pair<T>(qc[i], qc[i + CH / 2], a.rope.cos + r + N * i, a.rope.sin + r + N * i);
  }
  float q[D];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    T e[N];
    __builtin_memcpy(e, &qc[i], 16);
#pragma unroll
    for (int j = 0; j < N; ++j) q[N * i + j] = (float)e[j];
  }

  const float sl2e = a.scale * 1.4426950408889634f;
  const int bs_mask = (1 << a.log2_bs) - 1;
  const int64_t head_bytes = ((int64_t)1 << a.log2_bs) * RB;
  const int64_t blk_bytes = 2 * (int64_t)a.num_kv_heads * head_bytes, v_off = a.num_kv_heads * head_bytes;
  const int32_t* const table = a.block_tables + (int64_t)seq * a.max_nb;
  const uint32_t* const mask = a.mask + (int64_t)row * a.mask_words;
  float m = -INFINITY, l = 0.f, acc[D];
#pragma unroll
  for (int i = 0; i < D; ++i) acc[i] = 0.f;
  bool any = false;
  for (int p = lane; p < c + n; p += 64) {
    if (p >= c && !((mask[(p - c) >> 5] >> ((p - c) & 31)) & 1)) continue;
    const int64_t b = table[p >> a.log2_bs];
    if (b < 0 || b >= a.num_blocks) continue;      // host validates; stay inside the pool
    any = true;
    const char* const k = a.pool + b * blk_bytes + kvh * head_bytes + (int64_t)(p & bs_mask) * RB;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const vec16 v = ld16(k + 16 * i);
      T e[N];
      __builtin_memcpy(e, &v, 16);
#pragma unroll
      for (int j = 0; j < N; ++j) s = fmaf((float)e[j], q[N * i + j], s);
    }
    s *= sl2e;
    if (!(s <= m)) {                               // a larger score, or NaN
      const float f = m == -INFINITY ? 0.f : fast_exp2(m - s);
      l *= f;
#pragma unroll
      for (int i = 0; i < D; ++i) acc[i] *= f;
      m = s;
    }
    const float w = s == -INFINITY ? 0.f : fast_exp2(s - m);
    l += w;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const vec16 v = ld16(k + v_off + 16 * i);
      T e[N];
      __builtin_memcpy(e, &v, 16);
#pragma unroll
      for (int j = 0; j < N; ++j) acc[N * i + j] = fmaf(w, (float)e[j], acc[N * i + j]);
    }
  }
  float mm = m;
#pragma unroll
  for (int x = 1; x < 64; x *= 2) {
    const float o = __shfl_xor(mm, x);
    mm = mm != mm || o != o ? NAN : fmaxf(mm, o);
  }
  const float f = m == -INFINITY && mm == -INFINITY ? 0.f : fast_exp2(m - mm);
  l = group_sum<64>(l * f);
  const bool some = __any(any);
  const float inv = some ? 1.f / l : 0.f;
  char* const orow = a.out + (int64_t)row * a.out_row_bytes + (int64_t)head * RB;
#pragma unroll
  for (int i = 0; i < D; ++i) {
    const float s = group_sum<64>(m == -INFINITY ? 0.f : acc[i] * f);
    if (lane == i % 64) reinterpret_cast<T*>(orow)[i] = (T)(some ? s * inv : 0.f);
  }
}

template <typename Tag>
static void launch_rows(const tree_args& a, int num_rows, int head_dim, hipStream_t stream) {
  const dim3 grid(num_rows, a.num_heads);
  if (head_dim == 64) hipLaunchKernelGGL((tree_rows_kernel<Tag, 64>), grid, dim3(64), 0, stream, a);
  else hipLaunchKernelGGL((tree_rows_kernel<Tag, 128>), grid, dim3(64), 0, stream, a);
}

}  // namespace tb

extern "C" int32_t tb_tree_attention(const void* q, int64_t q_row_stride, const void* pool, int64_t num_blocks,
                                     void* out, int64_t out_row_stride, const int32_t* block_tables,
                                     int32_t max_blocks_per_seq, const int32_t* row_starts, const int32_t* cached,
                                     int32_t num_seqs, const int32_t* row_seq, int32_t num_rows,
                                     const uint32_t* mask, int32_t mask_words, int32_t num_heads,
                                     int32_t num_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                                     int32_t dtype, const int64_t* positions, const float* rope_cos,
                                     const float* rope_sin, int32_t rope_max_position, hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_rows >= 0 && num_seqs >= 0 && num_blocks > 0 && max_blocks_per_seq >= 0 && mask_words > 0);
  TB_CHECK_ARG(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 && num_heads <= 65535);
  TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16);
  TB_CHECK_ARG(block_size > 0 && (block_size & (block_size - 1)) == 0);
  if (head_dim != 64 && head_dim != 128) return TB_ERR_UNSUPPORTED;
  if (num_rows == 0) return TB_OK;
  TB_CHECK_ARG(q && pool && out && block_tables && row_starts && cached && row_seq && mask && num_seqs > 0);
  const int eb = dtype == TB_DTYPE_F32 ? 4 : 2;
  TB_CHECK_ARG(q_row_stride >= (int64_t)num_heads * head_dim && out_row_stride >= (int64_t)num_heads * head_dim);
  TB_CHECK_ARG((((uintptr_t)q | (uintptr_t)pool | (uintptr_t)out) & 15u) == 0);
  TB_CHECK_ARG((q_row_stride * eb) % 16 == 0 && (out_row_stride * eb) % 16 == 0);
  TB_CHECK_ARG((rope_cos == nullptr) == (rope_sin == nullptr));
  if (rope_cos) TB_CHECK_ARG(positions && rope_max_position > 0 && (((uintptr_t)rope_cos | (uintptr_t)rope_sin) & 15u) == 0);
  tree_args a{};
  a.q = (const char*)q;
  a.q_row_bytes = q_row_stride * eb;
  a.pool = (const char*)pool;
  a.num_blocks = num_blocks;
  a.out = (char*)out;
  a.out_row_bytes = out_row_stride * eb;
  a.block_tables = block_tables;
  a.max_nb = max_blocks_per_seq;
  a.row_starts = row_starts;
  a.cached = cached;
  a.row_seq = row_seq;
  a.mask = mask;
  a.mask_words = mask_words;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.rep = num_heads / num_kv_heads;
  a.log2_bs = __builtin_ctz(block_size);
  a.scale = scale;
  a.positions = positions;
  a.rope = rope_tables{rope_cos, rope_sin, rope_max_position};
  if (dtype == TB_DTYPE_F32) launch_rows<f32_t>(a, num_rows, head_dim, stream);
  else if (dtype == TB_DTYPE_F16) launch_rows<f16_t>(a, num_rows, head_dim, stream);
  else launch_rows<bf16_t>(a, num_rows, head_dim, stream);
  TB_RETURN_LAUNCH_STATUS();
}
