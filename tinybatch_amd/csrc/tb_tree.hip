// Attention for a tree of drafted tokens over the paged cache.
//
// Sequence b has c = cached[b] positions in its cache and n nodes (its rows of q), node j's
// K/V stored at position c + j of its block table. Node i sees the cached positions and the
// nodes of its mask (itself and its ancestors, or any set):
//   S_i = {0 .. c-1} + {c + j : bit j of mask[i]},
//   out[i][h] = sum_{t in S_i} e^(s_t - m) v_t / sum_{t in S_i} e^(s_t - m),  s_t = scale q[i][h] . k_t,
// with m the running maximum of the scores seen so far. A node that sees nothing gives 0.
// What a node does not see has no effect on it, also where it is infinite or NaN.
//
// Work: the n nodes and the rep query heads of a kv head make n * rep columns, column =
// node * rep + head, that read the same K/V rows whatever their masks. A workgroup of four
// waves takes 32 CW consecutive columns of a (sequence, kv head) and a part of the context, which
// it walks in chunks of CK positions through a ring of two in LDS: every wave loads a quarter of
// the next chunk (direct global->LDS loads) and computes on the present one, one barrier between.
// A wave holds 32 columns; with CW < 4 several waves hold the same ones, each a part of a
// chunk's positions, and join their softmax states in LDS at the end. A context cut into parts
// leaves a partial per part, joined by the workgroup of a (sequence, kv head, columns) that arrives
// last where there is little to join and the caller gives arrival counters, else by a second launch.
// Blocks of fewer than 16 positions (SMALL) give every row of a tile a block of its own; otherwise a tile has one,
// and its rows one base address. In blocks of 8 16 trees of 16 nodes behind 4000 positions at 32 / 8 heads of 128 take
// 50.4 us, in blocks of 16 45.6.
//
// Math per chunk and block of 32 columns (C rows are positions or dims, C columns the block's):
//   S^T[pos][col] = K[pos][:] . q[col][:]        A = K rows from LDS, B = q in registers
//   O^T[d][col]  += V^T[d][pos] . P^T[pos][col]  A = V^T from LDS, B = the S^T registers
// 16-bit: v_mfma_f32_32x32x16, V^T by LDS transpose reads; the weights P are rounded to the
// element type for the product, which takes both operands in one type (their lower halves would be a second
// product for each V), and their sum is taken of the rounded ones. fp32:
// v_mfma_f32_32x32x2_f32, nothing rounded further. The reference maximum of a column moves
// only when a score outgrows it by 8 (weights to 2^8), so that the accumulators are rescaled
// a few times per context. fp16 weights end at 2^-25: they refer to a maximum 7 lower (the largest one 2^7 to
// 2^15), so that the tail of 2^18 keys of a weight of 2^-25.4 beside one of 1 is there to 1.1% instead of
// missing; below 2^-32 of the dominant weight it still does.
#include <algorithm>
#include <cmath>
#include <exception>
#include <functional>
#include <type_traits>
#include <utility>
#include <vector>

#include "tb_stream.h"

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
  const int64_t* positions;    // [T], for the rotation of q
  rope_tables rope;
  const int4* work;            // three per workgroup, see tb_build_tree_work
  const int4* split;           // (row, first partial slot, parts, slots between parts)
  float* ws_acc;               // [slots][Hq][D]
  float* ws_ml;                // [slots][Hq][2]
  int64_t slots;
  uint32_t* arrivals;          // [units], zero between calls; null: tree_join_kernel joins
  float scale_log2e;           // > 0: the scale's size times log2(e), or 1 for a scale of 0
  float q_sign;                // 1, -1 or 0 (NaN: a NaN scale): multiplies q, so that masked scores stay -inf
};

// Whether node `row` of a tree of n nodes with `cached` positions before it sees anything.
__device__ __forceinline__ bool tree_sees(const uint32_t* mask, int cached, int n) {
  if (cached > 0) return true;
  for (int w = 0; 32 * w < n; ++w)
    if (mask[w] & (n - 32 * w >= 32 ? ~0u : (1u << (n - 32 * w)) - 1)) return true;
  return false;
}

// ---- column blocks over the matrix unit --------------------------------------------
template <typename Tag, int D>
struct tshape {
  static constexpr int EB = elem<Tag>::bytes;
  static constexpr int RB = EB * D;             // bytes per K or V row
  static constexpr int TB = 16 * RB;            // bytes of a 16-position tile
  static constexpr int PPR = RB / 16;           // 16-byte pieces per row
  static constexpr int RPL = 64 / PPR;          // rows per direct load
  static constexpr int QS = PPR / 2;            // 16-byte pieces of a lane's q (the other half's lane holds the rest)
  static constexpr int NB = D / 32;             // O^T blocks of 32 dims
  // K row r keeps its piece p in slot p ^ kswz(r), V row r in slot p ^ vswz(r), so that the operand
  // reads of 16 (K) and 32 (V, 16-bit transpose reads) lanes cover all 64 banks
  static __device__ __forceinline__ int kswz(int r) { return RB == 128 ? (r & 7) ^ ((r >> 3) & 1) : r & 15; }
  static __device__ __forceinline__ int vswz(int r) {
    return EB == 4 ? 0 : D == 64 ? 2 * (r & 3) : (0xCA60 >> (4 * (r & 3))) & 15;
  }
};

// The seen positions p0 .. p0 + 31 of a node (p0 a multiple of 32): the cached ones and its mask's bits.
__device__ __forceinline__ uint32_t tree_seen(const uint32_t* mask, int words, int cached, int limit, int p0) {
  const int off = p0 - cached, w = off >> 5;       // nodes off .. off + 31
  const uint32_t lo = w < 0 ? ~0u : w < words ? mask[w] : 0u;
  const uint32_t hi = w + 1 < 0 ? ~0u : w + 1 < words ? mask[w + 1] : 0u;
  const uint32_t seen = __builtin_amdgcn_alignbit(hi, lo, off & 31);
  return limit - p0 >= 32 ? seen : limit > p0 ? seen & ((1u << (limit - p0)) - 1) : 0u;
}
// The scores of unseen positions to -inf: register r holds position 8 (r / 4) + 4 half + r % 4.
__device__ __forceinline__ void tree_hide(float16_t& sc, uint32_t seen, int half) {
  const uint32_t mine = seen >> (4 * half);
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (!(mine & (1u << (8 * (r >> 2) + (r & 3))))) sc[r] = -INFINITY;
}
// Whether BYTES of V rows in LDS (a wave's reads) hold no infinity or NaN.
template <typename T, int BYTES>
__device__ __forceinline__ bool tree_finite(const char* v, int lane) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr uint32_t E = F32 ? 0x7F800000u : __is_same(T, _Float16) ? 0x7C00u : 0x7F80u;
  bool ok = true;
  for (int i = 0; i < BYTES / 1024; ++i) {
    const vec16 x = ld16(v + 1024 * i + 16 * lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      ok &= (x.w[j] & E) != E;
      if (!F32) ok &= ((x.w[j] >> 16) & E) != E;
    }
  }
  return __all(ok);
}
// O^T += V^T.P of 32 positions one by one, the unseen ones left out: a weight of 0 times an infinity is
// no 0. p(r): this lane's weight of register r.
template <typename Tag, int D, typename P>
__device__ __forceinline__ void tree_values_apart(float16_t (&acc)[D / 32], const char* v, uint32_t seen, int half,
                                                  P&& p) {
  using S = tshape<Tag, D>;
  using T = typename elem<Tag>::type;
  constexpr bool F32 = S::EB == 4;
#pragma unroll 1
  for (int pos = 0; pos < 32; ++pos) {
    const int reg = 4 * (pos >> 3) + (pos & 3);
    float mine = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) mine = r == reg ? p(r) : mine;
    const float other = __shfl_xor(mine, 32);
    const float w = half == ((pos >> 2) & 1) ? mine : other;
    if ((seen >> pos) & 1) {
#pragma unroll
      for (int b = 0; b < D / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {           // dims 32 b + 8 g + 4 half ..
          const char* const vp =
              v + pos * S::RB + (F32 ? 128 * b + 32 * g + 16 * half : 16 * ((4 * b + g) ^ S::vswz(pos)) + 8 * half);
          T e[4];
          __builtin_memcpy(e, __builtin_assume_aligned(vp, 8), 4 * sizeof(T));
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[b][4 * g + j] = fmaf(w, (float)e[j], acc[b][4 * g + j]);
        }
    }
  }
}
// Element i of a packed 16-bit operand.
template <typename T>
__device__ __forceinline__ float tree_unpack(su32x4_t x, int i) {
  T e[2];
  const uint32_t word = x[i >> 1];
  __builtin_memcpy(e, &word, 4);
  return (float)e[i & 1];
}
// q of a column rotated (RoPE at the node's position), its sign, complete on return.
template <typename Tag, int D, int QS>
__device__ __forceinline__ void tree_q(vec16 (&q)[QS], const tree_args& a, int row, int half) {
  using T = typename elem<Tag>::type;
  constexpr int E = 16 / sizeof(T);
  if (a.rope.cos) {
    const int64_t r = a.rope.row(a.positions[row], D / 2) + E * half;
#pragma unroll
    for (int s = 0; s < QS / 2; ++s)            // pieces s and s + QS/2 pair (dims i and i + D/2)
      rope_pair<T>(q[s], q[s + QS / 2], a.rope.cos + r + 2 * E * s, a.rope.sin + r + 2 * E * s);
  }
  if (a.q_sign != 1.f) {
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      T x[E];
      __builtin_memcpy(x, &q[s], 16);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = (T)((float)x[e] * a.q_sign);
      __builtin_memcpy(&q[s], x, 16);
    }
  }
#pragma unroll
  for (int s = 0; s < QS; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(q[s].w[i]));
}

// o += w x, rounded once: one form for the two joins below, which give the same bits.
__device__ __forceinline__ void tree_add(float4_t& o, float4_t x, float w) {
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = fmaf(x[j], w, o[j]);
}
// The join of a unit's parts by its last workgroup: what the others wrote is read past the L2s, which the
// XCDs do not share. Thread = 4 dims of a column.
template <typename Tag, int D, int CW>
__device__ __forceinline__ void tree_join_here(const tree_args& a, int row0, int cached, int nodes, int col0, int kvh,
                                               int first, int parts) {
  using T = typename elem<Tag>::type;
  constexpr int QPC = D / 4, BATCH = 8, ITEMS = 2;   // parts and columns of a thread in flight
  auto load2 = [](const float* p) {
    return __builtin_bit_cast(float2, __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  };
  const int items = min(32 * CW, nodes * a.rep - col0) * QPC;
  for (int i0 = threadIdx.x; i0 < items; i0 += 256 * ITEMS) {
    float M[ITEMS], L[ITEMS];
    float4_t o[ITEMS];
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) M[t] = -INFINITY, L[t] = 0.f, o[t] = float4_t{0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < parts; p0 += BATCH) {
      float2 ml[ITEMS][BATCH], lo[ITEMS][BATCH], hi[ITEMS][BATCH];
#pragma unroll
      for (int t = 0; t < ITEMS; ++t) {
        const int i = min(i0 + 256 * t, items - 1), col = col0 + i / QPC, node = col / a.rep;
        const int head = kvh * a.rep + col - node * a.rep;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const int64_t at = (int64_t)(first + min(p0 + k, parts - 1) * nodes + node) * a.num_heads + head;
          ml[t][k] = load2(a.ws_ml + at * 2);
          lo[t][k] = load2(a.ws_acc + at * D + 4 * (i % QPC));
          hi[t][k] = load2(a.ws_acc + at * D + 4 * (i % QPC) + 2);
        }
      }
#pragma unroll
      for (int t = 0; t < ITEMS; ++t) {
        float mb = M[t];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) mb = fmaxf(mb, ml[t][k].x);
        const float safe = mb == -INFINITY ? 0.f : mb, keep = fast_exp2(M[t] - safe);
        L[t] *= keep;
        o[t] *= keep;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const float w = p0 + k < parts ? fast_exp2(ml[t][k].x - safe) : 0.f;   // 0 for a part that saw nothing
          if (p0 + k < parts) {
            L[t] = fmaf(ml[t][k].y, w, L[t]);
            tree_add(o[t], float4_t{lo[t][k].x, lo[t][k].y, hi[t][k].x, hi[t][k].y}, w);
          }
        }
        M[t] = mb;
      }
    }
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
      const int i = i0 + 256 * t;
      if (i >= items) break;
      const int col = col0 + i / QPC, node = col / a.rep, head = kvh * a.rep + col - node * a.rep, row = row0 + node;
      float inv = 1.f / L[t];
      if (!(L[t] > 0.f) && !tree_sees(a.mask + (int64_t)row * a.mask_words, cached, nodes)) inv = 0.f;
      typedef T t4_t __attribute__((ext_vector_type(4)));
      t4_t x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (T)(o[t][j] * inv);
      st_through(a.out + (int64_t)row * a.out_row_bytes + ((int64_t)head * D + 4 * (i % QPC)) * sizeof(T), x);
    }
  }
}

// 32 CW columns: the four waves share chunks of CK positions, of which each loads a quarter. CW of them take
// 32 columns each, 4 / CW the same columns, each a part of a chunk's positions, joined at the end.
//
// What bounds it: with few columns the reads of K/V (48 chains of 4 to 8 nodes behind 8192 positions at 32 / 8 heads of
// 128, bf16: 1.9 GB in 293 to 309 us, 6.2 to 6.5 TB/s, the matrix unit busy 8% of the time). With many columns no unit
// by itself: a wave's LDS reads, products and softmax follow one another, behind a barrier a chunk, and hide only the
// other waves' of its SIMD. 16 trees of 64 nodes there, 80 GFLOP in 119 to 128 us (620 to 670 TFLOP/s; 137 to 151 once
// some ms of it have brought the clock down): matrix unit 29%, vector unit 26%, LDS 15%, 4.6 of 8 waves on a CU on
// average. 4 of 1024 nodes behind 25000 to 50000 positions: 47%, 42%, 25%, 6.8 of 8 (990 TFLOP/s behind 50000 to
// 100000). At head dim 64 32 trees of 20 to 30 nodes at 14 / 2 heads behind 512 to 4096 positions in 22 us: 10%, 18%,
// 5%, 3.4 of 8, waves waiting 46% of their time; 182 columns leave a quarter of two workgroups of 128 idle. fp32: 16
// trees of 26 nodes there behind 1000 to 2000 positions in 33 us, 66 TFLOP/s of a library's 153: matrix unit 40%, 4.5
// of 8 waves; at head dim 128 one wave a SIMD is all that the LDS has room for, and the matrix unit (44% for 8 of 32 at
// 32 / 8 heads) waits for its softmax. A single sequence: the launch, the block table and K/V reads one after the other
// (7.1 us in a graph for 5 nodes behind 600 positions).
// Why chunks are shared: with a ring of its own per wave, no barriers but a quarter of the bytes in flight per position
// loaded, the chains above took 343 us instead of 295. Rows that one workgroup of their sequence reads are loaded past
// the L2s' replacement (`once`: 297 us against 314), rows that several read through the L2 (16 trees of 64 nodes behind
// 8000 positions: 146 against 155). Sequences that share a prefix read its rows once each all the same (48 of 6 nodes
// behind the same 8192 positions 122 us, behind positions of their own 256). CK is what a ring of two leaves of the LDS
// to two workgroups (one at 512-byte rows); chunks of 32 positions in a ring of four, for one set of waves after the
// other, have half as much again under way, but 301 us against 291 for 48 chains behind 12000 positions, 27.4 against
// 21.7 for 4 trees of 24 nodes behind 4000.
template <typename Tag, int D, int CW, int CK, bool SMALL>
__global__ __launch_bounds__(256, D * elem<Tag>::bytes * CK < 32768 ? 2 : 1) void tree_columns_kernel(const tree_args a) {
  using S = tshape<Tag, D>;
  constexpr bool F32 = S::EB == 4;
  using T = typename elem<Tag>::type;
  constexpr int RB = S::RB, NB = S::NB, QS = S::QS, NW = 4, HALF = CK * RB, SLOT = 2 * HALF;
  constexpr int SETS = NW / CW, TL = CK / 32 / SETS;   // waves on a column; 32-position tiles a wave takes of a chunk
  constexpr int TILES = CK / 64;                // 16-position tiles a wave loads of a chunk
  constexpr int WS = 64 * (16 * NB + 2);        // floats of a wave's state
  constexpr int LDS = SETS > 1 && NW * WS * 4 > 2 * SLOT ? NW * WS * 4 : 2 * SLOT;
  static_assert(TL >= 1 && TILES >= 1, "a tile for every wave");
  constexpr float LIFT = std::is_same_v<T, _Float16> ? 7.f : 0.f;   // of the weights, in powers of two
  __shared__ __align__(1024) char lds[LDS];

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, lcol = lane & 31, half = lane >> 5;
  const int4 w0 = a.work[3 * blockIdx.x], w1 = a.work[3 * blockIdx.x + 1], w2 = a.work[3 * blockIdx.x + 2];
  const int row0 = w0.x, seq = w0.y, cached = w0.z, nodes = w0.w;
  if (nodes == 0) return;                       // a padding entry (whole workgroup)
  const int set = wave / CW;                    // its tiles start at position 32 TL set of a chunk
  const bool once = w2.y;                       // no other workgroup of its sequence reads these K/V rows
  const int col0 = w1.x + 32 * (wave % CW), kvh = w1.y, chunk0 = w1.z, chunks = w1.w;   // chunks of 32, chunk0 even
  const int limit = cached + nodes, ncols = nodes * a.rep;
  const int col = min(col0 + lcol, ncols - 1), my_row = col / a.rep, hd = kvh * a.rep + col - my_row * a.rep;

  vec16 q[QS];
  {
    const char* const qrow = a.q + (int64_t)(row0 + my_row) * a.q_row_bytes + (int64_t)hd * RB + 16 * half;
#pragma unroll
    for (int s = 0; s < QS; ++s) q[s] = ld16(qrow + 32 * s);
  }
  // ---- direct loads ----
  const int64_t head_bytes = ((int64_t)1 << a.log2_bs) * RB;
  const int64_t blk_bytes = 2 * (int64_t)a.num_kv_heads * head_bytes, v_off = a.num_kv_heads * head_bytes;
  const int sub_mask = SMALL ? 0 : (1 << (a.log2_bs - 4)) - 1, bs_mask = (1 << a.log2_bs) - 1;
  const int32_t* const table = a.block_tables + (int64_t)seq * a.max_nb;
  const char* const pool_kvh = a.pool + kvh * head_bytes;
  const int last_tile = (limit - 1) >> 4, tile0 = 2 * chunk0 + TILES * wave;
  const int lrow = lane / S::PPR, lpiece = lane % S::PPR;
  const int n = (32 * chunks + CK - 1) / CK;
  constexpr int IDS = SMALL ? 16 * TILES : TILES;   // block ids of a wave's part of a slot
  int id0 = 0;
  auto tile_of = [&](int k, int t) { return min(tile0 + CK / 16 * k + t, last_tile); };
  auto load_ids = [&](int k) {                  // lane j: block j % IDS (of a tile; SMALL: of a row) of slot k + j / IDS
    const int slot = k + lane / IDS, j = lane % IDS;
    const int tile = SMALL ? tile_of(slot, j / 16) : tile_of(slot, j);
    const int b = table[(SMALL ? min(16 * tile + j % 16, limit - 1) : 16 * tile) >> a.log2_bs];
    return (b < 0 || b >= a.num_blocks) ? 0 : b;   // host validates; stay inside the pool
  };
  int ids = load_ids(0);
  asm volatile("" : "+v"(ids));                 // the block ids have landed: no wait inside the loop
  auto issue = [&](int k) {
    if (k - id0 >= 64 / IDS) {                  // uniform, once per 64 or 32 slots (SMALL: 4 or 2)
      id0 = k;
      ids = load_ids(k);
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int tile = tile_of(k, t), rmax = limit - 1 - 16 * tile;   // rows past it repeat the last position
      char* const dst = lds + (k & 1) * SLOT + (TILES * wave + t) * S::TB;
      if constexpr (SMALL) {
#pragma unroll
        for (int i = 0; i < S::TB / 1024; ++i) {
          const int r = S::RPL * i + lrow, at = min(r, rmax);
          const int64_t b = __shfl(ids, IDS * (k - id0) + 16 * t + at);
          const char* const row = pool_kvh + b * blk_bytes + (int64_t)(at & bs_mask) * RB;
          s_dma16_l2p(row + 16 * (lpiece ^ S::kswz(r)), dst + 1024 * i);
          s_dma16_l2p(row + v_off + 16 * (lpiece ^ S::vswz(r)), dst + HALF + 1024 * i);
        }
      } else {
        const int64_t b = __builtin_amdgcn_readlane(ids, TILES * (k - id0) + t);
        const char* const base = pool_kvh + b * blk_bytes + (int64_t)(tile & sub_mask) * S::TB;
#pragma unroll
        for (int i = 0; i < S::TB / 1024; ++i) {
          const int r = S::RPL * i + lrow;
          const uint32_t row = (uint32_t)(min(r, rmax) * RB);
          const uint32_t ko = row + 16 * (lpiece ^ S::kswz(r)), vo = row + 16 * (lpiece ^ S::vswz(r));
          if (once) {
            s_dma16_s(ko, base, dst + 1024 * i);
            s_dma16_s(vo, base + v_off, dst + HALF + 1024 * i);
          } else {
            s_dma16_l2(ko, base, dst + 1024 * i);
            s_dma16_l2(vo, base + v_off, dst + HALF + 1024 * i);
          }
        }
      }
    }
  };
  issue(0);
  tree_q<Tag, D>(q, a, row0 + my_row, half);

  uint32_t ones = 0;                            // in a register: as a literal the bf16 dot product read it wrong
  if constexpr (!F32) ones = cmath<Tag>::ONES;
  asm volatile("" : "+v"(ones));
  float m = -INFINITY, l = 0.f;
  float16_t acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[b][r] = 0.f;
  uint32_t ka[QS], va[NB];
#pragma unroll
  for (int s = 0; s < QS; ++s) ka[s] = (uint32_t)(lcol * RB + 16 * ((2 * s + half) ^ S::kswz(lcol)));
  {
    const int li = lane & 15, rv = 4 * half + (li >> 2);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int c = 4 * b + 2 * ((lane >> 4) & 1) + ((li & 3) >> 1);
      va[b] = F32 ? (uint32_t)(HALF + 4 * half * RB + 128 * b + 4 * lcol)
                  : (uint32_t)(HALF + rv * RB + 16 * (c ^ S::vswz(rv)) + 8 * (li & 1));
    }
  }
  const float sl2e = a.scale_log2e;
  const bool busy = col0 < ncols;
  auto step = [&](int k, auto masked) {
    // the wave's loads of slot k have landed and its reads of slot k - 1 are done: behind the barrier
    // all of slot k is in LDS and the other one is free
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (k + 1 < n) issue(k + 1);
    if (!busy) return;
    const char* const base = lds + (k & 1) * SLOT + set * (32 * TL * RB);
    const int p0 = 32 * chunk0 + CK * k + 32 * TL * set;
    // ---- scores: operands read KG pieces ahead of their products ----
    float16_t sc[TL];
    if constexpr (!F32) {
#pragma unroll
      for (int t = 0; t < TL; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[t][r] = 0.f;
      constexpr int KG = 4 / TL;
      su32x4_t kf[2][KG][TL];
      auto read = [&](int g) {
#pragma unroll
        for (int i = 0; i < KG; ++i)
#pragma unroll
          for (int t = 0; t < TL; ++t)
            kf[g & 1][i][t] = *reinterpret_cast<const su32x4_t*>(base + ka[KG * g + i] + 32 * t * RB);
      };
      read(0);
#pragma unroll
      for (int g = 0; g < QS / KG; ++g) {
        if (g + 1 < QS / KG) read(g + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < KG; ++i)
#pragma unroll
          for (int t = 0; t < TL; ++t)
            sc[t] = cmath<Tag>::mfma(kf[g & 1][i][t], __builtin_bit_cast(su32x4_t, q[KG * g + i]), sc[t]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      float16_t d[TL][2];                       // two chains a tile
#pragma unroll
      for (int t = 0; t < TL; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) d[t][0][r] = d[t][1][r] = 0.f;
      vec16 kf[2][TL];
      auto read = [&](int s) {
#pragma unroll
        for (int t = 0; t < TL; ++t) kf[s & 1][t] = ld16(base + ka[s] + 32 * t * RB);
      };
      read(0);
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        if (s + 1 < QS) read(s + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < TL; ++t)
            d[t][i & 1] = __builtin_amdgcn_mfma_f32_32x32x2f32(bits_to_f32(kf[s & 1][t].w[i]), bits_to_f32(q[s].w[i]),
                                                               d[t][i & 1], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int t = 0; t < TL; ++t) sc[t] = d[t][0] + d[t][1];
    }
    // ---- online softmax ----
    uint32_t seen[TL];
    if constexpr (masked.value) {
#pragma unroll
      for (int t = 0; t < TL; ++t) {
        seen[t] = tree_seen(a.mask + (int64_t)(row0 + my_row) * a.mask_words, a.mask_words, cached, limit, p0 + 32 * t);
        tree_hide(sc[t], seen[t], half);
      }
    }
    float cm = max_f32(sc[0][0], sc[0][1]);
#pragma unroll
    for (int e = 2; e < 16 * TL; e += 2) cm = max3_f32(cm, sc[e >> 4][e & 15], sc[e >> 4][(e & 15) + 1]);
    cm *= sl2e;
    // (a score of size 2^24 or more is off by 1 and more itself: what its weight may pass 2^15 by is taken off)
    if (__any(cm > (LIFT > 0.f ? fmaf(fabsf(m), -0x1p-20f, m + (8.f + LIFT)) : m + 8.f))) {
      const float m_new = fmaxf(m, max_xor32(cm) - LIFT);
      const float alpha = fast_exp2(m - (m_new == -INFINITY ? 0.f : m_new));   // 0 while m = -inf
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] *= alpha;
    }
    const float neg_m = m == -INFINITY ? 0.f : -m;
    su32x4_t pb[2 * TL];                        // 16-bit P: B operands of 16 positions each
#pragma unroll
    for (int t = 0; t < TL; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[t][r] = fast_exp2(fmaf(sc[t][r], sl2e, neg_m));
    if constexpr (!F32) {
      float sum = 0.f;                          // of the chunk by itself: small weights count beside a large l
#pragma unroll
      for (int w = 0; w < 2 * TL; ++w) {
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = sc[w >> 1][8 * (w & 1) + j];
        pb[w] = smath<Tag>::pack8(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = cmath<Tag>::add2(pb[w][j], ones, sum);   // of the rounded P that multiplies V
      }
      l += sum;
    } else {
#pragma unroll
      for (int t = 0; t < TL; ++t) {
        const float16_t& p = sc[t];
        l += (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]))) +
             (((p[8] + p[9]) + (p[10] + p[11])) + ((p[12] + p[13]) + (p[14] + p[15])));
      }
    }
    // ---- values ----
    bool plain = true;
    if constexpr (masked.value) {
      plain = tree_finite<T, 32 * TL * RB>(base + HALF, lane);
      if (!plain) {
#pragma unroll
        for (int t = 0; t < TL; ++t)
          tree_values_apart<Tag, D>(acc, base + HALF + 32 * t * RB, seen[t], half, [&](int r) {
            if constexpr (F32) return sc[t][r];
            else return tree_unpack<T>(pb[2 * t + (r >> 3)], r & 7);
          });
      }
    }
    if (!plain) {
    } else if constexpr (F32) {
      float vf[2][NB];
      auto read = [&](int i) {                  // position register i of the wave's 16 TL
#pragma unroll
        for (int b = 0; b < NB; ++b)
          vf[i & 1][b] = *reinterpret_cast<const float*>(base + va[b] + (32 * (i >> 4) + 8 * ((i & 15) >> 2) + (i & 3)) * RB);
      };
      read(0);
#pragma unroll
      for (int i = 0; i < 16 * TL; ++i) {
        if (i + 1 < 16 * TL) read(i + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[i & 1][b], sc[i >> 4][i & 15], acc[b], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      uint2 vf[2][NB][2];
      auto read = [&](int w) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const char* const vp = base + va[b] + 16 * w * RB;
          vf[w & 1][b][0] = lds_read_tr16(vp);
          vf[w & 1][b][1] = lds_read_tr16(vp + 8 * RB);
        }
      };
      read(0);
#pragma unroll
      for (int w = 0; w < 2 * TL; ++w) {
        if (w + 1 < 2 * TL) read(w + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint2 lo = vf[w & 1][b][0], hi = vf[w & 1][b][1];
          acc[b] = cmath<Tag>::mfma(su32x4_t{lo.x, lo.y, hi.x, hi.y}, pb[w], acc[b]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // the slots that lie in the cache whole, then those with nodes: two loops, so that the mask costs the
  // long one neither instructions nor registers. The second is the slower one: a slot's mask words are loaded behind the
  // next slot's K/V and wait for those too, and with four column blocks of 16 bits at head dim 128 it spills 21 to 27
  // registers. Large trees behind short caches run in it: 8 of 512 nodes behind one position at 32 / 8 heads 103 us
  // (matrix unit 14%, vector unit 43%).
  const int plain = max(0, min(n, (cached - 32 * chunk0) / CK));
  int k = 0;
  for (; k < plain; ++k) step(k, std::false_type{});
  for (; k < n; ++k) step(k, std::true_type{});

  l = sum_xor32(l);
  const bool mine = col0 + lcol < ncols;
  const int slot = w2.x, row = row0 + my_row;   // slot < 0: the whole context, the output itself
  const float* all = nullptr;                   // the sets' states of these columns
  float f[SETS];
  if constexpr (SETS > 1) {
    float* const state = reinterpret_cast<float*>(lds) + lane;
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) state[wave * WS + 64 * (16 * b + r)] = acc[b][r];
    state[wave * WS + 64 * 16 * NB] = m;
    state[wave * WS + 64 * (16 * NB + 1)] = l;
    __syncthreads();
    all = state + (wave % CW) * WS;
    m = -INFINITY;
#pragma unroll
    for (int s = 0; s < SETS; ++s) m = fmaxf(m, all[s * CW * WS + 64 * 16 * NB]);
    const float safe = m == -INFINITY ? 0.f : m;
    l = 0.f;
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      f[s] = fast_exp2(all[s * CW * WS + 64 * 16 * NB] - safe);   // 0 for a set that saw nothing
      l += all[s * CW * WS + 64 * (16 * NB + 1)] * f[s];
    }
  }
  const bool here = slot >= 0 && a.arrivals != nullptr;   // the last workgroup joins the parts
  if (mine) {
    float inv = 1.f;
    if (slot < 0) {
      inv = 1.f / l;
      if (!(l > 0.f) && !tree_sees(a.mask + (int64_t)row * a.mask_words, cached, nodes)) inv = 0.f;
    }
    typedef T t4_t __attribute__((ext_vector_type(4)));
    const int64_t at = (int64_t)(slot + my_row) * a.num_heads + hd;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g) {             // dims 32 b + 8 g + 4 half ..: the group of set g % SETS
        float4_t o;
        if constexpr (SETS == 1) {
          o = float4_t{acc[b][4 * g], acc[b][4 * g + 1], acc[b][4 * g + 2], acc[b][4 * g + 3]};
        } else {
          if (g % SETS != set) continue;
          o = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < SETS; ++s) {
            const float* const x = all + s * CW * WS + 64 * (16 * b + 4 * g);
            o += float4_t{x[0], x[64], x[128], x[192]} * f[s];
          }
        }
        float* const partial = a.ws_acc + at * D + 32 * b + 8 * g + 4 * half;
        if (slot < 0) {
          t4_t t;
#pragma unroll
          for (int j = 0; j < 4; ++j) t[j] = (T)(o[j] * inv);
          st_through(a.out + (int64_t)row * a.out_row_bytes + (int64_t)hd * RB + (32 * b + 8 * g + 4 * half) * S::EB, t);
        } else if (here) {
          st_through(partial, o);
        } else {
          *reinterpret_cast<float4_t*>(partial) = o;
        }
      }
    if (slot >= 0 && half == 0 && set == 0) {
      if (here) st8_through(a.ws_ml + at * 2, make_float2(m, l));
      else *reinterpret_cast<float2*>(a.ws_ml + at * 2) = make_float2(m, l);
    }
  }
  if (!here) return;
  __shared__ uint32_t arrived;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wave's partials are in memory
  __syncthreads();
  const int parts = w2.w >> 16, part = w2.w & 0xFFFF;
  if (threadIdx.x == 0) {
    arrived = __hip_atomic_fetch_add(&a.arrivals[w2.z], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (arrived == (uint32_t)parts - 1)
      __hip_atomic_store(&a.arrivals[w2.z], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (arrived == (uint32_t)parts - 1)
    tree_join_here<Tag, D, CW>(a, row0, cached, nodes, w1.x, kvh, slot - part * nodes, parts);
}

// The partials of a row's parts joined: lane = 4 dims of a head, wave w the parts w, w + NW, ...; the waves'
// states meet in LDS. One wave up to 16 parts.
template <typename Tag, int D, int NW>
__global__ __launch_bounds__(64 * NW) void tree_join_kernel(const tree_args a) {
  using T = typename elem<Tag>::type;
  constexpr int QPH = D / 4, BATCH = 8;
  __shared__ float state[NW > 1 ? (NW - 1) * 64 * 6 : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = min(lane + 64 * (int)blockIdx.y, a.num_heads * QPH - 1);
  const int4 rec = a.split[blockIdx.x];
  const int row = rec.x, first = rec.y, parts = rec.z, step = rec.w;
  const int head = col / QPH, d4 = col - head * QPH;
  float M = -INFINITY, L = 0.f;
  float4_t o = float4_t{0.f, 0.f, 0.f, 0.f};
  for (int p0 = wave; p0 < parts; p0 += BATCH * NW) {
    float2 ml[BATCH];
    float4_t av[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      av[k] = float4_t{0.f, 0.f, 0.f, 0.f};
      if (p0 + k * NW < parts) {
        const int64_t at = (int64_t)(first + (p0 + k * NW) * step) * a.num_heads + head;
        ml[k] = *reinterpret_cast<const float2*>(a.ws_ml + at * 2);
        av[k] = *reinterpret_cast<const float4_t*>(a.ws_acc + at * D + 4 * d4);
      }
    }
    float mb = M;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) mb = fmaxf(mb, ml[k].x);
    const float safe = mb == -INFINITY ? 0.f : mb, keep = fast_exp2(M - safe);
    L *= keep;
    o *= keep;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const float w = fast_exp2(ml[k].x - safe);   // 0 for a part that saw nothing
      L = fmaf(ml[k].y, w, L);
      tree_add(o, av[k], w);
    }
    M = mb;
  }
  if constexpr (NW > 1) {
    if (wave > 0) {
      float* const s = state + (wave - 1) * 64 * 6 + lane;
      s[0] = M, s[64] = L, s[128] = o[0], s[192] = o[1], s[256] = o[2], s[320] = o[3];
    }
    __syncthreads();
    if (wave > 0) return;
    float mb = M;
#pragma unroll
    for (int w = 0; w < NW - 1; ++w) mb = fmaxf(mb, state[w * 64 * 6 + lane]);
    const float safe = mb == -INFINITY ? 0.f : mb, keep = fast_exp2(M - safe);
    L *= keep;
    o *= keep;
#pragma unroll
    for (int w = 0; w < NW - 1; ++w) {
      const float* const s = state + w * 64 * 6 + lane;
      const float f = fast_exp2(s[0] - safe);
      L = fmaf(s[64], f, L);
      tree_add(o, float4_t{s[128], s[192], s[256], s[320]}, f);
    }
  }
  if (lane + 64 * (int)blockIdx.y >= a.num_heads * QPH) return;
  float inv = 1.f / L;
  if (!(L > 0.f)) {
    const int seq = a.row_seq[row], r0 = a.row_starts[seq];
    if (!tree_sees(a.mask + (int64_t)row * a.mask_words, a.cached[seq], a.row_starts[seq + 1] - r0)) inv = 0.f;
  }
  typedef T t4_t __attribute__((ext_vector_type(4)));
  t4_t t;
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = (T)(o[j] * inv);
  st_through(a.out + (int64_t)row * a.out_row_bytes + ((int64_t)head * D + 4 * d4) * sizeof(T), t);
}

template <typename Tag, int D, bool SMALL>
static void launch_columns_as(const tree_args& a, int num_work, int blocks, hipStream_t stream) {
  const dim3 grid(num_work), block(256);
  if constexpr (tshape<Tag, D>::RB == 128)
    if (blocks == 1) hipLaunchKernelGGL((tree_columns_kernel<Tag, D, 1, 128, SMALL>), grid, block, 0, stream, a);
  if (blocks == 2) hipLaunchKernelGGL((tree_columns_kernel<Tag, D, 2, 64, SMALL>), grid, block, 0, stream, a);
  else if (blocks == 4) hipLaunchKernelGGL((tree_columns_kernel<Tag, D, 4, 64, SMALL>), grid, block, 0, stream, a);
}

template <typename Tag, int D>
static void launch_columns(const tree_args& a, int num_work, int blocks, int num_split, hipStream_t stream) {
  if (a.log2_bs < 4) launch_columns_as<Tag, D, true>(a, num_work, blocks, stream);
  else launch_columns_as<Tag, D, false>(a, num_work, blocks, stream);
  if (num_split > 0 && !a.arrivals) {
    const dim3 rows(num_split, (a.num_heads * (D / 4) + 63) / 64);
    // partial_slots / num_split: the parts of a row on average
    if (a.slots > 16 * (int64_t)num_split) hipLaunchKernelGGL((tree_join_kernel<Tag, D, 4>), rows, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((tree_join_kernel<Tag, D, 1>), rows, dim3(64), 0, stream, a);
  }
}

}  // namespace tb


// ---- the work list (host, no device call) ------------------------------------------
namespace {

// What a work list costs, in us, fitted to the times of 87 steps in every number of column blocks and cut
// (14 geometries and types, 1 to 100 sequences, contexts of 300 to 30000 positions, 2 to 128 nodes). Measured again on
// all of them, the list that it picks is 1.9% slower than the best cut on average, more than 5% in 11 and 26% in one
// (24 trees of 40 nodes at 14 / 2 heads of 64 in fp16, where two column blocks take 33.9 us and four 42.6). A round is a
// chunk of a workgroup. The blocks of a workgroup are part of the pick: few read K/V once more per 32 CW columns, but
// waste fewer columns and have their waves share a chunk's positions. 32 sequences of 26 nodes at 14 / 2 heads of 64 (182
// columns), 2000 positions: 19.3 us with two blocks against 21.9 with four, in fp32 (16 sequences) 32.8 against 45.8; 32
// of 32 nodes at 32 / 8 heads of 128, 8000 positions: 170 against 154. Up to 64 columns a third and fourth block would
// stand idle; one block pays in rows of 128 bytes alone (chunks of 128 positions fit the LDS twice): 64 of 4 nodes at
// 14 / 2 heads of 64, 16000 positions, 66 us against 69.
struct tree_price {
  int chunks_round;            // chunks of 32 positions in a round
  int on_cu;                   // workgroups a CU holds
  double full;                 // a CU's time for each round of a workgroup, when it holds on_cu of them
  int cus;
  double row_bytes;            // of a K or V row
};

// Chunks of a sequence's context.
inline int tree_chunks(int cached, int nodes) { return nodes > 0 ? (cached + nodes + 31) / 32 : 0; }

// A context of `chunks` in parts of up to `part` chunks (0: not cut), all of one length but the last: their
// length, a multiple of a round.
inline int tree_even(int chunks, int part, int round) {
  const int parts = part > 0 ? (chunks + part - 1) / part : 1;
  return ((chunks + parts - 1) / parts + round - 1) / round * round;
}

// What a call's partials may take. Without a bound the search cuts long contexts of large trees into hundreds of MB for
// what the price says is a few percent. Of 1500 random steps of up to 128 sequences and 130000 positions 63 are cut more
// coarsely for it, at a price 2.4% higher on average and 8.5% at most; 64 MiB would touch 111, up to 24%. Us a call without
// and with it, bf16, heads of 128: 4 trees of 1024 nodes at 32 / 8 behind 50000 to 100000 positions 4830 and 4904, 8 of
// 1024 at 64 / 8 behind 15000 to 30000 5829 and 5734, one of 773 at 40 / 40 behind 98000 1500 and 1472, 40 of 53 at 64 / 8
// behind 30000 to 60000 3908 and 4065.
constexpr double MOST_PARTIAL_BYTES = TB_TREE_MOST_PARTIAL_BYTES;

// The part length in rounds of least cost, and that cost; 0: no context is cut.
int tree_part_rounds(const tree_price& price, const int32_t* cached, const int32_t* nodes, int num_seqs, int rep,
                     int cols, int num_kv_heads, double slot_bytes, double& least) {
  constexpr double START = 4.9, START_ROUNDS = 1.8, ALONE = 1.38, BYTES_US = 6.8e6, JOIN = 0.71, JOIN_BATCH = 0.47,
                   PARTIAL_BYTES_US = 2.8e6;
  int most = 0;
  double kv_bytes = 0;
  for (int b = 0; b < num_seqs; ++b) {
    most = std::max(most, (tree_chunks(cached[b], nodes[b]) + price.chunks_round - 1) / price.chunks_round);
    kv_bytes += 64. * tree_chunks(cached[b], nodes[b]) * price.row_bytes * num_kv_heads;
  }
  std::vector<std::pair<int, int64_t>> pieces;   // (rounds, workgroups)
  auto cost = [&](int part) {
    pieces.clear();
    int64_t count = 0;
    double slots = 0;
    int most_parts = 1;
    for (int b = 0; b < num_seqs; ++b) {
      if (nodes[b] <= 0) continue;
      const int r = (tree_chunks(cached[b], nodes[b]) + price.chunks_round - 1) / price.chunks_round;
      const int even = tree_even(r, part, 1), parts = (r + even - 1) / even;
      const int64_t wgs = (int64_t)((nodes[b] * rep + cols - 1) / cols) * num_kv_heads;
      if (parts > 1) {
        pieces.push_back({even, wgs * (parts - 1)});
        slots += (double)parts * nodes[b];
        most_parts = std::max(most_parts, parts);
      }
      pieces.push_back({r - even * (parts - 1), wgs});
      count += wgs * parts;
    }
    if (slots * slot_bytes > MOST_PARTIAL_BYTES) return HUGE_VAL;
    // the longest first, each where a place is free first: a piece starts when those before it have
    // filled the places evenly
    std::sort(pieces.begin(), pieces.end(), std::greater<>());
    const bool alone = count <= price.cus;
    const double places = (double)price.cus * (alone ? 1 : price.on_cu);
    double end = 0, work = 0, seen = 0;
    for (const auto& [len, n] : pieces) {
      const double one = len + START_ROUNDS;
      const double first = seen < places ? 0 : work / places;
      const double last = seen + n - 1 < places ? 0 : (work + (n - 1) * one) / places;
      end = std::max(end, std::max(first, last) + one);
      work += n * one;
      seen += n;
    }
    const double t = end * price.full * (alone ? ALONE : price.on_cu);
    const double mem = kv_bytes / BYTES_US;
    double join = 0;
    if (slots > 0)
      join = JOIN + JOIN_BATCH * ((most_parts + 7) / (most_parts <= 16 ? 8 : 32)) + slots * slot_bytes / PARTIAL_BYTES_US;
    return START + std::cbrt(t * t * t + mem * mem * mem) + join;   // the two hide each other, less so where alike
  };
  int best = 0;
  least = cost(0);
  for (int part = 1; part < most; part += part < 6 ? 1 : part < 16 ? 2 : part < 32 ? 4 : part < 48 ? 8 : part < 96 ? 16 : 32) {
    const double c = cost(part);
    if (c < least) least = c, best = part;
  }
  return best;
}

struct tree_piece {
  int seq, kvh, chunk0, chunks, slot, groups, unit, order;   // order: part | parts << 16
};

// Whether a unit's last workgroup joins its parts. Its loads go past the L2s: for 4096 floats it takes 4 to 6 us, a
// launch 2 to 3, but 3 us more of the host, for which a short step's calls wait (12.7 us a call of two launches). So
// only little is joined there, more where the step is short and the parts come in one turn of loads. Us a call, there
// and by a launch: 13 nodes at 14 / 2 heads of 64, 600 positions, 10.5 and 12.7; 16 sequences of 18 nodes, 2000
// positions, 14.7 and 12.7; 8 of 13 in fp32 15.6 and 12.8; 8 nodes at 32 / 8 heads of 128 in 9 parts 15.6 and 12.6.
// Fewer than 2048 floats (less than one turn of the 256 threads' loads, two of four floats each) are joined there
// however long the step: 0.3 to 0.6 us more where the GPU is the slower side (16 sequences of 7 nodes at 8 / 2 heads of 64,
// 4000 positions, 12.9 and 12.4), 2.5 less where the host is (1 of 7, 600, 10.1 and 12.6). A full turn in a long step goes to
// the launch: 4 of 4 at 32 / 8 heads of 128, 4000 positions, 19.2 and 18.7 (in fp32 it would be better off there: 16 of 8 at
// 8 / 2 heads of 64, 4000 positions, 25.9 and 27.5).
constexpr int JOIN_HERE_FLOATS = 4096, JOIN_ALWAYS_FLOATS = 2048, JOIN_HERE_PARTS = 16;
constexpr double JOIN_HERE_US = 10;

}  // namespace

extern "C" int32_t tb_build_tree_work(const int32_t* cached, const int32_t* nodes, int32_t num_seqs,
                                      int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                                      int32_t num_cus, int32_t num_xcds, int32_t* work, int32_t work_capacity,
                                      int32_t* split, int32_t split_capacity, int32_t* counts) try {
  TB_CHECK_ARG(num_seqs >= 0 && num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0);
  TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16 && num_cus > 0 && num_xcds > 0 && counts);
  if (head_dim != 64 && head_dim != 128) return TB_ERR_UNSUPPORTED;
  TB_CHECK_ARG(num_seqs == 0 || (cached && nodes));
  const int rep = num_heads / num_kv_heads;
  int64_t rows = 0;
  int most_cols = 0;
  for (int b = 0; b < num_seqs; ++b) {
    TB_CHECK_ARG(cached[b] >= 0 && nodes[b] >= 0 && (int64_t)cached[b] + nodes[b] <= (1 << 30));
    TB_CHECK_ARG((int64_t)nodes[b] * rep < (1 << 28));
    most_cols = std::max(most_cols, nodes[b] * rep);
    rows += nodes[b];
  }
  TB_CHECK_ARG(rows < (1 << 30));
  const int row_bytes = head_dim * (dtype == TB_DTYPE_F32 ? 4 : 2);
  int blocks = 0, part = 0;
  double least = 0;
  for (const int n : {1, 2, 4}) {
    if (n == 1 ? most_cols > 32 || row_bytes != 128 : n == 4 && most_cols <= 64) continue;
    const double full = dtype == TB_DTYPE_F32 ? (head_dim == 64 ? (n == 2 ? 1.26 : 1.82) : n == 2 ? 3.43 : 5.61)
                        : head_dim == 128     ? (n == 2 ? 0.636 : 1.01)
                        : n == 1              ? 0.356
                        : n == 2              ? 0.353
                                              : 0.515;
    const tree_price price{n == 1 ? 4 : 2, row_bytes == 512 ? 1 : 2, full, num_cus, (double)row_bytes};
    double cost = 0;
    const int rounds = tree_part_rounds(price, cached, nodes, num_seqs, rep, 32 * n, num_kv_heads,
                                        (double)num_heads * (head_dim + 2) * 4, cost);
    if (blocks == 0 || cost < least) blocks = n, part = rounds * price.chunks_round, least = cost;
  }
  const int cols = 32 * blocks, round = blocks == 1 ? 4 : 2;
  std::vector<tree_piece> pieces;
  int64_t slots = 0, num_split = 0, row0 = 0, units = 0;
  bool here = true;
  const bool brief = least <= JOIN_HERE_US;
  std::vector<int32_t> first(num_seqs + 1);
  for (int b = 0; b < num_seqs; ++b) {
    first[b] = (int32_t)row0;
    row0 += nodes[b];
    const int all = tree_chunks(cached[b], nodes[b]);
    if (all == 0) continue;
    const int groups = (nodes[b] * rep + cols - 1) / cols, even = tree_even(all, part, round);
    const int parts = (all + even - 1) / even;
    const bool few = parts < (1 << 15);
    for (int i = 0; i < parts; ++i)
      for (int h = 0; h < num_kv_heads; ++h)
        pieces.push_back({b, h, even * i, std::min(even, all - even * i),
                          parts > 1 ? (int)(slots + (int64_t)i * nodes[b]) : -1, groups, (int)(units + h * groups),
                          few ? i | parts << 16 : 0});
    if (parts > 1) {
      const int floats = std::min(cols, nodes[b] * rep) * head_dim;   // of a part
      here &= parts <= JOIN_HERE_PARTS &&
              (floats < JOIN_ALWAYS_FLOATS || (brief && floats * ((parts + 7) / 8) <= JOIN_HERE_FLOATS));
      units += (int64_t)groups * num_kv_heads;
      for (int i = 0; i < nodes[b]; ++i, ++num_split)
        if (split && num_split < split_capacity) {
          int32_t* const s = split + 4 * num_split;
          s[0] = first[b] + i, s[1] = (int32_t)(slots + i), s[2] = parts, s[3] = nodes[b];
        }
      slots += (int64_t)parts * nodes[b];
    }
    TB_CHECK_ARG(slots < (1 << 30) && units < (1 << 30));
  }
  // longest first; the column groups of one piece, which read the same rows, on one XCD
  std::stable_sort(pieces.begin(), pieces.end(),
                   [](const tree_piece& x, const tree_piece& y) { return x.chunks > y.chunks; });
  std::vector<std::vector<std::pair<int, int>>> lists(num_xcds);
  std::vector<int64_t> load(num_xcds, 0);
  for (int i = 0; i < (int)pieces.size(); ++i) {
    const int x = (int)(std::min_element(load.begin(), load.end()) - load.begin());
    for (int g = 0; g < pieces[i].groups; ++g) lists[x].push_back({i, g});
    load[x] += (int64_t)pieces[i].groups * (pieces[i].chunks + 8);
  }
  size_t depth = 0;
  for (auto& l : lists) depth = std::max(depth, l.size());
  TB_CHECK_ARG(depth * num_xcds < ((size_t)1 << 30));
  const int64_t n = (int64_t)depth * num_xcds;
  counts[0] = (int32_t)n, counts[1] = (int32_t)num_split, counts[2] = (int32_t)slots, counts[3] = blocks;
  counts[4] = here ? (int32_t)units : 0;
  if (!work && !split) return TB_OK;
  TB_CHECK_ARG((n == 0 || work) && work_capacity >= n && (num_split == 0 || split) && split_capacity >= num_split);
  for (size_t j = 0; j < depth; ++j)
    for (int x = 0; x < num_xcds; ++x) {
      int32_t* const w = work + 12 * (j * num_xcds + x);
      std::fill(w, w + 12, 0);
      if (j >= lists[x].size()) continue;
      const tree_piece& p = pieces[lists[x][j].first];
      w[0] = first[p.seq], w[1] = p.seq, w[2] = cached[p.seq], w[3] = nodes[p.seq];
      w[4] = lists[x][j].second * cols, w[5] = p.kvh, w[6] = p.chunk0, w[7] = p.chunks;
      w[8] = p.slot, w[9] = p.groups == 1, w[10] = p.unit + lists[x][j].second, w[11] = p.order;
    }
  return TB_OK;
} catch (const std::exception&) {
  return TB_ERR_INVALID_ARG;
}

extern "C" int32_t tb_build_tree_rows(const int32_t* parents, const int32_t* row_starts, int32_t num_seqs,
                                      const int32_t* cached, const int32_t* block_tables,
                                      int32_t max_blocks_per_seq, int32_t block_size, int64_t num_blocks,
                                      uint32_t* mask, int32_t mask_words, int64_t* positions, int32_t* row_seq,
                                      int32_t* slot_mapping, int32_t* info) try {
  TB_CHECK_ARG(num_seqs >= 0 && row_starts && row_starts[0] == 0 && mask_words > 0 && info);
  std::fill(info, info + 4, 0);
  for (int b = 0; b < num_seqs; ++b)
    TB_CHECK_ARG(row_starts[b + 1] >= row_starts[b] && (row_starts[b + 1] - row_starts[b] + 31) / 32 <= mask_words);
  if (cached) {
    TB_CHECK_ARG(block_size > 0 && (block_size & (block_size - 1)) == 0 && num_blocks > 0 && max_blocks_per_seq >= 0);
    TB_CHECK_ARG((num_seqs == 0 || block_tables) && (row_starts[num_seqs] == 0 || slot_mapping));
  }
  if (row_starts[num_seqs] == 0 && !cached) return TB_OK;
  TB_CHECK_ARG(row_starts[num_seqs] == 0 || (parents && mask && positions && row_seq));
  auto fault = [&](int32_t reason, int64_t where, int32_t status) {
    info[2] = reason, info[3] = (int32_t)where;
    return status;
  };
  std::vector<int32_t> children, order, refusals;
  for (int b = 0; b < num_seqs; ++b) {
    const int row0 = row_starts[b], n = row_starts[b + 1] - row0, words = (n + 31) / 32;
    const int64_t start = cached ? cached[b] : 0;
    TB_CHECK_ARG(start >= 0 && start + n <= (1 << 30));
    children.assign(n, 0);
    order.assign(n, 0);                          // of a node among its siblings
    refusals.assign(n, 0);                       // below a node: until a child is kept, and from there on
    for (int i = 0; i < n; ++i) {
      const int p = parents[row0 + i], r = row0 + i;
      uint32_t* const m = mask + (int64_t)r * mask_words;
      if (i == 0 ? p != -1 : p < 0 || p >= i) return fault(TB_TREE_FAULT_PARENT, r, TB_ERR_INVALID_ARG);
      std::fill(m, m + mask_words, 0u);
      if (i > 0) {
        const uint32_t* const above = m - (int64_t)(i - p) * mask_words;
        std::copy(above, above + words, m);
        order[i] = children[p]++;
      }
      m[i >> 5] |= 1u << (i & 31);
      positions[r] = i > 0 ? positions[row0 + p] + 1 : start;
      row_seq[r] = b;
      info[1] = std::max<int32_t>(info[1], (int32_t)positions[r] + 1);
    }
    for (int i = n - 1; i >= 0; --i) {
      refusals[i] = std::max(refusals[i], children[i] - 1);
      if (i > 0) refusals[parents[row0 + i]] = std::max(refusals[parents[row0 + i]], order[i] + refusals[i]);
      else info[0] = std::max(info[0], refusals[0]);
    }
  }
  if (!cached) return TB_OK;
  // the blocks that nodes lie in, each with the offsets that they take there
  struct span {
    int32_t block, lo, hi;
    bool operator<(const span& o) const { return block != o.block ? block < o.block : lo < o.lo; }
  };
  std::vector<span> spans;
  std::vector<bool> taken(num_blocks, false);
  const int log2_bs = __builtin_ctz(block_size);
  for (int b = 0; b < num_seqs; ++b) {
    const int32_t* const table = block_tables + (int64_t)b * max_blocks_per_seq;
    const int row0 = row_starts[b], n = row_starts[b + 1] - row0, end = cached[b] + n;
    const int need = (int)(((int64_t)end + block_size - 1) >> log2_bs);
    if (need > max_blocks_per_seq) return fault(TB_TREE_FAULT_TABLE, b, TB_ERR_INDEX);
    for (int j = 0; j < need; ++j)
      if (table[j] < 0 || table[j] >= num_blocks) return fault(TB_TREE_FAULT_BLOCK, b, TB_ERR_INDEX);
    for (int p = cached[b]; p < end;) {
      const int block = table[p >> log2_bs], lo = p & (block_size - 1), hi = std::min(block_size, lo + end - p);
      if (((int64_t)block << log2_bs) + hi > INT32_MAX) return fault(TB_TREE_FAULT_SLOTS, b, TB_ERR_INVALID_ARG);
      for (int o = lo; o < hi; ++o) slot_mapping[row0 + p - cached[b] + o - lo] = (block << log2_bs) + o;
      spans.push_back({block, lo, hi});
      taken[block] = true;
      p += hi - lo;
    }
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].block == spans[i - 1].block && spans[i].lo < spans[i - 1].hi)
      return fault(TB_TREE_FAULT_SHARED, spans[i].block, TB_ERR_INVALID_ARG);
  // no node on a cached position, its own sequence's or another's
  for (int b = 0; b < num_seqs; ++b)
    for (int64_t j = 0; j << log2_bs < cached[b]; ++j) {
      const int block = block_tables[(int64_t)b * max_blocks_per_seq + j];
      if (!taken[block]) continue;
      const auto at = std::lower_bound(spans.begin(), spans.end(), span{block, 0, 0});
      if (at->lo < std::min<int64_t>(cached[b] - (j << log2_bs), block_size))
        return fault(TB_TREE_FAULT_CACHED, block, TB_ERR_INVALID_ARG);
    }
  return TB_OK;
} catch (const std::exception&) {
  return TB_ERR_INVALID_ARG;
}

extern "C" size_t tb_tree_attention_workspace_bytes(int32_t partial_slots, int32_t num_heads, int32_t head_dim) {
  if (partial_slots <= 0 || num_heads <= 0 || head_dim <= 0) return 0;
  return (size_t)partial_slots * num_heads * (head_dim + 2) * sizeof(float);
}

extern "C" int32_t tb_tree_attention(const void* q, int64_t q_row_stride, const void* pool, int64_t num_blocks,
                                     void* out, int64_t out_row_stride, const int32_t* block_tables,
                                     int32_t max_blocks_per_seq, const int32_t* row_starts, const int32_t* cached,
                                     int32_t num_seqs, const int32_t* row_seq, int32_t num_rows,
                                     const uint32_t* mask, int32_t mask_words, const int32_t* work,
                                     int32_t num_work, int32_t column_blocks, const int32_t* split_rows,
                                     int32_t num_split_rows, int32_t partial_slots, void* workspace,
                                     size_t workspace_bytes, uint32_t* arrivals, int32_t arrival_units,
                                     int32_t num_heads, int32_t num_kv_heads,
                                     int32_t head_dim, int32_t block_size, float scale,
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
  a.positions = positions;
  a.rope = rope_tables{rope_cos, rope_sin, rope_max_position};
  TB_CHECK_ARG(num_work >= 0 && num_split_rows >= 0 && num_split_rows <= num_rows && partial_slots >= 0);
  TB_CHECK_ARG((column_blocks == 1 && head_dim * eb == 128) || column_blocks == 2 || column_blocks == 4);
  TB_CHECK_ARG((num_split_rows == 0 || partial_slots > 0));
  if (num_work == 0) return TB_OK;
  TB_CHECK_ARG(work && ((uintptr_t)work & 15u) == 0 && (num_split_rows == 0 || split_rows) &&
               ((uintptr_t)split_rows & 15u) == 0);
  if (partial_slots > 0)
    TB_CHECK_ARG(workspace && ((uintptr_t)workspace & 15u) == 0 &&
                 workspace_bytes >= tb_tree_attention_workspace_bytes(partial_slots, num_heads, head_dim));
  TB_CHECK_ARG(!arrivals || (arrival_units > 0 && ((uintptr_t)arrivals & 3u) == 0));
  a.arrivals = partial_slots > 0 ? arrivals : nullptr;
  a.work = (const int4*)work;
  a.split = (const int4*)split_rows;
  a.ws_acc = (float*)workspace;
  a.slots = partial_slots;
  a.ws_ml = (float*)workspace + (size_t)partial_slots * num_heads * head_dim;
  const float s2 = fabsf(scale) * 1.4426950408889634f;
  a.scale_log2e = s2 > 0.f ? s2 : 1.f;
  a.q_sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : scale;   // 0, or a NaN
  const bool d64 = head_dim == 64;
  if (dtype == TB_DTYPE_F32)
    d64 ? launch_columns<f32_t, 64>(a, num_work, column_blocks, num_split_rows, stream)
        : launch_columns<f32_t, 128>(a, num_work, column_blocks, num_split_rows, stream);
  else if (dtype == TB_DTYPE_F16)
    d64 ? launch_columns<f16_t, 64>(a, num_work, column_blocks, num_split_rows, stream)
        : launch_columns<f16_t, 128>(a, num_work, column_blocks, num_split_rows, stream);
  else
    d64 ? launch_columns<bf16_t, 64>(a, num_work, column_blocks, num_split_rows, stream)
        : launch_columns<bf16_t, 128>(a, num_work, column_blocks, num_split_rows, stream);
  TB_RETURN_LAUNCH_STATUS();
}
