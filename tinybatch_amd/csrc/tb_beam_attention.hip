// Attention of one new token per beam over the paged cache.
//
// Row r (a beam of request g) sees the positions 0 .. row_ctx[r] - 1 of its block table; the leading
// shared[g] blocks of a request's rows are the same, c = shared[g] bs positions. Per row and query head
//   out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),  s_t = scale q . k_t,  m a maximum of the s_t,
// taken over 0 .. c - 1 and c .. row_ctx - 1 apart and joined: sums against different maxima m1, m2 add
// up after a factor of e^(m1 - m), e^(m2 - m).
//
// Work: the shared positions of a request are read once for all its rows: its beams and the rep query heads of
// a kv head make beams * rep columns, column = beam * rep + head, that meet the same K/V. The positions behind
// them make rep columns per row. Both are cut into parts of P positions (tb_beam_plan, on the GPU: the lengths are
// known there alone), a workgroup of four waves each, which walks its part in chunks of CK positions through a ring of
// two in LDS: every wave loads a quarter of the next chunk (direct global->LDS loads) and computes on the present
// one, one barrier between. A wave holds 32 columns; with CW < 4 sets of 32 several waves hold the same
// ones, each a part of a chunk's positions, and join their softmax states in LDS at the end. A row of one part
// is written at once, the parts of the others are joined by a second launch.
//
// Math per chunk and 32 columns (C rows are positions or dims, C columns the block's):
//   S^T[pos][col] = K[pos][:] . q[col][:]        A = K rows from LDS, B = q in registers
//   O^T[d][col]  += V^T[d][pos] . P^T[pos][col]  A = V^T from LDS, B = the S^T registers
// 16-bit: v_mfma_f32_32x32x16, V^T by LDS transpose reads; the weights P are rounded to the element type, which the
// product takes, and their sum is taken of the rounded ones. fp32: v_mfma_f32_32x32x2_f32, nothing rounded
// further. A column's reference maximum moves only when a score outgrows it by 8 (weights to 2^8), so that
// the accumulators are rescaled a few times per part. fp16 weights end at 2^-25: they refer to a maximum 7 lower.
//
// What bounds it: the K/V from memory where they are many (24 requests of 4 beams behind prompts of 1024 to 24000 positions at
// 32 / 8 heads of 128, bf16, 1.1 GB: 174 us, 6.4 TB/s, and 4.6 for the join); else a part's start, its chunks' latency and the join's launch
// (32 requests of 8 beams at 14 / 2 heads of 64, 57 MB: 14 + 4 us). Parts joined by the workgroup that ends last instead of
// by a launch: 21.3 us against 17 there, 24.7 against 16.6 for one request of 4 beams behind 8000 positions; a row's partials
// have to be in memory before they are counted, which the end of a launch does for all at once.
// fp32 over long contexts the waves: at 256 and 512 bytes a position's row a workgroup has places for 64 columns (OWN), and with up to
// 32 of them two of its four waves have none, while the products of the others take 16 times as long as in 16 bits. 16 requests of 4
// beams behind 4000 to 12000 positions: 14 / 2 heads of 64 58 us (164 MB, 2.8 TB/s; 16 bits: 18.3 and 4.5), 32 / 8 of 128 414 us (1.3 GB,
// 3.2 TB/s; 16 bits, bf16 as fp16: 102 to 104 and 6.4); one request of 4 behind 8000: 18.6 (14.1) and 41 (15.7).
#include <type_traits>

#include "tb_stream.h"

namespace tb {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_STEP = 128;                     // parts are multiples of it
// K/V of this many bytes are loaded past the caches' replacement, where one workgroup alone reads them: 1.1 GB (24 requests of 4
// beams at 32 / 8 heads of 128) 178 us against 190. Less may still lie in the 256 MB behind the L2s from the last time: 57 MB (32
// of 8 at 14 / 2 heads of 64, three such pools in turn) 16.7 us against 20.8.
constexpr int64_t PLAN_STREAM = (int64_t)256 << 20;
constexpr int PLAN_CUS = 256, PLAN_MOST = 2048;    // parts, over all kv heads: at least, where there is enough to read; at most

struct beam_args {
  const char* q;               // [R][Hq][D]
  int64_t q_row_bytes;
  const char* pool;            // [NB][2][Hkv][bs][D]
  int64_t num_blocks;
  char* out;                   // [R][Hq*D]
  int64_t out_row_bytes;
  const int32_t* block_tables; // [R][max_nb]
  int32_t max_nb, rows, beams;
  int32_t num_heads, num_kv_heads, rep;
  int32_t log2_bs;
  const int32_t* head;         // of the plan: {entries, P, whether K/V are loaded past the caches' replacement}
  const int4* entries;         // two per part
  const int4* row_parts;       // [R]: {first slot, parts} of the shared positions, {first slot, parts} of its own
  float* ws_acc;               // [slots][Hq][D]
  float* ws_ml;                // [slots][Hq][2]
  float scale_log2e;           // > 0: the scale's size times log2(e), or 1 for a scale of 0
  float q_sign;                // 1, -1 or 0 (NaN: a NaN scale): multiplies q
};

// ---- the plan -----------------------------------------------------------------------
struct plan_args {
  const int32_t* row_ctx;      // [R]
  const int32_t* shared;       // [R / beams]
  int32_t rows, beams, log2_bs, max_nb;
  int32_t col_blocks;          // workgroups that a part of shared positions takes for its columns
  int32_t own_blocks;          // the same of a row's own positions
  int32_t block_cols, own_cols;   // columns of one
  int32_t kv_heads, row_bytes;    // row_bytes: of a position's K and V of a kv head
  int32_t max_entries;
  int64_t max_slots;
  int32_t* head;               // {entries, P, whether the K/V are more than the caches behind the L2s hold}
  int4* entries;
  int4* row_parts;
};

// Sums over the workgroup, in every thread.
__device__ __forceinline__ int64_t plan_sum(int64_t x, int64_t* lds) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x += __shfl_xor(x, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = 0;
  for (int w = 0; w < PLAN_THREADS / 64; ++w) x += lds[w];
  return x;
}
// Exclusive running sum over the workgroup, and the whole.
__device__ __forceinline__ int plan_scan(int x, int (*waves)[PLAN_THREADS / 64], int turn, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int up = x;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int y = __shfl_up(up, o);
    if (lane >= o) up += y;
  }
  if (lane == 63) waves[turn & 1][wave] = up;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < PLAN_THREADS / 64; ++w) {
    if (w < wave) before += waves[turn & 1][w];
    total += waves[turn & 1][w];
  }
  return before + up - x;
}

// The length of the parts: a part has a start and an end (its first loads, its partials) that cost as much as a few hundred
// positions, and the last parts to run leave the GPU half empty, the longer the longer they are. Both weigh the
// same near 32 sqrt(bytes in all) bytes a part: bf16, 32 requests of 8 beams at 14 / 2 heads of 64 (51 MB of K/V) 17 us at
// parts of 900, 19 at 512, 23 at 256; 24 of 4 at 32 / 8 heads of 128 (1.1 GB) 191 us at 1920, 204 at 3840, 197 at 1024.
// With little to read, parts for every CU.
__device__ __forceinline__ int64_t plan_length(int64_t positions, const plan_args& a) {
  const int64_t all = positions * a.kv_heads;
  const int64_t even = (int64_t)(32.f * sqrtf((float)all / (float)a.row_bytes));
  int64_t P = min(even, all / PLAN_CUS);
  P = max(P, all / PLAN_MOST + 1);
  return (P + PLAN_STEP - 1) / PLAN_STEP * PLAN_STEP;
}

// Rows are looked at one a thread, requests by the thread of their first row, three times over (the bytes in all, the parts that these
// make, the entries): one workgroup, 10 to 12 us for 4 to 256 rows, 13.5 for 1000, once a step for all its layers.
__global__ __launch_bounds__(PLAN_THREADS) void beam_plan_kernel(const plan_args a) {
  __shared__ int64_t lds[PLAN_THREADS / 64];
  __shared__ int waves[2][PLAN_THREADS / 64];
  __shared__ int ctx[PLAN_THREADS], common[PLAN_THREADS], at[PLAN_THREADS], from[PLAN_THREADS];
  const int tid = threadIdx.x, K = a.beams, each = PLAN_THREADS / K * K;   // rows of whole requests
  const int bs = 1 << a.log2_bs;
  // rows i0 .. of the round: positions seen; the request's shared positions and its first row that sees any
  auto look = [&](int i0) {
    const int r = i0 + tid;
    const bool mine = tid < each && r < a.rows;
    __syncthreads();                               // (the round before has been read)
    ctx[tid] = mine ? max(0, min(a.row_ctx[r], a.max_nb << a.log2_bs)) : 0;   // (never beyond the row's table)
    const int given = mine && tid % K == 0 ? a.shared[r / K] : 0;
    __syncthreads();
    if (mine && tid % K == 0) {
      int least = INT32_MAX, live = -1;
      for (int k = K - 1; k >= 0; --k)
        if (ctx[tid + k] > 0) least = min(least, ctx[tid + k]), live = r + k;
      // whole blocks that every row which sees anything sees whole
      common[tid] = live < 0 || K == 1 ? 0 : max(0, min(given, least >> a.log2_bs)) * bs;
      from[tid] = live;
    }
    __syncthreads();
    return mine;
  };
  auto parts = [](int64_t n, int64_t P) { return (int)((max(n, (int64_t)0) + P - 1) / P); };
  int64_t all = 0;
  for (int i0 = 0; i0 < a.rows; i0 += each) {
    if (!look(i0)) continue;
    const int c = common[tid / K * K];
    all += (int64_t)max(0, ctx[tid] - c) * a.own_blocks + (tid % K == 0 ? (int64_t)c * a.col_blocks : 0);
  }
  all = plan_sum(all, lds);
  int64_t P = plan_length(all, a), shared_parts;
  for (;;) {                                       // longer parts until the partials fit
    int64_t shared = 0, own = 0;
    for (int i0 = 0; i0 < a.rows; i0 += each) {
      if (!look(i0)) continue;
      const int c = common[tid / K * K];
      own += parts(ctx[tid] - c, P);
      if (tid % K == 0) shared += parts(c, P);
    }
    shared_parts = plan_sum(shared, lds);
    if (shared_parts * K + plan_sum(own, lds) <= a.max_slots || P >= ((int64_t)1 << 31)) break;
    P *= 2;
  }
  // entries and slots: all requests' shared parts, which are the longer ones, then the rows' own
  auto put = [&](int64_t e, int row0, int n, int table, int64_t p0, int64_t p1, int col, int part, int shared) {
    if (e >= a.max_entries) return;
    a.entries[2 * e] = make_int4(row0, n, table, (int)p0);
    a.entries[2 * e + 1] = make_int4((int)p1, col, part, shared);
  };
  int part0 = 0, own0 = 0, turn = 0;
  for (int i0 = 0; i0 < a.rows; i0 += each) {
    const bool mine = look(i0);
    const int head = tid / K * K, c = mine ? common[head] : 0, n = ctx[tid], r = i0 + tid;
    const int shared = mine && tid == head ? parts(c, P) : 0, own = mine ? parts(n - c, P) : 0;
    int total;
    const int s = part0 + plan_scan(shared, waves, turn++, total);
    part0 += total;
    const int o = own0 + plan_scan(own, waves, turn++, total);
    own0 += total;
    at[tid] = s;
    __syncthreads();
    if (!mine) continue;
    const int first = at[head], mine_shared = parts(c, P);
    a.row_parts[r] = n > 0 ? make_int4(first * K + tid - head, mine_shared, (int)shared_parts * K + o, own) : make_int4(0, 0, 0, 0);
    for (int x = tid - head; x < mine_shared * a.col_blocks; x += K) {   // the request's threads in turn
      const int p = x / a.col_blocks, b = x - p * a.col_blocks;
      put((int64_t)(first + p) * a.col_blocks + b, i0 + head, K, from[head], p * P, min((p + 1) * P, (int64_t)c), b * a.block_cols,
          p, 1);
    }
    for (int x = 0; x < own * a.own_blocks; ++x) {
      const int p = x / a.own_blocks, b = x - p * a.own_blocks;
      put(shared_parts * a.col_blocks + (int64_t)(o + p) * a.own_blocks + b, r, 1, r, c + p * P, min(c + (p + 1) * P, (int64_t)n),
          b * a.own_cols, p, 0);
    }
  }
  if (tid == 0) {
    a.head[0] = (int)min(shared_parts * a.col_blocks + (int64_t)own0 * a.own_blocks, (int64_t)a.max_entries);
    a.head[1] = (int)min(P, (int64_t)INT32_MAX);
    a.head[2] = all * a.kv_heads * a.row_bytes >= PLAN_STREAM;
  }
}

// ---- columns over the matrix unit -----------------------------------------------------
// K row r keeps its 16-byte piece p in slot p ^ kswz(r), V row r in slot p ^ vswz(r), so that the operand
// reads of 16 (K) and 32 (V, 16-bit transpose reads) lanes cover all 64 banks.
template <typename Tag, int D>
struct bshape {
  static constexpr int EB = elem<Tag>::bytes;
  static constexpr int RB = EB * D;             // bytes per K or V row
  static constexpr int TB = 16 * RB;            // bytes of a 16-position tile
  static constexpr int PPR = RB / 16;           // 16-byte pieces per row
  static constexpr int RPL = 64 / PPR;          // rows per direct load
  static constexpr int QS = PPR / 2;            // 16-byte pieces of a lane's q (the other half's lane holds the rest)
  static constexpr int NB = D / 32;             // O^T blocks of 32 dims
  static constexpr int OWN = RB == 128 ? 1 : 2; // sets of 32 columns of a workgroup for a row's own positions
  static constexpr int chunk(int cw) { return cw == 1 ? 128 : 64; }
  static __device__ __forceinline__ int kswz(int r) { return RB == 128 ? (r & 7) ^ ((r >> 3) & 1) : r & 15; }
  static __device__ __forceinline__ int vswz(int r) {
    return EB == 4 ? 0 : D == 64 ? 2 * (r & 3) : (0xCA60 >> (4 * (r & 3))) & 15;
  }
  static constexpr int lds(int cw) {
    const int ring = 2 * 2 * chunk(cw) * RB, states = cw < 4 ? 4 * 64 * (16 * NB + 2) * 4 : 0;
    return ring > states ? ring : states;
  }
};

// One part: CW sets of 32 columns from col0 on, 4 / CW waves each.
template <typename Tag, int D, int CW>
__device__ __forceinline__ void beam_part(const beam_args& a, char* lds, const int4 e0, const int4 e1, int kvh) {
  using S = bshape<Tag, D>;
  constexpr bool F32 = S::EB == 4;
  using T = typename elem<Tag>::type;
  constexpr int CK = S::chunk(CW), RB = S::RB, NB = S::NB, QS = S::QS, HALF = CK * RB, SLOT = 2 * HALF;
  constexpr int SETS = 4 / CW, TL = CK / 32 / SETS;   // waves on a column; 32-position tiles a wave takes of a chunk
  constexpr int TILES = CK / 64;                // 16-position tiles a wave loads of a chunk
  constexpr int WS = 64 * (16 * NB + 2);        // floats of a wave's state
  static_assert(TL >= 1 && TILES >= 1, "a tile for every wave");
  constexpr float LIFT = std::is_same_v<T, _Float16> ? 7.f : 0.f;   // of the weights, in powers of two

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, lcol = lane & 31, half = lane >> 5;
  const int row0 = e0.x, nrows = e0.y, table_row = e0.z, p0 = e0.w, p1 = e1.x, part = e1.z;
  const int ncols = nrows * a.rep, col0 = e1.y + 32 * (wave % CW), set = wave / CW;
  const int col = min(col0 + lcol, ncols - 1), my_row = col / a.rep, hd = kvh * a.rep + col - my_row * a.rep;
  const bool busy = col0 < ncols, once = ncols <= 32 * CW && a.head[2];   // (no other workgroup reads these K/V rows)

  const int4 parts = a.row_parts[row0 + my_row];
  vec16 q[QS];
  {
    const char* const qrow = a.q + (int64_t)(row0 + my_row) * a.q_row_bytes + (int64_t)hd * RB + 16 * half;
#pragma unroll
    for (int s = 0; s < QS; ++s) q[s] = ld16(qrow + 32 * s);
  }
  // ---- direct loads ----
  const int64_t head_bytes = ((int64_t)1 << a.log2_bs) * RB;
  const int64_t blk_bytes = 2 * (int64_t)a.num_kv_heads * head_bytes, v_off = a.num_kv_heads * head_bytes;
  const int sub_mask = (1 << (a.log2_bs - 4)) - 1;
  const int32_t* const table = a.block_tables + (int64_t)table_row * a.max_nb;
  const char* const pool_kvh = a.pool + kvh * head_bytes;
  const int last_tile = (p1 - 1) >> 4, tile0 = (p0 >> 4) + TILES * wave;
  const int lrow = lane / S::PPR, lpiece = lane % S::PPR;
  const int n = (p1 - p0 + CK - 1) / CK;
  int id0 = 0;
  auto tile_of = [&](int k, int t) { return min(tile0 + CK / 16 * k + t, last_tile); };
  auto load_ids = [&](int k) {                  // lane j: the block of tile j % TILES of chunk k + j / TILES
    const int b = table[(16 * tile_of(k + lane / TILES, lane % TILES)) >> a.log2_bs];
    return (b < 0 || b >= a.num_blocks) ? 0 : b;   // stay inside the pool, whatever the table holds
  };
  int ids = load_ids(0);
  asm volatile("" : "+v"(ids));                 // the block ids have landed: no wait inside the loop
  auto issue = [&](int k) {
    if (k - id0 >= 64 / TILES) {                // uniform, once per 64 or 32 chunks
      id0 = k;
      ids = load_ids(k);
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int tile = tile_of(k, t), rmax = p1 - 1 - 16 * tile;   // rows past it repeat the last position
      char* const dst = lds + (k & 1) * SLOT + (TILES * wave + t) * S::TB;
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
  };
  issue(0);
  if (a.q_sign != 1.f) {
    constexpr int E = 16 / sizeof(T);
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
    for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(q[s].w[i]));   // q has landed before the loop

  uint32_t ones = 0;                            // in a register: as a literal the bf16 dot product read it wrong
  if constexpr (!F32) ones = cmath<Tag>::ONES;
  asm volatile("" : "+v"(ones));
  float m = -INFINITY, l = 0.f;
  float16_t acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[b][r] = 0.f;
  uint32_t ka[QS], va[NB];                      // LDS offsets of this lane's operands of tile 0
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
  auto step = [&](int k, auto last) {
    // the wave's loads of chunk k have landed and its reads of chunk k - 1 are done: behind the barrier
    // all of chunk k is in LDS and the other slot is free
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (k + 1 < n) issue(k + 1);
    if (!busy) return;
    const char* const base = lds + (k & 1) * SLOT + set * (32 * TL * RB);
    const int left = p1 - (p0 + CK * k + 32 * TL * set);   // positions of the part from the wave's first on
    if (last.value && left <= 0) return;
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
    // ---- online softmax; register r of tile t holds position 32 t + 8 (r / 4) + 4 half + r % 4 ----
    if constexpr (last.value) {
#pragma unroll
      for (int t = 0; t < TL; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * t + 8 * (r >> 2) + 4 * half + (r & 3) >= left) sc[t][r] = -INFINITY;
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
    if constexpr (F32) {
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
  int k = 0;
  for (; k < n - 1; ++k) step(k, std::false_type{});
  step(k, std::true_type{});

  // ---- the sets' states joined, the output or a partial ----
  l = sum_xor32(l);
  const bool mine = col0 + lcol < ncols;
  const int row = row0 + my_row;
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
      f[s] = fast_exp2(all[s * CW * WS + 64 * 16 * NB] - safe);   // 0 for a set without positions
      l += all[s * CW * WS + 64 * (16 * NB + 1)] * f[s];
    }
  }
  if (!mine) return;
  if (parts.y + parts.w == 0) return;           // a row that sees nothing, among rows that do
  const bool whole = parts.y + parts.w == 1;
  const int slot = e1.w ? parts.x + part * a.beams : parts.z + part;
  const float inv = whole ? 1.f / l : 1.f;
  typedef T t4_t __attribute__((ext_vector_type(4)));
  const int64_t at = (int64_t)slot * a.num_heads + hd;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {               // dims 32 b + 8 g + 4 half ..: the group of set g % SETS
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
      if (whole) {
        t4_t t;
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = (T)(o[j] * inv);
        st_through(a.out + (int64_t)row * a.out_row_bytes + (int64_t)hd * RB + (32 * b + 8 * g + 4 * half) * S::EB, t);
      } else {
        *reinterpret_cast<float4_t*>(a.ws_acc + at * D + 32 * b + 8 * g + 4 * half) = o;
      }
    }
  if (!whole && half == 0 && set == 0) *reinterpret_cast<float2*>(a.ws_ml + at * 2) = make_float2(m, l);
}

template <typename Tag, int D, int CW>
constexpr int BEAM_LDS = bshape<Tag, D>::lds(CW) > bshape<Tag, D>::lds(bshape<Tag, D>::OWN)
                             ? bshape<Tag, D>::lds(CW) : bshape<Tag, D>::lds(bshape<Tag, D>::OWN);

template <typename Tag, int D, int CW>
__global__ __launch_bounds__(256, (BEAM_LDS<Tag, D, CW> <= 81920 ? 2 : 1)) void beam_columns_kernel(const beam_args a) {
  using S = bshape<Tag, D>;
  __shared__ __align__(1024) char lds[BEAM_LDS<Tag, D, CW>];
  const int entry = blockIdx.x / a.num_kv_heads, kvh = blockIdx.x - entry * a.num_kv_heads;
  if (entry >= a.head[0]) return;
  const int4 e0 = a.entries[2 * entry], e1 = a.entries[2 * entry + 1];
  if (CW == S::OWN || e1.w) beam_part<Tag, D, CW>(a, lds, e0, e1, kvh);
  else beam_part<Tag, D, S::OWN>(a, lds, e0, e1, kvh);
}

// The parts of a row joined: thread = 4 dims of a head. Rows that see nothing give 0.
template <typename Tag, int D>
__global__ __launch_bounds__(256) void beam_join_kernel(const beam_args a) {
  using T = typename elem<Tag>::type;
  constexpr int QPH = D / 4, BATCH = 8;
  const int row = blockIdx.x, col = blockIdx.y * 256 + threadIdx.x;
  const int4 parts = a.row_parts[row];
  const int n = parts.y + parts.w;
  if (n == 1 || col >= a.num_heads * QPH) return;
  const int head = col / QPH, d4 = col - head * QPH;
  float M = -INFINITY, L = 0.f;
  float4_t o = float4_t{0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < n; p0 += BATCH) {
    float2 ml[BATCH];
    float4_t av[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      av[k] = float4_t{0.f, 0.f, 0.f, 0.f};
      const int p = p0 + k;
      if (p < n) {
        const int slot = p < parts.y ? parts.x + p * a.beams : parts.z + p - parts.y;
        const int64_t at = (int64_t)slot * a.num_heads + head;
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
      const float w = fast_exp2(ml[k].x - safe);
      L = fmaf(ml[k].y, w, L);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(av[k][j], w, o[j]);
    }
    M = mb;
  }
  const float inv = n ? 1.f / L : 0.f;
  typedef T t4_t __attribute__((ext_vector_type(4)));
  t4_t t;
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = (T)(o[j] * inv);
  st_through(a.out + (int64_t)row * a.out_row_bytes + ((int64_t)head * D + 4 * d4) * sizeof(T), t);
}

// What a plan of these sizes holds, the same for the plan's launch, the attention's and their callers.
struct beam_sizes {
  int cw, own;                 // sets of 32 columns of a workgroup: shared positions, a row's own
  int col_blocks, own_blocks;
  int64_t entries, slots, row_parts, list, plan_bytes;
  beam_sizes(int64_t rows, int64_t beams, int64_t heads, int64_t kv_heads, int64_t head_dim, int32_t dtype) {
    const int64_t rep = heads / kv_heads, cols = beams * rep, row_bytes = head_dim * (dtype == TB_DTYPE_F32 ? 4 : 2);
    own = row_bytes == 128 ? 1 : 2;
    cw = cols <= 32 * own ? own : cols <= 64 ? 2 : 4;
    col_blocks = (int)((cols + 32 * cw - 1) / (32 * cw));
    own_blocks = (int)((rep + 32 * own - 1) / (32 * own));
    const int64_t most_parts = PLAN_MOST / kv_heads + 1;   // but for a part of every request and row
    entries = rows / beams * col_blocks + rows * own_blocks + most_parts;
    const int64_t slot_bytes = heads * (head_dim + 2) * 4, least = 2 * rows;
    slots = TB_BEAM_PARTIAL_BYTES / slot_bytes;
    const int64_t most = most_parts * beams + least;   // a part of shared positions has a slot per beam
    if (slots > most) slots = most;
    if (slots < least) slots = least;
    row_parts = 64;
    list = row_parts + 16 * rows;
    plan_bytes = list + 32 * entries;
  }
};

template <typename Tag, int D>
static void launch_beams(const beam_args& a, const beam_sizes& z, hipStream_t stream) {
  const dim3 grid((unsigned)(z.entries * a.num_kv_heads)), block(256);
  if constexpr (bshape<Tag, D>::OWN == 1)
    if (z.cw == 1) hipLaunchKernelGGL((beam_columns_kernel<Tag, D, 1>), grid, block, 0, stream, a);
  if (z.cw == 2) hipLaunchKernelGGL((beam_columns_kernel<Tag, D, 2>), grid, block, 0, stream, a);
  if (z.cw == 4) hipLaunchKernelGGL((beam_columns_kernel<Tag, D, 4>), grid, block, 0, stream, a);
  const dim3 join(a.rows, (a.num_heads * (D / 4) + 255) / 256);
  hipLaunchKernelGGL((beam_join_kernel<Tag, D>), join, block, 0, stream, a);
}

static int32_t check_beams(int32_t rows, int32_t beams, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype,
                           int32_t block_size) {
  TB_CHECK_ARG(rows >= 0 && rows < (1 << 20) && beams > 0 && beams <= TB_BEAMS_MAX && rows % beams == 0);
  TB_CHECK_ARG(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 4096);
  TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16);
  TB_CHECK_ARG(block_size > 0 && (block_size & (block_size - 1)) == 0);
  if ((head_dim != 64 && head_dim != 128) || block_size < 16) return TB_ERR_UNSUPPORTED;
  return TB_OK;
}

}  // namespace tb

extern "C" size_t tb_beam_plan_bytes(int32_t num_rows, int32_t beams, int32_t num_heads, int32_t num_kv_heads,
                                     int32_t head_dim, int32_t dtype) {
  if (tb::check_beams(num_rows, beams, num_heads, num_kv_heads, head_dim, dtype, 16) != TB_OK) return 0;
  return (size_t)tb::beam_sizes(num_rows, beams, num_heads, num_kv_heads, head_dim, dtype).plan_bytes;
}

extern "C" size_t tb_beam_attention_workspace_bytes(int32_t num_rows, int32_t beams, int32_t num_heads,
                                                    int32_t num_kv_heads, int32_t head_dim, int32_t dtype) {
  if (tb::check_beams(num_rows, beams, num_heads, num_kv_heads, head_dim, dtype, 16) != TB_OK) return 0;
  const tb::beam_sizes z(num_rows, beams, num_heads, num_kv_heads, head_dim, dtype);
  return (size_t)(z.slots * num_heads * (head_dim + 2) * 4);
}

extern "C" int32_t tb_beam_plan(const int32_t* row_ctx, const int32_t* shared_blocks, int32_t num_rows, int32_t beams,
                                int32_t max_blocks_per_row, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                int32_t block_size, int32_t dtype, void* plan, size_t plan_bytes, hipStream_t stream) {
  using namespace tb;
  const int32_t st = check_beams(num_rows, beams, num_heads, num_kv_heads, head_dim, dtype, block_size);
  if (st != TB_OK) return st;
  TB_CHECK_ARG(max_blocks_per_row > 0 && (int64_t)max_blocks_per_row * block_size < ((int64_t)1 << 31));
  if (num_rows == 0) return TB_OK;
  const beam_sizes z(num_rows, beams, num_heads, num_kv_heads, head_dim, dtype);
  TB_CHECK_ARG(row_ctx && shared_blocks && plan && ((uintptr_t)plan & 15u) == 0 && plan_bytes >= (size_t)z.plan_bytes);
  TB_CHECK_ARG(z.entries * num_kv_heads < ((int64_t)1 << 31) && z.slots < ((int64_t)1 << 31));
  plan_args a;
  a.row_ctx = row_ctx, a.shared = shared_blocks, a.rows = num_rows, a.beams = beams;
  a.log2_bs = __builtin_ctz((unsigned)block_size), a.max_nb = max_blocks_per_row;
  a.col_blocks = z.col_blocks, a.own_blocks = z.own_blocks, a.block_cols = 32 * z.cw, a.own_cols = 32 * z.own;
  a.kv_heads = num_kv_heads, a.row_bytes = 2 * head_dim * (dtype == TB_DTYPE_F32 ? 4 : 2);
  a.max_entries = (int32_t)z.entries, a.max_slots = z.slots;
  char* const p = (char*)plan;
  a.head = (int32_t*)p, a.row_parts = (int4*)(p + z.row_parts), a.entries = (int4*)(p + z.list);
  hipLaunchKernelGGL(beam_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, stream, a);
  TB_RETURN_LAUNCH_STATUS();
}

extern "C" int32_t tb_beam_attention(const void* q, int64_t q_row_stride, const void* pool, int64_t num_blocks,
                                     void* out, int64_t out_row_stride, const int32_t* block_tables,
                                     int32_t max_blocks_per_row, int32_t num_rows, int32_t beams, int32_t num_heads,
                                     int32_t num_kv_heads, int32_t head_dim, int32_t block_size, float scale,
                                     int32_t dtype, const void* plan, size_t plan_bytes, void* workspace,
                                     size_t workspace_bytes, hipStream_t stream) {
  using namespace tb;
  const int32_t st = check_beams(num_rows, beams, num_heads, num_kv_heads, head_dim, dtype, block_size);
  if (st != TB_OK) return st;
  TB_CHECK_ARG(max_blocks_per_row > 0 && (int64_t)max_blocks_per_row * block_size < ((int64_t)1 << 31) && num_blocks > 0);
  if (num_rows == 0) return TB_OK;
  const int eb = dtype == TB_DTYPE_F32 ? 4 : 2;
  const int64_t width = (int64_t)num_heads * head_dim;
  TB_CHECK_ARG(q && pool && out && block_tables && plan && workspace);
  TB_CHECK_ARG(num_rows == 1 || (q_row_stride >= width && out_row_stride >= width));
  TB_CHECK_ARG((((uintptr_t)q | (uintptr_t)pool | (uintptr_t)out | (uintptr_t)plan | (uintptr_t)workspace) & 15u) == 0);
  TB_CHECK_ARG(num_rows == 1 || (q_row_stride * eb % 16 == 0 && out_row_stride * eb % 16 == 0));
  const beam_sizes z(num_rows, beams, num_heads, num_kv_heads, head_dim, dtype);
  const int64_t slot_rows = z.slots * num_heads;
  TB_CHECK_ARG(plan_bytes >= (size_t)z.plan_bytes && workspace_bytes >= (size_t)(slot_rows * (head_dim + 2) * 4));
  TB_CHECK_ARG(z.entries * num_kv_heads < ((int64_t)1 << 31));
  beam_args a;
  a.q = (const char*)q, a.q_row_bytes = q_row_stride * eb, a.pool = (const char*)pool, a.num_blocks = num_blocks;
  a.out = (char*)out, a.out_row_bytes = out_row_stride * eb, a.block_tables = block_tables;
  a.max_nb = max_blocks_per_row, a.rows = num_rows, a.beams = beams;
  a.num_heads = num_heads, a.num_kv_heads = num_kv_heads, a.rep = num_heads / num_kv_heads;
  a.log2_bs = __builtin_ctz((unsigned)block_size);
  const char* const p = (const char*)plan;
  a.head = (const int32_t*)p, a.row_parts = (const int4*)(p + z.row_parts), a.entries = (const int4*)(p + z.list);
  a.ws_acc = (float*)workspace, a.ws_ml = a.ws_acc + slot_rows * head_dim;
  const float size = scale < 0.f ? -scale : scale;
  a.scale_log2e = size > 0.f ? size * 1.4426950408889634f : 1.f;
  a.q_sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : scale;    // 0, or NaN
  if (dtype == TB_DTYPE_F32) {
    if (head_dim == 64) launch_beams<f32_t, 64>(a, z, stream);
    else launch_beams<f32_t, 128>(a, z, stream);
  } else if (dtype == TB_DTYPE_F16) {
    if (head_dim == 64) launch_beams<f16_t, 64>(a, z, stream);
    else launch_beams<f16_t, 128>(a, z, stream);
  } else {
    if (head_dim == 64) launch_beams<bf16_t, 64>(a, z, stream);
    else launch_beams<bf16_t, 128>(a, z, stream);
  }
  TB_RETURN_LAUNCH_STATUS();
}
