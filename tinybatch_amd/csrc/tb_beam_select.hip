// The best continuations of a request over its beams and the vocabulary.
//
// Beam k with score s_k and logits x_k: continuing with token v makes
//   c(k, v) = s_k + ((x_kv - m_k) - log S_k),  m_k = max_u x_ku,  S_k = sum_u e^(x_ku - m_k);
// a beam that has finished has one candidate, c(k, end) = s_k. Of a request's candidates the M
// largest are told; among equals the smaller beam's first, within a beam the larger logit (which c, rounded, may
// no longer show), then the smaller token.
//
// Three launches (in one, with the last workgroups to end going on, it was slower: 44 us against 33 for 32 requests of 8 beams,
// since code that does not fit the instruction cache is read again by every workgroup).
// Part 1 reads the logits once: a wave walks a run of tiles of 2048 bytes, writes the maxima of segments of the row (16 to 512
// tokens, so that a row has at most 1024, beyond 2^19 tokens several of these together) and adds up e^(x - r) against a reference r
// of the wave. Few beams: the GPU is filled by cutting rows into 16384 runs in all (8192: 26.3 us against 26.6 at 256 rows of
// 151936 in bf16, 45.3 against 44.3 at 192 rows of 128256 in fp32).
// Part 2, a workgroup per beam: its M best tokens by (x, v), which need no sum. They lie in its M best
// segments (the best tokens of the others are behind M better ones already): a threshold that at least
// M segment maxima reach and not many more, by bisection over the maxima in registers; the tokens of these segments from it up;
// their order by counting the better ones of each. Where these are many (flat rows), the M-th best of them by bisection first.
// Part 3, a workgroup per request: of its beams' lists the M best by c; up to 512 candidates find their places by halving
// the other beams' lists, of more the best ones are found by a threshold first.
// Sums of a wave's tiles, S, its logarithm and every c are in 64 bits: the order of two beams' candidates is decided
// by differences far below a float's step at the score's size.
//
// What bounds it: part 1 in fp32 the memory (192 rows, 98 MB, 18 us: 5.4 TB/s), in 16 bits the way through a wave, which has three
// tiles of a row of 151936: who counts, the first tile, its maximum, two more tiles, a sum over the lanes in 64 bits, each behind the
// one before (32 requests of 8 beams, bf16, 54 MB that count, 13.9 us: 3.9 TB/s; counted, a wave waits 69 % of its cycles, and the vector
// unit is busy 16300 of a CU's 27900 with 400 instructions a wave, half of them its tiles'). Parts 2 and 3 are chains
// of dependent steps of some 100 ns: 6 and 3 us for one request of 4 beams, 7 and 4 for 32 of 8 (M = 16), 11 and 10 for 4 of 48
// (M = 96, 150 segments a beam). In all, from a captured graph: one request 11.5 us, 32 requests 25.2, 4 of 48 beams 38.7.
#include "tb_common.h"

namespace tb {

constexpr int SELECT_LANE = 32, SELECT_TILE = 64 * SELECT_LANE;   // bytes of a lane and a wave at a time
constexpr int SELECT_SEGMENTS = 1024;              // of a row, at most
constexpr int SELECT_THREADS = 512;
constexpr int SELECT_LIST = 2048;                  // tokens from the threshold up that part 2 keeps in LDS
constexpr int MERGE_LIST = 512;                    // candidates that are ranked as they are; of more M + M / 2 + 8 at most
static_assert(MERGE_LIST == SELECT_THREADS, "a thread for every one");
constexpr float SELECT_MOST = 3.402823466e38f;

struct select_args {
  const char* logits;          // [rows][V]
  int64_t row_bytes;
  int32_t rows, beams, vocab;
  const float* scores;         // [rows]
  const uint8_t* finished;     // [rows] or null
  int32_t end_token;
  int32_t picks;               // M
  float* out_scores;           // [requests][M]
  int32_t* out_parents;
  int64_t* out_tokens;
  int32_t tiles, runs, per_run;   // tiles of a row, runs of a row, tiles of a run
  int32_t log2_lanes;          // 8 tokens 2^log2_lanes times: a segment, or the part of one in a tile
  int32_t tops;                // segment maxima that part 1 writes per row
  int32_t join, segments;      // of them in a segment (1 unless a segment is several tiles), segments of a row
  float* seg_max;              // [rows][tops]
  double2* sums;               // [rows][runs]: {S, r}, r -inf where nothing counts
  double2* norms;              // [rows]: {m, log S}
  float2* lists;               // [rows][M]: {x, token}, best first, then -inf
};

// A logit as it counts: NaN as -inf, +inf as the largest number.
__device__ __forceinline__ float select_logit(float x) { return x == x ? fminf(x, SELECT_MOST) : -INFINITY; }
__device__ __forceinline__ bool select_open(const select_args& a, int row) {   // whether the row's logits count
  return !(a.finished && a.finished[row]) && a.scores[row] > -INFINITY;
}

// 8 logits as they lie there. (Rows start at any element.)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) eight_logits {
  T v[8];
};

// Maximum over aligned groups of 2^N lanes, of numbers and infinities, or of whole numbers. (One instruction a step: the compiler
// makes a move and a three-operand maximum of a float's. A DPP source needs two wait states behind its writer.)
#define SELECT_MAX_DPP(TYPE, CTRL) \
  asm("s_nop 1\n\tv_max_" TYPE "_dpp %0, %1, %1 " CTRL " row_mask:0xf bank_mask:0xf" : "=v"(y) : "v"(x)); \
  x = y
#define SELECT_MAX_ROWS(TYPE)                                                   \
  if constexpr (N >= 1) { SELECT_MAX_DPP(TYPE, "quad_perm:[1,0,3,2]"); }        \
  if constexpr (N >= 2) { SELECT_MAX_DPP(TYPE, "quad_perm:[2,3,0,1]"); }        \
  if constexpr (N >= 3) { SELECT_MAX_DPP(TYPE, "row_half_mirror"); }            \
  if constexpr (N >= 4) { SELECT_MAX_DPP(TYPE, "row_mirror"); }
template <int N>
__device__ __forceinline__ float lanes_max(float x) {
  float y;
  SELECT_MAX_ROWS("f32")
  if constexpr (N >= 5) x = max_xor16(x);
  if constexpr (N >= 6) x = max_xor32(x);
  return x;
}
template <int N>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
  uint32_t y;
  SELECT_MAX_ROWS("u32")
  if constexpr (N >= 5) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((uint32_t)r[0], (uint32_t)r[1]);
  }
  if constexpr (N >= 6) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max((uint32_t)r[0], (uint32_t)r[1]);
  }
  return x;
}
#undef SELECT_MAX_ROWS
#undef SELECT_MAX_DPP

// Sum over the wave's lanes, in every lane.
__device__ __forceinline__ double lanes_sum(double x) {
  auto move = [](double v, auto&& f) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((int64_t)((uint64_t)f((uint32_t)(b >> 32)) << 32 | f((uint32_t)b)));
  };
  x += move(x, [](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, DPP_QUAD_XOR1, 0xf, 0xf, false); });
  x += move(x, [](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, DPP_QUAD_XOR2, 0xf, 0xf, false); });
  x += move(x, [](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, DPP_ROW_HALF_MIRROR, 0xf, 0xf, false); });
  x += move(x, [](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, DPP_ROW_MIRROR, 0xf, 0xf, false); });
  const int lane = threadIdx.x & 63;
  x += move(x, [&](uint32_t w) {
    const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return lane & 16 ? (uint32_t)r[0] : (uint32_t)r[1];
  });
  x += move(x, [&](uint32_t w) {
    const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return lane & 32 ? (uint32_t)r[0] : (uint32_t)r[1];
  });
  return x;
}

// One wave's run of a row whose logits count: tiles of 2048 bytes, 32 a lane. Terms are 2^(x l - c) with l = log2(e) and c = r l, both
// as floats, in one fused product each; what c lost is in the term of x = r as well, and the sum is divided by it: a row of
// one token sums to 1 exactly. From |r| = 2^16 on, where c could lose as much as the terms' size, they are 2^((x - r) l) (floats
// that far out differ by 0 or by more than counts, nearly). Both a subtraction and a product for every term, 8 tokens a lane and the
// reference found anew wherever a logit outgrew it by 1: 121 instructions for 8 tokens against 36, 16.6 us against 14.1 at 32
// requests of 8 beams in bf16.
template <typename T, int LANES>                   // 2^LANES lanes of a segment
__device__ __forceinline__ void select_run(const select_args& a, int row, int run, int lane) {
  constexpr int U = SELECT_LANE / sizeof(T), TILE = 64 * U, PER = 64 >> LANES;
  constexpr float LOG2E = 1.44269504088896f, FAR = 0x1p16f;
  constexpr float MOST = 50.f;                     // of a lane's terms: the reference moves when a logit outgrows it by log 50 at most
  const char* const at = a.logits + (int64_t)row * a.row_bytes;
  const int first = run * a.per_run, last = min(first + a.per_run, a.tiles), whole = min(last, a.vocab / TILE);
  const bool tells = (lane & ((1 << LANES) - 1)) == 0;
  float* const tops = a.seg_max + (int64_t)row * a.tops;
  float ref = -INFINITY, shift = NAN, unit = 1.f;   // r; -c, NaN: none or far; the term of x = r
  double sum = 0.;                                 // in units
  auto move = [&](float r) {
    const float c = r * LOG2E, was = unit;
    const bool near = fabsf(r) < FAR;
    shift = near ? -c : NAN;
    unit = near ? fast_exp2(fmaf(r, LOG2E, shift)) : 1.f;
    if (sum > 0.) sum *= exp((double)ref - (double)r) * ((double)unit / (double)was);
    ref = r;
  };
  auto most = [](const float(&x)[U]) {
    float top = fmaxf(x[0], x[1]);                 // (a NaN loses against a number)
#pragma unroll
    for (int i = 2; i < U; ++i) top = fmaxf(top, x[i]);
    return top;
  };
  auto add_up = [](auto&& term) {
    float part[2] = {term(0), term(1)};
#pragma unroll
    for (int i = 2; i < U; ++i) part[i & 1] += term(i);
    return part[0] + part[1];
  };
  auto add = [&](int t, float(&x)[U]) {
    float top = most(x);
    float part = add_up([&](int i) { return fast_exp2(fmaf(x[i], LOG2E, shift)); });
    if (__any(!(part <= MOST))) {                  // a logit outgrew the reference, or is none, or there is no reference
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = select_logit(x[i]);
      top = select_logit(top);
      const float r = lanes_max<6>(top);
      if (r > ref) move(r);
      part = 0.f;
      if (shift == shift) part = add_up([&](int i) { return fast_exp2(fmaf(x[i], LOG2E, shift)); });
      else if (ref > -INFINITY) part = add_up([&](int i) { return fast_exp2((x[i] - ref) * LOG2E); });
    }
    sum += (double)part;
    top = lanes_max<LANES>(top);
    if (tells && t * PER + (lane >> LANES) < a.tops) tops[t * PER + (lane >> LANES)] = top;
  };
  // whole tiles, the next one on its way while one is added up; the row's last, partial one by itself
  struct __attribute__((packed, aligned(sizeof(T)))) raw_t {
    T v[U];
  };
  raw_t next;
  auto fetch = [&](int t) {
    next = *reinterpret_cast<const raw_t*>(at + (int64_t)t * SELECT_TILE + SELECT_LANE * lane);
  };
  auto take = [&](float(&x)[U]) {
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = (float)next.v[i];
#pragma unroll
    for (int i = 0; i < U; ++i) asm volatile("" : "+v"(x[i]));   // (taken before the next load goes to the same registers)
  };
  if (first < whole) {
    fetch(first);
    float x[U];
    take(x);
    const float r = lanes_max<6>(most(x));
    if (fabsf(r) < FAR) move(r);
  }
  for (int t = first; t < whole; ++t) {
    float x[U];
    take(x);
    if (t + 1 < whole) fetch(t + 1);
    add(t, x);
  }
  if (whole < last) {
    float x[U];
    const int t0 = whole * TILE + U * lane;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      x[i] = (float)reinterpret_cast<const T*>(at)[min(t0 + i, a.vocab - 1)];
      if (t0 + i >= a.vocab) x[i] = -INFINITY;
    }
    add(whole, x);
  }
  sum = lanes_sum(sum);
  if (lane == 0) a.sums[(int64_t)row * a.runs + run] = make_double2(sum / (double)unit, (double)ref);
}

// A float's place among all floats, -inf 0x007FFFFF; -0 is 0.
__device__ __forceinline__ uint32_t select_order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float select_value(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
constexpr uint32_t ORDER_NONE = 0x007FFFFFu;       // of -inf

// A token's place among all of a row, larger ones first: its logit's order, then 2^30 - 1 - token, below 2^62: a positive double,
// which is compared in one instruction.
__device__ __forceinline__ double select_key(uint32_t order, int token) {
  return __longlong_as_double((int64_t)((uint64_t)order << 30 | (uint32_t)((1 << 30) - 1 - token)));
}

struct rows_lds {
  static constexpr int MOST = TB_BEAM_CANDIDATES_MAX + TB_BEAM_CANDIDATES_MAX / 2 + 8;
  double list[SELECT_LIST];                        // select_key
  uint32_t tops[SELECT_SEGMENTS];                  // orders of the segments' maxima
  double sums[SELECT_THREADS / 64];
  int picked[MOST], equal_of[MOST];
  int listed, counted;
};

// Part 2's tokens. They are looked at 512 at a time and wave: 64 >> log2_lanes segments side by side, or one of several tiles.
// each(place of the segment in `picked`, first token, how many of the 8 are not the piece's, x): as they lie there.
// TINY: rows of fewer than 8 tokens.
template <typename T, bool TINY, int AHEAD, typename F>
__device__ __forceinline__ void select_pieces(const select_args& a, const char* at, const int* picked, int n, int lane,
                                              int wave, F&& each) {
  constexpr int WAVES = SELECT_THREADS / 64;
  const int per = 64 >> a.log2_lanes, spot = lane >> a.log2_lanes, mine = lane & ((1 << a.log2_lanes) - 1);
  const int rounds = (n + WAVES * per - 1) / (WAVES * per) * a.join;   // of all waves
  for (int r0 = 0; r0 < rounds; r0 += AHEAD) {
    eight_logits<T> e[AHEAD];
    int p[AHEAD], t0[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {              // (past the end: the last round's again)
      const int r = min(r0 + u, rounds - 1), turn = r / a.join, j = r - turn * a.join;
      p[u] = (turn * WAVES + wave) * per + spot;
      const int segment = picked[min(p[u], rows_lds::MOST - 1)];
      t0[u] = p[u] < n ? (((segment * a.join + j) << a.log2_lanes) + mine) * 8 : a.vocab;
      if constexpr (TINY) {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[u].v[i] = reinterpret_cast<const T*>(at)[min(i, a.vocab - 1)];
      } else {                                     // 8 tokens inside the row: the last ones moved up
        e[u] = *reinterpret_cast<const eight_logits<T>*>(at + (int64_t)min(t0[u], a.vocab - 8) * sizeof(T));
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (r0 + u >= rounds) break;
      const int from = TINY ? 0 : min(t0[u], a.vocab - 8), skip = min(t0[u] - from, 8);
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = TINY && i >= a.vocab ? -INFINITY : (float)e[u].v[i];
      each(p[u], from, skip, x);
    }
  }
}

// Exclusive running sum of a wave's lanes, and its total.
__device__ __forceinline__ int select_scan(int x, int lane, int& total) {
  int up = x;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int y = __shfl_up(up, o);
    if (lane >= o) up += y;
  }
  total = __builtin_amdgcn_readlane(up, 63);
  return up - x;
}

// A row's list, by a workgroup of SELECT_THREADS.
template <typename T, bool TINY>
__device__ void select_list(const select_args& a, rows_lds& s, int row) {
  constexpr int WAVES = SELECT_THREADS / 64, WORDS = SELECT_SEGMENTS / 64;
  double* const list = s.list;
  int *const picked = s.picked, *const equal_of = s.equal_of;
  uint32_t* const tops = s.tops;
  int &listed = s.listed, &counted = s.counted;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), M = a.picks;
  float2* const out = a.lists + (int64_t)row * M;
  float first[SELECT_SEGMENTS / SELECT_THREADS];   // (of a row whose logits do not count: whatever is there)
#pragma unroll
  for (int i = 0; i < SELECT_SEGMENTS / SELECT_THREADS; ++i)
    first[i] = a.seg_max[(int64_t)row * a.tops + min((i * SELECT_THREADS + tid) * a.join, a.tops - 1)];
  const double2* const sums = a.sums + (int64_t)row * a.runs;
  const double2 part = sums[min(tid, a.runs - 1)];
  if (!select_open(a, row)) {                      // one candidate, the score itself, or none
    const bool one = a.finished && a.finished[row] && a.scores[row] > -INFINITY;
    for (int i = tid; i < M; i += SELECT_THREADS)
      out[i] = make_float2(one && i == 0 ? 0.f : -INFINITY, __int_as_float(a.end_token));
    if (tid == 0) a.norms[row] = make_double2(0., 0.);
    return;
  }
#pragma unroll
  for (int i = 0; i < SELECT_SEGMENTS / SELECT_THREADS; ++i) {
    const int seg = i * SELECT_THREADS + tid;
    float x = seg < a.segments ? select_logit(first[i]) : -INFINITY;
    for (int k = 1; k < a.join && seg * a.join + k < a.tops; ++k)
      x = fmaxf(x, select_logit(a.seg_max[(int64_t)row * a.tops + seg * a.join + k]));
    tops[seg] = select_order(x);
  }
  if (tid == 0) listed = 0;
  __syncthreads();
  uint32_t v[WORDS], mine = 0, mine2 = 0;          // every wave: all segments, lane l those of l + 64 i; its best and second best
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    v[i] = tops[64 * i + lane];
    mine2 = max(mine2, min(mine, v[i]));
    mine = max(mine, v[i]);
  }
  auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
  const uint32_t most = uniform(lanes_max<6>(mine));
  const float m = select_value(most);
  if (64 * wave < a.runs) {                        // S, a wave's part of the runs; their sum and its logarithm at the end
    double sum = 0.;
    if (m > -INFINITY) {
      if (tid < a.runs) sum = part.x * exp(part.y - (double)m);
      for (int r = tid + SELECT_THREADS; r < a.runs; r += SELECT_THREADS) sum += sums[r].x * exp(sums[r].y - (double)m);
    }
    sum = lanes_sum(sum);
    if (lane == 0) s.sums[wave] = sum;
  }
  // ---- the threshold: what M segments reach, or all above -inf do, and not many more ----
  auto reach = [&](uint32_t o) {
    uint64_t mask[WORDS];                          // (each in registers of its own: one register pair in turn waits 16 times)
    int c = 0;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) asm("v_cmp_le_u32 %0, %1, %2" : "=s"(mask[i]) : "s"(o), "v"(v[i]));
#pragma unroll
    for (int i = 0; i < WORDS; ++i) c += __popcll(mask[i]);
    return c;
  };
  // first the least of the best of as many groups of lanes as there are candidates wanted, at least (both of a lane's from 65 on)
  uint32_t least = M > 64 ? mine2 : mine;
  if (M <= 32) least = lanes_max<1>(least);
  if (M <= 16) least = max(least, (uint32_t)__shfl_xor((int)least, 2));
  if (M <= 8) least = max(least, (uint32_t)__shfl_xor((int)least, 4));
  uint32_t from = max(uniform(~lanes_max<6>(~least)), ORDER_NONE + 1), beyond = most + 1;
  int reached = reach(from), over = 0;             // segments that reach `from`, `beyond`
  const int few = M + M / 2 + 8;
  while (reached > few && beyond - from > 1) {
    const uint32_t mid = from + (beyond - from) / 2;
    const int c = reach(mid);
    if (c >= M) from = mid, reached = c;
    else beyond = mid, over = c;
  }
  // ---- these segments, in order; where many equal the threshold, the first ones of them ----
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  int n = 0;
  if (reached <= few) {
    int n0 = 0, n1 = 0;                            // before the wave's two words
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if (i == wave) n0 = n;
      if (i == wave + WAVES) n1 = n;
      n += __popcll(__ballot(v[i] >= from));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int seg = 64 * (wave + WAVES * h) + lane;
      const bool take = tops[seg] >= from;
      const uint64_t took = __ballot(take);
      if (take) picked[(h ? n1 : n0) + __popcll(took & below)] = seg;
    }
  } else {
    const int need = M - over;
    int equals = 0;
    for (int i = 0; i < WORDS; ++i) {
      const uint32_t o = tops[64 * i + lane];
      const uint64_t eq = __ballot(o == from);
      const bool take = o > from || (o == from && equals + (int)__popcll(eq & below) < need);
      const uint64_t took = __ballot(take);
      if (take && i % WAVES == wave) picked[n + __popcll(took & below)] = 64 * i + lane;
      equals += __popcll(eq);
      n += __popcll(took);
    }
  }
  __syncthreads();
  const char* const at = a.logits + (int64_t)row * a.row_bytes;
  // ---- the tokens from the threshold up ----
  const float threshold = select_value(from);
  select_pieces<T, TINY, 2>(a, at, picked, n, lane, wave, [&](int, int t, int skip, float(&x)[8]) {
    if (__any(skip > 0 && skip < 8)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < skip) x[i] = -INFINITY;
    }
    const float least = skip < 8 ? threshold : NAN;
    uint64_t reach[8];
    int total = 0;                                 // (of the wave, one addition for all)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      reach[i] = __ballot(x[i] >= least);          // (not NaN)
      total += __popcll(reach[i]);
    }
    if (total == 0) return;
    int place = 0;
    if (lane == 0) place = atomicAdd(&listed, total);
    place = __builtin_amdgcn_readfirstlane(place);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (reach[i] == 0) continue;
      const int mine = place + __popcll(reach[i] & (((uint64_t)1 << lane) - 1));
      if (x[i] >= least && mine < SELECT_LIST) list[mine] = select_key(select_order(select_logit(x[i])), t + i);
      place += __popcll(reach[i]);
    }
  });
  __syncthreads();
  int all = listed;
  if (all > SELECT_LIST) {
    // many of them (whole ranges of high or equal tokens): the M-th best token's value, what is above it, and as many
    // of its equals as are wanted, in order
    auto clean = [](float(&x)[8], int skip) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i < skip ? -INFINITY : select_logit(x[i]);
    };
    uint32_t t0 = from, t1 = most + 1;             // t0 is reached by M tokens, t1 by none
    while (t1 - t0 > 1) {
      const uint32_t mid = t0 + (t1 - t0) / 2;
      __syncthreads();
      if (tid == 0) counted = 0;
      __syncthreads();
      select_pieces<T, TINY, 1>(a, at, picked, n, lane, wave, [&](int, int, int skip, float(&x)[8]) {
        clean(x, skip);
        int c = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) c += select_order(x[i]) >= mid;
        if (c) atomicAdd(&counted, c);
      });
      __syncthreads();
      if (counted >= M) t0 = mid;
      else t1 = mid;
    }
    for (int i = tid; i < n; i += SELECT_THREADS) equal_of[i] = 0;
    if (tid == 0) listed = 0;
    __syncthreads();
    select_pieces<T, TINY, 1>(a, at, picked, n, lane, wave, [&](int p, int t, int skip, float(&x)[8]) {
      clean(x, skip);
      int c = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t o = select_order(x[i]);
        c += o == t0;
        if (o > t0) list[atomicAdd(&listed, 1)] = select_key(o, t + i);   // (fewer than M)
      }
      if (c) atomicAdd(&equal_of[p], c);
    });
    __syncthreads();
    if (wave == 0) {                               // running sums over the segments
      int base = 0;
      for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        int total;
        const int before = select_scan(i < n ? equal_of[i] : 0, lane, total);
        if (i < n) equal_of[i] = base + before;
        base += total;
      }
    }
    __syncthreads();
    const int over = listed, want = M - over, width = 1 << a.log2_lanes;
    int seen = 0, of = -1;                         // (segments of several tiles, one wave's: equals of the tiles before)
    select_pieces<T, TINY, 1>(a, at, picked, n, lane, wave, [&](int p, int t, int skip, float(&x)[8]) {
      clean(x, skip);
      int c = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) c += select_order(x[i]) == t0;
      int up = c;
      for (int o = 1; o < width; o *= 2) {
        const int y = __shfl_up(up, o);
        if ((lane & (width - 1)) >= o) up += y;
      }
      const int here = __shfl(up, (lane & ~(width - 1)) + width - 1);
      if (p != of) of = p, seen = 0;
      if (p < n) {
        int place = equal_of[p] + seen + up - c;
        for (int i = 0; i < 8; ++i)
          if (select_order(x[i]) == t0) {
            if (place < want) list[over + place] = select_key(t0, t + i);
            ++place;
          }
      }
      seen += here;
    });
    __syncthreads();
    all = M;
  }
  // ---- their order: how many are better, counted by a group of lanes for every entry ----
  if (tid == SELECT_THREADS - 1) {
    double sum = 0.;
    for (int w = 0; w < WAVES && 64 * w < a.runs; ++w) sum += s.sums[w];
    a.norms[row] = make_double2((double)m, log(sum));
  }
  for (int i = tid; i < M; i += SELECT_THREADS)
    if (i >= all) out[i] = make_float2(-INFINITY, 0.f);
  int share = 1;
  while (share < 64 && 2 * share * all <= SELECT_THREADS) share *= 2;
  for (int i = tid / share; i < all; i += SELECT_THREADS / share) {
    const double e = list[i];
    int c = 0;
#pragma unroll 8
    for (int j = tid % share; j < all; j += share) c += list[j] > e;
    for (int o = 1; o < share; o *= 2) c += __shfl_xor(c, o);
    const uint64_t key = (uint64_t)__double_as_longlong(e);
    const int token = (1 << 30) - 1 - (int)(key & ((1 << 30) - 1));
    if (tid % share == 0 && c < M) out[c] = make_float2(select_value((uint32_t)(key >> 30)), __int_as_float(token));
  }
}

// Part 3. A candidate's place in the order: larger value, then smaller beam, then the beam's own order.
struct merge_lds {
  double norms[TB_BEAMS_MAX][3];                   // m, log S, the score
  double value[MERGE_LIST];
  uint32_t place[MERGE_LIST];                      // beam << 8 | place in its list
  int ranks[MERGE_LIST];
  int waves[2][SELECT_THREADS / 64];
  uint32_t tops[SELECT_THREADS / 64], leasts[SELECT_THREADS / 64];
  int held;
};
// A double's place among all doubles.
__device__ __forceinline__ uint64_t merge_order(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.);
  return b >> 63 ? ~b : b | (uint64_t)1 << 63;
}

// A request's candidates from its beams' lists, by a workgroup of SELECT_THREADS.
__device__ void select_merge(const select_args& a, merge_lds& s, int request) {
  constexpr int EACH = TB_BEAMS_MAX * TB_BEAM_CANDIDATES_MAX / SELECT_THREADS, WAVES = SELECT_THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int M = a.picks, K = a.beams, row0 = request * K, all = K * M;
  const float2* const lists = a.lists + (int64_t)row0 * M;
  // the candidates of a thread, SELECT_THREADS behind each other: beam and place in its list
  const uint32_t k0 = tid / M, p0 = tid - k0 * M, dk = SELECT_THREADS / M, dp = SELECT_THREADS - dk * M;
  struct spot {
    uint32_t k, p;
  };
  auto next = [&](spot& x) {
    x.k += dk;
    x.p += dp;
    if (x.p >= (uint32_t)M) x.p -= M, ++x.k;
  };
  auto value = [&](spot at, float x) {             // -inf: none
    if (at.k >= (uint32_t)K || !(x > -INFINITY)) return -(double)INFINITY;
    return s.norms[at.k][2] + (((double)x - s.norms[at.k][0]) - s.norms[at.k][1]);
  };
  float mine[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (i * SELECT_THREADS < all) mine[i] = lists[min(i * SELECT_THREADS + tid, all - 1)].x;
  for (int i = tid; i < 2 * K; i += SELECT_THREADS) s.norms[i >> 1][i & 1] = (&a.norms[row0].x)[i];
  for (int i = tid; i < K; i += SELECT_THREADS) s.norms[i][2] = (double)a.scores[row0 + i];
  if (tid == 0) s.held = 0;
  s.ranks[tid] = 0;
  __syncthreads();
  int n;                                           // candidates in LDS
  if (all <= MERGE_LIST) {
    n = all;
    if (tid < n) {
      s.value[tid] = value({k0, p0}, mine[0]);
      s.place[tid] = k0 << 8 | p0;
    }
    __syncthreads();
    // how many are better: in its own list those before it, in another one by halving it
    const int groups = SELECT_THREADS / n, group = tid / n, i = tid - group * n;
    const double c = s.value[i];
    if (group < groups && c > -INFINITY) {
      const int k = s.place[i] >> 8, half = 1 << (31 - __clz(M));
      int better = group == 0 ? (int)(s.place[i] & 255) : 0;
      for (int other = group; other < K; other += groups) {
        if (other == k) continue;
        const double* const list = s.value + other * M;
        int lo = 0;
        for (int step = half; step; step >>= 1) {
          const double x = list[min(lo + step, M) - 1];
          const bool in = (lo + step <= M) & ((x > c) | ((x == c) & (other < k)));
          lo += in ? step : 0;
        }
        better += lo;
      }
      if (better) atomicAdd(&s.ranks[i], better);
    }
  } else {
    // by values rounded to fp32, which keeps their order but for new equals: what M candidates reach, or all there are do, and
    // not many more
    uint32_t v[EACH], top = 0;
    spot at = {k0, p0};
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      v[i] = 0;
      if (i * SELECT_THREADS < all) {
        const double x = value(at, mine[i]);
        if (x > -INFINITY) v[i] = select_order(fmaxf((float)x, -SELECT_MOST));
      }
      top = max(top, v[i]);
      next(at);
    }
    top = lanes_max<2>(top);                       // the best of every 4 threads: the least of these, which 128 candidates reach
    const uint32_t wave_top = lanes_max<6>(top), wave_least = ~lanes_max<6>(~top);
    if (lane == 0) s.tops[wave] = wave_top, s.leasts[wave] = wave_least;
    __syncthreads();
    uint32_t most = 0, least = ~0u;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) most = max(most, s.tops[w]), least = min(least, s.leasts[w]);
    int turn = 0;
    auto sum_up = [&](int c) {                     // over the waves
      if (lane == 0) s.waves[turn & 1][wave] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) c += s.waves[turn & 1][w];
      ++turn;
      return __builtin_amdgcn_readfirstlane(c);
    };
    auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
    uint64_t mask[EACH];
    auto reach = [&](uint32_t o) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) asm("v_cmp_le_u32 %0, %1, %2" : "=s"(mask[i]) : "s"(o), "v"(v[i]));
#pragma unroll
      for (int i = 0; i < EACH; ++i) c += __popcll(mask[i]);
      return c;
    };
    uint32_t from = max(uniform(least), 1u), beyond = uniform(most) + 1;
    int reached = sum_up(reach(from));
    const int few = M + M / 2 + 8;
    while (reached > few && beyond - from > 1) {
      const uint32_t mid = from + (beyond - from) / 2;
      const int c = sum_up(reach(mid));
      if (c >= M) from = mid, reached = c;
      else beyond = mid;
    }
    at = {k0, p0};
    if (reached <= MERGE_LIST) {
      const int c = reach(from);
      int to = 0;
      if (c && lane == 0) to = atomicAdd(&s.held, c);
      to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        if (mask[i]) {
          if (v[i] >= from) {
            const int x = to + __popcll(mask[i] & (((uint64_t)1 << lane) - 1));
            s.value[x] = value(at, mine[i]);
            s.place[x] = at.k << 8 | at.p;
          }
          to += __popcll(mask[i]);
        }
        next(at);
      }
      n = reached;
    } else {
      // many whose values round to one: by the values themselves the M best, of equals the first ones
      auto order = [&](int i, spot at) { return i * SELECT_THREADS < all ? merge_order(value(at, mine[i])) : 0; };
      uint64_t lo = merge_order(-(double)INFINITY) + 1, hi = ~(uint64_t)0;   // lo is reached by M, hi by fewer
      int over = 0;
      while (hi - lo > 1) {
        const uint64_t mid = lo + (hi - lo) / 2;
        int c = 0;
        at = {k0, p0};
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          c += __popcll(__ballot(order(i, at) >= mid));
          next(at);
        }
        c = sum_up(c);
        if (c >= M) lo = mid;
        else hi = mid, over = c;
      }
      int need = M - over;
      at = {k0, p0};
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const uint64_t o = order(i, at), equal = __ballot(o == lo);
        if (lane == 0) s.waves[turn & 1][wave] = __popcll(equal);
        __syncthreads();
        int before = 0, here = 0;
        for (int w = 0; w < WAVES; ++w) {
          if (w < wave) before += s.waves[turn & 1][w];
          here += s.waves[turn & 1][w];
        }
        ++turn;
        if (o > lo || (o == lo && before + (int)__popcll(equal & (((uint64_t)1 << lane) - 1)) < need)) {
          const int x = atomicAdd(&s.held, 1);
          s.value[x] = value(at, mine[i]);
          s.place[x] = at.k << 8 | at.p;
        }
        need -= here;
        next(at);
      }
      n = M;
    }
    __syncthreads();
    const int groups = SELECT_THREADS / max(n, 1), group = tid / max(n, 1), i = tid - group * n;
    if (n > 0 && group < groups) {                 // threads of a wave meet the same one at once
      const double c = s.value[i];
      const uint32_t place = s.place[i];
      int better = 0;
#pragma unroll 4
      for (int j = group; j < n; j += groups) {
        const double x = s.value[j];
        better += (x > c) | ((x == c) & (s.place[j] < place));
      }
      if (better) atomicAdd(&s.ranks[i], better);
    }
  }
  __syncthreads();
  if (tid == 0) s.held = 0;
  __syncthreads();
  const int64_t to = (int64_t)request * M;
  if (tid < n) {
    const double c = s.value[tid];
    const bool some = c > -INFINITY;
    const uint64_t there = __ballot(some);
    if (lane == 0) atomicAdd(&s.held, __popcll(there));
    const int rank = s.ranks[tid], k = s.place[tid] >> 8;
    if (some && rank < M) {
      a.out_scores[to + rank] = (float)c;
      a.out_parents[to + rank] = k;
      a.out_tokens[to + rank] = __float_as_int(lists[k * M + (int)(s.place[tid] & 255)].y);
    }
  }
  __syncthreads();
  for (int i = s.held + tid; i < M; i += SELECT_THREADS) {
    a.out_scores[to + i] = -INFINITY;
    a.out_parents[to + i] = -1;
    a.out_tokens[to + i] = -1;
  }
}

template <typename T, int LANES>
__global__ __launch_bounds__(256) void select_scan_kernel(const select_args a) {
  const int run = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  if (run < a.runs && select_open(a, blockIdx.y)) select_run<T, LANES>(a, blockIdx.y, run, threadIdx.x & 63);
}

template <typename T, bool TINY>
__global__ __launch_bounds__(SELECT_THREADS) void select_rows_kernel(const select_args a) {
  __shared__ rows_lds lds;
  select_list<T, TINY>(a, lds, blockIdx.x);
}

__global__ __launch_bounds__(SELECT_THREADS) void select_merge_kernel(const select_args a) {
  __shared__ merge_lds lds;
  select_merge(a, lds, blockIdx.x);
}

struct select_sizes {
  int32_t tiles, runs, per_run, log2_lanes, tops, join, segments;
  size_t norms, lists, maxima, all;                // of the workspace; the sums first
  select_sizes(int64_t rows, int64_t vocab, int64_t picks, int size) {
    const int64_t tile = SELECT_TILE / size;
    tiles = (int32_t)((vocab + tile - 1) / tile);
    // runs that fill the GPU twice
    const int64_t want = (16384 + rows - 1) / rows;
    per_run = (int32_t)((tiles + want - 1) / want);
    runs = (tiles + per_run - 1) / per_run;
    log2_lanes = 1;                                // (a lane's 16 tokens of 16 bits)
    while (log2_lanes < 6 && (vocab + (8 << log2_lanes) - 1) / (8 << log2_lanes) > SELECT_SEGMENTS) ++log2_lanes;
    tops = (int32_t)((vocab + (8 << log2_lanes) - 1) / (8 << log2_lanes));
    join = (tops + SELECT_SEGMENTS - 1) / SELECT_SEGMENTS;
    segments = (tops + join - 1) / join;
    norms = (size_t)rows * runs * 16;
    lists = norms + (size_t)rows * 16;
    maxima = lists + (size_t)rows * picks * 8;
    all = maxima + (size_t)rows * tops * 4;
  }
};

template <typename T, int LANES>
static void launch_select(const select_args& a, hipStream_t stream) {
  constexpr int MORE = sizeof(T) == 2 ? 1 : 0;     // of a lane's tokens: 8 << MORE
  if constexpr (LANES + MORE < 6)
    if (a.log2_lanes > LANES + MORE) return launch_select<T, LANES + 1>(a, stream);
  const dim3 block(SELECT_THREADS);
  hipLaunchKernelGGL((select_scan_kernel<T, LANES>), dim3((a.runs + 3) / 4, a.rows), dim3(256), 0, stream, a);
  if (a.vocab < 8) hipLaunchKernelGGL((select_rows_kernel<T, true>), dim3(a.rows), block, 0, stream, a);
  else hipLaunchKernelGGL((select_rows_kernel<T, false>), dim3(a.rows), block, 0, stream, a);
  hipLaunchKernelGGL(select_merge_kernel, dim3(a.rows / a.beams), block, 0, stream, a);
}

}  // namespace tb

extern "C" size_t tb_beam_select_workspace_bytes(int32_t num_rows, int32_t vocab, int32_t num_candidates) {
  if (num_rows <= 0 || vocab <= 0 || num_candidates <= 0) return 0;
  const size_t a = tb::select_sizes(num_rows, vocab, num_candidates, 2).all, b = tb::select_sizes(num_rows, vocab, num_candidates, 4).all;
  return a > b ? a : b;
}

extern "C" int32_t tb_beam_select(const void* logits, int64_t row_stride, int32_t vocab, int32_t dtype,
                                  const float* scores, const uint8_t* finished, int32_t end_token, int32_t num_rows,
                                  int32_t beams, int32_t num_candidates, float* out_scores, int32_t* out_parents,
                                  int64_t* out_tokens, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_rows >= 0 && num_rows <= 65535 && beams > 0 && beams <= TB_BEAMS_MAX && num_rows % beams == 0);
  TB_CHECK_ARG(vocab > 0 && vocab <= (1 << 30) && num_candidates > 0 && num_candidates <= TB_BEAM_CANDIDATES_MAX);
  TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16);
  TB_CHECK_ARG(!finished || (end_token >= 0 && end_token < vocab));
  if (num_rows == 0) return TB_OK;
  TB_CHECK_ARG(logits && scores && out_scores && out_parents && out_tokens && workspace);
  TB_CHECK_ARG(num_rows == 1 || row_stride >= vocab);
  const int size = dtype == TB_DTYPE_F32 ? 4 : 2;
  TB_CHECK_ARG((uintptr_t)logits % size == 0 && ((uintptr_t)workspace & 15u) == 0);
  const select_sizes z(num_rows, vocab, num_candidates, size);
  TB_CHECK_ARG(workspace_bytes >= z.all);
  select_args a;
  a.logits = (const char*)logits, a.row_bytes = row_stride * size, a.rows = num_rows, a.beams = beams, a.vocab = vocab;
  a.scores = scores, a.finished = finished, a.end_token = end_token, a.picks = num_candidates;
  a.out_scores = out_scores, a.out_parents = out_parents, a.out_tokens = out_tokens;
  a.tiles = z.tiles, a.runs = z.runs, a.per_run = z.per_run;
  a.log2_lanes = z.log2_lanes, a.tops = z.tops, a.join = z.join, a.segments = z.segments;
  char* const ws = (char*)workspace;
  a.sums = (double2*)ws, a.norms = (double2*)(ws + z.norms), a.lists = (float2*)(ws + z.lists);
  a.seg_max = (float*)(ws + z.maxima);
  if (dtype == TB_DTYPE_F32) launch_select<float, 1>(a, stream);
  else if (dtype == TB_DTYPE_F16) launch_select<_Float16, 0>(a, stream);
  else launch_select<__bf16, 0>(a, stream);
  TB_RETURN_LAUNCH_STATUS();
}
