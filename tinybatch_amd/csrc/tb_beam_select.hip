// The best continuations of a request over its beams and the vocabulary.
//
// Beam k with score s_k and logits x_k: continuing with token v makes
//   c(k, v) = s_k + ((x_kv - m_k) - log S_k),  m_k = max_u x_ku,  S_k = sum_u e^(x_ku - m_k);
// a beam that has finished has one candidate, c(k, end) = s_k. Of a request's candidates the M
// largest are told, the one of the smaller k V + v first among equals.
//
// Launch 1 reads the logits once: a wave walks a run of tiles of 512 tokens (8 a lane), keeps the tile's
// maximum (in memory) and the sum of e^(x - r) against a reference r per lane that moves only when a logit outgrows it by 8.
// Launch 2, a workgroup per request: the M best tiles by their maxima. A request's M best tokens
// lie in its M best tiles: the best tokens of the others are behind M better ones already. Then the M best
// tokens of those tiles.
// Sums of a wave's tiles, S, its logarithm and every c are in 64 bits: the order of two beams' candidates is decided
// by differences far below a float's step at the score's size.
#include "tb_common.h"

namespace tb {

constexpr int SELECT_TILE = 512;                   // tokens: 8 a lane
constexpr int SELECT_WAVES = 4;                    // of a workgroup of launch 1
constexpr int SELECT_THREADS = 1024;               // of launch 2

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
  float* tile_max;             // [rows][tiles]
  double2* sums;               // [rows][runs]: {S, r}
};

// A logit as it counts: NaN as -inf, +inf as the largest number.
__device__ __forceinline__ float select_logit(float x) {
  return x == x ? fminf(x, 3.402823466e38f) : -INFINITY;
}
__device__ __forceinline__ bool select_open(const select_args& a, int row) {   // whether the row's logits count
  return !(a.finished && a.finished[row]) && a.scores[row] > -INFINITY;
}

// 8 logits of a lane from token t0 on; past the vocabulary -inf.
template <typename T>
__device__ __forceinline__ void select_load(const char* row, int t0, int vocab, float (&x)[8]) {
  struct __attribute__((packed, aligned(sizeof(T)))) eight {
    T v[8];
  };
  if (t0 + 8 <= vocab) {
    const eight e = *reinterpret_cast<const eight*>(row + (int64_t)t0 * sizeof(T));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = select_logit((float)e.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = t0 + i < vocab ? select_logit((float)reinterpret_cast<const T*>(row)[t0 + i]) : -INFINITY;
  }
}

__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<DPP_QUAD_XOR1>(x));
  x = fmaxf(x, dpp<DPP_QUAD_XOR2>(x));
  x = fmaxf(x, dpp<DPP_ROW_HALF_MIRROR>(x));
  x = fmaxf(x, dpp<DPP_ROW_MIRROR>(x));
  x = max_xor16(x);
  return max_xor32(x);
}

template <typename T>
__global__ __launch_bounds__(64 * SELECT_WAVES) void select_scan_kernel(const select_args a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int run = blockIdx.x * SELECT_WAVES + wave, row = blockIdx.y;
  if (run >= a.runs || !select_open(a, row)) return;
  const char* const at = a.logits + (int64_t)row * a.row_bytes;
  const int first = run * a.per_run, last = min(first + a.per_run, a.tiles);
  float ref = -3.402823466e38f;
  double sum = 0.;
  for (int t = first; t < last; ++t) {
    float x[8];
    select_load<T>(at, t * SELECT_TILE + 8 * lane, a.vocab, x);
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    if (__any(top > ref + 8.f)) {
      const float r = fmaxf(ref, top);
      sum *= (double)expf(ref - r);
      ref = r;
    }
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) part += expf(x[i] - ref);
    sum += (double)part;
    top = wave_max(top);
    if (lane == 0) a.tile_max[(int64_t)row * a.tiles + t] = top;
  }
  // the lanes' sums against the largest reference
  const float r = wave_max(ref);
  sum *= exp((double)ref - (double)r);
#pragma unroll
  for (int o = 1; o < 64; o *= 2) sum += __shfl_xor(sum, o);
  if (lane == 0) a.sums[(int64_t)row * a.runs + run] = make_double2(sum, (double)r);
}

// A candidate and its place in the order: larger value, then smaller index.
struct cand {
  double c;
  int64_t at;
};
__device__ __forceinline__ bool better(const cand& x, const cand& y) { return x.c > y.c || (x.c == y.c && x.at < y.at); }
__device__ __forceinline__ cand better_of(const cand& x, const cand& y) { return better(x, y) ? x : y; }

// The workgroup's best candidate, in every thread.
__device__ __forceinline__ cand group_best(cand x, cand* lds, int turn) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    cand y;
    y.c = __shfl_xor(x.c, o);
    y.at = __shfl_xor(x.at, o);
    x = better_of(x, y);
  }
  cand* const mine = lds + 16 * (turn & 1);
  if ((threadIdx.x & 63) == 0) mine[threadIdx.x >> 6] = x;
  __syncthreads();
  x = mine[0];
  for (int w = 1; w < SELECT_THREADS / 64; ++w) x = better_of(x, mine[w]);
  return x;
}

template <typename T>
__global__ __launch_bounds__(SELECT_THREADS) void select_pick_kernel(const select_args a) {
  __shared__ cand lds[32];
  __shared__ double top[TB_BEAMS_MAX], norm[TB_BEAMS_MAX];   // m and log S of every beam
  __shared__ int64_t picked[TB_BEAM_CANDIDATES_MAX];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row0 = blockIdx.x * a.beams;
  const cand none = {-INFINITY, INT64_MAX};
  for (int k = wave; k < a.beams; k += SELECT_THREADS / 64) {
    const int row = row0 + k;
    float m = -INFINITY;
    double s = 0.;
    if (select_open(a, row)) {
      for (int t = lane; t < a.tiles; t += 64) m = fmaxf(m, a.tile_max[(int64_t)row * a.tiles + t]);
      m = wave_max(m);
      for (int r = lane; r < a.runs; r += 64) {
        const double2 x = a.sums[(int64_t)row * a.runs + r];
        s += x.x * (m == -INFINITY ? 0. : exp(x.y - (double)m));
      }
#pragma unroll
      for (int o = 1; o < 64; o *= 2) s += __shfl_xor(s, o);
    }
    if (lane == 0) top[k] = (double)m, norm[k] = log(s);
  }
  __syncthreads();
  auto value = [&](int k, float x) {               // c(k, .) of a logit
    return x == -INFINITY ? -INFINITY : (double)a.scores[row0 + k] + (((double)x - top[k]) - norm[k]);
  };
  // ---- the M best tiles ----
  int turn = 0;
  const int64_t all = (int64_t)a.beams * a.tiles;
  cand last = {INFINITY, -1};
  int n = 0;
  for (; n < a.picks; ++n) {
    cand best = none;
    for (int64_t i = tid; i < all; i += SELECT_THREADS) {
      const int k = (int)(i / a.tiles), t = (int)(i - (int64_t)k * a.tiles), row = row0 + k;
      cand x = none;
      if (select_open(a, row)) x = {value(k, a.tile_max[(int64_t)row * a.tiles + t]), i};
      else if (a.finished && a.finished[row] && t == 0) x = {(double)a.scores[row], i};
      if (x.c > -INFINITY && better(last, x)) best = better_of(best, x);
    }
    best = group_best(best, lds, turn++);
    if (best.at == INT64_MAX) break;
    last = best;
    if (tid == 0) picked[n] = best.at;
  }
  __syncthreads();
  // ---- the M best tokens of those tiles ----
  last = {INFINITY, -1};
  for (int o = 0; o < a.picks; ++o) {
    cand best = none;
    for (int p = wave; p < n; p += SELECT_THREADS / 64) {
      const int k = (int)(picked[p] / a.tiles), t = (int)(picked[p] - (int64_t)k * a.tiles), row = row0 + k;
      if (!select_open(a, row)) {
        const cand x = {(double)a.scores[row], (int64_t)k * a.vocab + a.end_token};
        if (better(last, x)) best = better_of(best, x);
        continue;
      }
      float x[8];
      select_load<T>(a.logits + (int64_t)row * a.row_bytes, t * SELECT_TILE + 8 * lane, a.vocab, x);
      for (int i = 0; i < 8; ++i) {
        const cand y = {value(k, x[i]), (int64_t)k * a.vocab + t * SELECT_TILE + 8 * lane + i};
        if (y.c > -INFINITY && better(last, y)) best = better_of(best, y);
      }
    }
    best = group_best(best, lds, turn++);
    last = best;
    if (tid == 0) {
      const int64_t at = (int64_t)blockIdx.x * a.picks + o;
      const bool some = best.at != INT64_MAX;
      a.out_scores[at] = some ? (float)best.c : -INFINITY;
      a.out_parents[at] = some ? (int32_t)(best.at / a.vocab) : -1;
      a.out_tokens[at] = some ? best.at % a.vocab : -1;
    }
  }
}

struct select_sizes {
  int32_t tiles, runs, per_run;
  size_t sums, all;
  select_sizes(int64_t rows, int64_t vocab) {
    tiles = (int32_t)((vocab + SELECT_TILE - 1) / SELECT_TILE);
    // as many runs as give every CU some 16 waves
    const int64_t want = (4096 + rows - 1) / rows;
    per_run = (int32_t)((tiles + want - 1) / want);
    runs = (tiles + per_run - 1) / per_run;
    sums = ((size_t)rows * tiles * 4 + 15) / 16 * 16;
    all = sums + (size_t)rows * runs * 16;
  }
};

template <typename T>
static void launch_select(const select_args& a, hipStream_t stream) {
  const dim3 grid((a.runs + SELECT_WAVES - 1) / SELECT_WAVES, a.rows);
  hipLaunchKernelGGL(select_scan_kernel<T>, grid, dim3(64 * SELECT_WAVES), 0, stream, a);
  hipLaunchKernelGGL(select_pick_kernel<T>, dim3(a.rows / a.beams), dim3(SELECT_THREADS), 0, stream, a);
}

}  // namespace tb

extern "C" size_t tb_beam_select_workspace_bytes(int32_t num_rows, int32_t vocab) {
  return num_rows > 0 && vocab > 0 ? tb::select_sizes(num_rows, vocab).all : 0;
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
  const select_sizes z(num_rows, vocab);
  TB_CHECK_ARG(workspace_bytes >= z.all);
  select_args a;
  a.logits = (const char*)logits, a.row_bytes = row_stride * size, a.rows = num_rows, a.beams = beams, a.vocab = vocab;
  a.scores = scores, a.finished = finished, a.end_token = end_token, a.picks = num_candidates;
  a.out_scores = out_scores, a.out_parents = out_parents, a.out_tokens = out_tokens;
  a.tiles = z.tiles, a.runs = z.runs, a.per_run = z.per_run;
  a.tile_max = (float*)workspace, a.sums = (double2*)((char*)workspace + z.sums);
  if (dtype == TB_DTYPE_F32) launch_select<float>(a, stream);
  else if (dtype == TB_DTYPE_F16) launch_select<_Float16>(a, stream);
  else launch_select<__bf16>(a, stream);
  TB_RETURN_LAUNCH_STATUS();
}
