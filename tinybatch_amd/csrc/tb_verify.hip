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
#include <algorithm>

#include "tb_common.h"

namespace tb {

// A call is a chain of launches. Launch 0: every workgroup of a sequence walks its tree until it
// needs a sum over the vocabulary, and sums its own stretch of the row; launch r + 1: every workgroup
// adds up launch r's stretches in order, goes on with the walk, and sums its stretch again. A
// chain, and drafts that were not drawn, need one sum whatever is refused; a tree of drawn
// drafts one more per refusal that has a sibling behind it: as many launches as the worst walk of the step's
// trees needs (max_refusals), up to MAX_ROUNDS, the rest by one workgroup at the end. What a later
// launch starts from (the state, the nodes' values, the sums) it loads at once.
// The end, by one workgroup per sequence, finds the border's stretch, thread and token: the
// workgroup of the last sum launch that arrives last where the caller gives arrival counters, else
// a launch of its own (a graph's replays may overlap, and then no counter is theirs alone).
//
// What bounds it: the reads of one target row, and one draft row, per sum where there are many sequences (64
// chains over 151936 fp32 tokens: 78 MB in 25 us, 16 us at a copy's rate; in 16 bits 39 MB in 19 us), the launches and
// their dependent loads where there are few (one sequence: 10 us in a graph, 14 to 15 on the host); each further sum of a
// drawn tree takes 3 to 7 us. 16 trees of 12 to 20 drawn nodes: 46 to 50 us, 39 to 42 in 16 bits, with up to six refusals.
// MAX_ROUNDS: a launch that turns out not to be needed costs 2 to 3 us, a sum that the end has to make up for
// 50: those trees with at most 5 launches 48 us on average and 107 at worst, with 6 or more 45 and 55; 3 trees of
// 15 to 60 nodes (walks of up to 8 refusals are possible, none needed 5) 32 with 5, 37 with 7, 40 with 9.
constexpr int SUM_THREADS = 256, FIND_CHUNKS = 8;   // chunks of a thread at the end: up to 64 tokens, a lane each
constexpr int MAX_ROUNDS = 6;
constexpr int MAX_STRETCHES = 64;
constexpr int MAX_STRETCH = 1 << 17;               // tokens whose refused ones are kept as bits in LDS

struct verify_state {
  double a;                    // the refusals' share of q so far (drafts drawn)
  int32_t cur, next, len;      // the reached node, the child to try next, the path's length
  int32_t round;               // the launch whose stretches sum up what is left at `cur`; -1: another test first
  int32_t row0, n;             // the sequence's rows
  float u;                     // the root's random number
};

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
  int32_t width, num_seqs;
  int32_t stretches;           // workgroups of a sequence
  verify_state* states;        // [launch][B]
  double* sums;                // [launch][B][stretches]
  int32_t* nodes;              // [B][5][width]: verify_tree's arrays
  uint32_t* arrivals;          // [B], zero between calls; null: the end is a launch of its own
};

template <int N>
__device__ __forceinline__ double scan64(double x, int lane) {   // inclusive, over the wave
#pragma unroll
  for (int o = 1; o < N; o *= 2) {
    const double y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}
__device__ __forceinline__ double sum64(double x) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) x += __shfl_xor(x, o);
  return x;
}

// A sequence's tree in LDS: what a walk looks at of every node.
struct verify_tree {
  int32_t *tok, *par;
  float *p, *q, *u;            // of the node's token in its parent's rows; its random number
  static constexpr size_t BYTES = 20;              // of a node
  static __host__ __device__ size_t bytes(int nodes) { return nodes * BYTES; }
  __device__ verify_tree(char* lds, int nodes)
      : tok((int32_t*)lds), par(tok + nodes), p((float*)(par + nodes)), q(p + nodes), u(q + nodes) {}
};

// A draft's entry as it counts: 0 where it is NaN or below 0. (The target's entries need none of it: a test and a
// weight ask for more than 0, which neither a NaN nor a value below 0 less something gives.)
template <typename T>
__device__ __forceinline__ float counted(T x) {
  return fmaxf((float)x, 0.f);
}

template <typename T>
__device__ __forceinline__ void load_tree(const verify_args& a, const verify_tree& t, int row0, int n) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int64_t x = a.tokens[row0 + i];
    const int par = a.parents[row0 + i];
    const bool known = x >= 0 && x < a.vocab && par >= 0 && par < n;
    t.tok[i] = known ? (int32_t)x : -1;
    t.par[i] = par;
    t.u[i] = a.uniforms[row0 + i];
    t.p[i] = known ? (float)((const T*)a.probs)[(row0 + par) * a.probs_stride + x] : 0.f;
    t.q[i] = known && a.draft ? counted(((const T*)a.draft)[(row0 + par) * a.draft_stride + x]) : 0.f;
  }
}
// The same from what launch 0 kept; entries past the sequence's nodes hold anything.
__device__ __forceinline__ void load_tree(const verify_args& a, const verify_tree& t, int seq, bool values) {
  const int32_t* const from = a.nodes + (int64_t)seq * 5 * a.width;
  for (int i = threadIdx.x; i < (values ? 5 : 2) * a.width; i += blockDim.x) t.tok[i] = from[i];
}

// The walk's view of a tree: trees of up to 64 nodes in registers, lane i node i (a test then takes
// some 100 cycles instead of 700), larger ones in LDS.
template <bool SMALL>
struct walk_nodes {
  const verify_tree& t;
  int n, lane, par, tok;
  float p, q, u;
  __device__ __forceinline__ walk_nodes(const verify_tree& t_, int n_, int lane_) : t(t_), n(n_), lane(lane_) {
    if constexpr (SMALL) {
      const int i = min(lane, n - 1);
      par = lane < n ? t.par[i] : -2;
      tok = t.tok[i], p = t.p[i], q = t.q[i], u = t.u[i];
    }
  }
  static __device__ __forceinline__ float at(float x, int i) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i));
  }
  __device__ __forceinline__ void get(int i, int& x, double& p_, double& q_, double& u_) const {
    if constexpr (SMALL)
      x = __builtin_amdgcn_readlane(tok, i), p_ = (double)at(p, i), q_ = (double)at(q, i), u_ = (double)at(u, i);
    else
      x = t.tok[i], p_ = (double)t.p[i], q_ = (double)t.q[i], u_ = (double)t.u[i];
  }
  // the first child of `cur` from row `from` on, or n
  __device__ __forceinline__ int child(int cur, int from) const {
    if constexpr (SMALL) {
      const uint64_t hit = __ballot(par == cur && lane >= from);
      return hit ? __ffsll((unsigned long long)hit) - 1 : n;
    } else {
      for (int i0 = from & ~63; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        const uint64_t hit = __ballot(i < n && i >= from && t.par[i < n ? i : 0] == cur);
        if (hit) return i0 + __ffsll((unsigned long long)hit) - 1;
      }
      return n;
    }
  }
  // whether a child of `cur` in rows [from, to) holds token x
  __device__ __forceinline__ bool holds(int cur, int x, int from, int to) const {
    if constexpr (SMALL) {
      return __ballot(par == cur && tok == x && lane >= from && lane < to) != 0;
    } else {
      bool any = false;
      for (int i0 = from & ~63; i0 < to; i0 += 64) {
        const int k = i0 + lane;
        any |= __ballot(k < to && k >= from && t.par[k < n ? k : 0] == cur && t.tok[k < n ? k : 0] == x) != 0;
      }
      return any;
    }
  }
};

// The walk from a state on, by one wave, until the path ends or a sum is needed; `s` is the sum
// at st.a. Nodes kept are written to path[] (LDS) as they come.
template <bool SMALL>
__device__ __forceinline__ void walk_as(const verify_tree& t, int n, bool drawn, double s, verify_state& st,
                                        int32_t* path, int lane, int launch) {
  const walk_nodes<SMALL> nodes(t, n, lane);
  int cur = __builtin_amdgcn_readfirstlane(st.cur);
  int i = nodes.child(cur, __builtin_amdgcn_readfirstlane(st.next)), first = i;   // cur's first child: refused tokens start there
  st.round = launch;
  while (i < n) {                                  // else every child refused, or none: the path ends at cur
    int x;
    double p, q, u;
    nodes.get(i, x, p, q, u);
    bool keep;
    if (drawn) {
      keep = u * q * s < p - st.a * q;
    } else {
      const bool again = nodes.holds(cur, x, first, i);   // a token refused before holds nothing
      keep = !again && p > 0. && u * s < p;
      if (!keep && !again && p > 0.) s -= p;
    }
    if (__builtin_amdgcn_readfirstlane(keep)) {
      cur = i;
      st.a = 0.;
      s = 1.;
      if (lane == 0) path[st.len] = i;
      ++st.len;
      i = first = nodes.child(cur, i + 1);
    } else {
      i = nodes.child(cur, i + 1);
      if (drawn) {                                 // the sum at the new a: for the next test or for the token
        st.a += s;
        if (i < n) st.round = -1;
        break;
      }
    }
  }
  st.cur = cur;
  st.next = i;
}
__device__ __forceinline__ void walk(const verify_tree& t, int n, bool drawn, double s, verify_state& st,
                                     int32_t* path, int lane, int launch) {
  if (n <= 64) walk_as<true>(t, n, drawn, s, st, path, lane, launch);
  else walk_as<false>(t, n, drawn, s, st, path, lane, launch);
}

// A row of the vocabulary in 16-byte chunks of the memory it lies in: chunk c holds tokens
// c E - shift .. + E - 1. What is left of a token: max(p - a q, 0) where the drafts were drawn (the draft's
// row is read chunk by chunk too where it is aligned alike; before a refusal a = 0, and the target's row
// stands in for it), otherwise p without the refused tokens.
template <typename T, bool DRAWN>
struct verify_row {
  static constexpr int E = 16 / sizeof(T);
  const char* p;               // the aligned chunk 0
  const T* q;                  // the draft's row, token 0
  int shift, vocab, chunks;
  bool alike;
  double a;
  const uint32_t* bits;        // refused tokens from chunk first on, a bit each; null: none
  int first;

  __device__ verify_row(const verify_args& v, int row, double a_) : vocab(v.vocab), bits(nullptr), first(0) {
    const T* const at = (const T*)v.probs + (int64_t)row * v.probs_stride;
    shift = (int)(((uintptr_t)at & 15) / sizeof(T));
    p = (const char*)((uintptr_t)at & ~(uintptr_t)15);
    chunks = (vocab + shift + E - 1) / E;
    draft(DRAWN && a_ != 0. ? (const T*)v.draft + (int64_t)row * v.draft_stride : at, a_);
  }
  __device__ __forceinline__ void draft(const T* q_, double a_) {
    q = q_, a = a_;
    alike = (((uintptr_t)q ^ (uintptr_t)shift * sizeof(T)) & 15) == 0;
  }
  // the row as it is
  __device__ __forceinline__ void whole() {
    bits = nullptr;
    draft((const T*)p + shift, 0.);
  }
  struct chunk {
    T p[E], q[DRAWN ? E : 1];
  };
  __device__ __forceinline__ chunk load(int c) const {
    chunk x;
    const vec16 v = ld16(p + (int64_t)c * 16);     // its 16 bytes hold a token of the row: inside its page
    __builtin_memcpy(x.p, &v, 16);
    if constexpr (DRAWN) {
      vec16 w;
      if (alike) {
        w = ld16((const char*)q - shift * (int)sizeof(T) + (int64_t)c * 16);
      } else {
        T e[E];
#pragma unroll
        for (int j = 0; j < E; ++j) e[j] = q[min(max(c * E - shift + j, 0), vocab - 1)];
        __builtin_memcpy(&w, e, 16);
      }
      __builtin_memcpy(x.q, &w, 16);
    }
    return x;
  }
  // what is left of a token whose values are x and y
  __device__ __forceinline__ double left(T x, T y, uint32_t gone) const {
    double w = (double)(float)x;
    if constexpr (DRAWN) w = fma(-a, (double)counted(y), w);
    else if (gone & 1) w = 0.;
    return w > 0. ? w : 0.;
  }
  // the refused tokens of chunk c
  __device__ __forceinline__ uint32_t gone(int c) const {
    const int bit = (c - first) * E;
    return !DRAWN && bits ? bits[bit >> 5] >> (bit & 31) : 0u;
  }
  __device__ __forceinline__ double weight(int i) const {
    if (i < 0 || i >= vocab) return 0.;
    const int c = (i + shift) / E;
    return left(((const T*)p)[i + shift], DRAWN ? q[i] : (T)0, gone(c) >> (i + shift - c * E));
  }
  __device__ __forceinline__ double sum(const chunk& x, int c) const {
    const bool edge = c == 0 || c == chunks - 1;
    const uint32_t no = gone(c);
    double s = 0.;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int i = c * E - shift + j;
      s += edge && (i < 0 || i >= vocab) ? 0. : left(x.p[j], x.q[DRAWN ? j : 0], no >> j);
    }
    return s;
  }
  // this thread's share of chunks [b, e): every nth from b + i on
  __device__ __forceinline__ double share(int b, int e, int i, int nth) const {
    constexpr int U = 4;                           // chunks in flight
    double s = 0.;
    for (int c = b + i; c < e; c += U * nth) {
      chunk x[U];
#pragma unroll
      for (int k = 0; k < U; ++k) x[k] = load(min(c + k * nth, e - 1));
#pragma unroll
      for (int k = 0; k < U; ++k) s += c + k * nth < e ? sum(x[k], c + k * nth) : 0.;
    }
    return s;
  }
  // the refused tokens among chunks [b, e) as bits; by all threads
  __device__ __forceinline__ void refuse(const verify_tree& t, int n, int cur, uint32_t* lds, int b, int e) {
    first = b;
    const int bit0 = b * E - shift, count = (e - b) * E;
    bool any = false;
    for (int k = threadIdx.x; k < n; k += blockDim.x) {
      const int x = t.tok[k] - bit0;
      any |= t.par[k] == cur && t.tok[k] >= 0 && x >= 0 && x < count;
    }
    bits = nullptr;
    if (!__syncthreads_or(any)) return;            // none of them lies here
    for (int k = threadIdx.x; k < (count + 31) / 32; k += blockDim.x) lds[k] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < n; k += blockDim.x) {
      const int x = t.tok[k] - bit0;
      if (t.par[k] == cur && t.tok[k] >= 0 && x >= 0 && x < count) atomicOr(&lds[x >> 5], 1u << (x & 31));
    }
    __syncthreads();
    bits = lds;
  }
};

__device__ __forceinline__ int stretch_begin(int chunks, int stretches, int g) {
  return (int)((int64_t)chunks * g / stretches);
}

// What the end of a call shares in LDS.
struct find_lds {
  double part[SUM_THREADS / 64], before;
  verify_state st;
  int32_t first, last;
  double chunk[SUM_THREADS * FIND_CHUNKS];         // sums of the stretch's chunks
};

// The end of a call for one sequence, by a workgroup: the walk's rest where its last sum was not
// the one for the token, and the token. `sum`: lane g's stretch g of the state's sum.
template <typename T, bool DRAWN>
__device__ __forceinline__ void verify_finish(const verify_args& a, int seq, verify_state st, double sum, const verify_tree& t,
                              int32_t* path, uint32_t* bits, find_lds& f) {
  constexpr int NT = SUM_THREADS, NW = NT / 64, E = verify_row<T, DRAWN>::E;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row0 = st.row0, n = st.n;
  int32_t* const acc = a.accepted + (int64_t)seq * a.width;
  int64_t* const out = a.out_tokens + (int64_t)seq * a.width;
  auto total = [&](double x) __attribute__((always_inline)) -> double {           // over the workgroup
    x = sum64(x);
    __syncthreads();
    if (lane == 0) f.part[wave] = x;
    __syncthreads();
    return sum64(lane < NW ? f.part[lane] : 0.);
  };
  // the first of the threads' ranges that passes the border, x this thread's sum: its thread and
  // what lies before it; the last one that holds anything where none passes
  auto pick = [&](double x, double border, double& before) __attribute__((always_inline)) -> int {
    const double run = scan64<64>(x, lane);
    __syncthreads();
    if (lane == 63) f.part[wave] = run;
    if (tid == 0) f.first = NT, f.last = -1;
    __syncthreads();
    double base = before;
#pragma unroll
    for (int w = 0; w < NW - 1; ++w) base += w < wave ? f.part[w] : 0.;
    const uint64_t past = __ballot(x > 0. && base + run > border), some = __ballot(x > 0.);
    if (lane == 0 && some) {
      if (past) atomicMin(&f.first, 64 * wave + __ffsll((unsigned long long)past) - 1);
      atomicMax(&f.last, 64 * wave + 63 - __clzll((long long)some));
    }
    __syncthreads();
    const int at = max(f.first < NT ? f.first : f.last, 0);
    if (tid == at) f.before = base + (run - x);
    __syncthreads();
    before = f.before;
    return at;
  };

  if (DRAWN && st.round < 0) {                     // the walk's rest: this workgroup sums all stretches
    const int len0 = st.len;
    do {
      const double s = sum64(sum);
      if (wave == 0) {
        walk(t, n, true, s, st, path, lane, 0);
        if (lane == 0) f.st = st;
      }
      __syncthreads();
      st = f.st;
      const verify_row<T, DRAWN> row(a, row0 + st.cur, st.a);
      for (int g = wave; g < a.stretches; g += NW) {
        const double x = sum64(row.share(stretch_begin(row.chunks, a.stretches, g),
                                         stretch_begin(row.chunks, a.stretches, g + 1), lane, 64));
        if (lane == 0) f.chunk[g] = x;
      }
      __syncthreads();
      sum = lane < a.stretches ? f.chunk[lane] : 0.;
      __syncthreads();
    } while (st.round < 0);
    for (int i = len0 + tid; i < st.len; i += NT) {
      acc[i] = path[i];
      out[i - 1] = a.tokens[row0 + path[i]];
    }
  }

  verify_row<T, DRAWN> row(a, row0 + st.cur, st.a);
  const double u = (double)st.u;
  int b = 0, e = row.chunks;
  double before = 0.;
  const double run = scan64<64>(sum, lane);
  double w = __shfl(run, 63), border = u * w;
  if (w > 0.) {                                    // the stretch
    const uint64_t some = __ballot(sum > 0.), past = __ballot(sum > 0. && run > border);
    const int g = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)some);
    b = stretch_begin(row.chunks, a.stretches, g), e = stretch_begin(row.chunks, a.stretches, g + 1);
    before = __shfl(run - sum, g);
    if constexpr (!DRAWN) row.refuse(t, n, st.cur, bits, b, e);
  } else {                                         // nothing is left: the row as it is
    row.whole();
    w = total(row.share(b, e, tid, NT));
    border = u * w;
  }
  int next = -1;
  if (w > 0.) {
    // by waves of neighbouring chunks, until a thread has a few neighbouring chunks of its own
    while (e - b > NT * FIND_CHUNKS) {
      const int step = (e - b + NW - 1) / NW, wb = min(e, b + wave * step), we = min(e, wb + step);
      const double x = sum64(row.share(wb, we, lane, 64));
      const int at = pick(lane == 0 ? x : 0., border, before) >> 6;
      b = min(e, b + at * step);
      e = min(e, b + step);
    }
    // the chunks' sums, read side by side, then summed by threads of neighbouring ones
    constexpr int U = 4;
    for (int c = b + tid; c < e; c += U * NT) {
      typename verify_row<T, DRAWN>::chunk x[U];
#pragma unroll
      for (int k = 0; k < U; ++k) x[k] = row.load(min(c + k * NT, e - 1));
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (c + k * NT < e) f.chunk[c + k * NT - b] = row.sum(x[k], c + k * NT);
    }
    __syncthreads();
    const int step = (e - b + NT - 1) / NT;
    double mine = 0.;
    for (int c = tid * step; c < min(e - b, (tid + 1) * step); ++c) mine += f.chunk[c];
    const int at = pick(mine, border, before);
    // that thread's tokens, one a lane
    if (wave == 0) {
      const int tb0 = min(e, b + at * step), te0 = min(e, tb0 + step), i = tb0 * E - row.shift + lane;
      const double y = i < te0 * E - row.shift ? row.weight(i) : 0., run = before + scan64<64>(y, lane);
      const uint64_t some = __ballot(y > 0.), past = __ballot(y > 0. && run > border);
      if (some) next = tb0 * E - row.shift + (past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)some));
    }
  }
  if (tid == 0) {
    out[st.len - 1] = (int64_t)next;
    a.num_accepted[seq] = st.len;
  }
}

// END: the last sum launch of a call with arrival counters; it ends the call.
template <typename T, bool DRAWN, bool END>
__global__ __launch_bounds__(SUM_THREADS) void verify_sum_kernel(const verify_args a, int launch) {
  extern __shared__ __align__(16) char lds[];
  __shared__ find_lds f;
  const int seq = blockIdx.x, g = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* const acc = a.accepted + (int64_t)seq * a.width;
  int64_t* const out = a.out_tokens + (int64_t)seq * a.width;
  const verify_tree t(lds, a.width);
  int32_t* const path = (int32_t*)(lds + verify_tree::bytes(a.width));
  uint32_t* const bits = (uint32_t*)(path + a.width);
  verify_state st;
  double s = 1., y = 0.;       // the sum that the walk goes on with; lane g's stretch g of the sum for the token
  bool summed = false;         // that one is there already
  if (launch > 0) {
    const int64_t before = (int64_t)(launch - 1) * a.num_seqs + seq;
    st = a.states[before];
    const double x = lane < a.stretches ? a.sums[before * a.stretches + lane] : 0.;
    load_tree(a, t, seq, true);
    summed = st.n <= 0 || st.round >= 0;
    if (summed) {
      if (g != 0) return;
      if (!END && tid == 0) a.states[before + a.num_seqs] = st;
      if (!END || st.n <= 0) return;
      if (lane < a.stretches) y = a.sums[((int64_t)st.round * a.num_seqs + seq) * a.stretches + lane];
    }
    s = sum64(x);
  } else {
    const int row0 = a.row_starts[seq], n = min(a.row_starts[seq + 1] - row0, a.width);
    st = verify_state{0., 0, 1, 1, 0, row0, n, 0.f};
    if (n > 0) load_tree<T>(a, t, row0, n);
    if (n <= 0) {
      if (g == 0) {
        for (int i = tid; i < a.width; i += SUM_THREADS) acc[i] = -1, out[i] = -1;
        if (tid == 0) {
          a.states[seq] = st;
          a.num_accepted[seq] = 0;
        }
      }
      return;
    }
  }
  __syncthreads();
  if (!summed) {
    const int row0 = st.row0, n = st.n, len0 = launch > 0 ? st.len : 0;
    if (wave == 0) {
      if (launch == 0) {
        st.u = t.u[0];
        if (lane == 0) path[0] = 0;
      }
      walk(t, n, DRAWN, s, st, path, lane, launch);
      if (lane == 0) f.st = st;
    }
    __syncthreads();
    st = f.st;
    verify_row<T, DRAWN> row(a, row0 + st.cur, st.a);
    const int b = stretch_begin(row.chunks, a.stretches, g), e = stretch_begin(row.chunks, a.stretches, g + 1);
    if constexpr (!DRAWN) row.refuse(t, n, st.cur, bits, b, e);
    const double x = sum64(row.share(b, e, tid, SUM_THREADS));
    if (lane == 0) f.part[wave] = x;
    __syncthreads();
    double* const sums = a.sums + ((int64_t)launch * a.num_seqs + seq) * a.stretches;
    if (tid == 0) {
      double w = 0.;
#pragma unroll
      for (int k = 0; k < SUM_THREADS / 64; ++k) w += f.part[k];
      if constexpr (END) {
        // past the L2s, which the XCDs do not share, and there before the arrival counts
        __hip_atomic_store((uint64_t*)&sums[g], __builtin_bit_cast(uint64_t, w), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint32_t before = __hip_atomic_fetch_add(&a.arrivals[seq], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        f.first = before == (uint32_t)a.stretches - 1;
        if (f.first) __hip_atomic_store(&a.arrivals[seq], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      } else {
        sums[g] = w;
      }
    }
    bool writes = g == 0;                          // of all workgroups, which went the same way
    if constexpr (END) {
      __syncthreads();
      if (!f.first) return;                        // the last one to arrive ends the call, and writes all of it
      writes = true;
    }
    if (writes) {
      if (launch == 0)
        for (int i = tid; i < a.width; i += SUM_THREADS) {
          if (i >= st.len) acc[i] = -1, out[i] = -1;
          else if (i == st.len - 1 && !END) out[i] = -1;
        }
      for (int i = len0 + tid; i < st.len; i += SUM_THREADS) {
        acc[i] = path[i];
        if (i > 0) out[i - 1] = a.tokens[row0 + path[i]];
      }
    }
    if constexpr (END) {
      if (lane < a.stretches)
        y = __builtin_bit_cast(double, __hip_atomic_load((uint64_t*)&sums[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    } else if (g == 0) {
      if (tid == 0) a.states[(int64_t)launch * a.num_seqs + seq] = st;
      if (launch == 0)
        for (int i = tid; i < 5 * a.width; i += SUM_THREADS) a.nodes[(int64_t)seq * 5 * a.width + i] = t.tok[i];
    }
  }
  if constexpr (END) {
    __syncthreads();
    verify_finish<T, DRAWN>(a, seq, st, y, t, path, bits, f);
  }
}

// The end as a launch of its own, after `launches` sum launches.
template <typename T, bool DRAWN>
__global__ __launch_bounds__(SUM_THREADS) void verify_find_kernel(const verify_args a, int launches) {
  extern __shared__ __align__(16) char lds[];
  __shared__ find_lds f;
  const int seq = blockIdx.x, lane = threadIdx.x & 63;
  const verify_state st = a.states[(int64_t)(launches - 1) * a.num_seqs + seq];
  const verify_tree t(lds, a.width);
  int32_t* const path = (int32_t*)(lds + verify_tree::bytes(a.width));
  // the sums: of launch 0 where there was no other, else where the state says
  double sum = lane < a.stretches ? a.sums[(int64_t)seq * a.stretches + lane] : 0.;
  if constexpr (!DRAWN) load_tree(a, t, seq, false);
  if (st.n <= 0) return;
  const bool pending = st.round < 0;
  if (launches > 1) {
    const int r = pending ? launches - 1 : st.round;
    sum = lane < a.stretches ? a.sums[((int64_t)r * a.num_seqs + seq) * a.stretches + lane] : 0.;
  }
  if (pending) load_tree(a, t, seq, true);
  __syncthreads();
  verify_finish<T, DRAWN>(a, seq, st, sum, t, path, (uint32_t*)(path + a.width), f);
}

// Workgroups of a sequence: about four per CU over the batch, few enough tokens for the end's threads
// (one step of FIND_CHUNKS chunks each, 16-byte chunks of fp32) and for the bits. Two per CU take 41.1 us instead
// of 40.9 for 16 trees and one 47.0; eight 28.4 instead of 24.7 for 64 chains, 23.1 instead of 16.9 for 32 trees.
static int verify_stretches(int num_seqs, int vocab) {
  const int fill = std::min(1024 / std::max(num_seqs, 1), std::max(vocab / 1024, 1));
  const int once = (vocab + SUM_THREADS * FIND_CHUNKS * 4 - 64) / (SUM_THREADS * FIND_CHUNKS * 4 - 64);
  const int bits = (vocab + MAX_STRETCH - 1) / MAX_STRETCH;
  return std::min(std::max({fill, std::min(once, 32), bits, 1}), MAX_STRETCHES);
}

static_assert(verify_tree::BYTES * TB_TREE_MAX_NODES + 4 * TB_TREE_MAX_NODES + MAX_STRETCH / 8 + 4 + sizeof(find_lds) <=
                  65536, "what a workgroup may ask for at its launch");

template <typename T, bool DRAWN>
static void launch_verify_as(const verify_args& a, int rounds, hipStream_t stream) {
  const int per = (a.vocab + 16 + a.stretches - 1) / a.stretches + 16;   // tokens of a stretch, at most
  const size_t lds = verify_tree::bytes(a.width) + 4 * (size_t)a.width + (DRAWN ? 0 : (size_t)(per / 32 + 1) * 4);
  const dim3 grid(a.num_seqs, a.stretches), block(SUM_THREADS);
  for (int r = 0; r < rounds + (a.arrivals ? 0 : 1); ++r)
    hipLaunchKernelGGL((verify_sum_kernel<T, DRAWN, false>), grid, block, lds, stream, a, r);
  if (a.arrivals) hipLaunchKernelGGL((verify_sum_kernel<T, DRAWN, true>), grid, block, lds, stream, a, rounds);
  else hipLaunchKernelGGL((verify_find_kernel<T, DRAWN>), dim3(a.num_seqs), block, lds, stream, a, rounds + 1);
}

template <typename T>
static void launch_verify(const verify_args& a, int rounds, hipStream_t stream) {
  if (a.draft) launch_verify_as<T, true>(a, rounds, stream);
  else launch_verify_as<T, false>(a, rounds, stream);
}

// The same walk for greedy targets: a child is kept where its token is the target's choice
// after its parent. One wave per sequence: the host's call (10.6 us) is longer than the launch (2.0 us in a graph for one
// chain of 6, 3.0 for 32 trees of 20 to 30 nodes).
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
// Bound by the scattered rows: 44 MB read and written in 13.5 us (3.3 TB/s) for 64 paths in 32 layers of 8 heads of
// 128, 9.1 us at a copy's rate; a step of one tree by its launch (2.7 us in a graph). Rows read 4 or 8 at a time ahead of
// their stores, non-temporal loads and stores past the L2 measured 14.5 to 21.7 us.
// path rises, so path[j] >= j: a thread that moves one 16-byte column of the rows in order never
// reads a row it has written, and no other thread touches its column. A position outside the table or
// a block outside the pool (a path that is none) is left out.
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
  auto slot = [&](int64_t pos) -> char* {
    const int64_t blk = pos >> log2_bs;
    const int64_t b = blk >= 0 && blk < max_nb ? table[blk] : -1;
    if (b < 0 || b >= num_blocks) return nullptr;
    return base + b * (2 * num_kv_heads) * head_bytes + (int64_t)(pos & (bs - 1)) * row_vecs * 16;
  };
  for (int j = 0; j < len; ++j) {
    const int i = path[j];
    if (i <= j) continue;                          // in its place already (or no node)
    const char* const from = slot((int64_t)c + i);
    char* const to = slot((int64_t)c + j);
    if (from && to) st16(to, ld16(from));
  }
}

}  // namespace tb

extern "C" size_t tb_tree_verify_workspace_bytes(int32_t num_seqs, int32_t vocab, int32_t width) {
  using namespace tb;
  if (num_seqs <= 0 || vocab <= 0 || width <= 0) return 0;
  return (size_t)num_seqs * ((MAX_ROUNDS + 1) * (sizeof(verify_state) + sizeof(double) * verify_stretches(num_seqs, vocab)) +
                             verify_tree::bytes(width));
}

extern "C" int32_t tb_tree_verify(const void* probs, int64_t probs_row_stride, const void* draft_probs,
                                  int64_t draft_row_stride, int32_t vocab, int32_t dtype, const int64_t* tokens,
                                  const float* uniforms, const int32_t* parents, const int32_t* row_starts,
                                  int32_t num_seqs, int32_t max_refusals, int32_t* accepted, int32_t* num_accepted,
                                  int64_t* out_tokens, int32_t width, void* workspace, size_t workspace_bytes,
                                  uint32_t* arrivals, int32_t arrival_units, hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_seqs >= 0 && vocab > 0 && width > 0 && max_refusals >= 0);
  TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16);
  if (width > TB_TREE_MAX_NODES || vocab > MAX_STRETCHES * (MAX_STRETCH - 64)) return TB_ERR_UNSUPPORTED;
  if (num_seqs == 0) return TB_OK;
  TB_CHECK_ARG(probs && tokens && uniforms && parents && row_starts && accepted && num_accepted && out_tokens);
  TB_CHECK_ARG(probs_row_stride >= vocab && (!draft_probs || draft_row_stride >= vocab));
  TB_CHECK_ARG(workspace && ((uintptr_t)workspace & 7u) == 0 &&
               workspace_bytes >= tb_tree_verify_workspace_bytes(num_seqs, vocab, width));
  TB_CHECK_ARG(!arrivals || (arrival_units >= num_seqs && ((uintptr_t)arrivals & 3u) == 0));
  const int stretches = verify_stretches(num_seqs, vocab);
  // sums that tests of later siblings need: none in a chain, or where the drafts were not drawn
  const int rounds = draft_probs ? std::min(max_refusals, MAX_ROUNDS) : 0;
  verify_state* const states = (verify_state*)workspace;
  double* const sums = (double*)(states + (size_t)(MAX_ROUNDS + 1) * num_seqs);
  const verify_args a{probs, probs_row_stride, draft_probs, draft_row_stride, vocab, tokens, uniforms, parents,
                      row_starts, accepted, num_accepted, out_tokens, width, num_seqs, stretches, states,
                      sums, (int32_t*)(sums + (size_t)(MAX_ROUNDS + 1) * num_seqs * stretches), arrivals};
  if (dtype == TB_DTYPE_F32) launch_verify<float>(a, rounds, stream);
  else if (dtype == TB_DTYPE_F16) launch_verify<_Float16>(a, rounds, stream);
  else launch_verify<__bf16>(a, rounds, stream);
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
