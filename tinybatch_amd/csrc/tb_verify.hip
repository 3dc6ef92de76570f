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

// A call is a chain of launches with no atomics between them. Launch 0: every workgroup
// of a sequence walks its tree until it needs a sum over the vocabulary, and sums its own
// stretch of the row; launch r + 1: every workgroup adds up launch r's stretches in order, goes on
// with the walk, and sums its stretch again; the last launch, one workgroup per sequence, finds
// the border's stretch, thread and token. A chain, and drafts that were not drawn, need one sum
// whatever is refused; a tree of drawn drafts one more per refusal that has a sibling
// behind it: up to MAX_ROUNDS of those in launches of their own, the rest in the last one. What
// a later launch starts from (the state, the nodes' values, the sums) it loads at once.
constexpr int SUM_THREADS = 256, FIND_THREADS = 512, FIND_CHUNKS = 4;
constexpr int MAX_ROUNDS = 5;
constexpr int MAX_STRETCHES = 64;
constexpr int MAX_STRETCH = 1 << 18;               // tokens whose refused ones are kept as bits in LDS

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
  static __host__ __device__ size_t bytes(int nodes) { return (size_t)nodes * 20; }
  __device__ verify_tree(char* lds, int nodes)
      : tok((int32_t*)lds), par(tok + nodes), p((float*)(par + nodes)), q(p + nodes), u(q + nodes) {}
};

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
    t.q[i] = known && a.draft ? (float)((const T*)a.draft)[(row0 + par) * a.draft_stride + x] : 0.f;
  }
}
// The same from what launch 0 kept; entries past the sequence's nodes hold anything.
__device__ __forceinline__ void load_tree(const verify_args& a, const verify_tree& t, int seq, bool values) {
  const int32_t* const from = a.nodes + (int64_t)seq * 5 * a.width;
  for (int i = threadIdx.x; i < (values ? 5 : 2) * a.width; i += blockDim.x) t.tok[i] = from[i];
}

// The walk from a state on, by one wave, until the path ends or a sum is needed; `s` is the sum
// at st.a. Nodes kept are written to path[] (LDS) as they come.
__device__ __forceinline__ void walk(const verify_tree& t, int n, bool drawn, double s, verify_state& st,
                                     int32_t* path, int lane, int launch) {
  auto child = [&](int from) -> int {              // the next child of st.cur from row `from` on, or n
    for (int i0 = from & ~63; i0 < n; i0 += 64) {
      const int i = i0 + lane;
      const uint64_t hit = __ballot(i < n && i >= from && t.par[i < n ? i : 0] == st.cur);
      if (hit) return i0 + __ffsll((unsigned long long)hit) - 1;
    }
    return n;
  };
  int i = child(st.next), first = i;               // `first`: st.cur's first child, where refused tokens start
  for (;;) {
    st.round = launch;
    st.next = i;
    if (i >= n) return;                            // every child refused, or none: the path ends at st.cur
    const double u = (double)t.u[i], p = (double)t.p[i], q = (double)t.q[i];
    bool keep;
    if (drawn) {
      keep = u * q * s < p - st.a * q;
    } else {
      // a token refused before holds nothing
      const int x = t.tok[i];
      bool again = false;
      for (int i0 = first & ~63; i0 < i; i0 += 64) {
        const int k = i0 + lane;
        again |= __ballot(k < i && k >= first && t.par[k] == st.cur && t.tok[k] == x) != 0;
      }
      keep = !again && p > 0. && u * s < p;
      if (!keep && !again && p > 0.) s -= p;
    }
    if (keep) {
      st.cur = i;
      st.a = 0.;
      s = 1.;
      if (lane == 0) path[st.len] = i;
      ++st.len;
      i = first = child(i + 1);
    } else {
      i = child(i + 1);
      if (drawn) {
        st.a += s;
        st.next = i;
        st.round = i < n ? -1 : launch;
        return;                                    // the sum at the new a: for the next test or for the token
      }
    }
  }
}

// A row of the vocabulary in 16-byte chunks of the memory it lies in: chunk c holds tokens
// c E - shift .. + E - 1. The draft's row is read chunk by chunk too where it is aligned alike.
template <typename T>
struct verify_row {
  static constexpr int E = 16 / sizeof(T);
  const char* p;               // the aligned chunk 0
  const T* q;                  // the draft's row, token 0; null without
  int shift, vocab, chunks;
  bool q_alike;
  double a;
  const uint32_t* bits;        // refused tokens from token bit0 on; null: none
  int bit0;

  __device__ verify_row(const verify_args& v, int row, double a_) : vocab(v.vocab), a(a_), bits(nullptr), bit0(0) {
    const uintptr_t at = (uintptr_t)((const T*)v.probs + (int64_t)row * v.probs_stride);
    shift = (int)((at & 15) / sizeof(T));
    p = (const char*)(at & ~(uintptr_t)15);
    chunks = (vocab + shift + E - 1) / E;
    q = v.draft && a_ != 0. ? (const T*)v.draft + (int64_t)row * v.draft_stride : nullptr;
    q_alike = ((uintptr_t)q & 15) == (at & 15);
  }
  struct chunk {
    T p[E], q[E];
  };
  __device__ __forceinline__ chunk load(int c) const {
    chunk x;
    const vec16 v = ld16(p + (int64_t)c * 16);     // its 16 bytes hold a token of the row: inside its page
    __builtin_memcpy(x.p, &v, 16);
    if (q) {
      if (q_alike) {
        const vec16 w = ld16((const char*)q - shift * (int)sizeof(T) + (int64_t)c * 16);
        __builtin_memcpy(x.q, &w, 16);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) x.q[j] = q[min(max(c * E - shift + j, 0), vocab - 1)];
      }
    }
    return x;
  }
  // what is left of the chunk's j-th token
  __device__ __forceinline__ double weight(const chunk& x, int c, int j, bool edge) const {
    double w = (double)(float)x.p[j];
    if (q) w = fma(-a, (double)(float)x.q[j], w);
    const int i = c * E - shift + j;
    if (edge && (i < 0 || i >= vocab)) return 0.;
    if (bits && ((bits[(i - bit0) >> 5] >> ((i - bit0) & 31)) & 1)) return 0.;
    return w > 0. ? w : 0.;
  }
  __device__ __forceinline__ double sum(const chunk& x, int c) const {
    const bool edge = c == 0 || c == chunks - 1;
    double s = 0.;
#pragma unroll
    for (int j = 0; j < E; ++j) s += weight(x, c, j, edge);
    return s;
  }
  // this thread's share of chunks [b, e): every nth from b + i on
  __device__ __forceinline__ double share(int b, int e, int i, int nth) const {
    constexpr int U = 4;                           // chunks in flight
    double s = 0.;
    int c = b + i;
    for (; c + (U - 1) * nth < e; c += U * nth) {
      chunk x[U];
#pragma unroll
      for (int k = 0; k < U; ++k) x[k] = load(c + k * nth);
#pragma unroll
      for (int k = 0; k < U; ++k) s += sum(x[k], c + k * nth);
    }
    for (; c < e; c += nth) s += sum(load(c), c);
    return s;
  }
  // the refused tokens among chunks [b, e) as bits; by all threads
  __device__ void refuse(const verify_tree& t, int n, int cur, uint32_t* lds, int b, int e) {
    bit0 = b * E - shift;
    const int count = (e - b) * E;
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

template <typename T>
__global__ __launch_bounds__(SUM_THREADS) void verify_sum_kernel(const verify_args a, int launch) {
  extern __shared__ __align__(16) char lds[];
  __shared__ double part[SUM_THREADS / 64];
  __shared__ verify_state shared;
  const int seq = blockIdx.x, g = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* const acc = a.accepted + (int64_t)seq * a.width;
  int64_t* const out = a.out_tokens + (int64_t)seq * a.width;
  const verify_tree t(lds, a.width);
  int32_t* const path = (int32_t*)(lds + verify_tree::bytes(a.width));
  verify_state st;
  double s = 1.;
  if (launch > 0) {
    const int64_t before = (int64_t)(launch - 1) * a.num_seqs + seq;
    st = a.states[before];
    const double x = lane < a.stretches ? a.sums[before * a.stretches + lane] : 0.;
    load_tree(a, t, seq, true);
    if (st.n <= 0 || st.round >= 0) {              // this sequence's sum is there already
      if (g == 0 && tid == 0) a.states[before + a.num_seqs] = st;
      return;
    }
    s = sum64(x);
  } else {
    const int row0 = a.row_starts[seq], n = min(a.row_starts[seq + 1] - row0, a.width);
    st = verify_state{0., 0, 1, 1, 0, row0, n, 0.f};
    if (n > 0) load_tree<T>(a, t, row0, n);
    if (g == 0)
      for (int i = tid; i < a.width; i += SUM_THREADS) acc[i] = -1, out[i] = -1;
    if (n <= 0) {
      if (g == 0 && tid == 0) {
        a.states[seq] = st;
        a.num_accepted[seq] = 0;
      }
      return;
    }
  }
  __syncthreads();
  const int row0 = st.row0, n = st.n, len0 = launch > 0 ? st.len : 0;
  if (wave == 0) {
    if (launch == 0) {
      st.u = t.u[0];
      if (lane == 0) path[0] = 0;
    }
    walk(t, n, a.draft != nullptr, s, st, path, lane, launch);
    if (lane == 0) shared = st;
  }
  __syncthreads();
  st = shared;
  verify_row<T> row(a, row0 + st.cur, st.a);
  const int b = stretch_begin(row.chunks, a.stretches, g), e = stretch_begin(row.chunks, a.stretches, g + 1);
  if (!a.draft) row.refuse(t, n, st.cur, (uint32_t*)(path + a.width), b, e);
  const double x = sum64(row.share(b, e, tid, SUM_THREADS));
  if (lane == 0) part[wave] = x;
  __syncthreads();
  if (tid == 0) {
    double w = 0.;
#pragma unroll
    for (int k = 0; k < SUM_THREADS / 64; ++k) w += part[k];
    a.sums[((int64_t)launch * a.num_seqs + seq) * a.stretches + g] = w;
  }
  if (g == 0) {
    for (int i = len0 + tid; i < st.len; i += SUM_THREADS) {
      acc[i] = path[i];
      if (i > 0) out[i - 1] = a.tokens[row0 + path[i]];
    }
    if (tid == 0) a.states[(int64_t)launch * a.num_seqs + seq] = st;
    if (launch == 0)
      for (int i = tid; i < 5 * a.width; i += SUM_THREADS) a.nodes[(int64_t)seq * 5 * a.width + i] = t.tok[i];
  }
}

// The last launch: the walk's rest where more sums are needed than there were launches, and the token.
template <typename T>
__global__ __launch_bounds__(FIND_THREADS) void verify_find_kernel(const verify_args a, int launches) {
  extern __shared__ __align__(16) char lds[];
  constexpr int NW = FIND_THREADS / 64, E = verify_row<T>::E;
  __shared__ double part[NW], before_s;
  __shared__ verify_state shared;
  __shared__ int32_t first, last, token;
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* const acc = a.accepted + (int64_t)seq * a.width;
  int64_t* const out = a.out_tokens + (int64_t)seq * a.width;
  verify_state st = a.states[(int64_t)(launches - 1) * a.num_seqs + seq];
  const verify_tree t(lds, a.width);
  int32_t* const path = (int32_t*)(lds + verify_tree::bytes(a.width));
  uint32_t* const bits = (uint32_t*)(path + a.width);
  // the sums: of launch 0 where there was no other, else where the state says
  double sum = lane < a.stretches ? a.sums[(int64_t)seq * a.stretches + lane] : 0.;
  if (!a.draft) load_tree(a, t, seq, false);
  if (st.n <= 0) return;
  const int row0 = st.row0, n = st.n;
  const bool pending = st.round < 0;
  if (launches > 1) {
    const int r = pending ? launches - 1 : st.round;
    sum = lane < a.stretches ? a.sums[((int64_t)r * a.num_seqs + seq) * a.stretches + lane] : 0.;
    if (pending) load_tree(a, t, seq, true);
  }
  __syncthreads();
  auto total = [&](double x) -> double {           // over the workgroup
    x = sum64(x);
    __syncthreads();
    if (lane == 0) part[wave] = x;
    __syncthreads();
    return sum64(lane < NW ? part[lane] : 0.);
  };
  // the first of the threads' ranges that passes the border, x this thread's sum: its thread and
  // what lies before it; the last one that holds anything where none passes
  auto pick = [&](double x, double border, double& before) -> int {
    const double run = scan64<64>(x, lane);
    __syncthreads();
    if (lane == 63) part[wave] = run;
    if (tid == 0) first = FIND_THREADS, last = -1;
    __syncthreads();
    const double head = scan64<NW>(lane < NW ? part[lane] : 0., lane);   // of the waves, inclusive
    const double base = before + (wave ? __shfl(head, wave - 1) : 0.);
    if (x > 0.) {
      if (base + run > border) atomicMin(&first, tid);
      atomicMax(&last, tid);
    }
    __syncthreads();
    const int at = first < FIND_THREADS ? first : last;
    if (tid == at) before_s = base + (run - x);
    __syncthreads();
    before = before_s;
    return at;
  };

  if (pending) {
    // the rest of the walk by this workgroup alone
    double s = sum64(sum);
    const int len0 = st.len;
    for (;;) {
      if (wave == 0) {
        walk(t, n, true, s, st, path, lane, launches);
        if (lane == 0) shared = st;
      }
      __syncthreads();
      st = shared;
      __syncthreads();
      if (st.round >= 0) break;
      const verify_row<T> row(a, row0 + st.cur, st.a);
      s = total(row.share(0, row.chunks, tid, FIND_THREADS));
    }
    for (int i = len0 + tid; i < st.len; i += FIND_THREADS) {
      acc[i] = path[i];
      out[i - 1] = a.tokens[row0 + path[i]];
    }
  }

  verify_row<T> row(a, row0 + st.cur, st.a);
  const double u = (double)st.u;
  int b = 0, e = row.chunks;
  double before = 0., border = 0., w;
  if (!pending) {                                  // the stretch, from its launch's sums
    const double x = sum, run = scan64<64>(x, lane);
    w = __shfl(run, 63);
    border = u * w;
    const uint64_t some = __ballot(x > 0.), past = __ballot(x > 0. && run > border);
    if (w > 0.) {
      const int g = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)some);
      b = stretch_begin(row.chunks, a.stretches, g), e = stretch_begin(row.chunks, a.stretches, g + 1);
      before = __shfl(run - x, g);
      if (!a.draft) row.refuse(t, n, st.cur, bits, b, e);
    }
  } else {
    w = total(row.share(b, e, tid, FIND_THREADS));
    border = u * w;
  }
  if (!(w > 0.)) {                                 // nothing is left: the row as it is
    row.q = nullptr;
    row.bits = nullptr;
    w = total(row.share(b, e, tid, FIND_THREADS));
    border = u * w;
  }
  int next = -1;
  if (w > 0.) {
    // by waves of neighbouring chunks, until a thread has a few neighbouring chunks of its own
    while (e - b > FIND_THREADS * FIND_CHUNKS) {
      const int step = (e - b + NW - 1) / NW, wb = min(e, b + wave * step), we = min(e, wb + step);
      const double x = sum64(row.share(wb, we, lane, 64));
      const int at = pick(lane == 0 ? x : 0., border, before) >> 6;
      b = min(e, b + at * step);
      e = min(e, b + step);
    }
    const int step = (e - b + FIND_THREADS - 1) / FIND_THREADS;
    const int tb = min(e, b + tid * step), te = min(e, tb + step);
    typename verify_row<T>::chunk x[FIND_CHUNKS];
#pragma unroll
    for (int k = 0; k < FIND_CHUNKS; ++k) x[k] = row.load(min(tb + k, row.chunks - 1));
    double mine = 0.;
#pragma unroll
    for (int k = 0; k < FIND_CHUNKS; ++k) mine += tb + k < te ? row.sum(x[k], tb + k) : 0.;
    const int at = pick(mine, border, before);
    if (tid == at) {
      int found = -1;
      double run = before;
#pragma unroll
      for (int k = 0; k < FIND_CHUNKS; ++k)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const int c = tb + k;
          const double y = c < te ? row.weight(x[k], c, j, true) : 0.;
          if (y > 0. && (found < 0 || !(run > border))) {
            run += y;
            found = c * E - row.shift + j;         // the last one so far; the first that passes stays
          }
        }
      token = found;
    }
    __syncthreads();
    next = token;
  }
  if (tid == 0) {
    out[st.len - 1] = (int64_t)next;
    a.num_accepted[seq] = st.len;
  }
}

// Workgroups of a sequence: about four per CU over the batch, and few enough tokens for the bits.
static int verify_stretches(int num_seqs, int vocab) {
  const int want = std::min(1024 / std::max(num_seqs, 1), std::max(vocab / 1024, 1));
  return std::min(std::max({want, (vocab + MAX_STRETCH - 1) / MAX_STRETCH, 1}), MAX_STRETCHES);
}

template <typename T>
static void launch_verify(const verify_args& a, int rounds, hipStream_t stream) {
  const int per = (a.vocab + 16 + a.stretches - 1) / a.stretches + 16;   // tokens of a stretch, at most
  const size_t lds = verify_tree::bytes(a.width) + 4 * (size_t)a.width + (a.draft ? 0 : (size_t)(per / 32 + 1) * 4);
  for (int r = 0; r <= rounds; ++r)
    hipLaunchKernelGGL((verify_sum_kernel<T>), dim3(a.num_seqs, a.stretches), dim3(SUM_THREADS), lds, stream, a, r);
  hipLaunchKernelGGL((verify_find_kernel<T>), dim3(a.num_seqs), dim3(FIND_THREADS), lds, stream, a, rounds + 1);
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

extern "C" size_t tb_tree_verify_workspace_bytes(int32_t num_seqs, int32_t vocab, int32_t width) {
  using namespace tb;
  if (num_seqs <= 0 || vocab <= 0 || width <= 0) return 0;
  return (size_t)num_seqs * ((MAX_ROUNDS + 1) * (sizeof(verify_state) + sizeof(double) * verify_stretches(num_seqs, vocab)) +
                             verify_tree::bytes(width));
}

extern "C" int32_t tb_tree_verify(const void* probs, int64_t probs_row_stride, const void* draft_probs,
                                  int64_t draft_row_stride, int32_t vocab, int32_t dtype, const int64_t* tokens,
                                  const float* uniforms, const int32_t* parents, const int32_t* row_starts,
                                  int32_t num_seqs, int32_t max_children, int32_t* accepted, int32_t* num_accepted,
                                  int64_t* out_tokens, int32_t width, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
  using namespace tb;
  TB_CHECK_ARG(num_seqs >= 0 && vocab > 0 && width > 0 && max_children >= 0);
  TB_CHECK_ARG(dtype >= TB_DTYPE_F32 && dtype <= TB_DTYPE_BF16);
  if (width > TB_TREE_MAX_NODES || vocab > MAX_STRETCHES * (MAX_STRETCH - 64)) return TB_ERR_UNSUPPORTED;
  if (num_seqs == 0) return TB_OK;
  TB_CHECK_ARG(probs && tokens && uniforms && parents && row_starts && accepted && num_accepted && out_tokens);
  TB_CHECK_ARG(probs_row_stride >= vocab && (!draft_probs || draft_row_stride >= vocab));
  TB_CHECK_ARG(workspace && ((uintptr_t)workspace & 7u) == 0 &&
               workspace_bytes >= tb_tree_verify_workspace_bytes(num_seqs, vocab, width));
  const int stretches = verify_stretches(num_seqs, vocab);
  // sums that tests of later siblings need: none in a chain, or where the drafts were not drawn
  const int rounds = draft_probs ? std::min(std::max(max_children - 1, 0), MAX_ROUNDS) : 0;
  verify_state* const states = (verify_state*)workspace;
  double* const sums = (double*)(states + (size_t)(MAX_ROUNDS + 1) * num_seqs);
  const verify_args a{probs, probs_row_stride, draft_probs, draft_row_stride, vocab, tokens, uniforms, parents,
                      row_starts, accepted, num_accepted, out_tokens, width, num_seqs, stretches, states,
                      sums, (int32_t*)(sums + (size_t)(MAX_ROUNDS + 1) * num_seqs * stretches)};
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
