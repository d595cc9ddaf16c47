// Trees of drafted tokens: depths and ancestor bits from parents, and the choice of the drafts that the target's
// probabilities take.
//
// The choice walks down from the root: at a node with target p and draft q its children are tried one after the other, each
// against what p has left after the rejected ones, norm(max(0, .. - q)) for each.  That residual after k rejections is
// max(0, p - a q) / S with a_0 = 0, S_0 = 1, a_{k+1} = a_k + S_k, S_k = sum max(0, p - a_k q): two numbers carry it, no row
// is ever written, and a rejection costs one pass over two rows for the next S.
//   max(0, max(0, p - a q) / S - q) = max(0, p - (a + S) q) / S
// Sums and comparisons are in 64 bits: a draw lies next to borders that are closer than 32-bit sums of a vocabulary.
// The first pass -- a chain has no other -- is one launch over all rows in pieces of 1024 tokens, each of whose blocks walks
// for itself; a second launch, a block for each sequence, goes on from there and draws the next token by the pieces' sums (for
// large vocabularies some more passes are launches like the first, see stages_of).
// Few sequences are launches and round trips: a chain of 6 over 131072 tokens 9.1 to 10.6 us among other calls, its kernels by
// themselves 4.0 + 6.4 at least.  Where siblings are rejected the passes come one after the other: 32 trees of 32 nodes over 32768
// tokens 28 to 31 us, up to 4 passes behind the first (5.3 + 23.6).
#include "kv_cache.h"

namespace rswa {
namespace {

constexpr int kMaxNodes = 1024;
constexpr int kPiece = 1024;  // tokens whose probabilities are summed by one wave

// Sequence b's rows, whatever cu_seqlens holds.
__device__ __forceinline__ void rows_of(const int32_t* cu, int b, int nodes, int64_t total, int64_t& row0, int& n) {
  row0 = 0;
  n = nodes;
  if (cu) {
    row0 = max((int64_t)0, min((int64_t)cu[b], total));
    n = (int)(max(row0, min((int64_t)cu[b + 1], total)) - row0);
  }
}

// ---- the tree ---------------------------------------------------------------------------------------------------
struct TreeKernelArgs {
  int32_t nodes, max_nodes, words;
  int64_t total;
  const int32_t* cu;
  const int32_t* parents;
  int64_t parents_st;
  int32_t* tree_parents;
  int32_t* depths;
  uint64_t* ancestors;
};

constexpr int kTreeThreads = 256;

// A block has a sequence.  A node's ancestors among the 64 nodes of its own word are found by walking up, and the first one
// of a lower word is remembered; the others are that one's, word by word.  (At most 63 + 15 steps through LDS in a row, where
// a walk up a chain of 1024 would be 1023.)  One tree of 32 nodes 2.0 us, 256 packed ones of up to 512 7.6; the call, with its
// three results, 6.2 and 7.2 among others.
__global__ __launch_bounds__(kTreeThreads) void draft_tree_kernel(const TreeKernelArgs a) {
  __shared__ int32_t up[kMaxNodes];   // the parent; -1: none, -2: the node is not there
  __shared__ int32_t out[kMaxNodes];  // the first ancestor of a lower word, -1 or -2 as the chain ends
  __shared__ uint64_t own[kMaxNodes]; // ancestors of its word, and itself
  const int b = blockIdx.x;
  int64_t row0;
  int n;
  rows_of(a.cu, b, a.nodes, a.total, row0, n);
  const int m = min(n, a.max_nodes);
  const int32_t* const parents = a.parents + (a.cu ? row0 : b * a.parents_st);
  const int64_t row = a.cu ? row0 : (int64_t)b * a.nodes;  // of what is written
  for (int i = threadIdx.x; i < m; i += kTreeThreads) {
    const int p = parents[i];
    up[i] = p >= -1 && p < i ? p : -2;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < m; i += kTreeThreads) {
    const int low = i & ~63;
    uint64_t bits = 0;
    int j = i;
    while (j >= low) {
      bits |= 1ull << (j & 63);
      j = up[j];
    }
    own[i] = bits;
    out[i] = j;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kTreeThreads) {
    int depth = -1, end = -2;
    if (i < m)
      for (int j = i; j >= 0; j = end) {
        depth += __popcll(own[j]);
        end = out[j];
      }
    const bool there = end == -1;
    a.tree_parents[row + i] = there ? up[i] : -2;
    a.depths[row + i] = there ? depth : -1;
    uint64_t* const to = a.ancestors + (row + i) * a.words;
    int j = there ? i : -1;
    for (int w = a.words - 1; w >= 0; w--) {
      const bool mine = j >= 64 * w;  // (j is of word w or a lower one; none: -1)
      to[w] = mine ? own[j] : 0;
      if (mine) j = out[j];
    }
  }
}

// ---- the choice -------------------------------------------------------------------------------------------------
struct VerifyArgs {
  int32_t batch, nodes, max_nodes, vocab, pieces, token_bytes, path_len;
  int64_t total;
  const int32_t* cu;
  const int32_t* parents;
  const void* tokens;
  const float* uniforms;
  int64_t parents_st, tokens_st, uniforms_st;
  const void* target;
  const void* draft;
  int64_t target_st[2], draft_st[2];
  int32_t* path;
  int32_t* accepted;
  void* next_token;
  // from one launch to the next: of `stage` launches behind the first
  double* sums;  // [stage][batch][pieces]
  struct Walk* walks;  // [stage][batch]
  int32_t stage;
};

// Where the walk of a sequence is: at node `cur`, whose children below `next` are tried, with the residual
// max(0, p - a q) / mass.
struct Walk {
  double a, mass;
  int32_t cur, next, count;  // count: nodes reached
  int32_t draw;              // no child is left to try
};

template <typename T>
__device__ __forceinline__ float positive(T v) {
  return fmaxf((float)v, 0.f);  // (0 for NaN)
}

// A sequence's nodes in LDS.
struct Nodes {
  int32_t parent[kMaxNodes];  // -2: nobody's child
  int32_t token[kMaxNodes];
  float p[kMaxNodes], q[kMaxNodes], u[kMaxNodes];  // the token's probabilities at the parent, and the node's number
  int32_t tried[kMaxNodes];   // tokens that were tried at a node
  int32_t n_tried;
};

template <typename T>
struct Sequence {
  const VerifyArgs& a;
  const T *target, *draft;
  int64_t row0;
  int b, n;
  __device__ __forceinline__ Sequence(const VerifyArgs& args, int b_) : a(args), b(b_) {
    rows_of(a.cu, b, a.nodes, a.total, row0, n);
    n = min(n, min(a.max_nodes, a.path_len));
    target = (const T*)a.target + (a.cu ? row0 * a.target_st[1] : b * a.target_st[0]);
    draft = a.draft ? (const T*)a.draft + (a.cu ? row0 * a.draft_st[1] : b * a.draft_st[0]) : nullptr;
  }
  __device__ __forceinline__ const T* p_row(int node) const { return target + node * a.target_st[1]; }
  __device__ __forceinline__ const T* q_row(int node) const { return draft ? draft + node * a.draft_st[1] : nullptr; }

  __device__ __forceinline__ void load(Nodes& s, int threads) const {
    const int32_t* const parents = a.parents + (a.cu ? row0 : b * a.parents_st);
    const float* const uniforms = a.uniforms + (a.cu ? row0 : b * a.uniforms_st);
    const int64_t at = a.cu ? row0 : b * a.tokens_st;
    for (int i = threadIdx.x; i < n; i += threads) {
      const int parent = parents[i];
      const int64_t x = a.token_bytes == 8 ? ((const int64_t*)a.tokens)[at + i] : ((const int32_t*)a.tokens)[at + i];
      const bool child = parent >= 0 && parent < i && x >= 0 && x < a.vocab;
      s.u[i] = uniforms[i];
      s.token[i] = (int)x;
      s.parent[i] = i == 0 ? parent : child ? parent : -2;
      s.p[i] = child ? positive(p_row(parent)[x]) : 0.f;
      s.q[i] = child && draft ? positive(q_row(parent)[x]) : 0.f;
    }
  }
};

// The first child of `node` from `from` on (n: none).
__device__ __forceinline__ int next_child(const Nodes& s, int node, int from, int n) {
  const int lane = threadIdx.x & 63;
  for (int i = from; i < n; i += 64) {
    const uint64_t mine = __builtin_amdgcn_ballot_w64(i + lane < n && s.parent[min(i + lane, n - 1)] == node);
    if (mine) return i + (int)__builtin_ctzll(mine);
  }
  return n;
}

// Without a draft: was the token tried at this node before, by a child below `i`?
__device__ __forceinline__ bool tried_before(const Nodes& s, int node, int i) {
  const int lane = threadIdx.x & 63;
  for (int j = node + 1; j < i; j += 64)
    if (__builtin_amdgcn_ballot_w64(j + lane < i && s.parent[min(j + lane, i)] == node && s.token[min(j + lane, i)] == s.token[i]))
      return true;
  return false;
}

// On to where a sum is wanted: the mass that a rejection leaves for the next child, or what the next token is drawn from.
// All lanes of a wave do the same; nodes reached go to `path` (null: not written).
template <bool DRAFT>
__device__ __forceinline__ void walk_on(const Nodes& s, Walk& w, int n, int32_t* path) {
  w.draw = 0;
  for (;;) {
    const int i = next_child(s, w.cur, w.next, n);
    if (i == n) {
      w.draw = 1;
      w.next = n;
      return;
    }
    w.next = i + 1;
    const double p = s.p[i], q = s.q[i], u = s.u[i];
    const double rest = DRAFT ? fmax(0.0, p - w.a * q) : tried_before(s, w.cur, i) ? 0.0 : p;
    if (DRAFT ? u * w.mass * q < rest : u * w.mass < rest) {
      if (path && threadIdx.x == 0) path[w.count] = i;
      w.count++;
      w.cur = i;
      w.a = 0.0;
      w.mass = 1.0;
    } else if (DRAFT) {
      w.a += w.mass;
      w.draw = next_child(s, w.cur, w.next, n) == n;  // (the sum wanted is that of what is drawn from)
      return;
    } else {
      w.mass = fmax(0.0, w.mass - rest);
    }
  }
}

// The tokens of the children of `node` below `next`, in any order.
__device__ __forceinline__ void list_tried(Nodes& s, int node, int next, int threads) {
  if (threadIdx.x == 0) s.n_tried = 0;
  __syncthreads();
  for (int i = node + 1 + threadIdx.x; i < next; i += threads)
    if (s.parent[i] == node) s.tried[atomicAdd(&s.n_tried, 1)] = s.token[i];
  __syncthreads();
}

// What is left at a node, r(x), for 16 bytes of tokens.  They are read from anywhere an element may lie; the last ones are
// the row's last 16 bytes, of which those ahead of x0 are not taken.
template <typename T, bool DRAFT>
struct Rest {
  static constexpr int N = 16 / sizeof(T);
  const T *p, *q;
  double a;
  int vocab;
  const int32_t* tried;
  int n_tried;
  typedef __attribute__((__vector_size__(16), aligned(sizeof(T)))) T Vec;
  struct Raw {
    Vec p, q;
  };
  __device__ __forceinline__ int base(int x0) const { return min(x0, vocab - N); }
  // vectors from x0 on, `step` apart, all on their way at once (of rows of N tokens or more)
  template <int M>
  __device__ __forceinline__ void load_row(int x0, int step, Raw (&v)[M]) const {
#pragma unroll
    for (int i = 0; i < M; i++) {
      v[i].p = *(const Vec*)(p + base(x0 + i * step));
      if constexpr (DRAFT) v[i].q = *(const Vec*)(q + base(x0 + i * step));
    }
  }
  template <int M>
  __device__ __forceinline__ void load(int x0, int step, Raw (&v)[M]) const {
    if (vocab >= N) {
      load_row(x0, step, v);
    } else {
#pragma unroll
      for (int i = 0; i < M; i++)
#pragma unroll 1
        for (int e = 0; e < N; e++) {
          const int x = max(0, base(x0 + i * step) + e);
          v[i].p[e] = p[x];
          if constexpr (DRAFT) v[i].q[e] = q[x];
        }
    }
  }
  // (of tokens base(x0) ..; 0 for those below x0)
  __device__ __forceinline__ void values(int x0, const Raw& v, double (&r)[N]) const {
    const int from = base(x0);
#pragma unroll
    for (int e = 0; e < N; e++) {
      r[e] = positive(v.p[e]);
      if constexpr (DRAFT) r[e] = fmax(0.0, r[e] - a * (double)positive(v.q[e]));
      r[e] = from + e >= x0 ? r[e] : 0.0;
    }
    if constexpr (!DRAFT)
      for (int i = 0; i < n_tried; i++) {
        const int at = tried[i] - from;
#pragma unroll
        for (int e = 0; e < N; e++) r[e] = at == e ? 0.0 : r[e];
      }
  }
};

// Sums over the lanes up to each, in the vector pipe (as wave_scan of floats).
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v) {
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  return __builtin_bit_cast(double, u32x2{(uint32_t)dpp_or_zero<CTRL, ROWS>((int)w[0]), (uint32_t)dpp_or_zero<CTRL, ROWS>((int)w[1])});
}
__device__ __forceinline__ double wave_scan(double v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ double of_lane(double v, int lane) {  // (the same lane for all)
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  return __builtin_bit_cast(double, u32x2{(uint32_t)__builtin_amdgcn_readlane((int)w[0], lane),
                                          (uint32_t)__builtin_amdgcn_readlane((int)w[1], lane)});
}
__device__ __forceinline__ double wave_sum(double v) { return of_lane(wave_scan(v), 63); }

// M pieces, `step` apart, as one wave has them ...
template <typename R>
constexpr int kTurns = kPiece / (64 * R::N);
template <int M, typename R>
__device__ __forceinline__ void load_pieces(const R& rest, int piece, int step, typename R::Raw (&v)[M][kTurns<R>]) {
#pragma unroll
  for (int m = 0; m < M; m++) rest.load((piece + m * step) * kPiece + lane_id() * R::N, 64 * R::N, v[m]);
}
// ... and their sums.
template <int M, typename R>
__device__ __forceinline__ void sum_pieces(const R& rest, int piece, int step, const typename R::Raw (&v)[M][kTurns<R>],
                                           double (&sum)[M]) {
#pragma unroll
  for (int m = 0; m < M; m++) {
    sum[m] = 0.0;
#pragma unroll
    for (int i = 0; i < kTurns<R>; i++) {
      double r[R::N];
      rest.values((piece + m * step) * kPiece + (lane_id() + i * 64) * R::N, v[m][i], r);
#pragma unroll
      for (int e = 0; e < R::N; e++) sum[m] += r[e];
    }
    sum[m] = wave_sum(sum[m]);
  }
}
template <typename R>
__device__ __forceinline__ double piece_sum(const R& rest, int piece) {
  typename R::Raw v[1][kTurns<R>];
  double sum[1];
  load_pieces(rest, piece, 0, v);
  sum_pieces(rest, piece, 0, v, sum);
  return sum[0];
}

constexpr int kFirstThreads = 256, kFirstPieces = kFirstThreads / 64;

// The walk as far as the first sum, and that sum over the waves' pieces.
template <typename T, bool DRAFT>
__global__ __launch_bounds__(kFirstThreads) void verify_first_kernel(const VerifyArgs a) {
  __shared__ Nodes s;
  const int b = blockIdx.y, piece = blockIdx.x * kFirstPieces + threadIdx.x / 64;
  const Sequence<T> seq(a, b);
  Walk w{0.0, 1.0, 0, 1, 0, 0};
  int32_t* const path = a.path + (int64_t)b * a.path_len;
  if (seq.n > 0) {
    seq.load(s, kFirstThreads);
    __syncthreads();
    if (s.parent[0] == -1) {
      if (blockIdx.x == 0 && threadIdx.x == 0) path[0] = 0;
      w.count = 1;
      walk_on<DRAFT>(s, w, seq.n, blockIdx.x == 0 ? path : nullptr);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.walks[b] = w;
  if (w.count == 0) return;
  if constexpr (!DRAFT) list_tried(s, w.cur, w.next, kFirstThreads);
  if (piece >= a.pieces) return;
  const Rest<T, DRAFT> rest{seq.p_row(w.cur), seq.q_row(w.cur), w.a, a.vocab, s.tried, DRAFT ? 0 : s.n_tried};
  const double sum = piece_sum(rest, piece);
  if ((threadIdx.x & 63) == 0) a.sums[(int64_t)b * a.pieces + piece] = sum;
}

// A lane's share of the sums of `pieces` pieces: as many as each in a row.
__device__ __forceinline__ double lane_total(const double* sums, int pieces) {
  const int per = (pieces + 63) / 64, lane = threadIdx.x & 63;
  double of = 0.0;
  for (int i = lane * per; i < min(pieces, (lane + 1) * per); i++) of += sums[i];
  return of;
}

// One rejection further, where that wants a sum: as the first launch, from where the one before it has come.
template <typename T>
__global__ __launch_bounds__(kFirstThreads) void verify_next_kernel(const VerifyArgs a) {
  __shared__ Nodes s;
  const int b = blockIdx.y, piece = blockIdx.x * kFirstPieces + threadIdx.x / 64;
  const Walk* const walks = a.walks + (int64_t)(a.stage - 1) * a.batch;
  const double* const sums = a.sums + ((int64_t)(a.stage - 1) * a.batch + b) * a.pieces;
  double* const to = a.sums + ((int64_t)a.stage * a.batch + b) * a.pieces;
  Walk w = walks[b];
  const bool wanted = w.count > 0 && !w.draw;
  const Sequence<T> seq(a, b);
  if (wanted) {
    seq.load(s, kFirstThreads);
    __syncthreads();
    w.mass = wave_sum(lane_total(sums, a.pieces));
    walk_on<true>(s, w, seq.n, blockIdx.x == 0 ? a.path + (int64_t)b * a.path_len : nullptr);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.walks[(int64_t)a.stage * a.batch + b] = w;
  if (piece >= a.pieces || w.count == 0) return;
  const double sum = wanted ? piece_sum(Rest<T, true>{seq.p_row(w.cur), seq.q_row(w.cur), w.a, a.vocab, nullptr, 0}, piece)
                            : sums[piece];
  if ((threadIdx.x & 63) == 0) to[piece] = sum;
}

constexpr int kRestThreads = 1024, kRestWaves = kRestThreads / 64;
constexpr int kMaxPieces = 4096;

// The rest of the walk, and the draw.
template <typename T, bool DRAFT>
__global__ __launch_bounds__(kRestThreads) void verify_rest_kernel(const VerifyArgs a) {
  using R = Rest<T, DRAFT>;
  constexpr int N = R::N;
  __shared__ Nodes s;
  __shared__ double sums[kMaxPieces];
  __shared__ double share[kRestWaves];
  __shared__ int found, last_positive;
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const Sequence<T> seq(a, b);
  int32_t* const path = a.path + (int64_t)b * a.path_len;
  // (all on their way at once: sums that the first launch has not written are not looked at)
  const float u_root = seq.n > 0 ? a.uniforms[a.cu ? seq.row0 : b * a.uniforms_st] : 0.f;
  const double* const known = a.sums + ((int64_t)a.stage * a.batch + b) * a.pieces;
  for (int i = threadIdx.x; i < a.pieces; i += kRestThreads) sums[i] = known[i];
  Walk w = a.walks[(int64_t)a.stage * a.batch + b];
  if (w.count > 0 && (!DRAFT || !w.draw)) seq.load(s, kRestThreads);
  if (threadIdx.x == 0) found = last_positive = -1;
  __syncthreads();
  // (all waves do the same)
  const int per = (a.pieces + 63) / 64;
  int drawn = -1;
  if (w.count > 0) {
    if constexpr (DRAFT) {
      // Rows of up to two pieces a wave stay in registers from one sibling to the next (32 trees of 32 nodes over 8192 tokens 23.8 ->
      // 18.9 us; the same rows over 32768 tokens and, with one more, read again, three inputs: 23.0 / 24.3, 19.4 / 21.6, 23.3 /
      // 27.0, 64 trees 34.0 / 37.2, 25.1 / 28.5, 29.0 / 33.8).
      auto rejections = [&](auto few) {
        [[maybe_unused]] typename R::Raw v[2][1][kTurns<R>];
        [[maybe_unused]] int held_node = -1;
        while (!w.draw) {
          w.mass = wave_sum(lane_total(sums, a.pieces));
          walk_on<DRAFT>(s, w, seq.n, path);
          const R rest{seq.p_row(w.cur), seq.q_row(w.cur), w.a, a.vocab, nullptr, 0};
          __syncthreads();
          if constexpr (few) {
            if (w.cur != held_node) {
#pragma unroll
              for (int m = 0; m < 2; m++)
                if (wave + m * kRestWaves < a.pieces)
                  rest.load_row((wave + m * kRestWaves) * kPiece + lane * N, 64 * N, v[m][0]);
            }
            held_node = w.cur;
#pragma unroll
            for (int m = 0; m < 2; m++)
              if (wave + m * kRestWaves < a.pieces) {
                double of[1];
                sum_pieces(rest, wave + m * kRestWaves, 0, v[m], of);
                if (lane == 0) sums[wave + m * kRestWaves] = of[0];
              }
          } else {
            for (int i = wave; i < a.pieces; i += 2 * kRestWaves) {  // (a piece behind the last: 0, as the row's end)
              typename R::Raw both[2][kTurns<R>];
              double of[2];
              load_pieces(rest, i, kRestWaves, both);
              sum_pieces(rest, i, kRestWaves, both, of);
              if (lane == 0) {
                sums[i] = of[0];
                if (i + kRestWaves < a.pieces) sums[i + kRestWaves] = of[1];
              }
            }
          }
          __syncthreads();
        }
      };
      if (a.pieces <= 2 * kRestWaves && a.vocab >= N)
        rejections(std::true_type{});
      else
        rejections(std::false_type{});
    } else {
      list_tried(s, w.cur, w.next, kRestThreads);
    }
    R rest{seq.p_row(w.cur), seq.q_row(w.cur), w.a, a.vocab, s.tried, DRAFT ? 0 : s.n_tried};
    double own = lane_total(sums, a.pieces), upto = wave_scan(own), all = of_lane(upto, 63);
    if (!(all > 0.0)) {  // nothing is left
      rest.a = 0.0;
      rest.n_tried = 0;
      __syncthreads();
      for (int i = wave; i < a.pieces; i += kRestWaves) {
        const double of = piece_sum(rest, i);
        if (lane == 0) sums[i] = of;
      }
      __syncthreads();
      own = lane_total(sums, a.pieces);
      upto = wave_scan(own);
      all = of_lane(upto, 63);
    }
    if (all > 0.0) {
      const double want = (double)u_root * all;
      // the piece: the first whose running sum is above, or the last that has anything
      const uint64_t past = __builtin_amdgcn_ballot_w64(upto > want && own > 0.0);
      const uint64_t any = __builtin_amdgcn_ballot_w64(own > 0.0);
      const int at = past ? (int)__builtin_ctzll(past) : 63 - (int)__builtin_clzll(any);
      double before = 0.0, upto_piece = at == 0 ? 0.0 : of_lane(upto, max(at - 1, 0));
      int piece = at * per;
      for (int i = at * per; i < min(a.pieces, (at + 1) * per); i++)
        if (sums[i] > 0.0) {
          before = upto_piece;
          piece = i;
          upto_piece += sums[i];
          if (upto_piece > want) break;
        }
      // the token: a thread has N tokens in a row
      const int x = piece * kPiece + threadIdx.x * N;
      const bool mine = (int)threadIdx.x * N < kPiece;
      double r[N], of = 0.0;
      if (mine) {
        typename R::Raw v[1];
        rest.load(x, 0, v);
        rest.values(x, v[0], r);
#pragma unroll
        for (int e = 0; e < N; e++) of += r[e];
      }
      const double in_wave = wave_scan(of);
      if (lane == 63) share[wave] = in_wave;
      __syncthreads();
      if (mine) {
        for (int i = 0; i < wave; i++) before += share[i];
        double sum = before + (in_wave - of);
        int first = -1, positive_at = -1;
#pragma unroll
        for (int e = 0; e < N; e++) {
          sum += r[e];
          if (r[e] > 0.0) {
            positive_at = rest.base(x) + e;
            if (sum > want && first < 0) first = positive_at;
          }
        }
        if (first >= 0) atomicMin((uint32_t*)&found, (uint32_t)first);  // (-1 is the largest)
        if (positive_at >= 0) atomicMax(&last_positive, positive_at);
      }
      __syncthreads();
      drawn = found != -1 ? found : last_positive;  // (the last: where roundings have the sums end short of their total)
    }
  }
  if (threadIdx.x == 0) {
    a.accepted[b] = w.count;
    if (a.token_bytes == 8)
      ((int64_t*)a.next_token)[b] = drawn;
    else
      ((int32_t*)a.next_token)[b] = drawn;
  }
  for (int i = w.count + threadIdx.x; i < a.path_len; i += kRestThreads) path[i] = -1;
}

int pieces_of(int vocab) { return (int)ceil_div(vocab, kPiece); }

// Launches between the first and the last: a pass over all compute units takes 4 us (2.5 if no sequence wants it), one by the
// last launch's block for a sequence 4.5 of 32768 tokens and 15 of 131072.  So three for large vocabularies and trees, of
// whose sequences some reject a few siblings: 8 sequences of 32 nodes over 131072 tokens 65 us without, 31 with three, 32 with
// five; 32 of 8 over 32768 22.0 and 24.8.  The same rows over 65535 tokens without and over 65536 with, three inputs: 32 of 32 nodes
// 37.2 / 27.8, 45.7 / 34.9, 38.9 / 29.1, 8 of 32 28.6 / 24.0, 38.2 / 26.7, 35.1 / 25.9, 8 of 16 21.2 / 22.1, 30.4 / 24.7, 21.2 / 22.1,
// one of 32 20.2 / 21.4, 10.6 / 19.0, 27.0 / 21.9, as rejections come.  (Between 32768 and 65536
// tokens launches have not been timed.)  Not for what is likely a chain, which rejects once (6 nodes over 131072 9.9, 19.0).
// Of a pack the mean count of nodes says which it is: its max_nodes is that of whole words of ancestors, 64 at least.
int stages_of(const rswa_verify_params* p) {
  const int64_t nodes = p->cu_seqlens ? ceil_div(p->total, std::max(1, p->batch)) : p->nodes;
  return p->draft && p->vocab >= 65536 && nodes > 8 ? 3 : 0;
}

uint64_t walk_bytes(const rswa_verify_params* p) {
  return (uint64_t)(stages_of(p) + 1) * p->batch * (sizeof(Walk) + 8 * (uint64_t)pieces_of(p->vocab));
}

template <typename T>
void launch_verify(VerifyArgs& a, int stages, hipStream_t stream) {
  const dim3 first((unsigned)ceil_div(a.pieces, kFirstPieces), (unsigned)a.batch), rest((unsigned)a.batch);
  if (a.draft) {
    hipLaunchKernelGGL((verify_first_kernel<T, true>), first, dim3(kFirstThreads), 0, stream, a);
    while (a.stage < stages) {
      a.stage++;
      hipLaunchKernelGGL((verify_next_kernel<T>), first, dim3(kFirstThreads), 0, stream, a);
    }
    hipLaunchKernelGGL((verify_rest_kernel<T, true>), rest, dim3(kRestThreads), 0, stream, a);
  } else {
    hipLaunchKernelGGL((verify_first_kernel<T, false>), first, dim3(kFirstThreads), 0, stream, a);
    hipLaunchKernelGGL((verify_rest_kernel<T, false>), rest, dim3(kRestThreads), 0, stream, a);
  }
}

}  // namespace
}  // namespace rswa

extern "C" int rswa_draft_tree(const rswa_tree_params* p, void* stream) {
  using namespace rswa;
  constexpr const char* who = "draft_tree";
  RSWA_REQUIRE(p, RSWA_ERR_INVALID, "%s: null parameters", who);
  RSWA_REQUIRE(p->batch >= 0 && p->nodes >= 0 && p->total >= 0, RSWA_ERR_INVALID, "%s: negative size", who);
  RSWA_REQUIRE(p->max_nodes >= 1 && p->max_nodes <= kMaxNodes, RSWA_ERR_UNSUPPORTED, "%s: max_nodes %d (1 to %d)", who,
               p->max_nodes, kMaxNodes);
  RSWA_REQUIRE(p->cu_seqlens || p->nodes <= p->max_nodes, RSWA_ERR_INVALID, "%s: %d nodes, max_nodes %d", who, p->nodes,
               p->max_nodes);
  RSWA_REQUIRE(p->total < (1ll << 31) && p->batch <= (1 << 20), RSWA_ERR_UNSUPPORTED, "%s: rows or batch too large", who);
  const int64_t rows = p->cu_seqlens ? p->total : (int64_t)p->batch * p->nodes;
  if (rows == 0 || p->batch == 0) return RSWA_OK;
  RSWA_REQUIRE(p->parents && p->tree_parents && p->depths && p->ancestors, RSWA_ERR_INVALID, "%s: null tensor", who);
  TreeKernelArgs a{};
  a.nodes = p->nodes;
  a.max_nodes = p->max_nodes;
  a.words = (p->max_nodes + 63) / 64;
  a.total = p->total;
  a.cu = p->cu_seqlens;
  a.parents = p->parents;
  a.parents_st = p->parents_stride;
  a.tree_parents = p->tree_parents;
  a.depths = p->depths;
  a.ancestors = (uint64_t*)p->ancestors;
  clear_launch_error();
  hipLaunchKernelGGL(draft_tree_kernel, dim3((unsigned)p->batch), dim3(kTreeThreads), 0, (hipStream_t)stream, a);
  return check_launch(who);
}

extern "C" uint64_t rswa_verify_drafts_workspace_bytes(const rswa_verify_params* p) {
  using namespace rswa;
  if (!p || p->batch <= 0 || p->vocab <= 0) return 0;
  return walk_bytes(p);
}

extern "C" int rswa_verify_drafts(const rswa_verify_params* p, void* stream) {
  using namespace rswa;
  constexpr const char* who = "verify_drafts";
  RSWA_REQUIRE(p, RSWA_ERR_INVALID, "%s: null parameters", who);
  RSWA_REQUIRE(p->dtype == RSWA_BF16 || p->dtype == RSWA_F16 || p->dtype == RSWA_F32, RSWA_ERR_UNSUPPORTED, "%s: dtype %d",
               who, p->dtype);
  RSWA_REQUIRE(p->token_bytes == 4 || p->token_bytes == 8, RSWA_ERR_UNSUPPORTED, "%s: tokens of %d bytes (4 or 8)", who,
               p->token_bytes);
  RSWA_REQUIRE(p->batch >= 0 && p->nodes >= 0 && p->total >= 0 && p->path_len >= 0, RSWA_ERR_INVALID, "%s: negative size",
               who);
  RSWA_REQUIRE(p->max_nodes >= 1 && p->max_nodes <= kMaxNodes, RSWA_ERR_UNSUPPORTED, "%s: max_nodes %d (1 to %d)", who,
               p->max_nodes, kMaxNodes);
  RSWA_REQUIRE(p->cu_seqlens || p->nodes <= p->max_nodes, RSWA_ERR_INVALID, "%s: %d nodes, max_nodes %d", who, p->nodes,
               p->max_nodes);
  RSWA_REQUIRE(p->path_len >= (p->cu_seqlens ? p->max_nodes : p->nodes), RSWA_ERR_INVALID, "%s: path_len %d is too short",
               who, p->path_len);
  RSWA_REQUIRE(p->vocab > 0, RSWA_ERR_INVALID, "%s: vocab %d", who, p->vocab);
  RSWA_REQUIRE(p->vocab <= kPiece * kMaxPieces, RSWA_ERR_UNSUPPORTED, "%s: vocab %d (at most %d)", who, p->vocab,
               kPiece * kMaxPieces);
  RSWA_REQUIRE(p->total < (1ll << 31) && p->batch < (1 << 16), RSWA_ERR_UNSUPPORTED, "%s: rows or batch too large", who);
  if (p->batch == 0) return RSWA_OK;
  const int64_t rows = p->cu_seqlens ? p->total : (int64_t)p->batch * p->nodes;
  RSWA_REQUIRE(p->accepted && p->next_token && (p->path || p->path_len == 0), RSWA_ERR_INVALID, "%s: null result", who);
  RSWA_REQUIRE(rows == 0 || (p->parents && p->tokens && p->uniforms && p->target), RSWA_ERR_INVALID, "%s: null tensor", who);
  RSWA_REQUIRE(p->workspace && (uintptr_t)p->workspace % 8 == 0 && p->workspace_bytes >= walk_bytes(p), RSWA_ERR_INVALID,
               "%s: workspace of %llu bytes, %llu needed (8-byte aligned)", who, (unsigned long long)p->workspace_bytes,
               (unsigned long long)walk_bytes(p));
  VerifyArgs a{};
  a.batch = p->batch;
  a.nodes = p->nodes;
  a.max_nodes = p->max_nodes;
  a.vocab = p->vocab;
  a.pieces = pieces_of(p->vocab);
  a.token_bytes = p->token_bytes;
  a.path_len = p->path_len;
  a.total = p->total;
  a.cu = p->cu_seqlens;
  a.parents = p->parents;
  a.tokens = p->tokens;
  a.uniforms = p->uniforms;
  a.parents_st = p->parents_stride;
  a.tokens_st = p->tokens_stride;
  a.uniforms_st = p->uniforms_stride;
  a.target = p->target;
  a.draft = p->draft;
  for (int i = 0; i < 2; i++) {
    a.target_st[i] = p->target_stride[i];
    a.draft_st[i] = p->draft_stride[i];
  }
  a.path = p->path;
  a.accepted = p->accepted;
  a.next_token = p->next_token;
  a.sums = (double*)p->workspace;
  const int stages = stages_of(p);
  a.walks = (Walk*)(a.sums + (int64_t)(stages + 1) * p->batch * a.pieces);
  clear_launch_error();
  hipStream_t st = (hipStream_t)stream;
  if (p->dtype == RSWA_F32)
    launch_verify<float>(a, stages, st);
  else if (p->dtype == RSWA_BF16)
    launch_verify<__bf16>(a, stages, st);
  else
    launch_verify<_Float16>(a, stages, st);
  return check_launch(who);
}

extern "C" uint64_t rswa_sizeof_tree_params(void) { return sizeof(rswa_tree_params); }
extern "C" uint64_t rswa_sizeof_verify_params(void) { return sizeof(rswa_verify_params); }
