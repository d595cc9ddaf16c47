// Band attention (window + sinks, causal from the sequence's end) of new queries over the 8-bit paged cache.
//
// A wave takes 64 keys at a time and 16 NT rows (a row is a token and one of the q heads that share the kv head):
//   S^T = K Q^T    A = K, straight from memory: lane l loads 16 bytes of key row l%16, widened in registers
//   P^T = exp2(S^T - max)
//   O^T += V^T P^T A = V^T, straight from memory too: a lane's 16 bytes are 16 keys of one dimension
// Which of the 64 keys is row m of the t-th S^T tile is free to choose, and key
// 16 (m/4) + 4 t + m%4 is the choice by which a lane's 16 scores are 16 consecutive keys -- those of its 16 bytes of
// V -- and already lie as the B operand of the second product wants them.  All 16 are of one group, so that a page's
// scale is one value per lane, folded into the widening.
// Bound by memory where rows are few: 64 sequences of 256 to 32768 keys, 32 / 8 heads of 128, 217 us, 5.1 TB/s.  The keys
// of long sequences are cut into chunks for the whole chip, whose partial results a second launch joins; one token
// against 4001 keys takes 6.8 + 3.9 us, each a launch and some five round trips to memory in a row.
//
// Queries that are nodes of a tree of drafted tokens (TreeArgs) are the same kernels: their own keys and values, in 16 bits,
// are up to 16 tiles more, of which ancestor bits say who sees whom.  One tree of 32 nodes against 4001 keys 18 us, 12.4 of the
// first kernel: finding its unit 1.6, rows, pages and first keys 2.5, nodes 2.8 (the blocks that have them), two tiles a wave
// 3.5, meeting in LDS 1.4.  64 trees of up to 24 with a window of 4092 (28 / 4 heads of 64, fp16) 83 us, bound by vector work and
// by the second, half-full round of blocks; 32 of 16 to 64, padded to 64, against 512 to 16384 keys 213, 2.3 us a tile (0.92
// PFLOP/s), the rest 13 us before and after each block's loop and unlike blocks.  Every row tile takes all tiles of its sequence's
// nodes, also those that none of its rows sees: one tree of 200 nodes against 4001 keys 54 us, of 1000 227 (as rows of a chunk, whose
// keys are cached, 39 and 90), 8 of 1000 883 (499).
#include "kv_cache.h"

namespace rswa {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxWords = 16;  // of a node's ancestors, at most

// Weights are taken 2^kLift times as large, and their sum with them, so that it cancels.  fp16: relative to the
// largest they reach down to 2^-38 then instead of 2^-24, below which a long cache's many small weights would be lost.
// bf16, whose values fill the range of the 32-bit sums: a million keys next to the largest value stay below infinity.
template <typename T>
constexpr float kLift = std::is_same_v<T, _Float16> ? 14.f : -20.f;

// The tiles of one row tile in one chunk: `n_a` from tile `a0`, then n_b from tile b0 (and of nodes n_d from tile d0).
struct TileList {
  int a0, n_a, b0, n_b, d0, n_d;
  __device__ __forceinline__ int operator[](int i) const { return i < n_a ? a0 + i : b0 + (i - n_a); }
  __device__ __forceinline__ int count() const { return n_a + n_b; }
};

template <typename Args>
__device__ __forceinline__ TileList chunk_tiles(const Args& a, const Unit& x, int first, int last) {
  int s0 = x.chunk_idx * x.chunk, s1 = s0 + x.chunk;
  TileList t;
  t.d0 = t.n_d = 0;
  if constexpr (std::is_same_v<Args, TreeArgs>) {
    t.d0 = min(s0, x.tiles.n_draft);
    t.n_d = last < 0 ? 0 : min(s1, x.tiles.n_draft) - t.d0;
    s0 = max(0, s0 - x.tiles.n_draft);
    s1 = max(0, s1 - x.tiles.n_draft);
  }
  t.a0 = min(s0, x.tiles.n_sink);
  t.n_a = min(s1, x.tiles.n_sink) - t.a0;
  int b0 = x.tiles.t_lo + max(0, s0 - x.tiles.n_sink);
  int b1 = x.tiles.t_lo + min(x.tiles.n_band, s1 - x.tiles.n_sink);
  // the band of these rows alone (its first tiles stay where sink keys are among them)
  if (a.window >= 0 && a.n_sink <= x.tiles.t_lo * kTileKeys) b0 = max(b0, max(0, first - a.window) / kTileKeys);
  b1 = min(b1, last < 0 ? 0 : last / kTileKeys + 1);
  t.b0 = b0;
  t.n_b = max(0, b1 - b0);
  if (last < 0) t.n_a = 0;
  return t;
}

// A lane's groups of a tile: K's rows l%16 are of group (l%16)/4, V's bytes and the scores of group l/16.
struct Pages {
  int k, v;  // ids as the table has them
};

// Where a kv head's keys and values of one sequence are.
template <int D>
struct Keys {
  const CacheArgs& a;
  const int32_t* table;
  const uint8_t *k, *v, *k_scale, *v_scale;
  int n_groups, per_page, col, hi;
  __device__ __forceinline__ Keys(const CacheArgs& args, const Unit& x, int hk, int lane)
      : a(args), table(args.table + (int64_t)x.b * args.table_st), k(args.k + times(hk, args.k_st[1])),
        v(args.v + times(hk, args.v_st[1])), k_scale(args.k_scale + times(hk, args.ks_st[1])),
        v_scale(args.v_scale + times(hk, args.vs_st[1])), n_groups((x.len + kGroupKeys - 1) / kGroupKeys),
        per_page(args.page_log2 - 4), col(lane & 15), hi(lane >> 4) {}
  __device__ __forceinline__ Pages pages(int tile) const {
    const int g = tile * 4;
    return {table[min(g + (col >> 2), n_groups - 1) >> per_page], table[min(g + hi, n_groups - 1) >> per_page]};
  }
  // (a page that is not there is read as page 0: within the pool, and masked)
  __device__ __forceinline__ bool there(int id) const { return (uint32_t)id < (uint32_t)a.num_pages; }
  // row l%16 of the t-th product, 16 bytes from hi * 16 on (and every 64 further)
  __device__ __forceinline__ const uint8_t* key_row(int tile, int t, int id) const {
    const int g = min(tile * 4 + (col >> 2), n_groups - 1) & ((1 << per_page) - 1);
    return k + times(there(id) ? id : 0, a.k_st[0]) + (g * kGroupKeys + 4 * t + (col & 3)) * D + hi * 16;
  }
  __device__ __forceinline__ int key_scale(int id) const { return k_scale[times(there(id) ? id : 0, a.ks_st[0])]; }
  // dimension l%16 (and every 16th further, 256 bytes each), the 16 keys of group hi
  __device__ __forceinline__ const uint8_t* values(int tile, int id) const {
    const int g = min(tile * 4 + hi, n_groups - 1) & ((1 << per_page) - 1);
    return v + times(there(id) ? id : 0, a.v_st[0]) + g * (kGroupKeys * D) + col * 16;
  }
  __device__ __forceinline__ int value_scale(int id) const { return v_scale[times(there(id) ? id : 0, a.vs_st[0])]; }
};

// Do all rows at positions first .. last see the whole tile from key j0 on?  (`here`: the lane's group has its page)
__device__ __forceinline__ bool whole_tile(const CacheArgs& a, int j0, bool here, int first, int last) {
  return j0 + kTileKeys - 1 <= first && (a.window < 0 || j0 >= last - a.window) &&
         __builtin_amdgcn_ballot_w64(!here) == 0;
}

// Bytes of a lane's 16 keys (from j on) that some row at positions first .. last sees.
__device__ __forceinline__ u32x4 seen_bytes(const CacheArgs& a, int j, bool here, int first, int last) {
  const int lo = a.window < 0 ? 0 : max(0, first - a.window);
  u32x4 keep;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    uint32_t mask = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int jj = j + 4 * w + e;
      mask |= here && jj <= last && (jj >= lo || jj < a.n_sink) ? 0xffu << (8 * e) : 0u;
    }
    keep[w] = mask;
  }
  return keep;
}

// A value that is not finite -- NaN, or a code whose value the type of the queries holds as infinite -- makes those rows
// not finite that see its key, and no others; but a weight of zero does not cancel it.  So in tiles that some rows see and
// others do not, the product is taken without such values, and where there were any, spoil() below gives them to their
// rows afterwards.  (In the loop there are no registers for that.)
//
// Half the value of a code of exponent field E at scale byte e is of exponent E + e - 135 and infinite from the type's
// largest exponent + 1 on (four significant bits: nothing lies between the largest finite value and that power of two).
// Codes below E = 1 are m * 2^-9 and reach E = 0 with m = 4, E = -1 with 2, E = -2 with 1.  Returned for each byte: 128
// less the least magnitude that is not finite, so that adding a magnitude carries into the byte's highest bit from there on.
template <typename T>
__device__ __forceinline__ uint32_t special_from(int e) {
  const int n = (std::is_same_v<T, __bf16> ? 128 : 16) + 135 - e;
  const int least = n > 0 ? min(8 * n, 0x7f) : 4 >> min(-n, 2);
  return (uint32_t)(0x80 - least) * 0x01010101u;
}
__device__ __forceinline__ uint32_t spread(uint32_t highest) {  // bytes' highest bits to all of their bits
  return highest | (highest - (highest >> 7));
}
__device__ __forceinline__ uint32_t special_bytes(uint32_t codes, uint32_t from) {
  return spread(((codes & 0x7f7f7f7fu) + from) & 0x80808080u);
}
template <int N>
__device__ __forceinline__ bool take_out_special(u32x4 (&codes)[N], uint32_t from) {
  uint32_t any = 0;
#pragma unroll
  for (int d = 0; d < N; d++)
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const uint32_t special = special_bytes(codes[d][q], from);
      codes[d][q] &= ~special;
      any |= special;
    }
  return __builtin_amdgcn_ballot_w64(any != 0) != 0;
}

// 16 NT rows of a wave from row r0 of the sequence on: B operands of Q (the dimensions in the order in which a lane of
// A holds K's), what each row sees, and the running softmax and output, O^T.
//
// Nodes of a tree (TREE) come behind all cached tokens, at positions that do not follow from the row: a node's is read
// from memory, where the mask needs it.  `first` is the last cached token, which all nodes see unless the window hides it,
// and `last` a bound on the nodes' positions.
template <typename T, int D, int NT, typename Args>
struct Rows {
  using V8 = typename Mma<T>::V8;
  static constexpr bool TREE = std::is_same_v<Args, TreeArgs>;
  static constexpr int C = D / 64;  // 16-byte pieces of a lane's key row
  static constexpr int ND = D / 16;
  V8 q[NT][C][2];
  int pos[NT];
  int first, last;  // positions of the first and the last row (last < 0: no rows)
  f32x4 acc[ND][NT];
  float m[NT], l[NT];
  float sc;

  __device__ __forceinline__ Rows(const Args& a, const Unit& x, int hk, int r0, int col, int hi) {
    const int shift = x.len - x.n_rows, n_flat = x.n_rows * a.group;  // shift: position of token 0
    if constexpr (TREE) {
      first = x.len - 1;
      last = r0 < n_flat ? first + x.n_rows : -1;
    } else {
      first = shift + quotient(min(r0, n_flat - 1), a.by_group);
      last = r0 < n_flat ? shift + quotient(min(r0 + NT * 16, n_flat) - 1, a.by_group) : -1;
    }
    sc = 2.f * a.scale_log2;  // (K at half its value)
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = r0 + nt * 16 + col;
      const int tok = quotient(min(r, n_flat - 1), a.by_group);
      const int head = hk * a.group + min(r, n_flat - 1) - tok * a.group;
      if constexpr (TREE) {
        const int depth = a.depths[(int64_t)x.b * a.depths_st + x.row0 + tok];
        pos[nt] = r < n_flat && depth >= 0 ? x.len + min(depth, x.n_rows - 1) : -1;
      } else {
        pos[nt] = r < n_flat ? shift + tok : -1;
      }
      const T* p = (const T*)a.q + (int64_t)x.b * a.q_st[0] + (int64_t)(x.row0 + tok) * a.q_st[1] +
                   (int64_t)head * a.q_st[2] + hi * 16;
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int h = 0; h < 2; h++) q[nt][c][h] = *(const V8*)(p + c * 64 + h * 8);
      m[nt] = -__builtin_inff();
      l[nt] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; d++) acc[d][nt] = f32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ bool whole(const CacheArgs& a, int j0, bool here) const {
    return whole_tile(a, j0, here, first, last);
  }
  // the last cached token that row nt may see
  __device__ __forceinline__ int upto(int nt) const { return TREE ? (pos[nt] < 0 ? -1 : first) : pos[nt]; }
  // scores of what a row does not see become -inf; j: the lane's first key
  __device__ __forceinline__ void mask(const CacheArgs& a, f32x4 (&s)[NT][4], int j, bool here) const {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int lo = a.window < 0 ? 0 : pos[nt] - a.window, end = upto(nt);
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int jj = j + 4 * t + e;
          const bool see = here && jj <= end && (jj >= lo || jj < a.n_sink);
          s[nt][t][e] = see ? s[nt][t][e] : -__builtin_inff();
        }
    }
  }
  // One tile's step of the running softmax (a row's scores are in the four lanes of its column): the maximum ...
  __device__ __forceinline__ void tops(const f32x4 (&s)[NT][4], float (&top)[NT]) const {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      // (NaN stays NaN, and its weights are: the other maximum would first quiet each score, an instruction apiece)
      float x = s[nt][0][0];
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) x = __builtin_elementwise_maximum(x, s[nt][t][e]);
      top[nt] = columns_max(x);
    }
  }
  // ... what it changes ...
  __device__ __forceinline__ void raise(const float (&top)[NT]) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      if (__builtin_amdgcn_ballot_w64(top[nt] > m[nt])) {
        const float m_new = __builtin_elementwise_maximum(m[nt], top[nt]);
        const float shrink = m[nt] == m_new ? 1.f : __builtin_amdgcn_exp2f((m[nt] - m_new) * sc);
        m[nt] = m_new;
        l[nt] *= shrink;
#pragma unroll
        for (int d = 0; d < ND; d++) acc[d][nt] *= shrink;
      }
    }
  }
  // ... and the weights, P^T (or half of them)
  template <bool HALF = false>
  __device__ __forceinline__ void weigh(const f32x4 (&s)[NT][4], V8 (&pf)[NT][2]) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const float base = m[nt] == -__builtin_inff() ? 0.f : __builtin_fmaf(m[nt], sc, -kLift<T>);
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nt][2 * h + e / 4][e % 4], sc, -base));
          sum += p[e];
        }
        if constexpr (HALF)
#pragma unroll
          for (int e = 0; e < 8; e++) p[e] *= 0.5f;
        // (weights are rounded to the type of the values' product: half a step of at most 1)
        pf[nt][h] = Mma<T>::pack(p);
      }
      l[nt] += sum;
    }
  }
  // nodes that are not there see nothing (tiles that all nodes see are not masked for them)
  __device__ __forceinline__ void leave_out() {
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
      if (pos[nt] < 0) {
        m[nt] = -__builtin_inff();
        l[nt] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; d++) acc[d][nt] = f32x4{0, 0, 0, 0};
      }
  }
};

// Dimensions 16 d .. of O^T: `up` and `down` (A operands) are 1 where a value is positive (negative) and infinite, or NaN,
// `sees` (B) where a row sees its key.
template <typename T, int D, int NT, typename Args, typename V8 = typename Mma<T>::V8>
__device__ __forceinline__ void add_specials(Rows<T, D, NT, Args>& w, int d, const V8 (&up)[2], const V8 (&down)[2],
                                             const V8 (&sees)[NT][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    f32x4 ups = {0, 0, 0, 0}, downs = {0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < 2; h++) {
      ups = Mma<T>::mfma16(up[h], sees[nt][h], ups);
      downs = Mma<T>::mfma16(down[h], sees[nt][h], downs);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float o = w.acc[d][nt][e];
      o = ups[e] > 0.f ? o + __builtin_inff() : o;
      w.acc[d][nt][e] = downs[e] > 0.f ? o - __builtin_inff() : o;
    }
  }
}

// What take_out_special() left out of tiles i, i + step, .., of those that rows at positions first .. last do not all
// see, for the rows that see it: two products of ones, 1 where a value is positive (negative) and infinite, or NaN, and 1
// where a row sees its key.  A row that has both is NaN.
template <typename T, int D, int NT, typename Args>
__device__ __forceinline__ void spoil(const Args& a, Rows<T, D, NT, Args>& w, const Keys<D>& keys, const TileList& list,
                                      int i, int step, int first, int last) {
  using V8 = typename Mma<T>::V8;
  const int n = list.count();
#pragma unroll 1
  for (; i < n; i += step) {
    const int tile = list[i], j = tile * kTileKeys + keys.hi * 16, id = keys.pages(tile).v;
    const bool here = keys.there(id);
    if (whole_tile(a, tile * kTileKeys, here, first, last)) continue;
    V8 sees[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int lo = a.window < 0 ? 0 : w.pos[nt] - a.window, end = w.upto(nt);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int jj = j + 8 * h + e;
          p[e] = here && jj <= end && (jj >= lo || jj < a.n_sink) ? 1.f : 0.f;
        }
        sees[nt][h] = Mma<T>::pack(p);
      }
    }
    const uint8_t* const from = keys.values(tile, id);
    const uint32_t specials = special_from<T>(keys.value_scale(id));
#pragma unroll
    for (int d = 0; d < D / 16; d++) {
      const u32x4 codes = *(const u32x4*)(from + d * 256);
      V8 up[2], down[2];  // (0x38 is the code of 1)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        uint32_t u[2], n[2];
#pragma unroll
        for (int q = 0; q < 2; q++) {
          const uint32_t c = codes[2 * h + q], below = spread(c & 0x80808080u);
          const uint32_t special = special_bytes(c, specials), nan = special_bytes(c, 0x01010101u);
          u[q] = ((special & ~below) | nan) & 0x38383838u;
          n[q] = ((special & below) | nan) & 0x38383838u;
        }
        up[h] = widen8<T>(u[0], u[1], 1.f);
        down[h] = widen8<T>(n[0], n[1], 1.f);
      }
      add_specials(w, d, up, down, sees);
    }
  }
}

// ---- the nodes' own keys and values, 64 to a tile, in their own type ------------------------------------------------
//
// As a tile of the cache: K from memory to the A operand, who sees whom from the nodes' ancestor bits.  Values lie in rows
// and are transposed through LDS, by the block together, into the operands that a tile of the cache is widened to.  The
// running softmax counts operands of the cache at half their value, so the nodes' scores are halved, and their weights for
// the product with V: exact, but for fp16 weights below 2^-27 of the largest, which are multiples of 2^-37 of it.

// Which of a lane's 16 nodes (from 64 tile + 16 hi on) does row nt see?  A bit for each.
template <typename T, int D, int NT>
__device__ __forceinline__ uint32_t seen_nodes(const TreeArgs& a, const Rows<T, D, NT, TreeArgs>& w, const Unit& x, int nt,
                                               int r0, int tile, int hi) {
  const int r = min(r0 + nt * 16 + (lane_id() & 15), x.n_rows * a.group - 1);
  const int64_t row = x.row0 + quotient(r, a.by_group);
  const int j = tile * kTileKeys + 16 * hi, left = max(0, min(16, x.n_rows - j));
  const uint64_t word = (uint64_t)a.ancestors[(int64_t)x.b * a.ancestors_st + row * a.words + tile];
  uint32_t bits = (uint32_t)(word >> (16 * hi)) & ((1u << left) - 1u);
  if (a.window >= 0 && x.n_rows - 1 > a.window) {  // (else no two depths are that far apart)
    const int32_t* const depths = a.depths + (int64_t)x.b * a.depths_st + x.row0;
#pragma unroll 1
    for (int e = 0; e < left; e++) {
      const int place = x.len + depths[j + e];
      if (place < w.pos[nt] - a.window && place >= a.n_sink) bits &= ~(1u << e);
    }
  }
  return w.pos[nt] < 0 ? 0u : bits;
}

template <typename T>
__device__ __forceinline__ bool not_finite(T v) {
  constexpr uint16_t exponent = std::is_same_v<T, __bf16> ? 0x7f80 : 0x7c00;
  return (__builtin_bit_cast(uint16_t, v) & exponent) == exponent;
}

// V^T of a tile of nodes as A operands in `ops` [D / 16][2][64 lanes], without values that are not finite; a byte of
// `special` for each wave says whether it found any.  A thread transposes 8 nodes of 4 dimensions.
template <typename T, int D>
__device__ __forceinline__ void stage_node_values(const TreeArgs& a, const Unit& x, int hk, int tile,
                                                  typename Mma<T>::V8* ops, uint32_t* special) {
  using V4 = typename Mma<T>::V4;
  using V8 = typename Mma<T>::V8;
  constexpr int LANES = D / 4;
  const int d0 = (int)threadIdx.x % LANES * 4, octet = (int)threadIdx.x / LANES;
  bool any = false;
  if (octet < 8) {
    const T* const p = (const T*)a.v_new + (int64_t)x.b * a.vn_st[0] + (int64_t)hk * a.vn_st[2] + d0;
    V4 v[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
      v[e] = *(const V4*)(p + (int64_t)(x.row0 + min(tile * kTileKeys + octet * 8 + e, x.n_rows - 1)) * a.vn_st[1]);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      V8 of;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const bool real = tile * kTileKeys + octet * 8 + e < x.n_rows, special_value = not_finite(v[e][i]);
        of[e] = real && !special_value ? v[e][i] : (T)0.f;
        any |= real && special_value;
      }
      const int d = d0 + i;
      ops[((d / 16) * 2 + (octet & 1)) * 64 + (octet >> 1) * 16 + d % 16] = of;
    }
  }
  const bool found = __builtin_amdgcn_ballot_w64(any) != 0;
  if (lane_id() == 0) ((uint8_t*)special)[threadIdx.x / 64] = found;
}

template <typename T, int D, int NT>
__device__ __forceinline__ void add_nodes(const TreeArgs& a, Rows<T, D, NT, TreeArgs>& w, const Unit& x, int hk, int r0,
                                          int tile, const typename Mma<T>::V8* ops) {
  using R = Rows<T, D, NT, TreeArgs>;
  using V8 = typename Mma<T>::V8;
  const int lane = lane_id(), col = lane & 15, hi = lane >> 4;
  const T* const p = (const T*)a.k_new + (int64_t)x.b * a.kn_st[0] + (int64_t)hk * a.kn_st[2] + hi * 16;
  uint32_t sees[NT];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) sees[nt] = seen_nodes(a, w, x, nt, r0, tile, hi);
  f32x4 s[NT][4];
#pragma unroll
  for (int t = 0; t < 4; t++) {
    const int key = min(tile * kTileKeys + 16 * (col >> 2) + 4 * t + (col & 3), x.n_rows - 1);
    const T* const row = p + (int64_t)(x.row0 + key) * a.kn_st[1];
    V8 kf[R::C][2];
#pragma unroll
    for (int c = 0; c < R::C; c++)
#pragma unroll
      for (int h = 0; h < 2; h++) kf[c][h] = *(const V8*)(row + c * 64 + h * 8);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      s[nt][t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < R::C; c++)
#pragma unroll
        for (int h = 0; h < 2; h++) s[nt][t] = Mma<T>::mfma16(kf[c][h], w.q[nt][c][h], s[nt][t]);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int e = 0; e < 4; e++) s[nt][t][e] = sees[nt] >> (4 * t + e) & 1 ? 0.5f * s[nt][t][e] : -__builtin_inff();
  V8 pf[NT][2];
  float top[NT];
  w.tops(s, top);
  w.raise(top);
  w.template weigh<true>(s, pf);
#pragma unroll
  for (int d = 0; d < R::ND; d++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const V8 vf = ops[(d * 2 + h) * 64 + lane];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) w.acc[d][nt] = Mma<T>::mfma16(vf, pf[nt][h], w.acc[d][nt]);
    }
}

// What stage_node_values() left out of a tile, for the rows that see it (as spoil()).
template <typename T, int D, int NT>
__device__ __forceinline__ void spoil_nodes(const TreeArgs& a, Rows<T, D, NT, TreeArgs>& w, const Unit& x, int hk, int r0,
                                            int tile) {
  using V8 = typename Mma<T>::V8;
  const int lane = lane_id(), col = lane & 15, hi = lane >> 4;
  V8 sees[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const uint32_t bits = seen_nodes(a, w, x, nt, r0, tile, hi);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; e++) p[e] = bits >> (8 * h + e) & 1 ? 1.f : 0.f;
      sees[nt][h] = Mma<T>::pack(p);
    }
  }
  const T* const p = (const T*)a.v_new + (int64_t)x.b * a.vn_st[0] + (int64_t)hk * a.vn_st[2] + col;
#pragma unroll
  for (int d = 0; d < D / 16; d++) {
    V8 up[2], down[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float u[8], n[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int key = tile * kTileKeys + 16 * hi + 8 * h + e;
        const float v = (float)p[(int64_t)(x.row0 + min(key, x.n_rows - 1)) * a.vn_st[1] + d * 16];
        const bool real = key < x.n_rows, nan = v != v;
        u[e] = real && (nan || v == __builtin_inff()) ? 1.f : 0.f;
        n[e] = real && (nan || v == -__builtin_inff()) ? 1.f : 0.f;
      }
      up[h] = Mma<T>::pack(u);
      down[h] = Mma<T>::pack(n);
    }
    add_specials(w, d, up, down, sees);
  }
}

// The kernel's arguments read again: those of the epilogue alone would be loaded ahead of the loop, where they crowd
// others out of the scalar registers.
template <typename Args>
__device__ __forceinline__ const Args& arguments_again() {
  auto p = (const __attribute__((address_space(4))) Args*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const Args*)p;
}

// Where row r's result goes: to the output, or to the join if the row has several chunks.
template <typename T, int D>
struct RowOut {
  T* out = nullptr;
  float* lse = nullptr;
  float* part = nullptr;
  float* part_ml = nullptr;
  __device__ __forceinline__ RowOut(const CacheArgs& a, const Unit& x, int hk, int r, bool direct) {
    if (r >= x.n_rows * a.group) return;
    if (direct) {
      const int tok = quotient(r, a.by_group), head = hk * a.group + r - tok * a.group;
      out = (T*)a.out + (int64_t)x.b * a.o_st[0] + (int64_t)(x.row0 + tok) * a.o_st[1] + (int64_t)head * a.o_st[2];
      if (a.lse)
        lse = a.lse + (int64_t)x.b * a.lse_st[0] + (int64_t)head * a.lse_st[1] + (int64_t)(x.row0 + tok) * a.lse_st[2];
    } else if (x.part >= 0 && x.part <= a.part_units - x.n_chunks) {  // (not so only of cu_seqlens that overlap)
      const int64_t at =
          (((int64_t)(x.part + x.chunk_idx) * a.heads_kv + hk) << a.row_log2) + (r - (x.row_tile << a.row_log2));
      part = a.part + at * D;
      part_ml = a.part_ml + at * 2;
    }
  }
  // four dimensions from d0 on
  __device__ __forceinline__ void put(int d0, f32x4 o, float inv) const {
    if (out) *(typename Mma<T>::V4*)(out + d0) = Mma<T>::pack4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    if (part) *(f32x4*)(part + d0) = o;
  }
  // the row's maximum in base 2, and the sum of its weights
  __device__ __forceinline__ void finish(float mx, float sum) const {
    if (lse) *lse = sum == 0.f ? -__builtin_inff() : (mx - kLift<T> + __log2f(sum)) * (1.f / kLog2e);
    if (part) *(f32x2*)part_ml = f32x2{mx, sum};
  }
  static __device__ __forceinline__ float inverse_of(float sum) { return sum == 0.f ? 0.f : 2.f / sum; }  // (V halved)
};

// A tile of `n` rows from r0 on none of whose nodes is there (padding): is it, and its results.  (Trees padded to twice
// their nodes, 32 sequences of 512 to 16384 keys, 64 nodes: 306 us without this and the order of the rows kernel's first
// loads, 239 with both.)
__device__ __forceinline__ bool no_nodes(const TreeArgs& a, const Unit& x, int r0, int n) {
  const int n_flat = x.n_rows * a.group;
  const int first = quotient(min(r0, n_flat - 1), a.by_group), last = quotient(min(r0 + n, n_flat) - 1, a.by_group);
  const int32_t* const depths = a.depths + (int64_t)x.b * a.depths_st + x.row0;
  uint64_t there = 0;
  for (int i = first; i <= last; i += 64) there |= __builtin_amdgcn_ballot_w64(depths[min(i + lane_id(), last)] >= 0);
  return there == 0;
}
template <typename T, int D>
__device__ __forceinline__ void put_nothing(const TreeArgs& a, const Unit& x, int hk, int r0, int n, int thread,
                                            int threads) {
#pragma unroll 1
  for (int at = thread; at < n * (D / 4); at += threads) {
    const int d0 = at % (D / 4) * 4;
    const RowOut<T, D> to(a, x, hk, r0 + at / (D / 4), x.n_chunks == 1);
    if (to.out) to.put(d0, f32x4{0, 0, 0, 0}, 0.f);
    if (d0 == 0) to.finish(-__builtin_inff(), 0.f);
  }
}

// Few rows: the four waves of a block have the same rows, each its own keys, and everything from memory to the output
// stays in registers; the waves meet in LDS at the end.
template <typename T, int D, int NT, typename Args>
__global__ __launch_bounds__(kThreads, (NT == 1 && !std::is_same_v<Args, TreeArgs>) ? 3 : 2) void cache_attn_kernel(
    const Args a) {
  using R = Rows<T, D, NT, Args>;
  using V8 = typename Mma<T>::V8;
  constexpr int KW = 4, ROWS = NT * 16, C = R::C, ND = R::ND;
  constexpr int LD = D + 4;
  __shared__ float lds[KW * ROWS * (LD + 2)];

  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int col = lane & 15, hi = lane >> 4;
  const int hk = blockIdx.x % a.heads_kv;
  Unit x;
  if (!find_unit<0>(a, blockIdx.x / a.heads_kv, x)) return;
  R w(a, x, hk, x.row_tile * ROWS, col, hi);
  const TileList list = chunk_tiles(a, x, w.first, w.last);
  const Keys<D> keys(a, x, hk, lane);
  u32x4 kb[4][C], vb[ND];
  int ke, ve;
  auto load_k = [&](int tile, int id) {
    ke = keys.key_scale(id);
    const uint8_t* p = keys.key_row(tile, 0, id);
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int c = 0; c < C; c++) kb[t][c] = *(const u32x4*)(p + t * 4 * D + c * 64);
  };
  auto load_v = [&](int tile, int id) {
    ve = keys.value_scale(id);
    const uint8_t* p = keys.values(tile, id);
#pragma unroll
    for (int d = 0; d < ND; d++) vb[d] = *(const u32x4*)(p + d * 256);
  };

  const int n = list.count();
  int i = R::TREE ? (wave - list.n_d) & (KW - 1) : wave;  // (waves that have a tile of nodes come last)
  Pages next{0, 0};
  bool here = false;  // the lane's group of the tile has its page
  if constexpr (R::TREE)
    if (no_nodes(a, x, x.row_tile * ROWS, ROWS))
      return put_nothing<T, D>(arguments_again<Args>(), x, hk, x.row_tile * ROWS, ROWS, threadIdx.x, kThreads);
  if (i < n) {
    const Pages now = keys.pages(list[i]);
    here = keys.there(now.v);
    next = keys.pages(list[min(i + KW, n - 1)]);
    load_k(list[i], now.k);
    load_v(list[i], now.v);
  }
  __shared__ uint32_t lds_special[R::TREE ? kMaxWords : 1];
  if constexpr (R::TREE) {
#pragma unroll 1
    for (int t = 0; t < list.n_d; t++) {
      if (t > 0) __syncthreads();
      stage_node_values<T, D>(a, x, hk, list.d0 + t, (V8*)lds, &lds_special[t]);
      __syncthreads();
      if (wave == (t & (KW - 1))) add_nodes(a, w, x, hk, x.row_tile * ROWS, list.d0 + t, (const V8*)lds);
    }
  }
  bool spoiled = false;  // (one token's rows see the same keys: nothing to tell apart)
  for (; i < n; i += KW) {
    const int j0 = list[i] * kTileKeys, tile_next = list[min(i + KW, n - 1)];
    const Pages after = keys.pages(list[min(i + 2 * KW, n - 1)]);
    f32x4 s[NT][4];
    const float kscale = half_scale(ke);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int t = 0; t < 4; t++) s[nt][t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
          const V8 kf = widen8<T>(kb[t][c][2 * h], kb[t][c][2 * h + 1], kscale);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) s[nt][t] = Mma<T>::mfma16(kf, w.q[nt][c][h], s[nt][t]);
        }
      }
    const bool more = i + KW < n;
    if (more) load_k(tile_next, next.k);
    const bool whole = w.whole(a, j0, here);
    if (!whole) w.mask(a, s, j0 + hi * 16, here);
    V8 pf[NT][2];
    float top[NT];
    w.tops(s, top);
    w.raise(top);
    w.weigh(s, pf);
    // what no row of the wave sees may hold anything, NaN and infinities included: a weight of zero does not cancel those
    if (!whole) {
      const u32x4 keep = seen_bytes(a, j0 + hi * 16, here, R::TREE ? w.first + 1 : w.first, R::TREE ? w.first : w.last);
#pragma unroll
      for (int d = 0; d < ND; d++) vb[d] &= keep;
      if (R::TREE ? a.window >= 0 : w.first != w.last) spoiled |= take_out_special(vb, special_from<T>(ve));
    }
    const float vscale = half_scale(ve);
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const V8 vf = widen8<T>(vb[d][2 * h], vb[d][2 * h + 1], vscale);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) w.acc[d][nt] = Mma<T>::mfma16(vf, pf[nt][h], w.acc[d][nt]);
      }
    if (more) load_v(tile_next, next.v);
    here = keys.there(next.v);
    next = after;
  }

  const Args& late = arguments_again<Args>();
  if (spoiled) spoil(late, w, keys, list, R::TREE ? (wave - list.n_d) & (KW - 1) : wave, KW, w.first, w.last);
  if constexpr (R::TREE) {
    for (int t = wave; t < list.n_d; t += KW)
      if (lds_special[t]) spoil_nodes(late, w, x, hk, x.row_tile * ROWS, list.d0 + t);
    w.leave_out();
    if (list.n_d > 0) __syncthreads();
  }
  float* ml = lds + KW * ROWS * LD;
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    w.l[nt] = columns_sum(w.l[nt]);
    const int row = wave * ROWS + nt * 16 + col;
#pragma unroll
    for (int d = 0; d < ND; d++) *(f32x4*)(lds + row * LD + d * 16 + hi * 4) = w.acc[d][nt];
    if (hi == 0) *(f32x2*)(ml + row * 2) = f32x2{w.m[nt], w.l[nt]};
  }
  __syncthreads();
#pragma unroll 1
  // (the thread's number anew: kept over the loop it would be the one register too many for a third block on the unit)
  for (int at = wave * 64 + lane_id(); at < ROWS * (D / 4); at += kThreads) {
    const int row = at / (D / 4), d0 = at % (D / 4) * 4;
    float mx = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < KW; k++) mx = fmaxf(mx, ml[(k * ROWS + row) * 2]);
    f32x4 o = {0, 0, 0, 0};
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < KW; k++) {
      const float mk = ml[(k * ROWS + row) * 2];
      const float f = mk == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((mk - mx) * w.sc);
      const f32x4 ok = *(const f32x4*)(lds + (k * ROWS + row) * LD + d0);
      sum += f * ml[(k * ROWS + row) * 2 + 1];
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] += f * ok[e];
    }
    const RowOut<T, D> to(late, x, hk, x.row_tile * ROWS + row, x.n_chunks == 1);
    to.put(d0, o, to.inverse_of(sum));
    if (d0 == 0) to.finish(mx * w.sc, sum);
  }
}

// Many rows: each wave has 16 NT of its own, and the block goes over the keys together.  A wave widens a quarter of
// each tile and leaves it in LDS as operands (lane after lane, so that reads and writes have no bank conflicts).  The
// loop is skewed so that matrix and vector work of a wave can run side by side: while the weights of tile i are
// computed the scores of tile i + 1 are multiplied, and while tile i's weights meet its values the next operands are
// widened, K two tiles ahead, V one, and the largest scores of tile i + 1 found (2.4 % less time than after the barrier);
// one barrier a tile.
// 2048 tokens of 32 / 8 heads against 32768 keys: 966 us, 1100 TFLOP/s (a library product of as many operations 873;
// each wave widening all of a tile for itself took a tenth longer, and so did the loop unskewed).  Of the time the matrix
// pipes are busy 49 %, the vector ones 52 %, both at once 15 %, and LDS 59 %: what bounds it is how the two waves of a SIMD
// (all that the registers allow) fill each other's gaps.
template <typename T, int D, int NT, typename Args>
__global__ __launch_bounds__(kThreads, 2) void cache_attn_rows_kernel(const Args a) {
  using R = Rows<T, D, NT, Args>;
  using V8 = typename Mma<T>::V8;
  constexpr int C = R::C, ND = R::ND, NV = ND / 4;
  constexpr int KF = 4 * C * 2, VF = ND * 2;  // operands of a tile
  __shared__ V8 k_ops[2][KF][64], v_ops[2][VF][64];
  __shared__ uint32_t any_special;

  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int col = lane & 15, hi = lane >> 4;
  const int hk = blockIdx.x % a.heads_kv;
  Unit x;
  if (!find_unit<0>(a, blockIdx.x / a.heads_kv, x)) return;
  const int r0 = x.row_tile * (4 * NT * 16);
  R w(a, x, hk, r0 + wave * (NT * 16), col, hi);
  // the block's rows
  const int shift = x.len - x.n_rows, n_flat = x.n_rows * a.group;
  const int first = R::TREE ? x.len - 1 : shift + quotient(r0, a.by_group);
  const int last = R::TREE ? first + x.n_rows : shift + quotient(min(r0 + 4 * NT * 16, n_flat) - 1, a.by_group);
  const TileList list = chunk_tiles(a, x, first, last);
  const Keys<D> keys(a, x, hk, lane);
  const int n = list.count();
  auto tile_at = [&](int i) { return list[min(i, n - 1)]; };  // (loads run past the end on the last tile)

  // the wave's quarter: product `wave` of K, dimensions 16 (NV wave) .. of V
  u32x4 kb[C], vb[NV];
  int ke = 0, ve = 0;
  auto load_k = [&](int tile, int id) {
    ke = keys.key_scale(id);
    const uint8_t* p = keys.key_row(tile, wave, id);
#pragma unroll
    for (int c = 0; c < C; c++) kb[c] = *(const u32x4*)(p + c * 64);
  };
  auto load_v = [&](int tile, int id) {
    ve = keys.value_scale(id);
    const uint8_t* p = keys.values(tile, id) + wave * (NV * 256);
#pragma unroll
    for (int d = 0; d < NV; d++) vb[d] = *(const u32x4*)(p + d * 256);
  };
  auto widen_k = [&](V8 (&to)[KF][64]) {
    const float f = half_scale(ke);
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int h = 0; h < 2; h++) to[(wave * C + c) * 2 + h][lane] = widen8<T>(kb[c][2 * h], kb[c][2 * h + 1], f);
  };
  // (what no row of the block sees may hold anything, NaN and infinities included: a weight of zero does not cancel those)
  bool spoiled = false;
  auto prepare_v = [&](int tile, int id) {
    const int j0 = tile * kTileKeys;
    const bool here = keys.there(id);
    if (whole_tile(a, j0, here, first, last)) return;
    const u32x4 keep = seen_bytes(a, j0 + hi * 16, here, R::TREE ? first + 1 : first, R::TREE ? first : last);
#pragma unroll
    for (int d = 0; d < NV; d++) vb[d] &= keep;
    spoiled |= take_out_special(vb, special_from<T>(ve));
  };
  auto widen_v = [&](V8 (&to)[VF][64]) {
    const float f = half_scale(ve);
#pragma unroll
    for (int d = 0; d < NV; d++) {
#pragma unroll
      for (int h = 0; h < 2; h++) to[(wave * NV + d) * 2 + h][lane] = widen8<T>(vb[d][2 * h], vb[d][2 * h + 1], f);
    }
  };

  f32x4 s0[NT][4], s1[NT][4];
  float top[NT];  // of the next tile's scores
  V8 kf[2][2], vf[2][2];
  // S^T of the tile whose operands are in `op`; they are read four products ahead, the first two before the call
  auto scores = [&](const V8 (&op)[KF][64], f32x4 (&z)[NT][4]) {
#pragma unroll
    for (int i = 0; i < 4 * C; i++) {
      const int t = i / C, c = i % C;
      if (i + 1 < 4 * C)
#pragma unroll
        for (int h = 0; h < 2; h++) kf[(i + 1) & 1][h] = op[(i + 1) * 2 + h][lane];
      if (c == 0)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) z[nt][t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) z[nt][t] = Mma<T>::mfma16(kf[i & 1][h], w.q[nt][c][h], z[nt][t]);
    }
  };

  auto hide = [&](f32x4 (&s)[NT][4], int i, const Pages& of) {
    const int j0 = tile_at(i) * kTileKeys;
    const bool here = keys.there(of.v);
    if (!w.whole(a, j0, here)) w.mask(a, s, j0 + hi * 16, here);
  };

  __shared__ uint32_t lds_special[R::TREE ? kMaxWords : 1];
  // Nodes' values go through the part of LDS that the first step writes, so that the first tiles' loads and the nodes' are
  // on their way together.
  auto& node_ops = v_ops[1];
  if constexpr (R::TREE)
    if (no_nodes(a, x, r0, 4 * NT * 16))
      return put_nothing<T, D>(arguments_again<Args>(), x, hk, r0, 4 * NT * 16, threadIdx.x, kThreads);
  if constexpr (R::TREE)
    if (list.n_d > 0) stage_node_values<T, D>(a, x, hk, list.d0, &node_ops[0][0], &lds_special[0]);
  if constexpr (R::TREE) {
    bool idle = true;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) idle = idle && __builtin_amdgcn_ballot_w64(w.pos[nt] >= 0) == 0;
    if (idle) {
      // A wave whose rows are all padding, or behind the last: its share of the operands, as below, and the same barriers (64
      // sequences of 12 nodes against 4001 keys, three waves of four with rows, 131 -> 110 us; 32 padded trees 220 -> 213).
      Pages p[4] = {};
      if (n > 0) {
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = keys.pages(tile_at(i));
        load_k(tile_at(0), p[0].k);
        load_v(tile_at(0), p[0].v);
        widen_k(k_ops[0]);
        load_k(tile_at(1), p[1].k);
        prepare_v(tile_at(0), p[0].v);
        widen_v(v_ops[0]);
        load_v(tile_at(1), p[1].v);
      }
#pragma unroll 1
      for (int t = 0; t < list.n_d; t++) {
        if (t > 0) {
          __syncthreads();
          stage_node_values<T, D>(a, x, hk, list.d0 + t, &node_ops[0][0], &lds_special[t]);
        }
        __syncthreads();
      }
      if (n > 0) {
        widen_k(k_ops[1]);
        load_k(tile_at(2), p[2].k);
        if (threadIdx.x == 0) any_special = 0;
        __syncthreads();
#pragma unroll 1
        for (int i = 0; i < n; i++) {
          const Pages after = keys.pages(tile_at(i + 4));
          prepare_v(tile_at(i + 1), p[1].v);
          __syncthreads();
          widen_k(k_ops[i & 1]);
          widen_v(v_ops[(i + 1) & 1]);
          load_k(tile_at(i + 3), p[3].k);
          load_v(tile_at(i + 2), p[2].v);
          p[0] = p[1];
          p[1] = p[2];
          p[2] = p[3];
          p[3] = after;
        }
        if (spoiled && lane == 0) any_special = 1;
        __syncthreads();
      }
      return put_nothing<T, D>(arguments_again<Args>(), x, hk, r0 + wave * (NT * 16), NT * 16, lane_id(), 64);
    }
  }
  Pages p[4] = {};  // of tiles i .. i + 3
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = keys.pages(tile_at(i));
    load_k(tile_at(0), p[0].k);
    load_v(tile_at(0), p[0].v);
    widen_k(k_ops[0]);
    load_k(tile_at(1), p[1].k);
    prepare_v(tile_at(0), p[0].v);
    widen_v(v_ops[0]);
    load_v(tile_at(1), p[1].v);
  }
  if constexpr (R::TREE) {
#pragma unroll 1
    for (int t = 0; t < list.n_d; t++) {
      if (t > 0) {
        __syncthreads();
        stage_node_values<T, D>(a, x, hk, list.d0 + t, &node_ops[0][0], &lds_special[t]);
      }
      __syncthreads();
      add_nodes(a, w, x, hk, r0 + wave * (NT * 16), list.d0 + t, &node_ops[0][0]);
    }
  }
  if (n > 0) {
    widen_k(k_ops[1]);
    load_k(tile_at(2), p[2].k);
    if (threadIdx.x == 0) any_special = 0;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; h++) kf[0][h] = k_ops[0][h][lane];
    scores(k_ops[0], s0);
    hide(s0, 0, p[0]);
    w.tops(s0, top);
  }
  // tile i, whose scores are in s and their largest in top; those of the next go to z
  auto step = [&](int i, f32x4 (&s)[NT][4], f32x4 (&z)[NT][4]) {
    const Pages after = keys.pages(tile_at(i + 4));
    prepare_v(tile_at(i + 1), p[1].v);
    // K of tile i + 1 and V of tile i are there; K of tile i and V of tile i - 1, in whose places the next go, are read
    __syncthreads();
    const auto& k_op = k_ops[(i + 1) & 1];
    const auto& v_op = v_ops[i & 1];
#pragma unroll
    for (int h = 0; h < 2; h++) kf[0][h] = k_op[h][lane];
    w.raise(top);

    __builtin_amdgcn_sched_barrier(0);
    V8 pf[NT][2];
    scores(k_op, z);
    w.weigh(s, pf);
#pragma unroll
    for (int h = 0; h < 2; h++) vf[0][h] = v_op[h][lane];
    // (a product, then vector work of the time it takes)
#pragma unroll
    for (int t = 0; t < 4 * C; t++) {
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
      for (int e = 0; e < 2 * NT; e++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    hide(z, i + 1, p[1]);

    // (products with little else between them: their wave goes first, the other fills the gaps; us for 2048 tokens against
    // 32768 keys without 1049, for all products 1031, for these 1009)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int d = 0; d < ND; d++) {
      if (d + 1 < ND)
#pragma unroll
        for (int h = 0; h < 2; h++) vf[(d + 1) & 1][h] = v_op[(d + 1) * 2 + h][lane];
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) w.acc[d][nt] = Mma<T>::mfma16(vf[d & 1][h], pf[nt][h], w.acc[d][nt]);
    }
    w.tops(z, top);
    widen_k(k_ops[i & 1]);
    widen_v(v_ops[(i + 1) & 1]);
    load_k(tile_at(i + 3), p[3].k);
    load_v(tile_at(i + 2), p[2].v);
#pragma unroll
    for (int d = 0; d < ND; d++) {
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
      for (int e = 0; e < 2 * NT; e++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);  // (1 or 3: 2 % more time)
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    p[0] = p[1];
    p[1] = p[2];
    p[2] = p[3];
    p[3] = after;
  };
  for (int i = 0; i < n; i += 2) {
    step(i, s0, s1);
    if (i + 1 < n) step(i + 1, s1, s0);
  }
  const Args& late = arguments_again<Args>();
  if (n > 0) {  // (each wave has looked at its quarter of the values)
    if (spoiled && lane == 0) any_special = 1;
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(any_special)) spoil(late, w, keys, list, 0, 1, first, last);
  }
  if constexpr (R::TREE) {
    for (int t = 0; t < list.n_d; t++)
      if (lds_special[t]) spoil_nodes(late, w, x, hk, r0 + wave * (NT * 16), list.d0 + t);
    w.leave_out();
  }
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    w.l[nt] = columns_sum(w.l[nt]);
    const RowOut<T, D> to(late, x, hk, r0 + wave * (NT * 16) + nt * 16 + col, x.n_chunks == 1);
    const float inv = to.inverse_of(w.l[nt]);
#pragma unroll
    for (int d = 0; d < ND; d++) to.put(d * 16 + hi * 4, w.acc[d][nt], inv);
    if (hi == 0) to.finish(w.m[nt] * w.sc, w.l[nt]);
  }
}

// Rows of several chunks: the partial results' sum with the weights of their maxima.  A thread has 4 dimensions of
// every P-th chunk of a row, 4 chunks at a time; where rows have many chunks (on average) P threads share a row and
// meet in LDS.  (A thread that went over all chunks one by one waited for each: 7.4 us for the 16 chunks of one token
// over 4001, 17 for 16 drafts of 5.)  A block does GROUPS groups of rows in turn: with chunks of a prompt, which mostly
// are not split, most blocks find nothing to do, and 4 groups are 5 us instead of 9; with drafts 7.5 instead of 4.
template <typename T, int D, int P, int GROUPS, typename Args>
__global__ __launch_bounds__(kThreads) void cache_join_kernel(const Args a) {
  constexpr int LANES = D / 4, ROWS = kThreads / LANES / P, N = 4;
  __shared__ f32x4 lds_o[P > 1 ? P : 1][ROWS * LANES];
  __shared__ f32x2 lds_ml[P > 1 ? P : 1][ROWS];
  const int hk = blockIdx.x % a.heads_kv;
  Unit x;
  if (!find_unit<ROWS * GROUPS>(a, blockIdx.x / a.heads_kv, x)) return;
  if (x.n_chunks == 1) return;
  const int lane = threadIdx.x % LANES, r0 = threadIdx.x / LANES % ROWS, part = threadIdx.x / LANES / ROWS, d0 = lane * 4;
#pragma unroll 1
  for (int g = 0; g < GROUPS; g++) {
    const int row = x.row + g * ROWS + r0;
    const int first = x.part + (row >> a.row_log2) * x.n_chunks;  // the row's first partial result
    const bool mine = row < x.n_rows * a.group && first >= 0 && first <= a.part_units - x.n_chunks;
    float mx = -__builtin_inff(), sum = 0.f;
    f32x4 o = {0, 0, 0, 0};
    // (mx, sum, o) of the chunks so far joined with others'
    auto add = [&](float m, float l, f32x4 v) {
      if (l == 0.f) return;  // (saw nothing; a maximum of -inf may also be that of scores that are all NaN, which l is then)
      const float m_new = fmaxf(mx, m);
      const float f0 = __builtin_amdgcn_exp2f(mx - m_new), f1 = __builtin_amdgcn_exp2f(m - m_new);
      mx = m_new;
      sum = sum * f0 + l * f1;
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = o[e] * f0 + v[e] * f1;
    };
    for (int c = mine ? part : x.n_chunks; c < x.n_chunks; c += P * N) {
      f32x2 ml[N];
      f32x4 v[N];
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int64_t at = (((int64_t)(first + min(c + i * P, x.n_chunks - 1)) * a.heads_kv + hk) << a.row_log2) +
                           (row & ((1 << a.row_log2) - 1));
        ml[i] = *(const f32x2*)(a.part_ml + at * 2);
        v[i] = *(const f32x4*)(a.part + at * D + d0);
      }
#pragma unroll
      for (int i = 0; i < N; i++)
        if (c + i * P < x.n_chunks) add(ml[i][0], ml[i][1], v[i]);
    }
    if constexpr (P > 1) {
      lds_o[part][r0 * LANES + lane] = o;
      if (lane == 0) lds_ml[part][r0] = f32x2{mx, sum};
      __syncthreads();
      if (part != 0) return;
#pragma unroll
      for (int i = 1; i < P; i++) add(lds_ml[i][r0][0], lds_ml[i][r0][1], lds_o[i][r0 * LANES + lane]);
    }
    if (mine) {
      const RowOut<T, D> to(a, x, hk, row, true);
      to.put(d0, o, to.inverse_of(sum));
      if (d0 == 0) to.finish(mx, sum);
    }
  }
}

// How a call is cut.  Rows of a sequence (on average, of a pack): up to 16 in one tile of a wave, more in two; the four
// waves of a block share the keys.  Above 64, if tiles of 128 rows are a block for every compute unit: each wave has 32
// rows of its own (us, shared keys / own rows, 32 / 8 heads: 32 sequences of 64 tokens against 1000 keys 78 / 52; 2 of
// 512 against 4096 96 / 90.  Half as many tiles as units: 1 of 512 against 1000 26 / 33, 4096 59 / 59, 32768 367 / 310, 16
// of 32 against 8000 120 / 116, 28 / 4 heads of 64, 3 of 200 against 8000 76 / 98; the host, which does not know the
// lengths, cannot tell these apart.  Fewer: 4 of 64 against 1000 20 / 34, 1 of 64 16 / 22).  All of these have sequences of
// equal counts.  Of a pack with unlike ones the mean chooses, which suits neither: 63 single tokens and a chunk of 512
// against 8000 keys each 280, the two parts in calls of their own 175 + 89; a chunk of 2048 580, apart 176 + 239.
constexpr int kMinChunk = 4;
struct Cut {
  int nt, wr, row_tile, wanted, min_chunk;
  int64_t row_tiles;   // at most, over all sequences
  int64_t part_units;  // at most
  int64_t grid;
};

// Nodes of trees (`words` != 0: tiles that a sequence's nodes are at most) are cut by the tiles of keys that a unit gets in
// a launch of two for each compute unit (32 / 8 heads of 128; us):
//   up to 20 with row tiles of 16: those.  One sequence of 32 nodes against 4001 keys 18.7 (tiles of 32: 20.3), 8 of 6 22 / 27, 2 of
//     32 21 / 24; with 32 tiles a unit, 4 of 32, 31 / 27
//   33 to 64 rows and a tile of 64 for every resident block: waves with 16 rows of their own.  64 sequences of 14 nodes
//     against 1000 keys 44 (shared keys: 61), of 12 against 4001 110 / 134, 128 of 16 against 512 to 4096 158 / 174; fewer, 16 of
//     12, 44 / 40
//   more rows, three quarters of tiles of 128 or more, of packs 128 or more, and from 24 tiles on: waves with 32 rows.  8 of 64
//     against 8000 91 (shared 101), 1 of 64 against 131072 165 / 192, 64 of 24 against 2000 102 / 117, a pack of 32 trees of 16 to 64
//     against 512 to 16384 201 / 245; with 8 tiles, 8 of 32, 51 / 37; packs of 32 trees of 11 to 44 against 2000 to 6000 145 / 136, of
//     64 of up to 24, 28 / 4 heads of 64, window 4092, 106 / 83
// The last are cut twice as fine where they are a block for every compute unit, since then sequences of unlike lengths are not
// evened by their splitting: 32 padded trees of 64 nodes against 512 to 16384 keys 239 -> 213, 16 128 -> 116 (equal lengths lose by
// it: 64 of 24 against 2000 102 -> 113).  Shared keys are not cut finer than once (the packed trees 83; twice as fine 91).
Cut cut_call(const rswa_cache_params* p, int words = 0) {
  Cut c;
  const int resident = 2 * kComputeUnits;
  const int64_t group = p->heads_q / p->heads_kv;
  const int64_t rows = p->cu_seqlens_q ? ceil_div(p->total_q * group, std::max(1, p->batch)) : p->seqlen_q * group;
  // tiles that a sequence's rows see at most: what its pages hold, or its rows' windows and the sinks; and its nodes
  int64_t most_tiles = ceil_div((int64_t)p->max_pages * p->page_size, kTileKeys);
  if (p->window_left >= 0) {
    const int64_t rows_seq = p->cu_seqlens_q ? p->total_q : p->seqlen_q;
    most_tiles = std::min(most_tiles, (p->window_left + rows_seq + kTileKeys - 2) / kTileKeys + 1 +
                                          ceil_div(p->num_sink, kTileKeys));
  }
  if (words) {
    most_tiles += p->cu_seqlens_q ? words : std::min<int64_t>(words, ceil_div(p->seqlen_q, kTileKeys));
    auto blocks = [&](int row_tile) { return p->batch * ceil_div(rows, row_tile) * p->heads_kv; };
    const bool filled = p->cu_seqlens_q ? rows >= 128 : 4 * rows >= 3 * 128 * ceil_div(rows, 128);
    const bool own = rows > 64 ? filled && blocks(128) * most_tiles >= 24 * resident : rows > 32 && blocks(64) >= resident;
    c.wr = own ? 4 : 1;
    c.nt = own ? (rows > 64 ? 2 : 1) : rows <= 16 || blocks(16) * most_tiles <= 20 * resident ? 1 : 2;
  } else {
    c.nt = rows <= 16 ? 1 : 2;
    const int64_t all_rows = (p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q) * p->heads_q;
    c.wr = rows <= 64 || all_rows < 128 * kComputeUnits ? 1 : 4;
  }
  c.row_tile = c.nt * 16 * c.wr;
  c.row_tiles = p->cu_seqlens_q ? p->total_q * group / c.row_tile + p->batch
                                : p->batch * ceil_div(p->seqlen_q * group, c.row_tile);
  // Units wanted: two for each compute unit, which holds three blocks of up to 16 rows (us, 512 / 1024 / 1536 / 2048 units:
  // one sequence of 131072 48 / 50 / 53 / 55, 128 of head_dim 64 56 / 59 / 62 / 60, 8 of 8192 28 / 28 / 30 / 30, 64 ragged
  // ones, which finer shares even out, 217 / 218 / 207 / 207) and two of more (16 x 5 drafts 37 / 43 / 45 / 46); where those
  // have more row tiles than that, whole rounds.
  int64_t rounds = (words ? c.wr : c.nt) == 1 ? 1 : std::min<int64_t>(4, ceil_div(c.row_tiles * p->heads_kv, resident));
  if (words && c.row_tile == 128 && c.row_tiles * p->heads_kv >= kComputeUnits) rounds = std::max<int64_t>(2, rounds);
  c.wanted = (int)rounds * resident;
  const int64_t per_head = ceil_div(c.wanted, p->heads_kv) + 1;
  const int64_t at_most = std::min(ceil_div(8 * per_head, 5), c.row_tiles * most_tiles);
  // few tiles are not split: the join costs what a wave's third tile does (one token: 512 keys 8.0 us whole, 10.1 in two
  // launches, 768 9.2 / 10.2, 1024 10.5 / 10.3; own rows: 500 keys 21.9 / 25.2, 1000 33.2 / 32.7)
  // (a table without columns has no tiles, and chunks of none could not be counted)
  c.min_chunk = most_tiles <= (c.wr == 1 ? 12 : 8) ? std::max(1, (int)most_tiles) : kMinChunk;
  c.part_units = most_tiles <= c.min_chunk ? 0 : at_most;
  c.grid = (c.row_tiles + std::min(per_head, c.row_tiles * most_tiles)) * p->heads_kv;
  return c;
}
uint64_t part_bytes(const Cut& c, const rswa_cache_params* p) {
  return (uint64_t)c.part_units * p->heads_kv * c.row_tile * (p->head_dim + 2) * 4;
}

template <typename T, int D, typename Args>
int launch_attn(const Args& a, const Cut& c, hipStream_t stream) {
  const dim3 grid((unsigned)c.grid), block(kThreads);
  clear_launch_error();
  constexpr bool TREE = std::is_same_v<Args, TreeArgs>;
  if (TREE && c.nt == 1 && c.wr == 4)
    hipLaunchKernelGGL((cache_attn_rows_kernel<T, D, TREE ? 1 : 2, Args>), grid, block, 0, stream, a);
  else if (c.nt == 1)
    hipLaunchKernelGGL((cache_attn_kernel<T, D, 1, Args>), grid, block, 0, stream, a);
  else if (c.wr == 1)
    hipLaunchKernelGGL((cache_attn_kernel<T, D, 2, Args>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((cache_attn_rows_kernel<T, D, 2, Args>), grid, block, 0, stream, a);
  if (int rc = check_launch("cache_attn")) return rc;
  if (c.part_units == 0) return RSWA_OK;
  // as many chunks a row (on average) as threads that may share one, or one thread for all
  constexpr int P = kThreads / (D / 4);
  const int64_t rows = a.cu ? a.total_q : (int64_t)a.batch * a.seqlen_q;
  auto join_blocks = [&](int64_t n) {  // of n rows each
    const int64_t per_head = a.cu ? rows * a.group / n + a.batch : a.batch * ceil_div((int64_t)a.seqlen_q * a.group, n);
    return dim3((unsigned)(per_head * a.heads_kv));
  };
  if (c.row_tiles * a.heads_kv * P <= c.wanted)
    hipLaunchKernelGGL((cache_join_kernel<T, D, P, 1, Args>), join_blocks(1), block, 0, stream, a);
  else if (c.wr == 1)
    hipLaunchKernelGGL((cache_join_kernel<T, D, 1, 1, Args>), join_blocks(P), block, 0, stream, a);
  else
    hipLaunchKernelGGL((cache_join_kernel<T, D, 1, 4, Args>), join_blocks(4 * P), block, 0, stream, a);
  return check_launch("cache_attn join");
}

// The rest of a call whose cache has been looked over.
template <typename Args>
int attention(const rswa_cache_params* p, int words, const char* who, Args& a, void* stream) {
  if (int rc = cache_query_args(p, who, a)) return rc;
  RSWA_REQUIRE(p->out, RSWA_ERR_INVALID, "%s: null tensor", who);
  RSWA_REQUIRE((uintptr_t)p->out % 16 == 0 && p->out_stride[0] % 8 == 0 && p->out_stride[1] % 8 == 0 &&
                   p->out_stride[2] % 8 == 0,
               RSWA_ERR_UNSUPPORTED, "%s: rows of out must be 16-byte aligned", who);
  const Cut c = cut_call(p, words);
  RSWA_REQUIRE(c.grid < (1ll << 31), RSWA_ERR_UNSUPPORTED, "%s: %lld blocks", who, (long long)c.grid);
  RSWA_REQUIRE(c.part_units == 0 || (p->workspace && (uintptr_t)p->workspace % 16 == 0 &&
                                     p->workspace_bytes >= part_bytes(c, p)),
               RSWA_ERR_INVALID, "%s: workspace of %llu bytes, %llu needed (16-byte aligned)", who,
               (unsigned long long)p->workspace_bytes, (unsigned long long)part_bytes(c, p));
  a.out = p->out;
  a.lse = p->lse;
  for (int i = 0; i < 3; i++) {
    a.o_st[i] = p->out_stride[i];
    a.lse_st[i] = p->lse_stride[i];
  }
  if (a.cu) a.o_st[0] = a.lse_st[0] = 0;
  a.row_log2 = __builtin_ctz((unsigned)c.row_tile);
  a.min_chunk = c.min_chunk;
  a.per_unit = (float)p->heads_kv / (float)c.wanted;
  a.part_units = (int)c.part_units;
  a.part = (float*)p->workspace;
  a.part_ml = a.part + (int64_t)c.part_units * p->heads_kv * c.row_tile * p->head_dim;
  hipStream_t st = (hipStream_t)stream;
  if (p->dtype == RSWA_BF16)
    return p->head_dim == 128 ? launch_attn<__bf16, 128>(a, c, st) : launch_attn<__bf16, 64>(a, c, st);
  return p->head_dim == 128 ? launch_attn<_Float16, 128>(a, c, st) : launch_attn<_Float16, 64>(a, c, st);
}

}  // namespace
}  // namespace rswa

extern "C" uint64_t rswa_cache_attn_workspace_bytes(const rswa_cache_params* p) {
  using namespace rswa;
  if (!p || p->heads_kv <= 0 || p->heads_q < p->heads_kv || p->page_size <= 0) return 0;
  return part_bytes(cut_call(p), p);
}

extern "C" int rswa_cache_attn(const rswa_cache_params* p, void* stream) {
  using namespace rswa;
  CacheArgs a;
  if (int rc = cache_args(p, "cache_attn", a)) return rc;
  const int64_t rows = p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q;
  if (rows == 0 || p->batch == 0) return RSWA_OK;
  return attention(p, 0, "cache_attn", a, stream);
}

extern "C" uint64_t rswa_cache_tree_attn_workspace_bytes(const rswa_draft_params* d) {
  using namespace rswa;
  if (!d || d->words <= 0 || d->words > kMaxWords) return 0;
  const rswa_cache_params* p = &d->cache;
  if (p->heads_kv <= 0 || p->heads_q < p->heads_kv || p->page_size <= 0) return 0;
  return part_bytes(cut_call(p, d->words), p);
}

extern "C" int rswa_cache_tree_attn(const rswa_draft_params* d, void* stream) {
  using namespace rswa;
  constexpr const char* who = "cache_tree_attn";
  TreeArgs a{};
  RSWA_REQUIRE(d, RSWA_ERR_INVALID, "%s: null parameters", who);
  const rswa_cache_params* p = &d->cache;
  if (int rc = cache_args(p, who, a)) return rc;
  const int64_t rows = p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q;
  if (rows == 0 || p->batch == 0) return RSWA_OK;
  RSWA_REQUIRE(d->words >= 1 && d->words <= kMaxWords, RSWA_ERR_UNSUPPORTED, "%s: %d words of ancestors (1 to %d)", who,
               d->words, kMaxWords);
  RSWA_REQUIRE(p->cu_seqlens_q || p->seqlen_q <= 64 * d->words, RSWA_ERR_INVALID, "%s: %d nodes, and ancestors of %d", who,
               p->seqlen_q, 64 * d->words);
  RSWA_REQUIRE(d->depths && d->ancestors, RSWA_ERR_INVALID, "%s: null tree", who);
  const void* x[2];
  int64_t st[2][3];
  if (int rc = cache_new_rows(p, who, x, st)) return rc;
  a.depths = d->depths;
  a.ancestors = d->ancestors;
  a.depths_st = a.cu ? 0 : d->depths_stride;
  a.ancestors_st = a.cu ? 0 : d->ancestors_stride;
  a.words = d->words;
  a.k_new = x[0];
  a.v_new = x[1];
  for (int i = 0; i < 3; i++) {
    a.kn_st[i] = st[0][i];
    a.vn_st[i] = st[1][i];
  }
  return attention(p, d->words, who, a, stream);
}

extern "C" uint64_t rswa_sizeof_draft_params(void) { return sizeof(rswa_draft_params); }
