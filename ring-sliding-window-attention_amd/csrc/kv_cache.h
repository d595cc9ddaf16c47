// What the kernels over the 8-bit paged cache share: its layout, the lookup of pages, the range of keys that
// queries see, and how a launch's blocks find their work without the host knowing any length.
//
// Register layouts of v_mfma_f32_16x16x32 (wave64): A (16 x 32): lane l holds row l%16, k = 8*(l/16) .. +7;
// B (32 x 16): lane l holds column l%16, the same k; C (16 x 16): lane l holds column l%16, rows 4*(l/16) .. +3.
#pragma once

#include "attn_common.h"

namespace rswa {

constexpr int kTileKeys = 64;   // keys that a wave takes at a time
constexpr int kGroupKeys = 16;  // keys of a group: 16 consecutive bytes for each dimension of V; never in two pages

// Kernel-side view of rswa_cache_params.
struct CacheArgs {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  // page, head (bytes); below 2^32, so that a page's place is one 32 x 32 -> 64 bit product, where one with a 64-bit
  // stride is three multiplications of 16 cycles
  uint32_t k_st[2], v_st[2];
  uint32_t ks_st[2], vs_st[2];
  const int32_t* table;
  int64_t table_st;
  const int32_t* lens;
  const int32_t* cu;  // null: dense
  int32_t num_pages, max_pages, page_log2;
  int32_t batch, heads_q, heads_kv, group;
  int32_t seqlen_q;  // dense
  int32_t total_q;   // packed
  int32_t window, n_sink;  // window < 0: unbounded
  FastDiv by_group;
  // rows
  const void* q;
  void* out;
  float* lse;
  int64_t q_st[3], o_st[3], lse_st[3];
  float scale_log2;  // softmax_scale * log2(e)
  // how the work is cut (see find_unit)
  int32_t row_log2;   // a unit's row tile has 2^row_log2 rows (token x grouped head)
  int32_t min_chunk;  // least tiles of a unit
  float per_unit;     // heads_kv / units wanted
  // partial results of units whose rows have several (workspace)
  float* part;        // [unit][row][D]
  float* part_ml;     // [unit][row][2]: maximum in base 2, sum
  int32_t part_units;
  // running sums of softmax weights
  float* weights;
  int64_t w_st[2];
  int32_t w_len;
};

// ... and of rswa_draft_params: queries that are nodes of a tree of drafted tokens.
struct TreeArgs : CacheArgs {
  const int32_t* depths;
  const int64_t* ancestors;
  int64_t depths_st, ancestors_st;  // sequence
  int32_t words;                    // of a node's ancestors, and tiles of 64 nodes that a sequence has at most
  const void* k_new;                // the nodes' own
  const void* v_new;
  int64_t kn_st[3], vn_st[3];
};

__device__ __forceinline__ int lane_id() {
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
}

// Sums over the lanes up to each (wave64), in the vector pipe: an exchange through LDS takes some 100 cycles, and a
// scan has six in a row.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_or_zero(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, true);
}
__device__ __forceinline__ int wave_scan(int x) {
  x += dpp_or_zero<0x111, 0xf>(x);  // from 1, 2, 4, 8 lanes below, within 16
  x += dpp_or_zero<0x112, 0xf>(x);
  x += dpp_or_zero<0x114, 0xf>(x);
  x += dpp_or_zero<0x118, 0xf>(x);
  x += dpp_or_zero<0x142, 0xa>(x);  // lane 15 of rows 0 and 2 to rows 1 and 3
  x += dpp_or_zero<0x143, 0xc>(x);  // lane 31 to rows 2 and 3
  return x;
}
__device__ __forceinline__ float wave_scan(float v) {
  auto from = [](int moved) { return __builtin_bit_cast(float, moved); };
  auto bits = [](float f) { return __builtin_bit_cast(int, f); };
  v += from(dpp_or_zero<0x111, 0xf>(bits(v)));
  v += from(dpp_or_zero<0x112, 0xf>(bits(v)));
  v += from(dpp_or_zero<0x114, 0xf>(bits(v)));
  v += from(dpp_or_zero<0x118, 0xf>(bits(v)));
  v += from(dpp_or_zero<0x142, 0xa>(bits(v)));
  v += from(dpp_or_zero<0x143, 0xc>(bits(v)));
  return v;
}
// The largest of all lanes' values, none below 0.
__device__ __forceinline__ float wave_max(float v) {
  int x = __float_as_int(v);  // (a positive float's bits grow with it)
  x = max(x, dpp_or_zero<0x111, 0xf>(x));
  x = max(x, dpp_or_zero<0x112, 0xf>(x));
  x = max(x, dpp_or_zero<0x114, 0xf>(x));
  x = max(x, dpp_or_zero<0x118, 0xf>(x));
  x = max(x, dpp_or_zero<0x142, 0xa>(x));
  x = max(x, dpp_or_zero<0x143, 0xc>(x));
  return __int_as_float(__builtin_amdgcn_readlane(x, 63));
}
__device__ __forceinline__ float last_lane(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Lanes l, l^16, l^32, l^48 with each other (the four that have a column of a 16 x 16 product).  A NaN stays one: the
// maximum that passes over NaN would first quiet its arguments, an instruction for each.
__device__ __forceinline__ float columns_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float m = __builtin_elementwise_maximum(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float columns_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return halfwave_sum(__uint_as_float(a[0]) + __uint_as_float(a[1]));
}

__device__ __forceinline__ uint64_t times(int n, uint32_t stride) { return (uint64_t)(uint32_t)n * stride; }

// Tokens that a sequence's row of the page table can hold at most bound its length: no lookup passes its end.
__device__ __forceinline__ int held_tokens(const CacheArgs& a, int len) {
  return max(0, min(len, a.max_pages << a.page_log2));
}

// A sequence as the device's tensors have it, and what it is taken for: a length that the table can hold, rows within
// the tensor whatever cu_seqlens holds.
struct Sequence {
  int len, cu0, cu1;
  __device__ __forceinline__ Sequence(const CacheArgs& a, int b) : len(a.lens[b]), cu0(0), cu1(0) {
    if (a.cu) {
      cu0 = a.cu[b];
      cu1 = a.cu[b + 1];
    }
  }
  __device__ __forceinline__ int tokens(const CacheArgs& a) const { return held_tokens(a, len); }
  __device__ __forceinline__ void rows(const CacheArgs& a, int& row0, int& n) const {
    row0 = a.cu ? max(0, min(cu0, a.total_q)) : 0;
    n = a.cu ? max(row0, min(cu1, a.total_q)) - row0 : a.seqlen_q;
  }
};

// The tiles that rows at positions first .. last (the end of the sequence) see: those of the sink keys ahead of the
// band, from tile 0 on, then n_band from tile t_lo on.  Ahead of them all, n_draft tiles of nodes.
struct SeenTiles {
  int n_sink, t_lo, n_band, n_draft;
  __device__ __forceinline__ int count() const { return n_draft + n_sink + n_band; }
};
__device__ __forceinline__ SeenTiles seen_tiles(const CacheArgs& a, int first, int last) {
  SeenTiles t{0, 0, 0, 0};
  if (last < 0) return t;
  const int lo = a.window < 0 ? 0 : max(0, first - a.window);
  t.t_lo = lo / kTileKeys;
  t.n_band = last / kTileKeys - t.t_lo + 1;
  t.n_sink = min((min(a.n_sink, lo) + kTileKeys - 1) / kTileKeys, t.t_lo);
  return t;
}
// ... and that a sequence's nodes do: all come behind its tokens, the first of them at position `len`.
__device__ __forceinline__ SeenTiles seen_tiles(const TreeArgs& a, int len, int nodes) {
  SeenTiles t{0, 0, 0, min((nodes + kTileKeys - 1) / kTileKeys, a.words)};
  if (len <= 0) return t;
  const int lo = a.window < 0 ? 0 : max(0, len - a.window);
  t.t_lo = lo / kTileKeys;
  t.n_band = (len - 1) / kTileKeys - t.t_lo + 1;  // (0 where the window holds no token and a tile ends with the last)
  t.n_sink = min((min(a.n_sink, lo) + kTileKeys - 1) / kTileKeys, t.t_lo);
  return t;
}

// Which sequence, row tile and share of its key tiles is unit `u`'s?
//
// The host knows no length.  Every wave reads all of them (64 at a time), sums the tiles of the whole call, and cuts
// the tiles of every row tile into chunks of as many as give the launch about the units it was sized for: sequences
// of any lengths make units of nearly one number of tiles, which the hardware then deals (for attention, that is; in the
// weights a row tile is all rows of a sequence, and units of long chunks take longer).  The grid is sized for the bound
//   sum over sequences of row_tiles * chunks <= units wanted / heads_kv + sum of row_tiles
// and what is beyond the last unit ends at once.  Rows of sequences with several chunks are joined from partial
// results; those sequences have at most 8/5 of the units wanted (with x = tiles / chunk, which is above 5/4 there,
// chunks < x + 3/4), which bounds the workspace.
// (The sum of tiles is taken in floating point, within 2^-16 of its value: less than the one unit that the host adds.)
struct Unit {
  int b, row, row_tile, chunk_idx, n_chunks;
  int row0, n_rows, len;
  int chunk;  // tiles
  int part;   // first of the row tile's n_chunks partial results
  SeenTiles tiles;
};

// JOIN > 0: units are JOIN rows from x.row on, and `part` is the sequence's first partial result.
template <int JOIN, typename Args>
__device__ __forceinline__ bool find_unit(const Args& a, int u, Unit& x) {
  constexpr bool TREE = std::is_same_v<Args, TreeArgs>;
  const int lane = lane_id();
  int row0 = 0, n = 0, len = 0, row_tiles = 0;
  SeenTiles t{0, 0, 0, 0};
  auto load = [&](int b) { return Sequence(a, min(b, a.batch - 1)); };
  auto take = [&](const Sequence& s, int b) {
    s.rows(a, row0, n);
    len = s.tokens(a);
    n = b < a.batch ? n : 0;
    row_tiles = (n * a.group + (1 << a.row_log2) - 1) >> a.row_log2;  // (below 2^30 rows)
    if constexpr (TREE)
      t = n > 0 ? seen_tiles(a, len, n) : SeenTiles{0, 0, 0, 0};
    else
      t = n > 0 ? seen_tiles(a, len - n, len - 1) : SeenTiles{0, 0, 0, 0};
  };
  // (fused by hand: attention and join must come to the same chunk)
  float total = 0.f;
  Sequence next = load(lane);
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const Sequence s = next;
    if (a.batch > 64) next = load(b0 + 64 + lane);
    take(s, b0 + lane);
    total = __builtin_fmaf((float)row_tiles, (float)t.count(), total);
  }
  total = last_lane(wave_scan(total));
  x.chunk = max(a.min_chunk, (int)__builtin_ceilf(total * a.per_unit));
  int before = 0, before_part = 0;
  if (a.batch > 64) next = load(lane);
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) {
      const Sequence s = next;
      next = load(b0 + 64 + lane);
      take(s, b0 + lane);
    }
    // (up to a quarter more in one chunk rather than a small one behind it)
    const int chunks = max(1, (t.count() + x.chunk - 1 - x.chunk / 4) / x.chunk);
    const int units = JOIN ? (n * a.group + JOIN - 1) / JOIN : row_tiles * chunks;
    const int parts = chunks > 1 ? row_tiles * chunks : 0;
    const int su = wave_scan(units), sp = wave_scan(parts);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + su > u);
    if (past) {
      const int at = __builtin_ctzll(past);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };
      x.b = b0 + at;
      x.n_chunks = of(chunks);
      const int in_seq = u - before - (of(su) - of(units));
      // (not so only of cu_seqlens that overlap, whose units can be more than 31 bits count)
      if (in_seq < 0 || in_seq >= of(units)) return false;
      x.row = in_seq * JOIN;
      const int tile = JOIN ? 0 : in_seq / x.n_chunks;
      x.chunk_idx = JOIN ? 0 : in_seq - tile * x.n_chunks;
      // (the last rows, which see the most keys, first, so that the launch ends on small units: 8192 tokens from empty 665 us
      // from the first row on, 617 from the last; 4 sequences of 2048 239 / 222)
      x.row_tile = JOIN ? 0 : of(row_tiles) - 1 - tile;
      x.chunk = (of(t.count()) + x.n_chunks - 1) / x.n_chunks;
      x.part = before_part + of(sp) - of(parts) + x.row_tile * x.n_chunks;
      x.row0 = of(row0);
      x.n_rows = of(n);
      x.len = of(len);
      x.tiles.n_sink = of(t.n_sink);
      x.tiles.t_lo = of(t.t_lo);
      x.tiles.n_band = of(t.n_band);
      x.tiles.n_draft = TREE ? of(t.n_draft) : 0;
      return true;
    }
    before += __builtin_amdgcn_readlane(su, 63);
    before_part += __builtin_amdgcn_readlane(sp, 63);
  }
  return false;
}

// Of rows that lie behind `held` tokens of their sequences: sequence b, its rows, and which of the pages that they touch
// (u, from 0 on; below 0: none) is slot u's.  `pages`: of a sequence at most (dense).
__device__ __forceinline__ void touched_page(const CacheArgs& c, int pages, const FastDiv& by_pages, int& u, int& b,
                                             int& row0, int& n) {
  if (c.cu) {
    // sequence b owns the slots from cu[b] / page_size + 2 b on: n tokens touch at most n / page_size + 2 pages.
    // (a search 64 ways at a time, as locate_packed)
    const int lane = lane_id();
    int lo = 0, cnt = c.batch;
    for (;;) {
      const int step = (cnt + 63) >> 6;
      const int i = min(lo + lane * step, lo + cnt - 1);
      const int slot = (max(0, min(c.cu[i], c.total_q)) >> c.page_log2) + 2 * i;
      // (none: rows ahead of the first sequence; the count is unsigned)
      const int at = max((int)__popcll(__builtin_amdgcn_ballot_w64(lane * step < cnt && slot <= u)) - 1, 0);
      lo += at * step;
      if (step == 1) break;
      cnt = min(step, cnt - at * step);
    }
    b = __builtin_amdgcn_readfirstlane(lo);
    Sequence(c, b).rows(c, row0, n);
    u -= (row0 >> c.page_log2) + 2 * b;
  } else {
    b = quotient(u, by_pages);
    u -= b * pages;
    row0 = 0;
    n = c.seqlen_q;
  }
}

// Two e4m3 codes (the low or the high half of a word) times a power of two, in the matrix operand's type: one
// instruction, exact as long as the value fits the type.
template <typename T, bool HIGH>
__device__ __forceinline__ uint32_t widen2(uint32_t codes, float scale) {
  if constexpr (std::is_same_v<T, __bf16>)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HIGH));
}
template <typename T>
__device__ __forceinline__ typename Mma<T>::V8 widen8(uint32_t lo, uint32_t hi, float scale) {
  u32x4 r = {widen2<T, false>(lo, scale), widen2<T, true>(lo, scale), widen2<T, false>(hi, scale),
             widen2<T, true>(hi, scale)};
  return __builtin_bit_cast(typename Mma<T>::V8, r);
}

// Half of the power of two that scale byte `e` stands for.  Operands are taken at half their value (and scores and
// outputs doubled, which costs nothing): rounding to e4m3 can raise a value just below the 16-bit type's largest
// past it, and half of that is always there.  What it costs: fp16 operands below 2^-20 are
// multiples of 2^-23, where the type has 2^-24 (off by 2^-24 at most).
__device__ __forceinline__ float half_scale(int e) {
  return __builtin_bit_cast(float, (uint32_t)(max(e, 1) - 1) << 23);
}

// Byte of the least 2^e with amax <= 448 * 2^e (448 = 1.75 * 2^8), -120 <= e <= 120.
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return max(7, min(247, e));
}
__device__ __forceinline__ float inverse(int e) {  // 2^(127 - e)
  return __builtin_bit_cast(float, (uint32_t)max(0, 254 - e) << 23);
}

// Four codes of fp32 values within +-448 (rounded to the nearest, ties to even; non-finite ones to NaN).
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
// Four codes times f <= 1, rounded anew.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return codes4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}

// Checks of rswa_cache_params that every call makes, and the kernels' view of them.
int cache_args(const rswa_cache_params* p, const char* who, CacheArgs& a);
int cache_query_args(const rswa_cache_params* p, const char* who, CacheArgs& a);
// Rows that a call's new keys and values are, or go to.
int cache_new_rows(const rswa_cache_params* p, const char* who, const void* (&x)[2], int64_t (&st)[2][3]);

}  // namespace rswa
