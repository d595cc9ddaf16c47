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
#include "kv_cache.h"

namespace rswa {
namespace {

constexpr int kThreads = 256;

// Weights are taken 2^kLift times as large, and their sum with them, so that it cancels.  fp16: relative to the
// largest they reach down to 2^-38 then instead of 2^-24, below which a long cache's many small weights would be lost.
// bf16, whose values fill the range of the 32-bit sums: a million keys next to the largest value stay below infinity.
template <typename T>
constexpr float kLift = std::is_same_v<T, _Float16> ? 14.f : -20.f;

// The tiles of one row tile in one chunk: `n_a` from tile `a0`, then n_b from tile b0.
struct TileList {
  int a0, n_a, b0, n_b;
  __device__ __forceinline__ int operator[](int i) const { return i < n_a ? a0 + i : b0 + (i - n_a); }
  __device__ __forceinline__ int count() const { return n_a + n_b; }
};

__device__ __forceinline__ TileList chunk_tiles(const CacheArgs& a, const Unit& x, int first, int last) {
  const int s0 = x.chunk_idx * x.chunk, s1 = s0 + x.chunk;
  TileList t;
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
template <typename T, int D, int NT>
struct Rows {
  using V8 = typename Mma<T>::V8;
  static constexpr int C = D / 64;  // 16-byte pieces of a lane's key row
  static constexpr int ND = D / 16;
  V8 q[NT][C][2];
  int pos[NT];
  int first, last;  // positions of the first and the last row (last < 0: no rows)
  f32x4 acc[ND][NT];
  float m[NT], l[NT];
  float sc;

  __device__ __forceinline__ Rows(const CacheArgs& a, const Unit& x, int hk, int r0, int col, int hi) {
    const int shift = x.len - x.n_rows, n_flat = x.n_rows * a.group;  // shift: position of token 0
    first = shift + quotient(min(r0, n_flat - 1), a.by_group);
    last = r0 < n_flat ? shift + quotient(min(r0 + NT * 16, n_flat) - 1, a.by_group) : -1;
    sc = 2.f * a.scale_log2;  // (K at half its value)
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = r0 + nt * 16 + col;
      const int tok = quotient(min(r, n_flat - 1), a.by_group);
      const int head = hk * a.group + min(r, n_flat - 1) - tok * a.group;
      pos[nt] = r < n_flat ? shift + tok : -1;
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
  // scores of what a row does not see become -inf; j: the lane's first key
  __device__ __forceinline__ void mask(const CacheArgs& a, f32x4 (&s)[NT][4], int j, bool here) const {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int lo = a.window < 0 ? 0 : pos[nt] - a.window;
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int jj = j + 4 * t + e;
          const bool see = here && jj <= pos[nt] && (jj >= lo || jj < a.n_sink);
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
  // ... and the weights, P^T
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
        // (weights are rounded to the type of the values' product: half a step of at most 1)
        pf[nt][h] = Mma<T>::pack(p);
      }
      l[nt] += sum;
    }
  }
};

// What take_out_special() left out of tiles i, i + step, .., of those that rows at positions first .. last do not all
// see, for the rows that see it: two products of ones, 1 where a value is positive (negative) and infinite, or NaN, and 1
// where a row sees its key.  A row that has both is NaN.
template <typename T, int D, int NT>
__device__ __forceinline__ void spoil(const CacheArgs& a, Rows<T, D, NT>& w, const Keys<D>& keys, const TileList& list,
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
      const int lo = a.window < 0 ? 0 : w.pos[nt] - a.window;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int jj = j + 8 * h + e;
          p[e] = here && jj <= w.pos[nt] && (jj >= lo || jj < a.n_sink) ? 1.f : 0.f;
        }
        sees[nt][h] = Mma<T>::pack(p);
      }
    }
    const uint8_t* const from = keys.values(tile, id);
    const uint32_t specials = special_from<T>(keys.value_scale(id));
#pragma unroll
    for (int d = 0; d < Rows<T, D, NT>::ND; d++) {
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
  }
}

// The kernel's arguments read again: those of the epilogue alone would be loaded ahead of the loop, where they crowd
// others out of the scalar registers.
__device__ __forceinline__ const CacheArgs& arguments_again() {
  auto p = (const __attribute__((address_space(4))) CacheArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const CacheArgs*)p;
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

// Few rows: the four waves of a block have the same rows, each its own keys, and everything from memory to the output
// stays in registers; the waves meet in LDS at the end.
template <typename T, int D, int NT>
__global__ __launch_bounds__(kThreads, NT == 1 ? 3 : 2) void cache_attn_kernel(const CacheArgs a) {
  using R = Rows<T, D, NT>;
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
  int i = wave;
  Pages next{0, 0};
  bool here = false;  // the lane's group of the tile has its page
  if (i < n) {
    const Pages now = keys.pages(list[i]);
    here = keys.there(now.v);
    next = keys.pages(list[min(i + KW, n - 1)]);
    load_k(list[i], now.k);
    load_v(list[i], now.v);
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
      const u32x4 keep = seen_bytes(a, j0 + hi * 16, here, w.first, w.last);
#pragma unroll
      for (int d = 0; d < ND; d++) vb[d] &= keep;
      if (w.first != w.last) spoiled |= take_out_special(vb, special_from<T>(ve));
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

  const CacheArgs& late = arguments_again();
  if (spoiled) spoil(late, w, keys, list, wave, KW, w.first, w.last);
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
template <typename T, int D, int NT>
__global__ __launch_bounds__(kThreads, 2) void cache_attn_rows_kernel(const CacheArgs a) {
  using R = Rows<T, D, NT>;
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
  const int first = shift + quotient(r0, a.by_group);
  const int last = shift + quotient(min(r0 + 4 * NT * 16, n_flat) - 1, a.by_group);
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
    const u32x4 keep = seen_bytes(a, j0 + hi * 16, here, first, last);
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
  const CacheArgs& late = arguments_again();
  if (n > 0) {  // (each wave has looked at its quarter of the values)
    if (spoiled && lane == 0) any_special = 1;
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(any_special)) spoil(late, w, keys, list, 0, 1, first, last);
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
template <typename T, int D, int P, int GROUPS>
__global__ __launch_bounds__(kThreads) void cache_join_kernel(const CacheArgs a) {
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
Cut cut_call(const rswa_cache_params* p) {
  Cut c;
  const int64_t group = p->heads_q / p->heads_kv;
  const int64_t rows = p->cu_seqlens_q ? ceil_div(p->total_q * group, std::max(1, p->batch)) : p->seqlen_q * group;
  c.nt = rows <= 16 ? 1 : 2;
  const int64_t all_rows = (p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q) * p->heads_q;
  c.wr = rows <= 64 || all_rows < 128 * kComputeUnits ? 1 : 4;
  c.row_tile = c.nt * 16 * c.wr;
  c.row_tiles = p->cu_seqlens_q ? p->total_q * group / c.row_tile + p->batch
                                : p->batch * ceil_div(p->seqlen_q * group, c.row_tile);
  // Units wanted: two for each compute unit, which holds three blocks of up to 16 rows (us, 512 / 1024 / 1536 / 2048 units:
  // one sequence of 131072 48 / 50 / 53 / 55, 128 of head_dim 64 56 / 59 / 62 / 60, 8 of 8192 28 / 28 / 30 / 30, 64 ragged
  // ones, which finer shares even out, 217 / 218 / 207 / 207) and two of more (16 x 5 drafts 37 / 43 / 45 / 46); where those
  // have more row tiles than that, whole rounds.
  const int resident = 2 * kComputeUnits;
  c.wanted =
      c.nt == 1 ? resident : (int)std::min<int64_t>(4, ceil_div(c.row_tiles * p->heads_kv, resident)) * resident;
  const int64_t per_head = ceil_div(c.wanted, p->heads_kv) + 1;
  // tiles that a sequence's rows see at most: what its pages hold, or its rows' windows and the sinks
  int64_t most_tiles = ceil_div((int64_t)p->max_pages * p->page_size, kTileKeys);
  if (p->window_left >= 0) {
    const int64_t rows_seq = p->cu_seqlens_q ? p->total_q : p->seqlen_q;
    most_tiles = std::min(most_tiles, (p->window_left + rows_seq + kTileKeys - 2) / kTileKeys + 1 +
                                          ceil_div(p->num_sink, kTileKeys));
  }
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

template <typename T, int D>
int launch_attn(CacheArgs& a, const Cut& c, hipStream_t stream) {
  const dim3 grid((unsigned)c.grid), block(kThreads);
  clear_launch_error();
  if (c.nt == 1)
    hipLaunchKernelGGL((cache_attn_kernel<T, D, 1>), grid, block, 0, stream, a);
  else if (c.wr == 1)
    hipLaunchKernelGGL((cache_attn_kernel<T, D, 2>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((cache_attn_rows_kernel<T, D, 2>), grid, block, 0, stream, a);
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
    hipLaunchKernelGGL((cache_join_kernel<T, D, P, 1>), join_blocks(1), block, 0, stream, a);
  else if (c.wr == 1)
    hipLaunchKernelGGL((cache_join_kernel<T, D, 1, 1>), join_blocks(P), block, 0, stream, a);
  else
    hipLaunchKernelGGL((cache_join_kernel<T, D, 1, 4>), join_blocks(4 * P), block, 0, stream, a);
  return check_launch("cache_attn join");
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
  if (int rc = cache_query_args(p, "cache_attn", a)) return rc;
  RSWA_REQUIRE(p->out, RSWA_ERR_INVALID, "cache_attn: null tensor");
  RSWA_REQUIRE((uintptr_t)p->out % 16 == 0 && p->out_stride[0] % 8 == 0 && p->out_stride[1] % 8 == 0 &&
                   p->out_stride[2] % 8 == 0,
               RSWA_ERR_UNSUPPORTED, "cache_attn: rows of out must be 16-byte aligned");
  const Cut c = cut_call(p);
  RSWA_REQUIRE(c.grid < (1ll << 31), RSWA_ERR_UNSUPPORTED, "cache_attn: %lld blocks", (long long)c.grid);
  RSWA_REQUIRE(c.part_units == 0 || (p->workspace && (uintptr_t)p->workspace % 16 == 0 &&
                                     p->workspace_bytes >= part_bytes(c, p)),
               RSWA_ERR_INVALID, "cache_attn: workspace of %llu bytes, %llu needed (16-byte aligned)",
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
