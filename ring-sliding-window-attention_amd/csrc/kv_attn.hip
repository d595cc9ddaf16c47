// Band attention (window + sinks, causal from the sequence's end) of new queries over the 8-bit paged cache.
//
// A wave takes 64 keys at a time and 16 NT rows (a row is a token and one of the q heads that share the kv head):
//   S^T = K Q^T    A = K, straight from memory: lane l loads 16 bytes of key row l%16, widened in registers
//   P^T = exp2(S^T - max)
//   O^T += V^T P^T A = V^T, straight from memory too: a lane's 16 bytes are 16 keys of one dimension
// Nothing goes through LDS: which of the 64 keys is row m of the t-th S^T tile is free to choose, and key
// 16 (m/4) + 4 t + m%4 is the choice by which a lane's 16 scores are 16 consecutive keys -- those of its 16 bytes of
// V -- and already lie as the B operand of the second product wants them.  All 16 are of one group, so that a page's
// scale is one value per lane, folded into the widening.
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

template <typename T, int D, int NT, int WR>
__global__ __launch_bounds__(kThreads, 2) void cache_attn_kernel(const CacheArgs a) {
  using V8 = typename Mma<T>::V8;
  constexpr int KW = 4 / WR;  // waves that share a row tile's keys
  constexpr int ROWS = NT * 16 * WR;
  constexpr int C = D / 64;   // 16-byte pieces of a lane's key row
  constexpr int ND = D / 16;
  constexpr int LD = D + 4;
  __shared__ float lds[KW > 1 ? KW * ROWS * (LD + 2) : 1];

  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int col = lane & 15, hi = lane >> 4;
  const int hk = blockIdx.x % a.heads_kv;
  Unit x;
  if (!find_unit<0>(a, blockIdx.x / a.heads_kv, x)) return;

  const int wr = wave / KW, kw = wave % KW;
  const int r0 = x.row_tile * ROWS + wr * (NT * 16);  // the wave's first row
  const int shift = x.len - x.n_rows;                 // position of token 0
  const int n_flat = x.n_rows * a.group;

  // its rows' tokens, first and last
  const int tok0 = quotient(min(r0, n_flat - 1), a.by_group);
  const int tok1 = quotient(min(r0 + NT * 16, n_flat) - 1, a.by_group);
  const bool some = r0 < n_flat;
  const int first = shift + tok0, last = some ? shift + tok1 : -1;
  const TileList list = chunk_tiles(a, x, first, last);
  const int lo_all = a.window < 0 ? 0 : max(0, first - a.window);

  // B operand: rows of Q, the dimensions in the order in which a lane of A holds K's
  V8 qf[NT][C][2];
  int pos[NT], lo[NT];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    const int r = r0 + nt * 16 + col;
    const int tok = quotient(min(r, n_flat - 1), a.by_group);
    const int head = hk * a.group + min(r, n_flat - 1) - tok * a.group;
    pos[nt] = r < n_flat ? shift + tok : -1;
    lo[nt] = a.window < 0 ? 0 : pos[nt] - a.window;
    const T* q = (const T*)a.q + (int64_t)x.b * a.q_st[0] + (int64_t)(x.row0 + tok) * a.q_st[1] +
                 (int64_t)head * a.q_st[2] + hi * 16;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
      for (int h = 0; h < 2; h++) qf[nt][c][h] = *(const V8*)(q + c * 64 + h * 8);
  }

  const int32_t* table = a.table + (int64_t)x.b * a.table_st;
  const int n_groups = (x.len + kGroupKeys - 1) / kGroupKeys;
  const int per_page = a.page_log2 - 4;
  auto page_ids = [&](int tile) {
    const int g = tile * 4;
    Pages p;
    p.k = table[min(g + (col >> 2), n_groups - 1) >> per_page];
    p.v = table[min(g + hi, n_groups - 1) >> per_page];
    return p;
  };
  const uint8_t* const k_head = a.k + (int64_t)hk * a.k_st[1];
  const uint8_t* const v_head = a.v + (int64_t)hk * a.v_st[1];
  const uint8_t* const ks_head = a.k_scale + (int64_t)hk * a.ks_st[1];
  const uint8_t* const vs_head = a.v_scale + (int64_t)hk * a.vs_st[1];
  // (a page that is not there is read as page 0: within the pool, and masked)
  auto there = [&](int id) { return (uint32_t)id < (uint32_t)a.num_pages; };
  const int in_page = (1 << per_page) - 1;

  u32x4 kb[4][C], vb[ND];
  int ke, ve;
  auto load_k = [&](int tile, int id) {
    const int page = there(id) ? id : 0;
    const int g = min(tile * 4 + (col >> 2), n_groups - 1) & in_page;
    const uint8_t* p = k_head + (int64_t)page * a.k_st[0] + (g * kGroupKeys + (col & 3)) * D + hi * 16;
    ke = ks_head[(int64_t)page * a.ks_st[0]];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int c = 0; c < C; c++) kb[t][c] = *(const u32x4*)(p + t * 4 * D + c * 64);
  };
  auto load_v = [&](int tile, int id) {
    const int page = there(id) ? id : 0;
    const int g = min(tile * 4 + hi, n_groups - 1) & in_page;
    const uint8_t* p = v_head + (int64_t)page * a.v_st[0] + g * (kGroupKeys * D) + col * 16;
    ve = vs_head[(int64_t)page * a.vs_st[0]];
#pragma unroll
    for (int d = 0; d < ND; d++) vb[d] = *(const u32x4*)(p + d * 256);
  };

  f32x4 acc[ND][NT];
  float m[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; nt++) {
    m[nt] = -__builtin_inff();
    l[nt] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; d++) acc[d][nt] = f32x4{0, 0, 0, 0};
  }
  const float sc = 2.f * a.scale_log2;  // (K at half its value)

  const int n = list.count();
  int i = kw;
  Pages now{0, 0}, next{0, 0};
  if (i < n) {
    now = page_ids(list[i]);
    next = page_ids(list[min(i + KW, n - 1)]);
    load_k(list[i], now.k);
    load_v(list[i], now.v);
  }
  for (; i < n; i += KW) {
    const int tile = list[i], tile_next = list[min(i + KW, n - 1)];
    const Pages after = page_ids(list[min(i + 2 * KW, n - 1)]);

    // S^T
    f32x4 s[NT][4];
    const float kscale = half_scale(ke);
#pragma unroll
    for (int t = 0; t < 4; t++) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++) s[nt][t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const V8 kf = widen8<T>(kb[t][c][2 * h], kb[t][c][2 * h + 1], kscale);
#pragma unroll
          for (int nt = 0; nt < NT; nt++) s[nt][t] = Mma<T>::mfma16(kf, qf[nt][c][h], s[nt][t]);
        }
    }
    const bool here = there(now.v);
    const bool more = i + KW < n;
    if (more) load_k(tile_next, next.k);

    // masks, where a row sees part of the tile or a page is missing
    const int j0 = tile * kTileKeys;
    const bool whole = j0 + kTileKeys - 1 <= first && (a.window < 0 || j0 >= last - a.window) &&
                       __builtin_amdgcn_ballot_w64(!here) == 0;
    if (!whole) {
      const int j = j0 + hi * 16;
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int jj = j + 4 * t + e;
            const bool see = here && jj <= pos[nt] && (jj >= lo[nt] || jj < a.n_sink);
            s[nt][t][e] = see ? s[nt][t][e] : -__builtin_inff();
          }
    }

    // softmax: a row's scores are in the four lanes of its column
    V8 pf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float top = s[nt][0][0];
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) top = fmaxf(top, s[nt][t][e]);
      top = columns_max(top);
      if (__builtin_amdgcn_ballot_w64(top > m[nt])) {
        const float m_new = fmaxf(m[nt], top);
        const float shrink = m[nt] == m_new ? 1.f : __builtin_amdgcn_exp2f((m[nt] - m_new) * sc);
        m[nt] = m_new;
        l[nt] *= shrink;
#pragma unroll
        for (int d = 0; d < ND; d++) acc[d][nt] *= shrink;
      }
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

    // what no row of the wave sees may hold anything, NaN codes included: a weight of zero does not cancel those
    if (!whole) {
      const int j = j0 + hi * 16;
      u32x4 keep;
#pragma unroll
      for (int wd = 0; wd < 4; wd++) {
        uint32_t mask = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int jj = j + 4 * wd + e;
          mask |= here && jj <= last && (jj >= lo_all || jj < a.n_sink) ? 0xffu << (8 * e) : 0u;
        }
        keep[wd] = mask;
      }
#pragma unroll
      for (int d = 0; d < ND; d++) vb[d] &= keep;
    }
    const float vscale = half_scale(ve);
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const V8 vf = widen8<T>(vb[d][2 * h], vb[d][2 * h + 1], vscale);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) acc[d][nt] = Mma<T>::mfma16(vf, pf[nt][h], acc[d][nt]);
      }
    if (more) load_v(tile_next, next.v);
    now = next;
    next = after;
  }

#pragma unroll
  for (int nt = 0; nt < NT; nt++) l[nt] = columns_sum(l[nt]);

  // Row r's result: written if the row has one chunk, else left for the join.  d0: first of 4 dimensions.
  const bool direct = x.n_chunks == 1;
  if (!direct && x.part + x.n_chunks > a.part_units) return;  // (cu_seqlens that overlap: more units than rows make)
  const int unit = (x.part + x.chunk_idx) * a.heads_kv + hk;
  auto store = [&](int r, int d0, f32x4 o, float mx, float sum) {
    if (r >= n_flat) return;
    if (direct) {
      const int tok = quotient(r, a.by_group), head = hk * a.group + r - tok * a.group;
      const float inv = sum == 0.f ? 0.f : 2.f / sum;  // (V at half its value)
      T* out = (T*)a.out + (int64_t)x.b * a.o_st[0] + (int64_t)(x.row0 + tok) * a.o_st[1] + (int64_t)head * a.o_st[2];
      *(typename Mma<T>::V4*)(out + d0) = Mma<T>::pack4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
      if (d0 == 0 && a.lse)
        a.lse[(int64_t)x.b * a.lse_st[0] + (int64_t)head * a.lse_st[1] + (int64_t)(x.row0 + tok) * a.lse_st[2]] =
            sum == 0.f ? -__builtin_inff() : (mx * sc - kLift<T> + __log2f(sum)) * (1.f / kLog2e);
    } else {
      const int64_t at = (int64_t)unit * ROWS + (r - x.row_tile * ROWS);
      *(f32x4*)(a.part + at * D + d0) = o;
      if (d0 == 0) *(f32x2*)(a.part_ml + at * 2) = f32x2{mx * sc, sum};
    }
  };

  if constexpr (KW == 1) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int d = 0; d < ND; d++) store(r0 + nt * 16 + col, d * 16 + hi * 4, acc[d][nt], m[nt], l[nt]);
  } else {
    float* ml = lds + KW * ROWS * LD;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int row = (kw * WR + wr) * (NT * 16) + nt * 16 + col;
#pragma unroll
      for (int d = 0; d < ND; d++) *(f32x4*)(lds + row * LD + d * 16 + hi * 4) = acc[d][nt];
      if (hi == 0) *(f32x2*)(ml + row * 2) = f32x2{m[nt], l[nt]};
    }
    __syncthreads();
#pragma unroll 1
    for (int at = threadIdx.x; at < ROWS * (D / 4); at += kThreads) {
      const int row = at / (D / 4), d0 = at % (D / 4) * 4;
      float mx = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < KW; w++) mx = fmaxf(mx, ml[(w * ROWS + row) * 2]);
      f32x4 o = {0, 0, 0, 0};
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < KW; w++) {
        const float mw = ml[(w * ROWS + row) * 2];
        const float f = mw == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((mw - mx) * sc);
        const f32x4 ow = *(const f32x4*)(lds + (w * ROWS + row) * LD + d0);
        sum += f * ml[(w * ROWS + row) * 2 + 1];
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += f * ow[e];
      }
      store(x.row_tile * ROWS + row, d0, o, mx, sum);
    }
  }
}

// Rows of several chunks: the partial results' sum with the weights of their maxima.  A thread has 4 dimensions of
// every P-th chunk of a row, 4 chunks at a time; where rows have many chunks (on average) P threads share a row and
// meet in LDS.  (A thread that went over all chunks one by one waited for each: 7.4 us for the 16 chunks of one token
// over 4001, 17 for 16 drafts of 5.)
template <typename T, int D, int P>
__global__ __launch_bounds__(kThreads) void cache_join_kernel(const CacheArgs a) {
  constexpr int LANES = D / 4, ROWS = kThreads / LANES / P, N = 4;
  __shared__ f32x4 lds_o[P > 1 ? P : 1][ROWS * LANES];
  __shared__ f32x2 lds_ml[P > 1 ? P : 1][ROWS];
  const int hk = blockIdx.x % a.heads_kv;
  Unit x;
  if (!find_unit<ROWS>(a, blockIdx.x / a.heads_kv, x)) return;
  if (x.n_chunks == 1 || x.part + x.n_chunks > a.part_units) return;
  const int lane = threadIdx.x % LANES, r = threadIdx.x / LANES % ROWS, part = threadIdx.x / LANES / ROWS;
  const int d0 = lane * 4;
  const int row = x.row + r - x.row_tile * a.row_tile;
  const bool mine = x.row + r < x.n_rows * a.group;
  float mx = -__builtin_inff(), sum = 0.f;
  f32x4 o = {0, 0, 0, 0};
  // (mx, sum, o) of the chunks so far joined with others'
  auto add = [&](float m, float l, f32x4 v) {
    if (m == -__builtin_inff()) return;  // (nothing seen: v was not written)
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
      const int64_t at = ((int64_t)(x.part + min(c + i * P, x.n_chunks - 1)) * a.heads_kv + hk) * a.row_tile + row;
      ml[i] = *(const f32x2*)(a.part_ml + at * 2);
      v[i] = *(const f32x4*)(a.part + at * D + d0);
    }
#pragma unroll
    for (int i = 0; i < N; i++)
      if (c + i * P < x.n_chunks) add(ml[i][0], ml[i][1], v[i]);
  }
  if constexpr (P > 1) {
    lds_o[part][r * LANES + lane] = o;
    if (lane == 0) lds_ml[part][r] = f32x2{mx, sum};
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int i = 1; i < P; i++) add(lds_ml[i][r][0], lds_ml[i][r][1], lds_o[i][r * LANES + lane]);
  }
  if (!mine) return;
  const int tok = quotient(x.row + r, a.by_group), head = hk * a.group + x.row + r - tok * a.group;
  const float inv = sum == 0.f ? 0.f : 2.f / sum;
  T* out = (T*)a.out + (int64_t)x.b * a.o_st[0] + (int64_t)(x.row0 + tok) * a.o_st[1] + (int64_t)head * a.o_st[2];
  *(typename Mma<T>::V4*)(out + d0) = Mma<T>::pack4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (d0 == 0 && a.lse)
    a.lse[(int64_t)x.b * a.lse_st[0] + (int64_t)head * a.lse_st[1] + (int64_t)(x.row0 + tok) * a.lse_st[2]] =
        sum == 0.f ? -__builtin_inff() : (mx - kLift<T> + __log2f(sum)) * (1.f / kLog2e);
}

// How a call is cut.  Rows of a sequence (on average, of a pack): up to 16 in one tile of a wave, up to 32 in two;
// the four waves of a block then share the keys.  More: each wave has 32 rows of its own.
struct Cut {
  int nt, wr, row_tile, wanted;
  int64_t row_tiles;   // at most, over all sequences
  int64_t part_units;  // at most
  int64_t grid;
};
Cut cut_call(const rswa_cache_params* p) {
  Cut c;
  const int64_t group = p->heads_q / p->heads_kv;
  const int64_t rows = p->cu_seqlens_q ? ceil_div(p->total_q * group, std::max(1, p->batch)) : p->seqlen_q * group;
  c.nt = rows <= 16 ? 1 : 2;
  c.wr = rows <= 64 ? 1 : 4;
  c.row_tile = c.nt * 16 * c.wr;
  c.wanted = kComputeUnits * (c.nt == 1 ? 3 : 2) * 2;
  c.row_tiles = p->cu_seqlens_q ? p->total_q * group / c.row_tile + p->batch
                                : p->batch * ceil_div(p->seqlen_q * group, c.row_tile);
  const int64_t per_head = ceil_div(c.wanted, p->heads_kv) + 1;
  const int64_t most_tiles = ceil_div((int64_t)p->max_pages * p->page_size, kTileKeys);
  const int64_t at_most = std::min(2 * per_head, c.row_tiles * most_tiles);
  c.part_units = most_tiles <= 4 ? 0 : at_most;
  c.grid = (c.row_tiles + std::min(per_head, c.row_tiles * most_tiles)) * p->heads_kv;
  return c;
}
constexpr int kMinChunk = 4;

uint64_t part_bytes(const Cut& c, const rswa_cache_params* p) {
  return (uint64_t)c.part_units * p->heads_kv * c.row_tile * (p->head_dim + 2) * 4;
}

template <typename T, int D>
int launch_attn(CacheArgs& a, const Cut& c, hipStream_t stream) {
  const dim3 grid((unsigned)c.grid), block(kThreads);
  clear_launch_error();
  if (c.nt == 1)
    hipLaunchKernelGGL((cache_attn_kernel<T, D, 1, 1>), grid, block, 0, stream, a);
  else if (c.wr == 1)
    hipLaunchKernelGGL((cache_attn_kernel<T, D, 2, 1>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((cache_attn_kernel<T, D, 2, 4>), grid, block, 0, stream, a);
  if (int rc = check_launch("cache_attn")) return rc;
  if (c.part_units == 0) return RSWA_OK;
  // as many chunks a row (on average) as threads that may share one, or one thread for all
  constexpr int P = kThreads / (D / 4);
  const int64_t rows = a.cu ? a.total_q : (int64_t)a.batch * a.seqlen_q;
  if (c.row_tiles * a.heads_kv * P <= c.wanted) {
    hipLaunchKernelGGL((cache_join_kernel<T, D, P>), dim3((unsigned)(rows * a.heads_q)), block, 0, stream, a);
  } else {
    const int64_t groups = a.cu ? rows * a.group / P + a.batch : a.batch * ceil_div((int64_t)a.seqlen_q * a.group, P);
    hipLaunchKernelGGL((cache_join_kernel<T, D, 1>), dim3((unsigned)(groups * a.heads_kv)), block, 0, stream, a);
  }
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
  a.row_tile = c.row_tile;
  a.min_chunk = kMinChunk;
  a.per_unit = (float)p->heads_kv / (float)c.wanted;
  a.part_units = (int)c.part_units;
  a.part = (float*)p->workspace;
  a.part_ml = a.part + (int64_t)c.part_units * p->heads_kv * c.row_tile * p->head_dim;
  hipStream_t st = (hipStream_t)stream;
  if (p->dtype == RSWA_BF16)
    return p->head_dim == 128 ? launch_attn<__bf16, 128>(a, c, st) : launch_attn<__bf16, 64>(a, c, st);
  return p->head_dim == 128 ? launch_attn<_Float16, 128>(a, c, st) : launch_attn<_Float16, 64>(a, c, st);
}
