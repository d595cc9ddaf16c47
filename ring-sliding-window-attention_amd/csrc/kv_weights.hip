// Sums of the softmax weights of every cached key over a call's rows, added to running sums.
//
// A wave keeps up to 16 NR rows as matrix operands in registers and goes over the keys, 64 at a time: S = Q K^T with
// the keys as columns, exp2(S - lse), and a sum over rows that needs no exchange until a tile's end.  V is not read.
// Few rows: each wave has keys of its own, and K is read once.  More: the four waves of a block share the keys, with
// rows of their own; their sums meet in LDS, in a fixed order, and rows beyond 64 NR come in further rounds over the
// block's keys, whether those rows see them or not: what a window or the sequence's end hides is computed and masked
// (2048 tokens from an empty cache 184 us whatever the window; against 8192 or 32768 keys with a window of 1000 261).
// 32 tokens of as many sequences of 1024 to 16384 keys, 32 / 8 heads: 45 us, 4.2 TB/s, bound by memory.  64 tokens
// against 32001 keys: 28 us, 600 TFLOP/s, of which 8 are blocks' starts and ends (eight tiles each); 700
// TFLOP/s against 200000, bound by issuing vector instructions: an exponential, at a quarter of their rate, for each
// 2 x 128 operations.  (Keys in registers and rows from memory 64 us, waiting for rows 16 at a time.)  Units are equal
// shares of key tiles, not of rows: a pack's long chunk is left to the few blocks that have its keys (63 single tokens
// and a chunk of 2048 against 8000 keys each 6600 us, in calls of their own 117 + 357).
#include "kv_cache.h"

namespace rswa {
namespace {

constexpr int kThreads = 256;

template <typename T, int D, int NR, int RW>
__global__ __launch_bounds__(kThreads, 2) void cache_weights_kernel(const CacheArgs a) {
  using V8 = typename Mma<T>::V8;
  constexpr int KW = 4 / RW;  // waves with keys of their own
  constexpr int C = D / 64;
  __shared__ float lds[2][RW > 1 ? RW * kTileKeys : 1];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int col = lane & 15, hi = lane >> 4;
  const int hk = blockIdx.x % a.heads_kv;
  Unit x;
  if (!find_unit<0>(a, blockIdx.x / a.heads_kv, x)) return;
  const int shift = x.len - x.n_rows, n_flat = x.n_rows * a.group;
  const int rw = wave / KW, kw = wave % KW;
  const float sc = 2.f * a.scale_log2;
  const int32_t* table = a.table + (int64_t)x.b * a.table_st;
  const int n_groups = (x.len + kGroupKeys - 1) / kGroupKeys;
  const int per_page = a.page_log2 - 4, in_page = (1 << per_page) - 1;
  const uint8_t* const k_head = a.k + times(hk, a.k_st[1]);
  const uint8_t* const ks_head = a.k_scale + times(hk, a.ks_st[1]);
  float* const w = a.weights + (int64_t)x.b * a.w_st[0] + (int64_t)hk * a.w_st[1];
  const T* const q_seq = (const T*)a.q + (int64_t)x.b * a.q_st[0] + (int64_t)x.row0 * a.q_st[1] + hi * 16;
  const float* const lse_seq = a.lse + (int64_t)x.b * a.lse_st[0] + (int64_t)x.row0 * a.lse_st[2];

  const int s0 = x.chunk_idx * x.chunk, s1 = min(s0 + x.chunk, x.tiles.count());
  auto tile_of = [&](int slot) { return slot < x.tiles.n_sink ? slot : x.tiles.t_lo + slot - x.tiles.n_sink; };

  // B: column `col` of the t-th product is key 16 (col/4) + 4 t + col%4 of the tile, so that a lane's keys are of one
  // group: one page id and one scale
  auto page_id = [&](int slot) {
    return table[min(tile_of(min(slot, s1 - 1)) * 4 + (col >> 2), n_groups - 1) >> per_page];
  };
  // Of many rows two sets of registers, the next tile's loaded ahead of this one's products (behind the last tile that one
  // again: a branch here makes the compiler wait for more than it must).  us without / with it, 32 / 8 heads, in bursts of
  // 20 calls, which run at lower clocks than calls among others: 64 tokens against 4000 keys 11.9 / 12.6, 32001 32.6 / 31.3,
  // 200000 155 / 148; 2 sequences of 512 against 4096 100 / 95.
  constexpr int BUFS = NR > 1 ? 2 : 1;
  u32x4 kbs[BUFS][4][C];
  int kes[BUFS];
  auto load_keys = [&](u32x4 (&kb)[4][C], int& ke, int tile, int id) {
    const int page = (uint32_t)id < (uint32_t)a.num_pages ? id : 0;
    const int g = min(tile * 4 + (col >> 2), n_groups - 1) & in_page;
    const uint8_t* p = k_head + times(page, a.k_st[0]) + (g * kGroupKeys + (col & 3)) * D + hi * 16;
    ke = ks_head[times(page, a.ks_st[0])];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int c = 0; c < C; c++) kb[t][c] = *(const u32x4*)(p + t * 4 * D + c * 64);
  };

  for (int round = 0; round < n_flat; round += 16 * NR * RW) {
    // A: lane l has row l%16 of each row tile; its results are rows 4 (l/16) .. +3
    const int first_row = round + rw * (16 * NR);
    V8 q[NR][C][2];
    float base[NR][4];
#pragma unroll
    for (int i = 0; i < NR; i++) {
      const int r0 = first_row + 16 * i, r = min(r0 + col, n_flat - 1);
      const int tok = quotient(r, a.by_group), head = hk * a.group + r - tok * a.group;
      const T* p = q_seq + (int64_t)tok * a.q_st[1] + (int64_t)head * a.q_st[2];
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int h = 0; h < 2; h++) q[i][c][h] = *(const V8*)(p + c * 64 + h * 8);
      // rows that are none, or saw nothing, add nothing: exp2(x - inf)
      const float lse = lse_seq[(int64_t)head * a.lse_st[1] + (int64_t)tok * a.lse_st[2]];
      const float mine = r0 + col < n_flat && lse != -__builtin_inff() ? lse * kLog2e : __builtin_inff();
#pragma unroll
      for (int e = 0; e < 4; e++) base[i][e] = __shfl(mine, hi * 4 + e);
    }
    const int first = shift + quotient(min(first_row, n_flat - 1), a.by_group);  // positions of the wave's rows
    const int last = shift + quotient(min(first_row + 16 * NR, n_flat) - 1, a.by_group);

    int slot = s0 + kw;
    if (slot >= s1) return;  // (RW > 1: all waves or none)
    int id = page_id(slot), id_next = page_id(slot + KW);
    load_keys(kbs[0], kes[0], tile_of(slot), id);
    auto step = [&](int slot, u32x4 (&kb)[4][C], int& ke, u32x4 (&kb_next)[4][C], int& ke_next) {
      const int tile = tile_of(slot), j0 = tile * kTileKeys;
      const int id_after = page_id(slot + 2 * KW);
      const bool here = (uint32_t)id < (uint32_t)a.num_pages;
      if (BUFS > 1) load_keys(kb_next, ke_next, tile_of(min(slot + KW, s1 - 1)), id_next);
      const float scale = half_scale(ke);
      const int key = j0 + 16 * (col >> 2) + (col & 3);  // of product 0
      // (lane l takes product l/16's column at the end; the sum so far is read here, a round trip to memory ahead)
      const int at = 16 * (col >> 2) + 4 * hi + (col & 3);
      const bool mine_to_add = rw == 0 && j0 + at < min(x.len, a.w_len);
      const float so_far = mine_to_add ? w[j0 + at] : 0.f;
      float sum[4] = {0, 0, 0, 0};
      // (one test for the tile: with one for each product's rows nothing could be scheduled past the next)
      auto add_rows = [&](auto whole) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
          V8 kf[C][2];
#pragma unroll
          for (int c = 0; c < C; c++) {
            kf[c][0] = widen8<T>(kb[t][c][0], kb[t][c][1], scale);
            kf[c][1] = widen8<T>(kb[t][c][2], kb[t][c][3], scale);
          }
          f32x4 s[NR];
#pragma unroll
          for (int i = 0; i < NR; i++) {
            s[i] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
              for (int h = 0; h < 2; h++) s[i] = Mma<T>::mfma16(q[i][c][h], kf[c][h], s[i]);
          }
#pragma unroll
          for (int i = 0; i < NR; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              float z = __builtin_fmaf(s[i][e], sc, -base[i][e]);
              if constexpr (!decltype(whole)::value) {
                const int j = key + 4 * t;
                const int pos = shift + quotient(min(first_row + 16 * i + hi * 4 + e, n_flat - 1), a.by_group);
                const bool see = here & (j <= pos) & ((a.window < 0) | (j >= pos - a.window) | (j < a.n_sink));
                z = see ? z : -__builtin_inff();  // (last of all: a row whose lse is NaN leaves what it does not see alone)
              }
              sum[t] += __builtin_amdgcn_exp2f(z);
            }
        }
      };
      if (j0 + kTileKeys - 1 <= first && (a.window < 0 || j0 >= last - a.window) &&
          __builtin_amdgcn_ballot_w64(!here) == 0)
        add_rows(std::true_type{});
      else
        add_rows(std::false_type{});
      if (BUFS == 1 && slot + KW < s1) load_keys(kb, ke, tile_of(slot + KW), id_next);
      id = id_next;
      id_next = id_after;
#pragma unroll
      for (int t = 0; t < 4; t++) sum[t] = columns_sum(sum[t]);
      float mine = hi == 0 ? sum[0] : hi == 1 ? sum[1] : hi == 2 ? sum[2] : sum[3];
      if constexpr (RW > 1) {
        // (two buffers: a wave that writes the next tile's has passed the barrier behind the reads of this one's last)
        float* const buf = lds[(slot - s0) & 1];
        buf[rw * kTileKeys + lane] = mine;
        __syncthreads();
        mine = 0.f;
        if (rw == 0)
#pragma unroll
          for (int i = 0; i < RW; i++) mine += buf[i * kTileKeys + lane];
      }
      if (mine_to_add) w[j0 + at] = so_far + mine;
    };
    for (; slot < s1; slot += BUFS * KW) {
      step(slot, kbs[0], kes[0], kbs[BUFS - 1], kes[BUFS - 1]);
      if (BUFS > 1 && slot + KW < s1) step(slot + KW, kbs[BUFS - 1], kes[BUFS - 1], kbs[0], kes[0]);
    }
    if constexpr (RW > 1) __syncthreads();
  }
}

// Rows of a sequence (on average, of a pack): up to 16, up to 64, more.  What either side of the first line takes is the
// rows' registers: with 16 rows a unit holds four blocks, which memory wants; what the second saves is keys widened once
// for each 64 rows.
template <typename T, int D>
void launch_weights(const CacheArgs& a, int64_t rows, int64_t grid, hipStream_t stream) {
  const dim3 blocks((unsigned)grid), threads(kThreads);
  if (rows <= 16)
    hipLaunchKernelGGL((cache_weights_kernel<T, D, 1, 1>), blocks, threads, 0, stream, a);
  else if (rows <= 64)
    hipLaunchKernelGGL((cache_weights_kernel<T, D, 4, 1>), blocks, threads, 0, stream, a);
  else
    hipLaunchKernelGGL((cache_weights_kernel<T, D, 4, 4>), blocks, threads, 0, stream, a);
}

}  // namespace
}  // namespace rswa

extern "C" int rswa_cache_weights(const rswa_cache_params* p, void* stream) {
  using namespace rswa;
  CacheArgs a;
  if (int rc = cache_args(p, "cache_weights", a)) return rc;
  const int64_t rows = p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q;
  if (rows == 0 || p->batch == 0 || p->max_pages == 0) return RSWA_OK;
  if (int rc = cache_query_args(p, "cache_weights", a)) return rc;
  RSWA_REQUIRE(p->weights_len >= 0, RSWA_ERR_INVALID, "cache_weights: negative size");
  RSWA_REQUIRE(p->lse && (p->weights || p->weights_len == 0), RSWA_ERR_INVALID, "cache_weights: null tensor");
  if (p->weights_len == 0) return RSWA_OK;
  a.lse = p->lse;
  for (int i = 0; i < 3; i++) a.lse_st[i] = p->lse_stride[i];
  if (a.cu) a.lse_st[0] = 0;
  a.weights = p->weights;
  a.w_st[0] = p->weights_stride[0];
  a.w_st[1] = p->weights_stride[1];
  a.w_len = p->weights_len;
  a.row_log2 = 30;  // a unit has all rows of its sequence
  const int64_t per_seq = ceil_div(rows, p->batch) * a.group;
  // Units wanted: as many as a compute unit holds of few rows, in one round and a half; of many rows one round, since
  // each block reads all its rows anew (64 tokens against 32001 keys: 6 for each compute unit 46 us, 2 33)
  const int64_t wanted = kComputeUnits * (per_seq <= 16 ? 6 : 2);
  a.min_chunk = per_seq > 64 ? 1 : 4;
  a.per_unit = (float)p->heads_kv / (float)wanted;
  const int64_t per_head = ceil_div(wanted, p->heads_kv) + 1;
  const int64_t most_tiles = ceil_div((int64_t)p->max_pages * p->page_size, kTileKeys);
  const int64_t grid = (p->batch + std::min(per_head, p->batch * most_tiles)) * p->heads_kv;
  RSWA_REQUIRE(grid < (1ll << 31), RSWA_ERR_UNSUPPORTED, "cache_weights: %lld blocks", (long long)grid);
  hipStream_t st = (hipStream_t)stream;
  clear_launch_error();
  if (p->dtype == RSWA_BF16)
    p->head_dim == 128 ? launch_weights<__bf16, 128>(a, per_seq, grid, st) : launch_weights<__bf16, 64>(a, per_seq, grid, st);
  else
    p->head_dim == 128 ? launch_weights<_Float16, 128>(a, per_seq, grid, st)
                       : launch_weights<_Float16, 64>(a, per_seq, grid, st);
  return check_launch("cache_weights");
}
