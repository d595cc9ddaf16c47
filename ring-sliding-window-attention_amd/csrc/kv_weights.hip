// Sums of the softmax weights of every cached key over a call's rows, added to running sums.
//
// A wave keeps 64 keys as matrix operands in registers and goes over the rows, 16 at a time: S = Q K^T with the keys as
// columns, exp2(S - lse), and a sum over rows that needs no exchange until the end.  K is read once, V not at all.
// Few rows (one tile of 16): each wave has keys of its own.  More: the four waves of a block share the keys and take
// every fourth row tile; their sums meet in LDS, in a fixed order.
#include "kv_cache.h"

namespace rswa {
namespace {

constexpr int kThreads = 256;

template <typename T, int D, int RW>
__global__ __launch_bounds__(kThreads, 2) void cache_weights_kernel(const CacheArgs a) {
  using V8 = typename Mma<T>::V8;
  constexpr int KW = 4 / RW;  // waves with keys of their own
  constexpr int C = D / 64;
  __shared__ float lds[RW > 1 ? RW * kTileKeys : 1];
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
  const uint8_t* const k_head = a.k + (int64_t)hk * a.k_st[1];
  const uint8_t* const ks_head = a.k_scale + (int64_t)hk * a.ks_st[1];
  float* const w = a.weights + (int64_t)x.b * a.w_st[0] + (int64_t)hk * a.w_st[1];
  const T* const q_seq = (const T*)a.q + (int64_t)x.b * a.q_st[0] + (int64_t)x.row0 * a.q_st[1];
  const float* const lse_seq = a.lse + (int64_t)x.b * a.lse_st[0] + (int64_t)x.row0 * a.lse_st[2];

  const int s0 = x.chunk_idx * x.chunk, s1 = min(s0 + x.chunk, x.tiles.count());
  for (int slot = s0 + kw; slot < s1; slot += KW) {
    const int tile = slot < x.tiles.n_sink ? slot : x.tiles.t_lo + slot - x.tiles.n_sink;
    const int j0 = tile * kTileKeys;
    // column `col` of the t-th product is key j0 + 16 t + col: one group, one page, one scale
    V8 kf[4][C][2];
    bool here[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const int g = min(tile * 4 + t, n_groups - 1);
      const int id = table[g >> per_page];
      here[t] = (uint32_t)id < (uint32_t)a.num_pages;
      const int page = here[t] ? id : 0;
      const uint8_t* p = k_head + (int64_t)page * a.k_st[0] + ((g & in_page) * kGroupKeys + col) * D + hi * 16;
      const float scale = half_scale(ks_head[(int64_t)page * a.ks_st[0]]);
#pragma unroll
      for (int c = 0; c < C; c++) {
        const u32x4 r = *(const u32x4*)(p + c * 64);
        kf[t][c][0] = widen8<T>(r[0], r[1], scale);
        kf[t][c][1] = widen8<T>(r[2], r[3], scale);
      }
    }
    float sum[4] = {0, 0, 0, 0};
    // rows whose token sees the tile's first key or a later one
    const int tok_first = max(0, j0 - shift);
    const bool sinks = j0 < a.n_sink;
    const int tok_last = a.window < 0 || sinks ? x.n_rows - 1
                                               : (int)min((int64_t)x.n_rows - 1, (int64_t)j0 + kTileKeys - 1 + a.window - shift);
    const int rt0 = tok_first * a.group / 16, rt1 = tok_last < 0 ? 0 : ((tok_last + 1) * a.group + 15) / 16;
    for (int rt = rt0 + rw; rt < rt1; rt += RW) {
      // A: row r = 16 rt + l%16;  the lane's results are rows 16 rt + 4 (l/16) .. +3
      const int r = min(rt * 16 + col, n_flat - 1);
      const int tok = quotient(r, a.by_group);
      const T* q = q_seq + (int64_t)tok * a.q_st[1] + (int64_t)(hk * a.group + r - tok * a.group) * a.q_st[2] + hi * 16;
      V8 qf[C][2];
#pragma unroll
      for (int c = 0; c < C; c++)
#pragma unroll
        for (int h = 0; h < 2; h++) qf[c][h] = *(const V8*)(q + c * 64 + h * 8);
      float base[4];
      int pos[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int re = rt * 16 + hi * 4 + e, rc = min(re, n_flat - 1);
        const int te = quotient(rc, a.by_group);
        const float lse = lse_seq[(int64_t)(hk * a.group + rc - te * a.group) * a.lse_st[1] + (int64_t)te * a.lse_st[2]];
        pos[e] = re < n_flat && lse != -__builtin_inff() ? shift + te : -1;
        base[e] = lse * kLog2e;
      }
#pragma unroll
      for (int t = 0; t < 4; t++) {
        f32x4 s = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
          for (int h = 0; h < 2; h++) s = Mma<T>::mfma16(qf[c][h], kf[t][c][h], s);
        const int j = j0 + 16 * t + col;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const bool see = here[t] && j <= pos[e] && (a.window < 0 || j >= pos[e] - a.window || j < a.n_sink);
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], sc, -base[e]));
          sum[t] += see ? p : 0.f;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 4; t++) sum[t] = columns_sum(sum[t]);
    // lane l takes key l of the tile
    float mine = hi == 0 ? sum[0] : hi == 1 ? sum[1] : hi == 2 ? sum[2] : sum[3];
    if constexpr (RW > 1) {
      lds[rw * kTileKeys + lane] = mine;
      __syncthreads();
      mine = 0.f;
#pragma unroll
      for (int i = 0; i < RW; i++) mine += lds[i * kTileKeys + lane];
      __syncthreads();
    }
    if (rw == 0 && j0 + lane < min(x.len, a.w_len)) w[j0 + lane] += mine;
  }
}

template <typename T, int D>
void launch_weights(const CacheArgs& a, bool share, int64_t grid, hipStream_t stream) {
  if (share)
    hipLaunchKernelGGL((cache_weights_kernel<T, D, 4>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((cache_weights_kernel<T, D, 1>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a);
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
  RSWA_REQUIRE(p->lse && p->weights, RSWA_ERR_INVALID, "cache_weights: null tensor");
  RSWA_REQUIRE(p->weights_len >= 0, RSWA_ERR_INVALID, "cache_weights: negative size");
  a.lse = p->lse;
  for (int i = 0; i < 3; i++) a.lse_st[i] = p->lse_stride[i];
  if (a.cu) a.lse_st[0] = 0;
  a.weights = p->weights;
  a.w_st[0] = p->weights_stride[0];
  a.w_st[1] = p->weights_stride[1];
  a.w_len = p->weights_len;
  a.row_tile = INT32_MAX;  // a unit has all rows of its sequence
  const bool share = ceil_div(rows, p->batch) * a.group > 16;
  const int64_t wanted = kComputeUnits * 6;
  a.min_chunk = share ? 1 : 4;
  a.per_unit = (float)p->heads_kv / (float)wanted;
  const int64_t per_head = ceil_div(wanted, p->heads_kv) + 1;
  const int64_t most_tiles = ceil_div((int64_t)p->max_pages * p->page_size, kTileKeys);
  const int64_t grid = (p->batch + std::min(per_head, p->batch * most_tiles)) * p->heads_kv;
  RSWA_REQUIRE(grid < (1ll << 31), RSWA_ERR_UNSUPPORTED, "cache_weights: %lld blocks", (long long)grid);
  hipStream_t st = (hipStream_t)stream;
  clear_launch_error();
  if (p->dtype == RSWA_BF16)
    p->head_dim == 128 ? launch_weights<__bf16, 128>(a, share, grid, st) : launch_weights<__bf16, 64>(a, share, grid, st);
  else
    p->head_dim == 128 ? launch_weights<_Float16, 128>(a, share, grid, st)
                       : launch_weights<_Float16, 64>(a, share, grid, st);
  return check_launch("cache_weights");
}
