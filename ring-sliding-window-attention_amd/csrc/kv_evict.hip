// Eviction from the 8-bit paged cache by running sums of softmax weights.
//
// Two launches.  The first chooses, a block per (sequence, kv head): the least weight that stays is found by its bits,
// eight at a time from the highest (counts in LDS), then each wave walks a part of the sequence in order and writes
// the kept tokens' numbers behind those of the waves before it.  The second moves: a block makes a new page of one kv
// head, gathers its tokens from wherever they lie, and writes them at the scale that fits them.
#include "kv_cache.h"

namespace rswa {
namespace {

constexpr int kSelectThreads = 1024;

struct EvictArgs {
  CacheArgs c;
  int32_t budget, n_recent;
  const int32_t* new_table;
  int64_t new_table_st;
  int32_t new_max_pages;
  int32_t* new_lens;
  float* new_weights;
  int32_t* kept;
};

// A weight's bits as an unsigned number that grows with it; NaN below everything.
__device__ __forceinline__ uint32_t ordered(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);  // (-0 as 0)
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelectThreads) void cache_select_kernel(const EvictArgs a) {
  constexpr int WAVES = kSelectThreads / 64;
  __shared__ uint32_t hist[256];
  __shared__ uint32_t chosen[2];  // digit, how many are still to be found among its weights
  __shared__ int count[WAVES][2];
  const CacheArgs& c = a.c;
  const int b = blockIdx.x / c.heads_kv, hk = blockIdx.x % c.heads_kv;
  const int len = held_tokens(c, b);
  const int stay = min(len, a.budget);
  const float* w = c.weights + (int64_t)b * c.w_st[0] + (int64_t)hk * c.w_st[1];
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  float* new_w = a.new_weights + (int64_t)blockIdx.x * c.w_len;
  // (tokens without a weight of their own have none)
  auto weight = [&](int j) { return j < c.w_len ? w[j] : 0.f; };

  if (hk == 0 && threadIdx.x == 0) a.new_lens[b] = stay;
  for (int r = stay + threadIdx.x; r < a.budget; r += kSelectThreads) kept[r] = -1;
  for (int r = stay + threadIdx.x; r < c.w_len; r += kSelectThreads) new_w[r] = 0.f;
  if (len <= a.budget) {
    for (int j = threadIdx.x; j < len; j += kSelectThreads) {
      kept[j] = j;
      if (j < c.w_len) new_w[j] = weight(j);
    }
    return;
  }
  // of tokens c0 .. c1 - 1 the `find` with the largest weights
  const int c0 = c.n_sink, c1 = len - a.n_recent;
  int find = a.budget - c.n_sink - a.n_recent;
  uint32_t least = 0;  // bits of the least weight that stays, known from the top
  if (find > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      for (int j = c0 + threadIdx.x; j < c1; j += kSelectThreads) {
        const uint32_t o = ordered(weight(j));
        if (shift == 24 || (o >> (shift + 8)) == (least >> (shift + 8))) atomicAdd(&hist[(o >> shift) & 255], 1u);
      }
      __syncthreads();
      if (threadIdx.x < 64) {
        // lane l: digits 255 - 4 l - 0 .. 3, from the largest down
        uint32_t n[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          n[i] = hist[255 - 4 * threadIdx.x - i];
          sum += n[i];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
          const uint32_t t = __shfl_up(incl, s);
          if ((int)threadIdx.x >= s) incl += t;
        }
        uint32_t above = incl - sum;
        if (above < (uint32_t)find && incl >= (uint32_t)find) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if (above < (uint32_t)find && above + n[i] >= (uint32_t)find) {
              chosen[0] = 255 - 4 * threadIdx.x - i;
              chosen[1] = find - above;
            }
            above += n[i];
          }
        }
      }
      __syncthreads();
      least |= chosen[0] << shift;
      find = chosen[1];
      __syncthreads();
    }
  }
  // `find` of the weights equal to `least` stay: the earliest
  const bool any = a.budget > c.n_sink + a.n_recent;
  const int lane = lane_id(), wave = threadIdx.x / 64;
  const int part = ((len + WAVES - 1) / WAVES + 63) & ~63;
  const int p0 = min(len, wave * part), p1 = min(len, p0 + part);
  auto kind = [&](int j, bool& sure, bool& equal) {
    sure = equal = false;
    if (j >= p1) return;
    if (j < c0 || j >= c1) {
      sure = true;
    } else if (any) {
      const uint32_t o = ordered(weight(j));
      sure = o > least;
      equal = o == least;
    }
  };
  int n_sure = 0, n_equal = 0;
  for (int j = p0; j < p1; j += 64) {
    bool sure, equal;
    kind(j + lane, sure, equal);
    n_sure += __popcll(__builtin_amdgcn_ballot_w64(sure));
    n_equal += __popcll(__builtin_amdgcn_ballot_w64(equal));
  }
  if (lane == 0) {
    count[wave][0] = n_sure;
    count[wave][1] = n_equal;
  }
  __syncthreads();
  int at = 0, equals = 0;  // kept, and equal ones seen, before this wave's part
  for (int i = 0; i < wave; i++) {
    at += count[i][0];
    equals += count[i][1];
  }
  at += min(equals, find);
  const uint64_t below = (1ull << lane) - 1;
  for (int j = p0; j < p1; j += 64) {
    bool sure, equal;
    kind(j + lane, sure, equal);
    const uint64_t eq = __builtin_amdgcn_ballot_w64(equal);
    const bool keep = sure || (equal && equals + __popcll(eq & below) < find);
    const uint64_t k = __builtin_amdgcn_ballot_w64(keep);
    const int r = at + __popcll(k & below);
    if (keep && r < a.budget) {
      kept[r] = j + lane;
      if (r < c.w_len) new_w[r] = weight(j + lane);
    }
    at += __popcll(k);
    equals += __popcll(eq);
  }
}

// One new page of one kv head.  Keys, then values: lane l of a wave has place l%16 of a group, so that tokens that
// lay side by side are read from the same 16 bytes and written to the same 16 bytes.
template <int D>
__global__ __launch_bounds__(256) void cache_move_kernel(const EvictArgs a) {
  __shared__ uint32_t amax[2];
  __shared__ int64_t from[256];     // (source page << 8) + place, -1: none
  __shared__ uint8_t ks[256], vs[256];
  const CacheArgs& c = a.c;
  const int page_size = 1 << c.page_log2;
  const int hk = blockIdx.x % c.heads_kv;
  const int b = blockIdx.x / c.heads_kv / a.new_max_pages, np = blockIdx.x / c.heads_kv % a.new_max_pages;
  const int len = held_tokens(c, b), stay = min(len, a.budget);
  const int r0 = np << c.page_log2;
  const int n = min(page_size, stay - r0);  // tokens of the page
  if (n <= 0) return;
  const int id = a.new_table[(int64_t)b * a.new_table_st + np];
  if ((uint32_t)id >= (uint32_t)c.num_pages) return;
  const int t = threadIdx.x;
  if (t < 2) amax[t] = 0;
  if (t < n) {
    const int j = a.kept[((int64_t)b * c.heads_kv + hk) * a.budget + r0 + t];
    // (weights that another stream changes during the choice may leave numbers out: nothing is looked up by those)
    const int sp = (uint32_t)j < (uint32_t)len ? c.table[(int64_t)b * c.table_st + (j >> c.page_log2)] : -1;
    const bool here = (uint32_t)sp < (uint32_t)c.num_pages;
    from[t] = here ? ((int64_t)sp << 8) + (j & (page_size - 1)) : -1;
    ks[t] = here ? c.k_scale[(int64_t)sp * c.ks_st[0] + (int64_t)hk * c.ks_st[1]] : 0;
    vs[t] = here ? c.v_scale[(int64_t)sp * c.vs_st[0] + (int64_t)hk * c.vs_st[1]] : 0;
  }
  __syncthreads();
  const uint8_t* const k_head = c.k + (int64_t)hk * c.k_st[1];
  const uint8_t* const v_head = c.v + (int64_t)hk * c.v_st[1];
  // largest finite magnitude: of a code the bits without the sign, NaN (0x7f) passed over
  auto value = [](uint32_t code, int e) {
    const uint32_t m = code & 0x7fu;
    const float f = __builtin_amdgcn_cvt_f32_fp8((int)(m == 0x7fu ? 0u : m), 0);
    return __builtin_ldexpf(f, e - 127);
  };
  float mk = 0.f, mv = 0.f;
  for (int i = t; i < n * (D / 4); i += 256) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const int64_t f = from[r];
    if (f < 0) continue;
    const uint32_t w = *(const uint32_t*)(k_head + (f >> 8) * c.k_st[0] + (f & 255) * D + d);
#pragma unroll
    for (int e = 0; e < 4; e++) mk = fmaxf(mk, value(w >> (8 * e), ks[r]));
  }
  for (int i = t; i < ((n + 15) & ~15) * D; i += 256) {
    const int r = i / (16 * D) * 16 + (i & 15), d = i / 16 % D;
    if (r >= n || from[r] < 0) continue;
    const int64_t f = from[r];
    const int s = (int)(f & 255);
    mv = fmaxf(mv, value(v_head[(f >> 8) * c.v_st[0] + (s >> 4) * (16 * D) + d * 16 + (s & 15)], vs[r]));
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    mk = fmaxf(mk, __shfl_xor(mk, s));
    mv = fmaxf(mv, __shfl_xor(mv, s));
  }
  if (lane_id() == 0) {
    atomicMax(&amax[0], __builtin_bit_cast(uint32_t, mk));
    atomicMax(&amax[1], __builtin_bit_cast(uint32_t, mv));
  }
  __syncthreads();
  const int ke = scale_byte(__builtin_bit_cast(float, amax[0])), ve = scale_byte(__builtin_bit_cast(float, amax[1]));
  if (t == 0) {
    const_cast<uint8_t*>(c.k_scale)[(int64_t)id * c.ks_st[0] + (int64_t)hk * c.ks_st[1]] = (uint8_t)ke;
    const_cast<uint8_t*>(c.v_scale)[(int64_t)id * c.vs_st[0] + (int64_t)hk * c.vs_st[1]] = (uint8_t)ve;
  }
  uint8_t* const k_new = const_cast<uint8_t*>(k_head) + (int64_t)id * c.k_st[0];
  uint8_t* const v_new = const_cast<uint8_t*>(v_head) + (int64_t)id * c.v_st[0];
  for (int i = t; i < n * (D / 4); i += 256) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const int64_t f = from[r];
    uint32_t w = 0;
    if (f >= 0) {
      w = *(const uint32_t*)(k_head + (f >> 8) * c.k_st[0] + (f & 255) * D + d);
      if (ks[r] != ke) w = rescale4(w, __builtin_ldexpf(1.f, ks[r] - ke));
    }
    *(uint32_t*)(k_new + r * D + d) = w;
  }
  for (int i = t; i < ((n + 15) & ~15) * D; i += 256) {
    const int r = i / (16 * D) * 16 + (i & 15), d = i / 16 % D;
    if (r >= n) continue;
    const int64_t f = from[r];
    uint32_t w = 0;
    if (f >= 0) {
      const int s = (int)(f & 255);
      w = v_head[(f >> 8) * c.v_st[0] + (s >> 4) * (16 * D) + d * 16 + (s & 15)];
      if (vs[r] != ve) w = rescale4(w, __builtin_ldexpf(1.f, vs[r] - ve));
    }
    v_new[(r >> 4) * (16 * D) + d * 16 + (r & 15)] = (uint8_t)w;
  }
}

}  // namespace
}  // namespace rswa

extern "C" int rswa_cache_evict(const rswa_cache_params* p, void* stream) {
  using namespace rswa;
  EvictArgs a;
  if (int rc = cache_args(p, "cache_evict", a.c)) return rc;
  if (p->batch == 0) return RSWA_OK;
  RSWA_REQUIRE(p->budget > 0, RSWA_ERR_INVALID, "cache_evict: budget %d", p->budget);
  RSWA_REQUIRE(p->num_sink >= 0 && p->num_recent >= 0 && (int64_t)p->num_sink + p->num_recent <= p->budget,
               RSWA_ERR_INVALID, "cache_evict: %d sinks and %d recent tokens in a budget of %d", p->num_sink,
               p->num_recent, p->budget);
  RSWA_REQUIRE(p->num_pages > 0 && p->weights_len >= 0 && p->new_max_pages >= 0, RSWA_ERR_INVALID,
               "cache_evict: a cache without pages, or a negative size");
  RSWA_REQUIRE((p->weights && p->new_weights || p->weights_len == 0) && p->new_page_table && p->new_seqlens && p->kept,
               RSWA_ERR_INVALID, "cache_evict: null tensor");
  RSWA_REQUIRE(p->new_page_table != p->page_table, RSWA_ERR_INVALID,
               "cache_evict: the new pages must be others than the old ones");
  const int64_t most = std::min<int64_t>(p->budget, (int64_t)p->max_pages * p->page_size);
  RSWA_REQUIRE((int64_t)p->new_max_pages * p->page_size >= most, RSWA_ERR_INVALID,
               "cache_evict: a row of new_page_table holds %lld tokens, %lld may stay",
               (long long)p->new_max_pages * p->page_size, (long long)most);
  a.c.weights = p->weights;
  a.c.w_st[0] = p->weights_stride[0];
  a.c.w_st[1] = p->weights_stride[1];
  a.c.w_len = p->weights_len;
  a.c.n_sink = p->num_sink;
  a.budget = p->budget;
  a.n_recent = p->num_recent;
  a.new_table = p->new_page_table;
  a.new_table_st = p->new_page_table_stride;
  a.new_max_pages = (int32_t)ceil_div(most, p->page_size);
  a.new_lens = p->new_seqlens;
  a.new_weights = p->new_weights;
  a.kept = p->kept;
  const int64_t heads = (int64_t)p->batch * p->heads_kv, blocks = heads * a.new_max_pages;
  RSWA_REQUIRE(blocks < (1ll << 31), RSWA_ERR_UNSUPPORTED, "cache_evict: %lld blocks", (long long)blocks);
  hipStream_t st = (hipStream_t)stream;
  clear_launch_error();
  hipLaunchKernelGGL(cache_select_kernel, dim3((unsigned)heads), dim3(kSelectThreads), 0, st, a);
  if (int rc = check_launch("cache_evict select")) return rc;
  if (blocks == 0) return RSWA_OK;
  if (p->head_dim == 128)
    hipLaunchKernelGGL((cache_move_kernel<128>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((cache_move_kernel<64>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  return check_launch("cache_evict move");
}
