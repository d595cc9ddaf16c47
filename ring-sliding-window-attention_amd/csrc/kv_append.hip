// New keys and values into the 8-bit paged cache.
//
// A block takes one page of one kv head, the first half of its threads the keys, the second the values.  A thread has
// 16 tokens (a group) of 8 dimensions: 16 loads of 16 bytes, all in flight before the first use, hold the whole page in
// registers, so that its largest value is known before the first code is made and memory is read once.  Keys leave as
// 8 bytes a row, values as 16 bytes a dimension (the transpose is byte permutations).  Bound by memory: prompts of
// 31500 tokens together, 8 heads of 128, 194 MB in 43 us, 4.5 TB/s (values stored a byte at a time 60 us).
#include "kv_cache.h"

namespace rswa {
namespace {

struct AppendArgs {
  CacheArgs c;
  const void* x[2];  // new keys, values
  int64_t x_st[2][3];
  int32_t pages;     // dense: pages that a sequence's new tokens touch at most
  int32_t work;      // blocks with work
  FastDiv by_pages, by_heads;
};

template <typename T, int D>
__global__ void cache_append_kernel(const AppendArgs a) {
  using V8 = typename Mma<T>::V8;
  constexpr int LANES = D / 8;
  __shared__ uint32_t amax[2];
  const CacheArgs& c = a.c;
  const int page_size = 1 << c.page_log2;
  // Hardware deals block ids to the 8 XCDs in turn; each takes an eighth of the work in a row here, so that the heads of
  // a page, whose rows of the input lie side by side, are read by one.
  const int id0 = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  if (id0 >= a.work) return;
  int u = quotient(id0, a.by_heads), b, row0, n;
  const int hk = id0 - u * c.heads_kv;
  // sequence, and which of its touched pages
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
    b = quotient(u, a.by_pages);
    u -= b * a.pages;
    row0 = 0;
    n = c.seqlen_q;
  }
  if (u < 0) return;
  const int start = max(0, c.lens[b]);
  const int in_seq = (start >> c.page_log2) + u;  // page of the sequence
  if (in_seq >= c.max_pages) return;
  const int from = u == 0 ? start & (page_size - 1) : 0;     // first place written
  const int i0 = (in_seq << c.page_log2) + from - start;     // its token among the new ones
  const int count = min(page_size - from, n - i0);
  if (count <= 0) return;
  const int id = c.table[(int64_t)b * c.table_st + in_seq];

  const int half = blockDim.x / 2;
  const int which = threadIdx.x >= half;
  const int t = threadIdx.x - which * half;
  const int d0 = t % LANES * 8, g = t / LANES;  // 8 dimensions, group of 16 places
  const bool mine = g < (page_size >> 4);       // (blocks of small pages have threads left over)
  const int lo = max(0, from - g * 16), hi = min(16, from + count - g * 16);  // its places written: lo <= e < hi

  // (read ahead of the page's number, on which nothing of it depends)
  const T* x = (const T*)a.x[which] + (int64_t)b * a.x_st[which][0] + (int64_t)hk * a.x_st[which][2] + d0 +
               (int64_t)(row0 + i0 + g * 16 - from) * a.x_st[which][1];  // (of place 0, which may be none of them)
  V8 v[16];
  if (mine && lo == 0 && hi == 16) {
#pragma unroll
    for (int e = 0; e < 16; e++) v[e] = __builtin_nontemporal_load((const V8*)(x + e * a.x_st[which][1]));
  } else {
#pragma unroll
    for (int e = 0; e < 16; e++) {
      v[e] = V8{};
      if (mine && e >= lo && e < hi) v[e] = *(const V8*)(x + e * a.x_st[which][1]);
    }
  }
  if ((uint32_t)id >= (uint32_t)c.num_pages) return;
  uint8_t* const scale = which ? const_cast<uint8_t*>(c.v_scale) + times(id, c.vs_st[0]) + times(hk, c.vs_st[1])
                               : const_cast<uint8_t*>(c.k_scale) + times(id, c.ks_st[0]) + times(hk, c.ks_st[1]);
  const int was = from > 0 ? *scale : 0;
  if (threadIdx.x < 2) amax[threadIdx.x] = 0;
  float most = 0.f;
#pragma unroll
  for (int e = 0; e < 16; e++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float y = __builtin_fabsf((float)v[e][i]);
      most = y < __builtin_inff() ? fmaxf(most, y) : most;
    }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) most = fmaxf(most, __shfl_xor(most, s));  // (a wave has keys or values)
  __syncthreads();
  // (a positive float's bits grow with it)
  if (lane_id() == 0) atomicMax(&amax[which], __builtin_bit_cast(uint32_t, most));
  __syncthreads();
  const int e_new = max(was, scale_byte(__builtin_bit_cast(float, amax[which])));
  const float inv = inverse(e_new);
  const bool grown = from > 0 && e_new > was;
  // 2^(was - e_new): zero where that is below the least normal number, as every code times it is
  const float shrink = grown && e_new - was < 127 ? __builtin_bit_cast(float, (uint32_t)(127 - (e_new - was)) << 23) : 0.f;
  if (!mine) return;
  if (t == 0) *scale = (uint8_t)e_new;

  uint32_t code[16][2];
#pragma unroll
  for (int e = 0; e < 16; e++)
#pragma unroll
    for (int h = 0; h < 2; h++)
      code[e][h] = codes4((float)v[e][4 * h] * inv, (float)v[e][4 * h + 1] * inv, (float)v[e][4 * h + 2] * inv,
                          (float)v[e][4 * h + 3] * inv);
  const int old = min(16, from - g * 16);  // places e < old hold tokens from before
  if (!which) {
    uint8_t* k = const_cast<uint8_t*>(c.k) + times(id, c.k_st[0]) + times(hk, c.k_st[1]) + g * 16 * D + d0;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      if (e >= lo && e < hi) {
        *(u32x2*)(k + e * D) = u32x2{code[e][0], code[e][1]};
      } else if (grown && e < old) {
        const u32x2 w = *(const u32x2*)(k + e * D);
        *(u32x2*)(k + e * D) = u32x2{rescale4(w[0], shrink), rescale4(w[1], shrink)};
      }
    }
  } else {
    uint8_t* vp = const_cast<uint8_t*>(c.v) + times(id, c.v_st[0]) + times(hk, c.v_st[1]) + (g * D + d0) * 16;
    const bool full = lo == 0 && hi == 16;
    if (full) {
      // 4 tokens x 4 dimensions are transposed by byte permutations
#pragma unroll
      for (int h = 0; h < 2; h++) {
        u32x4 w[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const uint32_t c0 = code[4 * q][h], c1 = code[4 * q + 1][h], c2 = code[4 * q + 2][h], c3 = code[4 * q + 3][h];
          const uint32_t lo01 = __builtin_amdgcn_perm(c1, c0, 0x05010400u), hi01 = __builtin_amdgcn_perm(c1, c0, 0x07030602u);
          const uint32_t lo23 = __builtin_amdgcn_perm(c3, c2, 0x05010400u), hi23 = __builtin_amdgcn_perm(c3, c2, 0x07030602u);
          w[0][q] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
          w[1][q] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
          w[2][q] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
          w[3][q] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) *(u32x4*)(vp + (4 * h + i) * 16) = w[i];
      }
    } else if (grown && old > 0) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        u32x4 w = *(const u32x4*)(vp + i * 16);
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const uint32_t again = rescale4(w[q], shrink);
          uint32_t r = 0;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int at = 4 * q + e;
            const uint32_t fresh = code[at][i / 4] >> (8 * (i % 4));
            const uint32_t byte = at >= lo && at < hi ? fresh : at < old ? again >> (8 * e) : w[q] >> (8 * e);
            r |= (byte & 0xffu) << (8 * e);
          }
          w[q] = r;
        }
        *(u32x4*)(vp + i * 16) = w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (e >= lo && e < hi)
#pragma unroll
          for (int i = 0; i < 8; i++) vp[i * 16 + e] = (uint8_t)(code[e][i / 4] >> (8 * (i % 4)));
    }
  }
}

// One token per sequence (dense): a wave has the key or the value of one head.  The same as above in a tenth of the
// code: such a launch waits for little but memory, and that includes its instructions (one sequence or 128 of 8 heads:
// 3.5 us, the kernel above 7.5).
template <typename T, int D>
__global__ __launch_bounds__(64) void cache_append_token_kernel(const AppendArgs a) {
  constexpr int E = D / 64;  // elements of a lane
  typedef __attribute__((__vector_size__(E * sizeof(T)))) T VE;
  const CacheArgs& c = a.c;
  const int which = blockIdx.x & 1, u = blockIdx.x >> 1, lane = threadIdx.x;
  const int b = quotient(u, a.by_heads), hk = u - b * c.heads_kv;
  const int start = max(0, c.lens[b]);
  const VE x = *(const VE*)((const T*)a.x[which] + (int64_t)b * a.x_st[which][0] + (int64_t)hk * a.x_st[which][2] +
                            lane * E);
  const int page_size = 1 << c.page_log2, in_seq = start >> c.page_log2, from = start & (page_size - 1);
  if (in_seq >= c.max_pages) return;
  const int id = c.table[(int64_t)b * c.table_st + in_seq];
  if ((uint32_t)id >= (uint32_t)c.num_pages) return;
  uint8_t* const scale = which ? const_cast<uint8_t*>(c.v_scale) + times(id, c.vs_st[0]) + times(hk, c.vs_st[1])
                               : const_cast<uint8_t*>(c.k_scale) + times(id, c.ks_st[0]) + times(hk, c.ks_st[1]);
  uint8_t* const page = which ? const_cast<uint8_t*>(c.v) + times(id, c.v_st[0]) + times(hk, c.v_st[1])
                              : const_cast<uint8_t*>(c.k) + times(id, c.k_st[0]) + times(hk, c.k_st[1]);
  const int was = from > 0 ? *scale : 0;
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const float y = __builtin_fabsf((float)x[i]);
    most = y < __builtin_inff() ? fmaxf(most, y) : most;
  }
  const int e_new = max(was, scale_byte(wave_max(most)));
  const float inv = inverse(e_new);
  const uint32_t code = codes4((float)x[0] * inv, (float)x[E - 1] * inv, 0.f, 0.f);
  if (from > 0 && e_new > was) {  // the tokens from before at the new scale
    const float f = e_new - was < 127 ? __builtin_bit_cast(float, (uint32_t)(127 - (e_new - was)) << 23) : 0.f;
    const int words = which ? (from + 15) / 16 * 4 * D : from * D / 4;
#pragma unroll 1
    for (int i = lane; i < words; i += 64) {
      const int left = which ? from - (i / (4 * D) * 16 + (i & 3) * 4) : 4;  // tokens from before in this word
      uint32_t* const w = (uint32_t*)page + i;
      const uint32_t again = left > 0 ? rescale4(*w, f) : 0u;
      if (left >= 4) *w = again;
#pragma unroll
      for (int k = 0; k < 3; k++)
        if (left < 4 && k < left) ((uint8_t*)w)[k] = (uint8_t)(again >> (8 * k));
    }
  }
  if (lane == 0) *scale = (uint8_t)e_new;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int d = lane * E + i;
    page[which ? from / 16 * (16 * D) + d * 16 + from % 16 : from * D + d] = (uint8_t)(code >> (8 * i));
  }
}

}  // namespace
}  // namespace rswa

extern "C" int rswa_cache_append(const rswa_cache_params* p, void* stream) {
  using namespace rswa;
  AppendArgs a;
  if (int rc = cache_args(p, "cache_append", a.c)) return rc;
  const int64_t rows = p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q;
  if (rows == 0 || p->batch == 0 || p->max_pages == 0) return RSWA_OK;
  RSWA_REQUIRE(p->new_k && p->new_v, RSWA_ERR_INVALID, "cache_append: null tensor");
  a.x[0] = p->new_k;
  a.x[1] = p->new_v;
  for (int i = 0; i < 3; i++) {
    a.x_st[0][i] = p->new_k_stride[i];
    a.x_st[1][i] = p->new_v_stride[i];
  }
  for (int w = 0; w < 2; w++) {
    RSWA_REQUIRE((uintptr_t)a.x[w] % 16 == 0 && a.x_st[w][0] % 8 == 0 && a.x_st[w][1] % 8 == 0 && a.x_st[w][2] % 8 == 0,
                 RSWA_ERR_UNSUPPORTED, "cache_append: rows of new_k and new_v must be 16-byte aligned");
    if (p->cu_seqlens_q) a.x_st[w][0] = 0;
  }
  a.pages = (int32_t)((p->seqlen_q + p->page_size - 2) / p->page_size + 1);
  const int64_t slots =
      p->cu_seqlens_q ? p->total_q / p->page_size + 2 * (int64_t)p->batch : (int64_t)p->batch * a.pages;
  const int64_t blocks = slots * p->heads_kv;
  RSWA_REQUIRE(blocks < (1ll << 30), RSWA_ERR_UNSUPPORTED, "cache_append: %lld blocks", (long long)blocks);
  a.work = (int32_t)blocks;
  a.by_pages = fast_div((uint32_t)a.pages);
  a.by_heads = fast_div((uint32_t)p->heads_kv);
  const int threads = 2 * std::max(64, p->page_size / 16 * (p->head_dim / 8));
  clear_launch_error();
  const bool tokens = !p->cu_seqlens_q && p->seqlen_q == 1;
  auto go = [&](auto t, auto d) {
    if (tokens) {
      hipLaunchKernelGGL((cache_append_token_kernel<decltype(t), decltype(d)::value>), dim3((unsigned)(2 * blocks)),
                         dim3(64), 0, (hipStream_t)stream, a);
      return;
    }
    hipLaunchKernelGGL((cache_append_kernel<decltype(t), decltype(d)::value>),
                       dim3((unsigned)(ceil_div(blocks, 8) * 8)), dim3(threads), 0, (hipStream_t)stream, a);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (p->dtype == RSWA_BF16)
    p->head_dim == 128 ? go(__bf16{}, D128{}) : go(__bf16{}, D64{});
  else
    p->head_dim == 128 ? go(_Float16{}, D128{}) : go(_Float16{}, D64{});
  return check_launch("cache_append");
}
