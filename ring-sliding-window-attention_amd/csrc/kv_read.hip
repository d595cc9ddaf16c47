// Cached keys and values back in 16 bits: the inverse of an append.
//
// A block takes one page of one kv head, the first half of its threads the keys, the second the values.  A thread has 16
// tokens (a group) of 8 dimensions: of the keys 8 bytes a token, of the values 16 bytes a dimension, which byte
// permutations put in rows.  A code times its page's power of two is exact in 32 bits and rounded once.
// Bound by memory, of which two thirds are written: prefixes of 31300 tokens together, 8 heads of 128, 193 MB in 33 us, 5.8
// TB/s with the codes partly in the last-level cache.  The values go past the caches (through them 47 us, and with
// codes that do not stay there 56).
#include <algorithm>

#include "kv_cache.h"

namespace rswa {
namespace {

struct ReadArgs {
  CacheArgs c;
  void* x[2];  // keys, values
  int64_t x_st[2][3];
  int32_t pages;  // dense: pages that a sequence's rows touch at most
  int32_t work;   // blocks with work
  FastDiv by_pages, by_heads;
};

// Eight values of codes in two words.
template <typename T>
__device__ __forceinline__ typename Mma<T>::V8 values8(uint32_t lo, uint32_t hi, int exponent) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo, true);
  const auto c = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, true);
  const float f[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  typename Mma<T>::V8 r;
#pragma unroll
  for (int i = 0; i < 8; i++) r[i] = (T)__builtin_ldexpf(f[i], exponent);
  return r;
}

template <typename T, int D>
__global__ void cache_read_kernel(const ReadArgs a) {
  using V8 = typename Mma<T>::V8;
  constexpr int LANES = D / 8;
  const CacheArgs& c = a.c;
  const int page_size = 1 << c.page_log2;
  // (an eighth of the work in a row for each XCD: the heads of a page, whose rows lie side by side, are written by one)
  const int id0 = (int)(blockIdx.x & 7) * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3);
  if (id0 >= a.work) return;
  int u = quotient(id0, a.by_heads), b, row0, n;
  const int hk = id0 - u * c.heads_kv;
  touched_page(c, a.pages, a.by_pages, u, b, row0, n);
  if (u < 0) return;
  const int start = max(0, c.lens[b]), in_page = start & (page_size - 1);
  const int64_t in_seq = (int64_t)(start >> c.page_log2) + u;  // page of the sequence
  const int from = u == 0 ? in_page : 0;                       // first place read
  const int64_t i0 = u == 0 ? 0 : ((int64_t)u << c.page_log2) - in_page;  // its row
  const int count = (int)min((int64_t)(page_size - from), n - i0);
  if (count <= 0) return;
  const int id = in_seq < c.max_pages ? c.table[(int64_t)b * c.table_st + in_seq] : -1;
  const bool there = (uint32_t)id < (uint32_t)c.num_pages;

  const int half = blockDim.x / 2;
  const int which = threadIdx.x >= half;
  const int t = threadIdx.x - which * half;
  const int d0 = t % LANES * 8, g = t / LANES;  // 8 dimensions, group of 16 places
  const int lo = max(0, from - g * 16), hi = min(16, from + count - g * 16);  // its places read: lo <= e < hi
  if (g >= (page_size >> 4) || lo >= hi) return;
  T* const x = (T*)a.x[which] + (int64_t)b * a.x_st[which][0] + (int64_t)hk * a.x_st[which][2] + d0 +
               (row0 + i0 + g * 16 - from) * a.x_st[which][1];  // (of place 0, which may be none of them)
  u32x2 codes[16];
  int exponent = 0;
  if (!there) {
#pragma unroll
    for (int e = 0; e < 16; e++) codes[e] = u32x2{0, 0};
  } else if (!which) {
    const uint8_t* const k = c.k + times(id, c.k_st[0]) + times(hk, c.k_st[1]) + g * 16 * D + d0;
#pragma unroll
    for (int e = 0; e < 16; e++) codes[e] = *(const u32x2*)(k + e * D);
    exponent = c.k_scale[times(id, c.ks_st[0]) + times(hk, c.ks_st[1])] - 127;
  } else {
    const uint8_t* const v = c.v + times(id, c.v_st[0]) + times(hk, c.v_st[1]) + (g * D + d0) * 16;
    u32x4 w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = *(const u32x4*)(v + i * 16);
    exponent = c.v_scale[times(id, c.vs_st[0]) + times(hk, c.vs_st[1])] - 127;
    // 4 dimensions x 4 tokens are transposed by byte permutations
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const uint32_t c0 = w[4 * h][q], c1 = w[4 * h + 1][q], c2 = w[4 * h + 2][q], c3 = w[4 * h + 3][q];
        const uint32_t lo01 = __builtin_amdgcn_perm(c1, c0, 0x05010400u), hi01 = __builtin_amdgcn_perm(c1, c0, 0x07030602u);
        const uint32_t lo23 = __builtin_amdgcn_perm(c3, c2, 0x05010400u), hi23 = __builtin_amdgcn_perm(c3, c2, 0x07030602u);
        codes[4 * q][h] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
        codes[4 * q + 1][h] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
        codes[4 * q + 2][h] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
        codes[4 * q + 3][h] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
      }
  }
#pragma unroll
  for (int e = 0; e < 16; e++)
    if (e >= lo && e < hi)
      __builtin_nontemporal_store(values8<T>(codes[e][0], codes[e][1], exponent), (V8*)(x + e * a.x_st[which][1]));
}

// ---- rows that share an element ----
// They are written by many blocks at once, so that none may.  A row's address is a sum of counts times strides: two rows meet
// where the difference of two such sums, with the counts' differences in their ranges, is below head_dim.  It is looked for from the
// largest stride down, as far as the smaller ones reach: of dimensions that lie inside one another a count or two at each.
struct Differences {
  typedef __int128 wide;  // (strides and counts are the caller's)
  struct Step {
    wide by, lo, hi;  // lo .. hi times `by`
  };
  Step of[6];
  wide lo_behind[7], hi_behind[7];  // what the steps from each on reach
  int n = 0, looked = 0, dim;
  explicit Differences(int dim_) : dim(dim_) {}

  void add(wide by, wide lo, wide hi, bool join) {
    if (by < 0) {
      by = -by;
      std::swap(lo, hi);
      lo = -lo;
      hi = -hi;
    }
    for (int i = 0; join && i < n; i++)
      if (of[i].by == by) {
        of[i].lo += lo;
        of[i].hi += hi;
        return;
      }
    of[n++] = {by, lo, hi};
  }
  // Is from + some sum below `dim`?  (`other`: of counts that are not all 0)
  bool found(wide from, bool other) {
    std::sort(of, of + n, [](const Step& a, const Step& b) { return a.by > b.by; });
    lo_behind[n] = hi_behind[n] = 0;
    for (int i = n - 1; i >= 0; i--) {
      lo_behind[i] = lo_behind[i + 1] + of[i].by * of[i].lo;
      hi_behind[i] = hi_behind[i + 1] + of[i].by * of[i].hi;
    }
    return look(0, from, other);
  }
  bool look(int i, wide from, bool other) {
    if (++looked > 4096) return true;  // (refused unproven: no layout of tensors in use comes near it)
    if (i == n) return !other && from < dim && -from < dim;
    const Step& s = of[i];
    wide lo = s.lo, hi = s.hi;
    if (s.by > 0) {
      const wide least = -dim + 1 - from - hi_behind[i + 1], most = dim - 1 - from - lo_behind[i + 1];
      const auto down = [&](wide v) { return v >= 0 ? v / s.by : -((-v + s.by - 1) / s.by); };
      lo = std::max(lo, -down(-least));
      hi = std::min(hi, down(most));
    }
    for (wide c = lo; c <= hi; c++)
      if (look(i + 1, from + c * s.by, other && c == 0)) return true;
    return false;
  }
};

bool rows_meet(const rswa_cache_params* p) {
  const bool packed = p->cu_seqlens_q != nullptr;
  const int64_t count[3] = {packed ? 1 : p->batch, packed ? p->total_q : p->seqlen_q, p->heads_kv};
  for (int64_t c : count)
    if (c <= 0) return false;
  Differences both(p->head_dim);
  for (const int64_t* st : {p->new_k_stride, p->new_v_stride}) {
    Differences own(p->head_dim);
    for (int d = 0; d < 3; d++)
      if (count[d] > 1) {
        own.add(st[d], 1 - count[d], count[d] - 1, false);
        st == p->new_k_stride ? both.add(st[d], 1 - count[d], 0, true) : both.add(st[d], 0, count[d] - 1, true);
      }
    if (own.found(0, true)) return true;
  }
  // (elements of two bytes, and of addresses that are 16-byte aligned, or refused before)
  const intptr_t apart = (intptr_t)p->new_v - (intptr_t)p->new_k;
  return both.found(apart / 2, false);
}

}  // namespace
}  // namespace rswa

extern "C" int rswa_cache_read_rows_meet(const rswa_cache_params* p) { return p && rswa::rows_meet(p); }

extern "C" int rswa_cache_read(const rswa_cache_params* p, void* stream) {
  using namespace rswa;
  constexpr const char* who = "cache_read";
  ReadArgs a;
  if (int rc = cache_args(p, who, a.c)) return rc;
  const int64_t rows = p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q;
  if (rows == 0 || p->batch == 0) return RSWA_OK;
  const void* x[2];
  if (int rc = cache_new_rows(p, who, x, a.x_st)) return rc;
  RSWA_REQUIRE(!rows_meet(p), RSWA_ERR_INVALID, "%s: rows of new_k and new_v, which are written, overlap", who);
  for (int w = 0; w < 2; w++) a.x[w] = const_cast<void*>(x[w]);
  a.pages = (int32_t)((p->seqlen_q + (int64_t)p->page_size - 2) / p->page_size + 1);
  const int64_t slots =
      p->cu_seqlens_q ? p->total_q / p->page_size + 2 * (int64_t)p->batch : (int64_t)p->batch * a.pages;
  const int64_t blocks = slots * p->heads_kv;
  RSWA_REQUIRE(blocks < (1ll << 30), RSWA_ERR_UNSUPPORTED, "%s: %lld blocks", who, (long long)blocks);
  a.work = (int32_t)blocks;
  a.by_pages = fast_div((uint32_t)a.pages);
  a.by_heads = fast_div((uint32_t)p->heads_kv);
  const int threads = 2 * std::max(64, p->page_size / 16 * (p->head_dim / 8));
  clear_launch_error();
  auto go = [&](auto t, auto d) {
    hipLaunchKernelGGL((cache_read_kernel<decltype(t), decltype(d)::value>),
                       dim3((unsigned)(ceil_div(blocks, 8) * 8)), dim3(threads), 0, (hipStream_t)stream, a);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (p->dtype == RSWA_BF16)
    p->head_dim == 128 ? go(__bf16{}, D128{}) : go(__bf16{}, D64{});
  else
    p->head_dim == 128 ? go(_Float16{}, D128{}) : go(_Float16{}, D64{});
  return check_launch(who);
}
