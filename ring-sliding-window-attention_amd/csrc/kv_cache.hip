// Checks that the calls over the 8-bit paged cache share.
#include "kv_cache.h"

namespace rswa {

int cache_args(const rswa_cache_params* p, const char* who, CacheArgs& a) {
  RSWA_REQUIRE(p, RSWA_ERR_INVALID, "%s: null parameters", who);
  RSWA_REQUIRE(p->dtype == RSWA_BF16 || p->dtype == RSWA_F16, RSWA_ERR_UNSUPPORTED, "%s: dtype %d", who, p->dtype);
  RSWA_REQUIRE(p->head_dim == 64 || p->head_dim == 128, RSWA_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", who,
               p->head_dim);
  RSWA_REQUIRE(p->batch >= 0 && p->heads_kv > 0 && p->heads_q > 0 && p->num_pages >= 0 && p->max_pages >= 0 &&
                   p->seqlen_q >= 0 && p->total_q >= 0,
               RSWA_ERR_INVALID, "%s: negative size", who);
  RSWA_REQUIRE(p->heads_q % p->heads_kv == 0, RSWA_ERR_INVALID, "%s: heads_q %d is no multiple of heads_kv %d", who,
               p->heads_q, p->heads_kv);
  RSWA_REQUIRE(p->heads_q <= (1 << 16) && p->batch <= (1 << 20), RSWA_ERR_UNSUPPORTED, "%s: heads or batch too large",
               who);
  RSWA_REQUIRE(p->page_size >= 16 && p->page_size <= 256 && (p->page_size & (p->page_size - 1)) == 0,
               RSWA_ERR_UNSUPPORTED, "%s: page_size %d (16, 32, 64, 128 or 256)", who, p->page_size);
  RSWA_REQUIRE((int64_t)p->max_pages * p->page_size < (1 << 28), RSWA_ERR_UNSUPPORTED,
               "%s: a row of the page table holds 2^28 tokens or more", who);
  const int64_t rows = p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q;
  RSWA_REQUIRE(rows * p->heads_q < (1ll << 30), RSWA_ERR_UNSUPPORTED, "%s: 2^30 (row, head) pairs or more", who);
  RSWA_REQUIRE(p->batch == 0 || p->seqlens, RSWA_ERR_INVALID, "%s: null seqlens", who);
  RSWA_REQUIRE(p->batch == 0 || p->max_pages == 0 || p->page_table, RSWA_ERR_INVALID, "%s: null page_table", who);
  RSWA_REQUIRE(p->num_pages > 0 || rows == 0, RSWA_ERR_INVALID, "%s: a cache without pages", who);
  RSWA_REQUIRE(p->num_pages == 0 || (p->k && p->v && p->k_scale && p->v_scale), RSWA_ERR_INVALID, "%s: null cache", who);
  RSWA_REQUIRE((uintptr_t)p->k % 16 == 0 && (uintptr_t)p->v % 16 == 0, RSWA_ERR_UNSUPPORTED,
               "%s: k and v must be 16-byte aligned", who);
  for (const int64_t* st : {p->k_stride, p->v_stride, p->k_scale_stride, p->v_scale_stride})
    RSWA_REQUIRE(st[0] >= 0 && st[0] < (1ll << 32) && st[1] >= 0 && st[1] < (1ll << 32), RSWA_ERR_UNSUPPORTED,
                 "%s: strides of the cache must be below 4 GiB", who);
  for (int i = 0; i < 2; i++)
    RSWA_REQUIRE(p->k_stride[i] % 16 == 0 && p->v_stride[i] % 16 == 0, RSWA_ERR_UNSUPPORTED,
                 "%s: strides of k and v must be multiples of 16 bytes", who);

  a = CacheArgs{};
  a.k = (const uint8_t*)p->k;
  a.v = (const uint8_t*)p->v;
  a.k_scale = (const uint8_t*)p->k_scale;
  a.v_scale = (const uint8_t*)p->v_scale;
  for (int i = 0; i < 2; i++) {
    a.k_st[i] = (uint32_t)p->k_stride[i];
    a.v_st[i] = (uint32_t)p->v_stride[i];
    a.ks_st[i] = (uint32_t)p->k_scale_stride[i];
    a.vs_st[i] = (uint32_t)p->v_scale_stride[i];
  }
  a.table = p->page_table;
  a.table_st = p->page_table_stride;
  a.lens = p->seqlens;
  a.cu = p->cu_seqlens_q;
  a.num_pages = p->num_pages;
  a.max_pages = p->max_pages;
  a.page_log2 = __builtin_ctz((unsigned)p->page_size);
  a.batch = p->batch;
  a.heads_q = p->heads_q;
  a.heads_kv = p->heads_kv;
  a.group = p->heads_q / p->heads_kv;
  a.seqlen_q = p->seqlen_q;
  a.total_q = (int32_t)p->total_q;
  a.by_group = fast_div((uint32_t)a.group);
  return RSWA_OK;
}

// What attention and weights read besides: queries, mask, scale.
int cache_query_args(const rswa_cache_params* p, const char* who, CacheArgs& a) {
  RSWA_REQUIRE(p->softmax_scale > 0.f && p->softmax_scale < __builtin_inff(), RSWA_ERR_INVALID,
               "%s: softmax_scale must be positive and finite", who);
  // Every block reads all lengths (find_unit), so that part of a call's time grows with the square of the batch: attention
  // of one token against 64 keys, 8 kv heads, 0.14 ms for 1024 sequences, 1.4 for 4096, 19 for 16384, 75 for 32768; weights
  // a tenth less.  The limit is eight times the last, 0.6 s.
  RSWA_REQUIRE((double)p->batch * p->batch * p->heads_kv <= 0x1p36, RSWA_ERR_UNSUPPORTED,
               "%s: %d sequences of %d kv heads (batch^2 * heads_kv must not exceed 2^36)", who, p->batch, p->heads_kv);
  RSWA_REQUIRE(p->num_sink >= 0, RSWA_ERR_INVALID, "%s: num_sink %d", who, p->num_sink);
  RSWA_REQUIRE(p->q, RSWA_ERR_INVALID, "%s: null tensor", who);
  RSWA_REQUIRE((uintptr_t)p->q % 16 == 0 && p->q_stride[0] % 8 == 0 && p->q_stride[1] % 8 == 0 &&
                   p->q_stride[2] % 8 == 0,
               RSWA_ERR_UNSUPPORTED, "%s: rows of q must be 16-byte aligned", who);
  a.q = p->q;
  for (int i = 0; i < 3; i++) a.q_st[i] = p->q_stride[i];
  if (a.cu) a.q_st[0] = 0;
  a.window = p->window_left < 0 || p->window_left >= (1 << 28) ? -1 : p->window_left;
  a.n_sink = p->num_sink;
  a.scale_log2 = p->softmax_scale * kLog2e;
  return RSWA_OK;
}

int cache_new_rows(const rswa_cache_params* p, const char* who, const void* (&x)[2], int64_t (&st)[2][3]) {
  RSWA_REQUIRE(p->new_k && p->new_v, RSWA_ERR_INVALID, "%s: null tensor", who);
  x[0] = p->new_k;
  x[1] = p->new_v;
  for (int i = 0; i < 3; i++) {
    st[0][i] = p->new_k_stride[i];
    st[1][i] = p->new_v_stride[i];
  }
  for (int w = 0; w < 2; w++) {
    RSWA_REQUIRE((uintptr_t)x[w] % 16 == 0 && st[w][0] % 8 == 0 && st[w][1] % 8 == 0 && st[w][2] % 8 == 0,
                 RSWA_ERR_UNSUPPORTED, "%s: rows of new_k and new_v must be 16-byte aligned", who);
    if (p->cu_seqlens_q) st[w][0] = 0;
  }
  return RSWA_OK;
}

}  // namespace rswa

extern "C" uint64_t rswa_sizeof_cache_params(void) { return sizeof(rswa_cache_params); }
