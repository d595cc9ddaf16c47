// Eviction from the 8-bit paged cache by running sums of softmax weights.
//
// Two launches: the first chooses, for each sequence and kv head, the second moves what stays into the new pages.
// 32 sequences of 2176 tokens cut to 2048, 8 heads of 128: 10 + 53 us (275 MB, 5 TB/s).  4 of 20000 to
// 32768 cut to 4096: 24 + 30 us; one in six tokens stays, so that nearly every group of 16 has one and all of V is read
// (the price of V in groups, which the attention reads as they are).
#include "kv_cache.h"

namespace rswa {
namespace {

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

// Weights as unsigned numbers that grow with them.  0: no token, 1: NaN, the largest: a token that stays whatever its
// weight (none is that of a weight).
constexpr uint32_t kStays = ~0u;
__device__ __forceinline__ uint32_t ordered(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);  // (-0 as 0)
  if ((u & 0x7fffffffu) > 0x7f800000u) return 1;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A block has one sequence's kv head, a wave of it a part of the tokens in a row, which it keeps in registers (those
// beyond 32 a lane are read again in each pass).  The bits of the least weight that stays are found from the highest
// down: a histogram of the first 11 (sign, exponent and two more: with eight, all weights meet in a few counters), a
// list of the weights that share the digit found, and two more digits from that list.  What bounds it is the one
// compute unit that a block runs on (32000 tokens, thousands of cycles: loads 12, histogram 11, list 7, two digits 7,
// writing 8, of 50); parts of one sequence on several would need a launch for each step, 3 to 4 us apiece.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void cache_select_kernel(const EvictArgs a) {
  constexpr int WAVES = THREADS / 64, N = 32, BINS = 2048, COPIES = THREADS / 256, LIST = THREADS * 8;
  constexpr int MINE = BINS / THREADS;  // bins of a thread
  __shared__ __attribute__((aligned(16))) uint32_t hist[COPIES][BINS];
  __shared__ uint32_t list[LIST];
  __shared__ uint32_t listed;
  __shared__ uint32_t chosen[2];  // digit, how many are still to be found among its weights
  __shared__ int count[WAVES][2], missing[WAVES][2];
  __shared__ uint32_t sums[WAVES];
  const CacheArgs& c = a.c;
  const int b = blockIdx.x / c.heads_kv, hk = blockIdx.x % c.heads_kv;
  const int len = held_tokens(c, c.lens[b]);
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int32_t* const table = c.table + (int64_t)b * c.table_st;
  const float* w = c.weights + (int64_t)b * c.w_st[0] + (int64_t)hk * c.w_st[1];
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  float* new_w = a.new_weights + (int64_t)blockIdx.x * c.w_len;

  int c0 = c.n_sink, c1 = len - a.n_recent;  // the others
  const int steps = (len + THREADS - 1) / THREADS;
  const int p0 = wave * steps * 64 + lane;  // a lane's first token
  // (loads first and without branches, so that they are all in flight; tokens without a weight of their own have 0)
  const int last = max(0, c.w_len - 1);
  if (c.w_len == 0) w = (const float*)c.lens;  // (any place that can be read)
  const int n_pages = (len + (1 << c.page_log2) - 1) >> c.page_log2;
  auto there = [&](int id) { return (uint32_t)id < (uint32_t)c.num_pages; };
  const int first_id = (int)threadIdx.x < n_pages ? table[threadIdx.x] : 0;
  auto load = [&](int i) { return w[min(p0 + i * 64, last)]; };
  auto number = [&](int i, float x) -> uint32_t {
    const int j = p0 + i * 64;
    uint32_t o = ordered(j < c.w_len ? x : 0.f);
    o = (uint32_t)(j - c0) < (uint32_t)(c1 - c0) ? o : kStays;
    return j < len ? o : 0;
  };
  uint32_t mine[N];
  float raw[N] = {};
  if (len > a.budget)
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += 8)
      if (i0 < steps)
#pragma unroll
        for (int i = i0; i < i0 + 8; i++) raw[i] = load(i);

  // Tokens whose page is not there are not kept: how many, and how many of them are sinks or recent ones.  (The table's
  // entries are on their way together with the weights.)
  int gone = 0, gone_stays = 0;
  auto look = [&](int p, int id) {
    if (there(id)) return;
    const int lo = p << c.page_log2, hi = min(lo + (1 << c.page_log2), len);
    gone += hi - lo;
    gone_stays += max(0, min(hi, c0) - lo) + max(0, hi - max(lo, c1));  // (of use only where c0 <= c1)
  };
  if ((int)threadIdx.x < n_pages) look(threadIdx.x, first_id);
  for (int p = threadIdx.x + THREADS; p < n_pages; p += THREADS) look(p, table[p]);
  gone = wave_scan(gone);
  gone_stays = wave_scan(gone_stays);
  if (lane == 63) {
    missing[wave][0] = gone;
    missing[wave][1] = gone_stays;
  }
  __syncthreads();
  gone = gone_stays = 0;
#pragma unroll
  for (int i = 0; i < WAVES; i++) {
    gone += missing[i][0];
    gone_stays += missing[i][1];
  }
  const int stay = min(len - gone, a.budget);
  if (hk == 0 && threadIdx.x == 0) a.new_lens[b] = stay;
  for (int r = stay + threadIdx.x; r < a.budget; r += THREADS) kept[r] = -1;
  for (int r = stay + threadIdx.x; r < c.w_len; r += THREADS) new_w[r] = 0.f;  // (the others: see the move)
  if (gone == 0 && len <= a.budget) {
    for (int j = threadIdx.x; j < len; j += THREADS) kept[j] = j;
    return;
  }
  const bool all = len - gone <= a.budget;  // all that are there
  if (all) c0 = c1 = 0;
  int find = all ? 0 : a.budget - (c.n_sink + a.n_recent - gone_stays);  // so many of the others stay

  for (int i = threadIdx.x; i < COPIES * BINS / 4; i += THREADS) ((u32x4*)hist)[i] = u32x4{0, 0, 0, 0};
  if (threadIdx.x == 0) listed = 0;
#pragma unroll
  for (int i0 = 0; i0 < N; i0 += 8)
    if (i0 < steps)
#pragma unroll
      for (int i = i0; i < i0 + 8; i++) mine[i] = i < steps ? number(i, raw[i]) : 0;
  auto has_page = [&](int i) { return there(table[min(p0 + i * 64, len - 1) >> c.page_log2]); };
  if (gone > 0)
#pragma unroll
    for (int i = 0; i < N; i++)
      if (i < steps && !has_page(i)) mine[i] = 0;
  // all of a wave's weights, eight steps without a branch at a time (those beyond its part are 0)
  auto each = [&](auto f) {
#pragma unroll
    for (int i0 = 0; i0 < N; i0 += 8)
      if (i0 < steps)
#pragma unroll
        for (int i = i0; i < i0 + 8; i++) f(i, mine[i]);
    for (int i = N; i < steps; i++) f(i, gone > 0 && !has_page(i) ? 0u : number(i, load(i)));
  };

  uint32_t least = all ? 0 : kStays - 1;  // below every token's number, or above every weight: none of the others stays
  if (find > 0) {
    // the digit of the find-th largest, from the counts in so many copies
    auto choose = [&](int copies) {
      uint32_t n[MINE], sum = 0;
      const int top = BINS - 1 - MINE * (int)threadIdx.x;  // thread t: MINE bins, from BINS - 1 - MINE t down
#pragma unroll
      for (int k = 0; k < MINE; k++) {
        n[k] = 0;
        for (int i = 0; i < copies; i++) n[k] += hist[i][top - k];
        sum += n[k];
      }
      uint32_t incl = (uint32_t)wave_scan((int)sum);
      if (lane == 63) sums[wave] = incl;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WAVES; i++) incl += i < wave ? sums[i] : 0;
      uint32_t above = incl - sum;
      if (above < (uint32_t)find && incl >= (uint32_t)find) {
#pragma unroll
        for (int k = 0; k < MINE; k++) {
          if (above < (uint32_t)find && above + n[k] >= (uint32_t)find) {
            chosen[0] = top - k;
            chosen[1] = find - above;
          }
          above += n[k];
        }
      }
      __syncthreads();
      find = chosen[1];
      return chosen[0];
    };
    auto weighs = [](uint32_t o) { return o - 1 < kStays - 1; };
    __syncthreads();
    each([&](int, uint32_t o) {
      if (weighs(o)) atomicAdd(&hist[wave % COPIES][o >> 21], 1u);
    });
    __syncthreads();
    const uint32_t digit = choose(COPIES);
    each([&](int, uint32_t o) {
      if (weighs(o) && o >> 21 == digit) {
        const uint32_t at = atomicAdd(&listed, 1u);  // (in any order: only counted)
        if (at < LIST) list[at] = o;
      }
    });
    least = digit << 21;
#pragma unroll 1
    for (int shift = 10; shift >= 0; shift -= 10) {
      const uint32_t mask = shift ? 2047 : 1023;
      for (int i = threadIdx.x; i < BINS / 4; i += THREADS) ((u32x4*)hist)[i] = u32x4{0, 0, 0, 0};
      __syncthreads();
      const uint32_t known = shift ? ~0u << 21 : ~0u << 10;
      auto tally = [&](uint32_t o) {
        if ((o & known) == least) atomicAdd(&hist[0][(o >> shift) & mask], 1u);
      };
      if (listed <= LIST)
        for (uint32_t i = threadIdx.x; i < listed; i += THREADS) tally(list[i]);
      else
        each([&](int, uint32_t o) {
          if (weighs(o)) tally(o);
        });
      __syncthreads();
      least |= choose(1) << shift;
    }
  }
  // stays: a larger weight; and `find` of the equal ones, the earliest
  int n_sure = 0, n_equal = 0;
  each([&](int, uint32_t o) {
    n_sure += __popcll(__builtin_amdgcn_ballot_w64(o > least));
    n_equal += __popcll(__builtin_amdgcn_ballot_w64(o == least));
  });
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
  auto below = [](uint64_t m, int n) {  // n and the lanes of m below this one
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, n));
  };
  each([&](int i, uint32_t o) {
    bool keep = o > least;
    const uint64_t eq = __builtin_amdgcn_ballot_w64(o == least);
    if (eq) {
      keep = keep || (o == least && below(eq, equals) < find);
      equals += __popcll(eq);
    }
    const uint64_t k = __builtin_amdgcn_ballot_w64(keep);
    const int r = below(k, at);
    if (keep && r < a.budget) kept[r] = p0 + i * 64;
    at += __popcll(k);
  });
}

// Largest finite magnitude among codes.  A magnitude's code grows with it; one more than the seven bits, modulo 128,
// is 0 for NaN and 1 .. 127 for the others, and two such bytes are compared at a time.
struct LargestCode {
  uint32_t even = 0, odd = 0;
  typedef __attribute__((__vector_size__(2 * sizeof(uint16_t)))) uint16_t u16x2;
  static __device__ __forceinline__ uint32_t max2(uint32_t x, uint32_t y) {
    const u16x2 p = __builtin_bit_cast(u16x2, x), q = __builtin_bit_cast(u16x2, y);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(p, q));
  }
  __device__ __forceinline__ void add(uint32_t codes) {
    even = max2(even, ((codes & 0x007f007fu) + 0x00010001u) & 0x007f007fu);
    odd = max2(odd, (((codes >> 8) & 0x007f007fu) + 0x00010001u) & 0x007f007fu);
  }
  // ... times the power of two of scale byte e
  __device__ __forceinline__ float value(int e) const {
    const uint32_t m = max2(even, odd), code = max(m & 0xffffu, m >> 16);
    return __builtin_ldexpf(__builtin_amdgcn_cvt_f32_fp8((int)(code == 0 ? 0 : code - 1), 0), e - 127);
  }
};

// Moves the kept tokens into new pages.  A block makes one new page of one kv head; a wave has 64 tokens of its keys or
// of its values.  Keys are rows to copy.  Of the values a lane has one or two dimensions, 16 tokens of which are 16
// bytes: it reads the old groups that hold kept tokens one after the other, and since which bytes of a word stay is
// the same for all lanes, one byte permutation with a scalar selector closes the gaps and one shift appends what is
// left.  The words wait in LDS until the page's largest value, and with it the new scale, is known.
// (Reading the values byte by byte, twice, and storing them so, took 195 us for 32 sequences cut from 2176 to 2048.)
template <int D>
__global__ __launch_bounds__(512, 4) void cache_move_kernel(const EvictArgs a) {
  constexpr int DL = D / 64;          // dimensions of a lane of a value wave
  constexpr int ROW = 16 + 1;         // words of 64 tokens, and one against bank conflicts
  constexpr int PIECES = D / 16, PER = 64 / PIECES, STEPS = 64 / PER;  // 16-byte pieces of a key row; rows of a load
  // of each wave, base: keys: of each row; values: of each old group; -1: its page is not there.  info: keys: scale byte;
  // values: which tokens of the group stay, scale byte << 16.  Behind them the words of the value waves.
  extern __shared__ int64_t shared[];
  const int waves = blockDim.x / 64;
  int64_t(*const base)[64] = (int64_t(*)[64])shared;
  uint32_t(*const info)[64] = (uint32_t(*)[64])(shared + waves * 64);
  uint32_t* const packed = (uint32_t*)(shared + waves * 96);
  __shared__ uint32_t amax[2];
  const CacheArgs& c = a.c;
  const int page_size = 1 << c.page_log2;
  const int hk = blockIdx.x % c.heads_kv;
  const int b = blockIdx.x / c.heads_kv / a.new_max_pages, np = blockIdx.x / c.heads_kv % a.new_max_pages;
  const int len = held_tokens(c, c.lens[b]), stay = a.new_lens[b];
  const int r0 = np << c.page_log2;
  const int n_page = min(page_size, stay - r0);  // tokens of the page
  if (n_page <= 0) return;
  const int id = a.new_table[(int64_t)b * a.new_table_st + np];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int half = waves / 2;
  const bool values = wave >= half;
  const int sub = (values ? wave - half : wave) * 64;  // first place of the wave's tokens
  const int n = max(0, min(64, n_page - sub));

  // lane l: the wave's token l
  int j = -1, sp = -1, e = 0;
  if (threadIdx.x < 2) amax[threadIdx.x] = 0;
  info[wave][lane] = 0;
  if (lane < n) {
    j = a.kept[((int64_t)b * c.heads_kv + hk) * a.budget + r0 + sub + lane];
    // (weights that another stream changes during the choice may leave numbers out: nothing is looked up by those)
    const bool one = (uint32_t)j < (uint32_t)len;
    if (one) sp = c.table[(int64_t)b * c.table_st + (j >> c.page_log2)];
    const int r = r0 + sub + lane;
    if (!values && r < c.w_len)
      a.new_weights[((int64_t)b * c.heads_kv + hk) * c.w_len + r] =
          one && j < c.w_len ? c.weights[(int64_t)b * c.w_st[0] + (int64_t)hk * c.w_st[1] + j] : 0.f;
    if ((uint32_t)sp >= (uint32_t)c.num_pages) sp = -1;
    if (sp >= 0)
      e = values ? c.v_scale[times(sp, c.vs_st[0]) + times(hk, c.vs_st[1])]
                 : c.k_scale[times(sp, c.ks_st[0]) + times(hk, c.ks_st[1])];
  }
  if ((uint32_t)id >= (uint32_t)c.num_pages) return;
  const int slot = j & (page_size - 1);
  uint64_t starts = 0;  // values: tokens that are the first of their old group
  if (!values) {
    if (lane < n) {
      base[wave][lane] = sp < 0 ? -1 : (int64_t)times(sp, c.k_st[0]) + slot * D;
      info[wave][lane] = (uint32_t)e;
    }
  } else {
    const int before = __shfl_up(j, 1);
    const bool start = lane < n && (lane == 0 || (j >> 4) != (before >> 4));
    starts = __builtin_amdgcn_ballot_w64(start);
    const int group = __popcll(starts & (~0ull >> (63 - lane))) - 1;
    if (start) base[wave][group] = sp < 0 ? -1 : (int64_t)times(sp, c.v_st[0]) + (slot >> 4) * (16 * D);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // (the zeros above)
    if (lane < n) atomicOr(&info[wave][group], (1u << (j & 15)) | ((uint32_t)e << 16));
  }
  __syncthreads();

  float most = 0.f;
  u32x4 rows[STEPS];
  uint32_t* const words = packed + (values ? wave - half : 0) * (D * ROW);
  const uint8_t* const head = values ? c.v + times(hk, c.v_st[1]) : c.k + times(hk, c.k_st[1]);
  if (!values) {
    const int piece = lane % PIECES * 16;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
      const int r = i * PER + lane / PIECES;
      rows[i] = u32x4{0, 0, 0, 0};
      if (r < n && base[wave][r] >= 0) rows[i] = *(const u32x4*)(head + base[wave][r] + piece);
    }
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
      const int r = i * PER + lane / PIECES;
      LargestCode top;
#pragma unroll
      for (int q = 0; q < 4; q++) top.add(rows[i][q]);
      if (r < n) most = fmaxf(most, top.value((int)info[wave][r]));
    }
  } else {
    // lane m: selector that closes the gaps of a word of which the tokens of the mask m stay
    uint32_t closes = 0;
    int taken = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (lane >> i & 1) closes |= (uint32_t)i << (8 * taken++);
    closes |= 0x0c0c0c0cu << (8 * (taken & 3)) & (taken == 4 ? 0u : ~0u);
    const int groups = __popcll(starts);
    const int64_t at = base[wave][lane];  // (lane g: old group g)
    const uint32_t inf = info[wave][lane];
    constexpr int AHEAD = 4;
    u32x4 x[AHEAD][DL];  // groups g .. g + 3, in turn
    auto load = [&](int g, u32x4(&y)[DL]) {
      const int64_t from = ((int64_t)__builtin_amdgcn_readlane((int)(at >> 32), g) << 32) |
                           (uint32_t)__builtin_amdgcn_readlane((int)at, g);
#pragma unroll
      for (int i = 0; i < DL; i++)
        y[i] = from < 0 ? u32x4{0, 0, 0, 0} : *(const u32x4*)(head + from + (lane + 64 * i) * 16);
    };
    uint32_t part[DL] = {};
    int fill = 0, word = 0;  // bytes in `part`, words written
#pragma unroll
    for (int k = 0; k < AHEAD; k++)
      if (k < groups) load(k, x[k]);
    auto group = [&](int g, u32x4(&x)[DL]) {
      const uint32_t which = (uint32_t)__builtin_amdgcn_readlane((int)inf, g);
      LargestCode top;
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const int m = which >> (4 * q) & 15;
        if (m == 0) continue;
        const uint32_t sel = (uint32_t)__builtin_amdgcn_readlane((int)closes, m);
        const int bytes = __builtin_popcount(m);
#pragma unroll
        for (int i = 0; i < DL; i++) {
          const uint32_t y = __builtin_amdgcn_perm(0u, x[i][q], sel);
          top.add(y);
          const uint64_t wide = ((uint64_t)y << (8 * fill)) | part[i];
          part[i] = (uint32_t)wide;
          if (fill + bytes >= 4) {
            words[(lane + 64 * i) * ROW + word] = part[i];
            part[i] = (uint32_t)(wide >> 32);
          }
        }
        fill += bytes;
        if (fill >= 4) {
          fill -= 4;
          word++;
        }
      }
      most = fmaxf(most, top.value((int)(which >> 16)));
      if (g + AHEAD < groups) load(g + AHEAD, x);
    };
    for (int g = 0; g < groups; g += AHEAD)
#pragma unroll
      for (int k = 0; k < AHEAD; k++)
        if (g + k < groups) group(g + k, x[k]);
    if (fill > 0)
#pragma unroll
      for (int i = 0; i < DL; i++) words[(lane + 64 * i) * ROW + word] = part[i];
  }
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) most = fmaxf(most, __shfl_xor(most, s));
  if (lane == 0) atomicMax(&amax[values], __float_as_uint(most));
  __syncthreads();
  const int e_new = scale_byte(__uint_as_float(amax[values]));
  if (!values) {
    if (threadIdx.x == 0)
      const_cast<uint8_t*>(c.k_scale)[times(id, c.ks_st[0]) + times(hk, c.ks_st[1])] = (uint8_t)e_new;
    uint8_t* const to = const_cast<uint8_t*>(head) + times(id, c.k_st[0]) + (int64_t)sub * D + lane % PIECES * 16;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
      const int r = i * PER + lane / PIECES;
      if (r >= n) continue;
      const int was = (int)info[wave][r];
      if (was != e_new) {
        const float f = __builtin_ldexpf(1.f, was - e_new);
#pragma unroll
        for (int q = 0; q < 4; q++) rows[i][q] = rescale4(rows[i][q], f);
      }
      *(u32x4*)(to + r * D) = rows[i];
    }
    return;
  }
  if (wave == half && lane == 0)
    const_cast<uint8_t*>(c.v_scale)[times(id, c.vs_st[0]) + times(hk, c.vs_st[1])] = (uint8_t)e_new;
  uint8_t* const to = const_cast<uint8_t*>(head) + times(id, c.v_st[0]) + (int64_t)(sub / 16) * (16 * D);
  const float f = __builtin_ldexpf(1.f, e - e_new);  // lane l: token l's
  const bool change = __builtin_amdgcn_ballot_w64(lane < n && e != e_new) != 0;
  for (int g = 0; g * 16 < n; g++) {
    u32x4 y[DL];
#pragma unroll
    for (int i = 0; i < DL; i++)
#pragma unroll
      for (int q = 0; q < 4; q++) y[i][q] = words[(lane + 64 * i) * ROW + g * 4 + q];
    if (change) {
#pragma unroll
      for (int q = 0; q < 4; q++) {
        float ft[4];
#pragma unroll
        for (int t = 0; t < 4; t++)
          ft[t] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), g * 16 + q * 4 + t));
#pragma unroll
        for (int i = 0; i < DL; i++) {
          const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)y[i][q], false);
          const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)y[i][q], true);
          y[i][q] = codes4(lo[0] * ft[0], lo[1] * ft[1], hi[0] * ft[2], hi[1] * ft[3]);
        }
      }
    }
    const int left = n - g * 16;
#pragma unroll
    for (int i = 0; i < DL; i++) {
      uint8_t* const p = to + g * (16 * D) + (lane + 64 * i) * 16;
      if (left >= 16) {
        *(u32x4*)p = y[i];
      } else {  // places behind the last token stay as they are
#pragma unroll
        for (int t = 0; t < 16; t++)
          if (t < left) p[t] = (uint8_t)(y[i][t / 4] >> (8 * (t % 4)));
      }
    }
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
  RSWA_REQUIRE((p->weights && p->new_weights || p->weights_len == 0) && (p->new_page_table || p->new_max_pages == 0) &&
                   p->new_seqlens && p->kept,
               RSWA_ERR_INVALID, "cache_evict: null tensor");
  RSWA_REQUIRE(p->new_page_table != p->page_table || p->new_max_pages == 0, RSWA_ERR_INVALID,
               "cache_evict: the new pages must be others than the old ones");
  // (blocks of other heads still read these while one writes its results)
  RSWA_REQUIRE(p->new_seqlens != p->seqlens && (p->new_weights != p->weights || p->weights_len == 0), RSWA_ERR_INVALID,
               "cache_evict: the new lengths and weights must be others than the old ones");
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
  // 32 weights a lane are in registers; the blocks of short sequences are smaller, so that a unit has eight of them
  // (64 sequences of 21 to 87 tokens, 32 heads: 48 us with 1024 threads, 14 with 256)
  if ((int64_t)p->max_pages * p->page_size <= 8192)
    hipLaunchKernelGGL(cache_select_kernel<256>, dim3((unsigned)heads), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(cache_select_kernel<1024>, dim3((unsigned)heads), dim3(1024), 0, st, a);
  if (int rc = check_launch("cache_evict select")) return rc;
  if (blocks == 0) return RSWA_OK;
  const int waves = std::max(1, p->page_size / 64);  // of keys, and as many of values
  const size_t lds = (size_t)waves * (2 * 64 * (8 + 4) + p->head_dim * 17 * 4);
  if (p->head_dim == 128)
    hipLaunchKernelGGL((cache_move_kernel<128>), dim3((unsigned)blocks), dim3(waves * 128), lds, st, a);
  else
    hipLaunchKernelGGL((cache_move_kernel<64>), dim3((unsigned)blocks), dim3(waves * 128), lds, st, a);
  return check_launch("cache_evict move");
}
