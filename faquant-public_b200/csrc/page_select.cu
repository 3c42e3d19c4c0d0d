// K12 -- which pages a query attends to: bounds of the pages' keys, and the pages of the
// greatest bounds of a score.
//
// Bounds. For a page and kv head, over the page's tokens (those below the sequence's length):
//   lo_d = min K_d, hi_d = max K_d,   stored as floor(lo_d / 2^e), ceil(hi_d / 2^e) in 8 bits,
// e the least exponent that holds them all in -127 .. 127. The values of the cache are exact in
// bf16, so minimum and maximum are exact and the bounds depend on the page's tokens alone, not on
// the steps in which they came: a page that a step wrote to is read anew as a whole (4.6 bits
// per value of K), which also forgets tokens that were taken back.
// Score. sum_d max(q_d lo_d, q_d hi_d) = sum_d (q_d >= 0 ? q_d hi_d : q_d lo_d) is at least
// q . K of every token of the page; the greatest over the query heads of the kv head counts. With
// q in 8 bits too (one exponent for the group, so that its heads can be compared) the sums are
// whole numbers below 2^21 times 2^e: exact in fp32 in any order, so that the same pages
// are taken by every kernel, batch and split.
// The products of 16 pages with 8 query heads are mma.sync m16n8k32 of 8-bit numbers, [lo | hi] times
// [negative | positive entries of q], whose lanes load 16 bytes of a page's row each.
// Selection. The first pages and the token's last ones, then the greatest scores, ties to the
// lowest column: a search for the count-th greatest key, then one pass in order.
//
// Measured (one B200): bounds of a step's pages 2.6 to 3.8 us. Selection for one token of 8 kv heads among 512 pages 7.6 us
// and for 32 sequences of 1 .. 1000 pages 13.7, both chains of loads that wait for one another (cu, lens, table,
// bounds), then the search; for 512 tokens of 64 query heads on 8 kv heads among 512 pages 62 us: some 7300
// instructions per token and kv head at 14 warps an SM (the scores take 37 us, the search 16). With dp4a in
// place of the 8-bit products they took 17.6, 32 and 227.
#include "kv_pages.cuh"

namespace faq {
namespace kvp {

__host__ __device__ constexpr int bounds_bytes(int d) { return 2 * d + 16; }  // lo, hi, exponent, 15 unused

// The least e with a <= 127 * 2^e (0 for a = 0), a >= 0 a finite fp32.
__device__ __forceinline__ int shared_exponent(float a) {
  if (a == 0.0f) return 0;
  int more = 0;
  if (a < 1e-30f) {  // towards the subnormals of bf16
    a *= 18446744073709551616.0f;  // 2^64
    more = 64;
  }
  return exponent_of(a) - 6 + ((__float_as_uint(a) & 0x7FFFFFu) > 0x7E0000u) - more;
}

__device__ __forceinline__ uint32_t min2_bf16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max2_bf16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

struct BoundsParams {
  Pages p;
  int64_t total;  // new tokens
  uint8_t* bounds;
};

// As the slots of blocks (kv_cache.cu): n new tokens touch at most n / page_size + 2 pages, so
// sequence b's pages get the slots from cu[b] / page_size + 2 b on.
__device__ __forceinline__ int64_t first_page_slot(const Pages& p, int b) {
  return (p.cu[b] >> p.page_shift) + 2 * static_cast<int64_t>(b);
}
__host__ __device__ inline int64_t page_slots_of(int64_t total, int64_t batch, int shift) { return (total >> shift) + 2 * batch; }

// A CTA takes a page of one kv head, its warps the page's blocks in turn.
constexpr int BOUNDS_WARPS = 4;
template <int NG>
__global__ void __launch_bounds__(32 * BOUNDS_WARPS) key_bounds_kernel(BoundsParams w) {
  constexpr int D = 64 * NG;
  __shared__ uint32_t s_lo[BOUNDS_WARPS][D / 2], s_hi[BOUNDS_WARPS][D / 2];
  __shared__ float s_top[BOUNDS_WARPS];
  grid_dependency_wait();
  allow_dependent_launch();
  const Pages& p = w.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t slot = blockIdx.x / p.kv_heads;
  const int head = static_cast<int>(blockIdx.x - slot * p.kv_heads);
  const int lo = last_of(p.batch, [&](int i) { return first_page_slot(p, i) <= slot; });
  const int c0 = p.cu[lo], c1 = p.cu[lo + 1];
  if (c0 < 0 || c1 <= c0 || c1 > w.total || slot < first_page_slot(p, lo)) {
    if (tid == 0) check_rows(p, lo, w.total);
    return;
  }
  const int64_t len = p.lens[lo], first = len - (c1 - c0);  // position of the first new token
  const int64_t col = (first > 0 ? first >> p.page_shift : 0) + (slot - first_page_slot(p, lo));
  const int64_t pos = col << p.page_shift;
  if (pos >= len) return;
  const int64_t page = page_of(p, lo, static_cast<int>(pos));
  if (page < 0) return;
  const int live = static_cast<int>(std::min<int64_t>(len - pos, int64_t(1) << p.page_shift));
  const uint8_t* src = p.base + page * p.page_stride + block_in_page<NG>(p, 0, head, static_cast<int>(pos));
  uint32_t mn[NG][2][4], mx[NG][2][4];  // [group][unit][pair]: channels 8 (2 t + unit) .. of the lane's t
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mn[g][i >> 2][i & 3] = 0x7F807F80u;  // infinity
      mx[g][i >> 2][i & 3] = 0xFF80FF80u;
    }
  const Expand expand;
  for (int blk = warp; blk * BLOCK < live; blk += BOUNDS_WARPS) {
    KBlock<NG> x;
    x.load(src + static_cast<int64_t>(blk) * block_bytes(NG), lane);
    x.each(expand, lane, [&](int token, int g, int unit, const uint32_t (&row)[4]) {
      if (blk * BLOCK + token < live) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          mn[g][unit & 1][i] = min2_bf16(mn[g][unit & 1][i], row[i]);
          mx[g][unit & 1][i] = max2_bf16(mx[g][unit & 1][i], row[i]);
        }
      }
    });
  }
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t a = mn[g][i >> 2][i & 3], b = mx[g][i >> 2][i & 3];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        a = min2_bf16(a, __shfl_xor_sync(0xffffffffu, a, o));
        b = max2_bf16(b, __shfl_xor_sync(0xffffffffu, b, o));
      }
      if (lane < 4) {
        s_lo[warp][32 * g + 8 * lane + i] = a;
        s_hi[warp][32 * g + 8 * lane + i] = b;
      }
    }
  __syncthreads();
  float low = 0.0f, high = 0.0f;
  if (tid < D) {
    uint32_t a = s_lo[0][tid >> 1], b = s_hi[0][tid >> 1];
#pragma unroll
    for (int k = 1; k < BOUNDS_WARPS; ++k) {
      a = min2_bf16(a, s_lo[k][tid >> 1]);
      b = max2_bf16(b, s_hi[k][tid >> 1]);
    }
    low = __uint_as_float(tid & 1 ? a & 0xFFFF0000u : a << 16);
    high = __uint_as_float(tid & 1 ? b & 0xFFFF0000u : b << 16);
  }
  float top = fmaxf(fabsf(low), fabsf(high));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < BOUNDS_WARPS; ++k) top = fmaxf(top, s_top[k]);
  const int e = shared_exponent(top);
  uint8_t* dst = w.bounds + (page * p.kv_heads + head) * bounds_bytes(D);
  if (tid < D) {
    const float unit = pow2f(-e);
    dst[tid] = static_cast<uint8_t>(static_cast<int8_t>(floorf(low * unit)));
    dst[D + tid] = static_cast<uint8_t>(static_cast<int8_t>(ceilf(high * unit)));
  }
  if (tid < 16) dst[2 * D + tid] = tid == 0 ? static_cast<uint8_t>(static_cast<int8_t>(e)) : 0;
}

struct SelectParams {
  Pages p;  // its base is not read
  const uint8_t* bounds;
  const __nv_bfloat16* q;
  int64_t qt, qh;
  int64_t total;
  int group;
  int count, first, last;
  int32_t* out;   // [total, kv_heads, count]
  float* scores;  // the same, or null
  int slots;      // log2 of the columns of a product that a token's heads take: 3 to 0
  int key_ld;     // keys of a token in shared memory
  bool vec;       // q can be read 16 bytes at a time
};

constexpr int SELECT_WARPS = 8, SELECT_THREADS = 32 * SELECT_WARPS;
constexpr int MAX_COLUMNS = 32768;  // pages of a sequence whose keys fit in shared memory
constexpr int MAX_GROUP = 128;
constexpr int WARP_COLUMNS = 256;   // keys that one warp searches
constexpr int SELECT_KEY_BYTES = 96 << 10;  // of a CTA whose warps have a token each: two to an SM
constexpr int HELD = 16;            // keys of a lane that it holds in registers while it searches

// The greatest-first order of fp32 as an order of whole numbers; 0 and 2^32 - 1 are no number's.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float number_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ void mma_s8_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight query heads in 8 bits, as the B operand of the products with the pages' bounds: column
// lane / 4, and per 64 bytes of the bounds [lo | hi] the lane's 16 from 16 (lane % 4) on; lo meets
// the negative entries, hi the others. (The order of the channels in a product is free.)
template <int NG>
struct Query {
  uint4 b[2 * NG];
  int e;  // the exponent of the lane's column
  // rows: the lane's column's query, heads stride `step` apart to further passes; `slots` as above
  __device__ __forceinline__ float top_of(const __nv_bfloat16* row, int lane, bool vec) const {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 2 * NG; ++j) {
      Raw<__nv_bfloat16> r;
      float v[8];
      r.load(row + 64 * (j >> 1) + 16 * (lane & 3) + 8 * (j & 1), vec);
      r.values(v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (fabsf(v[i]) < INFINITY) top = fmaxf(top, fabsf(v[i]));
    }
    return top;
  }
  __device__ __forceinline__ void round(const __nv_bfloat16* row, int lane, bool vec) {
    const float u0 = pow2f(-(e / 2)), u1 = pow2f(e / 2 - e);  // 2^-e passes fp32's range
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      uint32_t pos[4], neg[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        Raw<__nv_bfloat16> r;
        float v[8];
        r.load(row + 64 * j + 16 * (lane & 3) + 8 * h, vec);
        r.values(v);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t x = 0, y = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = v[4 * w + i];
            const int n = fabsf(a) < INFINITY ? __float2int_rn(a * u0 * u1) : 0;  // what is not finite does not count
            x |= static_cast<uint32_t>(max(n, 0) & 255) << (8 * i);
            y |= static_cast<uint32_t>(min(n, 0) & 255) << (8 * i);
          }
          pos[2 * h + w] = x;
          neg[2 * h + w] = y;
        }
      }
      b[j] = make_uint4(neg[0], neg[1], neg[2], neg[3]);
      b[NG + j] = make_uint4(pos[0], pos[1], pos[2], pos[3]);
    }
  }
};

// The bounds of 16 pages from column c0 on as the A operand: rows lane / 4 and 8 further.
template <int NG>
struct PageRows {
  uint4 a[2][2 * NG];
  int e[2];
  bool ok[2];
  // entry: the table's entry of column c0 + lane % 16 (-1 from `columns` on), loaded ahead
  static __device__ __forceinline__ int entry(const int32_t* row, int c0, int columns, int lane) {
    const int c = c0 + (lane & 15);
    return c < columns ? row[c] : -1;
  }
  __device__ __forceinline__ void load(const SelectParams& w, int head, int entry, int lane) {
    constexpr int D = 64 * NG;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int page = __shfl_sync(0xffffffffu, entry, (lane >> 2) + 8 * h);
      ok[h] = page >= 0 && page < w.p.num_pages;
      const uint8_t* src = w.bounds + (static_cast<int64_t>(ok[h] ? page : 0) * w.p.kv_heads + head) * bounds_bytes(D);
#pragma unroll
      for (int j = 0; j < 2 * NG; ++j) a[h][j] = *reinterpret_cast<const uint4*>(src + 64 * j + 16 * (lane & 3));
      e[h] = static_cast<int8_t>(src[2 * D]);
    }
  }
  // key(k, slot, c, value) is called, by one lane each, for the columns below `columns` and the tokens' slots
  // (0 .. 7 >> slots) of q[k] with the greatest score of the token's heads, 0 for a page that is not there.
  // Two sums per product, so that its steps do not all wait for one another; the lanes of a page that hold a
  // token's columns halve what they hold at each exchange of their maxima.
  template <int K, typename F>
  __device__ __forceinline__ void score(const SelectParams& w, const Query<NG> (&q)[K], int c0, int columns, int lane,
                                        F&& key) const {
    const int g = lane >> 2, t = lane & 3;
    int v[K][2][2];  // [product][row lane / 4 or 8 further][column 2 t or the next]
#pragma unroll
    for (int k = 0; k < K; ++k) {
      int acc[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int j = 0; j < 2 * NG; ++j) {
        mma_s8_16832(acc[0], a[0][j].x, a[1][j].x, a[0][j].y, a[1][j].y, q[k].b[j].x, q[k].b[j].y);
        mma_s8_16832(acc[1], a[0][j].z, a[1][j].z, a[0][j].w, a[1][j].w, q[k].b[j].z, q[k].b[j].w);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k][i >> 1][i & 1] = acc[0][i] + acc[1][i];
    }
    auto give = [&](int k, int slot, int h, int value) {
      const int c = c0 + g + 8 * h;
      const float unit = pow2f(min(max(h ? e[1] : e[0], -100), 100));
      if (c < columns) key(k, slot, c, (h ? ok[1] : ok[0]) ? order_key(static_cast<float>(value) * unit) : 0u);
    };
    if (w.slots == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) give(k, 2 * t + (i & 1), i >> 1, v[k][i >> 1][i & 1]);
      return;
    }
    int x[K][2], y[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) x[k][h] = max(v[k][h][0], v[k][h][1]);
    if (w.slots == 1) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) give(k, t, h, x[k][h]);
      return;
    }
    const int h = t & 1;  // the lane keeps this row
#pragma unroll
    for (int k = 0; k < K; ++k) y[k] = max(h ? x[k][1] : x[k][0], __shfl_xor_sync(0xffffffffu, h ? x[k][0] : x[k][1], 1));
    if (w.slots == 2) {
#pragma unroll
      for (int k = 0; k < K; ++k) give(k, t >> 1, h, y[k]);
      return;
    }
    if constexpr (K == 2) {
      const int k = t >> 1;  // and this product
      give(k, 0, h, max(k ? y[1] : y[0], __shfl_xor_sync(0xffffffffu, k ? y[0] : y[1], 2)));
    } else {
      const int z = max(y[0], __shfl_xor_sync(0xffffffffu, y[0], 2));
      if (t < 2) give(0, 0, h, z);
    }
  }
  // A page that the table does not hold is reported, once per row of it.
  __device__ __forceinline__ void report(int c0, int columns, int lane) const {
    if ((!ok[0] && c0 + (lane >> 2) < columns) || (!ok[1] && c0 + (lane >> 2) + 8 < columns))
      atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
  }
};

// What a token's search knows.
struct Wanted {
  int columns;  // visible pages
  int count, first, last;
  __device__ __forceinline__ bool forced(int c) const { return c < first || c >= columns - last; }
};

// The `count` greatest keys, bit by bit, by one warp or by all of a CTA (WARPS): warp k has the k-th
// equal part of the columns, in rounds of 32. The pages that are always taken have no part in the search.
struct SearchScratch {
  int sum[2][SELECT_WARPS], part[2][SELECT_WARPS];
};
template <int WARPS>
__device__ __forceinline__ void take(const uint32_t* keys, const Wanted& w, int eq, int32_t* out, float* scores,
                                     SearchScratch* scratch) {
  const int lane = threadIdx.x & 31, warp = WARPS > 1 ? threadIdx.x >> 5 : 0;
  const int rounds = (w.columns + 32 * WARPS - 1) / (32 * WARPS), c0 = warp * rounds * 32 + lane;
  const bool few = rounds <= HELD;
  int turn = 0;
  auto all = [&](int n) {  // the sum over the lanes of all warps
    n = __reduce_add_sync(0xffffffffu, n);
    if constexpr (WARPS > 1) {
      turn ^= 1;
      if (lane == 0) scratch->sum[turn][warp] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) n += scratch->sum[turn][k];
    }
    return n;
  };
  uint32_t held[HELD], top = 0, low = 0xFFFFFFFFu;  // of the choices
  int always = 0, others = 0;
  auto key_at = [&](int c) -> uint32_t { return c < w.columns ? keys[c] : 0; };
  auto count_in = [&](uint32_t key, bool forced) -> uint32_t {  // the key as a choice, 0: it is none
    always += key != 0 && forced;
    if (key == 0 || forced) return 0;
    ++others;
    top = max(top, key);
    low = min(low, key);
    return key;
  };
  if (few) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = i < rounds ? count_in(key_at(c0 + 32 * i), w.forced(c0 + 32 * i)) : 0;
  } else {
    for (int i = 0; i < rounds; ++i) count_in(key_at(c0 + 32 * i), w.forced(c0 + 32 * i));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  if constexpr (WARPS > 1) {
    if (lane == 0) {
      scratch->part[0][warp] = static_cast<int>(top);
      scratch->part[1][warp] = static_cast<int>(low);
    }
  }
  const int found_both = all(always | others << 16);  // at most 32768 of the others: their sum passes no bit of 32
  always = found_both & 0xFFFF;
  others = static_cast<int>(static_cast<uint32_t>(found_both) >> 16);
  if constexpr (WARPS > 1) {
    for (int k = 0; k < WARPS; ++k) {
      top = max(top, static_cast<uint32_t>(scratch->part[0][k]));
      low = min(low, static_cast<uint32_t>(scratch->part[1][k]));
    }
    __syncthreads();  // the parts are written again
  }
  const int need = max(w.count - always, 0);
  // taken are the keys above the limit and the first `ties` of those equal to it
  uint32_t limit = 0;
  int ties = 0;
  if (need == 0) {
    limit = 0xFFFFFFFFu;
  } else if (others > need) {
    const int first_bit = 31 - __clz(top ^ low);  // the keys agree above it; -1: they are one
    uint32_t found = first_bit < 0 ? top : top & ~((2u << first_bit) - 1);
    int above = 0;
    bool exact = false;
    for (int bit = first_bit; bit >= 0 && !exact; --bit) {
      const uint32_t at = found | (1u << bit);
      int n = 0;
      if (few) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) n += held[i] >= at;
      } else {
        for (int i = 0; i < rounds; ++i) n += !w.forced(c0 + 32 * i) && key_at(c0 + 32 * i) >= at;
      }
      n = all(n);
      if (n >= need) found = at; else above = n;
      exact = n == need;
    }
    limit = exact ? found - 1 : found;
    ties = exact ? 0 : need - above;
  }
  // where this warp's part of the list begins
  int at = 0, equal = 0;
  if constexpr (WARPS > 1) {
    int sure = 0, same = 0;
    for (int i = 0; i < rounds; ++i) {
      const int c = c0 + 32 * i;
      const uint32_t key = key_at(c);
      const bool f = w.forced(c);
      sure += key != 0 && (f || key > limit);
      same += key != 0 && !f && key == limit;
    }
    sure = __reduce_add_sync(0xffffffffu, sure);
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0) {
      scratch->part[0][warp] = sure;
      scratch->part[1][warp] = same;
    }
    __syncthreads();
    for (int k = 0; k < warp; ++k) {
      at += scratch->part[0][k];
      equal += scratch->part[1][k];
    }
    at += min(equal, ties);
  }
  const uint32_t below = (1u << lane) - 1;
  for (int i = 0; i < rounds; ++i) {
    const int c = c0 + 32 * i;
    const uint32_t key = key_at(c);
    const bool f = w.forced(c), same = ties > 0 && !f && key == limit;
    bool taken = key != 0 && (f || key > limit);
    if (ties > 0) {
      const uint32_t vs = __ballot_sync(0xffffffffu, same);
      taken = taken || (same && equal + __popc(vs & below) < ties);
      equal += __popc(vs);
    }
    const uint32_t vt = __ballot_sync(0xffffffffu, taken);
    if (vt == 0) continue;
    const int mine = at + __popc(vt & below);
    if (taken && mine < w.count) {
      out[mine] = c;
      if (scores != nullptr) scores[mine] = ldexpf(number_of(key), eq);
    }
    at += __popc(vt);
  }
  const int listed = min(always + min(others, need), w.count);
  for (int i = listed + (WARPS > 1 ? static_cast<int>(threadIdx.x) : lane); i < w.count; i += 32 * WARPS) {
    out[i] = -1;
    if (scores != nullptr) scores[i] = -INFINITY;
  }
}

// The exponent of column lane / 4's token, from its heads' greatest magnitudes: `passes` times 8 of them.
template <int NG>
__device__ __forceinline__ int query_exponent(const Query<NG>& q, const SelectParams& w, const __nv_bfloat16* heads, int first,
                                              int lane) {
  float top = 0.0f;
  for (int h = first; h < w.group; h += 8) top = fmaxf(top, q.top_of(heads + h * w.qh, lane, w.vec));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  for (int o = 0; o < w.slots; ++o) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4 << o));
  return shared_exponent(top);
}

// Few rows: a cluster of `split` CTAs per token and kv head. Their warps score the pages in turn; the keys
// meet in the first CTA, which searches them.
template <int NG>
__global__ void __launch_bounds__(SELECT_THREADS, 2) select_pages_cta_kernel(SelectParams w, int split) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ SearchScratch s_search;
  const Pages& p = w.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (split > 1) cluster_sync();  // the first CTA is there to be written to
  grid_dependency_wait();
  allow_dependent_launch();
  const int rank = static_cast<int>(blockIdx.x % split);
  const int64_t unit = blockIdx.x / split, token = unit / p.kv_heads;
  const int head = static_cast<int>(unit - token * p.kv_heads);
  if (blockIdx.x == 0) check_batch(p, w.total, tid, SELECT_THREADS);
  int b;
  int64_t pos;
  if (!find_token(p, token, w.total, b, pos)) return;  // the whole cluster
  Wanted want = {0, w.count, w.first, w.last};
  if (pos >= 0) {
    want.columns = static_cast<int>(std::min<int64_t>((pos >> p.page_shift) + 1, p.table_cols));
    if (tid == 0 && (pos >> p.page_shift) >= p.table_cols) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
  }
  const __nv_bfloat16* heads = w.q + token * w.qt + static_cast<int64_t>(head) * w.group * w.qh;
  const int32_t* row = p.table + b * p.table_ld;
  const uint32_t dst = split > 1 ? mapa_shared(smem_addr(s_keys), 0) : smem_addr(s_keys);
  const int begin = 16 * (warp + SELECT_WARPS * rank), step = 16 * SELECT_WARPS * split;
  PageRows<NG> rows;  // the first pages' loads fly while q is rounded
  rows.load(w, head, PageRows<NG>::entry(row, begin, want.columns, lane), lane);
  int entry = PageRows<NG>::entry(row, begin + step, want.columns, lane);
  Query<NG> q[1];
  q[0].e = query_exponent(q[0], w, heads, min(lane >> 2, w.group - 1), lane);
  for (int h = 0; h < w.group; h += 8) {
    q[0].round(heads + min(h + (lane >> 2), w.group - 1) * w.qh, lane, w.vec);
    if (h > 0) {
      rows.load(w, head, PageRows<NG>::entry(row, begin, want.columns, lane), lane);
      entry = PageRows<NG>::entry(row, begin + step, want.columns, lane);
    }
    for (int c0 = begin; c0 < want.columns; c0 += step) {
      const PageRows<NG> now = rows;
      if (c0 + step < want.columns) rows.load(w, head, entry, lane);
      entry = PageRows<NG>::entry(row, c0 + 2 * step, want.columns, lane);
      now.report(c0, want.columns, lane);
      now.score(w, q, c0, want.columns, lane, [&](int, int, int c, uint32_t key) {
        const uint32_t at = dst + 4 * c;  // a column's passes are one lane's
        if (h > 0) {
          uint32_t old;
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(old) : "r"(at) : "memory");
          key = max(key, old);
        }
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(key) : "memory");
      });
    }
  }
  if (split > 1) cluster_sync(); else __syncthreads();
  if (rank > 0) return;
  const int64_t list = unit * w.count;
  int32_t* out = w.out + list;
  float* scores = w.scores == nullptr ? nullptr : w.scores + list;
  if (want.columns > WARP_COLUMNS)
    take<SELECT_WARPS>(s_keys, want, q[0].e, out, scores, &s_search);
  else if (warp == 0)
    take<1>(s_keys, want, q[0].e, out, scores, nullptr);
}

// Many rows: a warp per kv head and two products' columns, 16 >> slots tokens: the heads of several tokens
// share a product, and two products a page's bounds.
constexpr int PRODUCTS = 2;
template <int NG>
__global__ void __launch_bounds__(SELECT_THREADS, 2) select_pages_warp_kernel(SelectParams w) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  const Pages& p = w.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_wait();
  allow_dependent_launch();
  if (blockIdx.x == 0) check_batch(p, w.total, tid, SELECT_THREADS);
  const int each = 8 >> w.slots, tokens = PRODUCTS * each;
  const int64_t block = blockIdx.x / p.kv_heads, token0 = (block * SELECT_WARPS + warp) * tokens;
  const int head = static_cast<int>(blockIdx.x - block * p.kv_heads);
  uint32_t* keys = s_keys + static_cast<int64_t>(warp) * tokens * w.key_ld;
  const int column = (lane >> 2) & ((1 << w.slots) - 1);  // the lane's head of a pass
  int done = 0;  // tokens of the group that have been looked at
  while (done < tokens && token0 + done < w.total) {
    // a run of tokens of one sequence
    int b;
    int64_t pos;
    if (!find_token(p, token0 + done, w.total, b, pos)) {
      ++done;
      continue;
    }
    const int run = static_cast<int>(std::min<int64_t>(p.cu[b + 1] - (token0 + done), tokens - done));
    const int64_t last = pos + run - 1;
    const int columns = last < 0 ? 0 : static_cast<int>(std::min<int64_t>((last >> p.page_shift) + 1, p.table_cols));
    if (lane == 0 && last >= 0 && (last >> p.page_shift) >= p.table_cols) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
    const int32_t* row = p.table + b * p.table_ld;
    const __nv_bfloat16* heads[PRODUCTS];
    Query<NG> q[PRODUCTS];
#pragma unroll
    for (int k = 0; k < PRODUCTS; ++k) {  // columns of other tokens repeat one of the run
      const int64_t token = token0 + min(max(k * each + (lane >> 2 >> w.slots), done), done + run - 1);
      heads[k] = w.q + token * w.qt + static_cast<int64_t>(head) * w.group * w.qh;
      q[k].e = query_exponent(q[k], w, heads[k], min(column, w.group - 1), lane);
    }
    for (int h = 0; h < w.group; h += 8) {
#pragma unroll
      for (int k = 0; k < PRODUCTS; ++k) q[k].round(heads[k] + min(h + column, w.group - 1) * w.qh, lane, w.vec);
      auto step = [&](const PageRows<NG>& rows, int c0) {
        rows.report(c0, columns, lane);
        rows.score(w, q, c0, columns, lane, [&](int k, int slot, int c, uint32_t key) {
          uint32_t* at = keys + static_cast<int64_t>(k * each + slot) * w.key_ld + c;
          *at = h > 0 ? max(key, *at) : key;
        });
      };
      PageRows<NG> rows[2];  // the next 16 pages' are loaded while these are multiplied
      int entry = PageRows<NG>::entry(row, 16, columns, lane);
      rows[0].load(w, head, PageRows<NG>::entry(row, 0, columns, lane), lane);
      for (int c0 = 0; c0 < columns; c0 += 32) {
        if (c0 + 16 < columns) rows[1].load(w, head, entry, lane);
        entry = PageRows<NG>::entry(row, c0 + 32, columns, lane);
        step(rows[0], c0);
        if (c0 + 16 >= columns) break;
        if (c0 + 32 < columns) rows[0].load(w, head, entry, lane);
        entry = PageRows<NG>::entry(row, c0 + 48, columns, lane);
        step(rows[1], c0 + 16);
      }
    }
    __syncwarp();
    for (int i = done; i < done + run; ++i) {
      const int64_t at = pos + i - done, list = ((token0 + i) * p.kv_heads + head) * w.count;
      const Wanted want = {at < 0 ? 0 : static_cast<int>(std::min<int64_t>((at >> p.page_shift) + 1, p.table_cols)), w.count,
                           w.first, w.last};
      const int k = i / each, e = __shfl_sync(0xffffffffu, k == 0 ? q[0].e : q[1].e, (i - k * each) << w.slots << 2);
      take<1>(keys + static_cast<int64_t>(i) * w.key_ld, want, e, w.out + list, w.scores == nullptr ? nullptr : w.scores + list,
              nullptr);
    }
    __syncwarp();
    done += run;
  }
}

}  // namespace kvp
}  // namespace faq

extern "C" int faq_hif4_key_bounds(const void* pages, int64_t num_pages, int64_t page_stride, int page_size,
                                   int64_t kv_heads, int d, const int32_t* table, int64_t table_ld, int64_t table_cols,
                                   const int32_t* cu, const int32_t* lens, int64_t batch, int64_t total, void* bounds,
                                   void* stream) {
  using namespace faq;
  using namespace faq::kvp;
  BoundsParams w;
  const int rc = make_pages(w.p, pages, num_pages, page_stride, page_size, kv_heads, d, table, table_ld, table_cols, cu,
                            lens, batch);
  if (rc) return rc;
  FAQ_CHECK_ARG(total >= 0 && total < (int64_t(1) << 31), "bad token count");
  if (total == 0) return FAQ_OK;
  FAQ_CHECK_ARG(bounds && aligned16(bounds), "bounds must be 16-byte aligned");
  w.total = total;
  w.bounds = static_cast<uint8_t*>(bounds);
  const int64_t blocks = page_slots_of(total, batch, w.p.page_shift) * kv_heads;
  FAQ_CHECK_ARG(blocks < (int64_t(1) << 31), "too many tokens for one call");
  auto kern = d == 64 ? key_bounds_kernel<1> : key_bounds_kernel<2>;
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(blocks)), 32 * BOUNDS_WARPS, 0, stream, w));
  return launch_status("key_bounds_kernel");
}

extern "C" int faq_hif4_select_pages(const void* q, int64_t total, int64_t heads, int64_t q_token_stride,
                                     int64_t q_head_stride, const void* bounds, int64_t num_pages, int page_size,
                                     int64_t kv_heads, int d, const int32_t* table, int64_t table_ld,
                                     int64_t table_cols, const int32_t* cu, const int32_t* lens, int64_t batch,
                                     int64_t count, int64_t first, int64_t last, int32_t* selected, float* scores,
                                     void* stream) {
  using namespace faq;
  using namespace faq::kvp;
  SelectParams w;
  // the pages themselves are not read: the bounds stand in for them in the checks
  const int rc = make_pages(w.p, bounds, num_pages, int64_t(1) << 40, page_size, kv_heads, d, table, table_ld, table_cols, cu,
                            lens, batch);
  if (rc) return rc;
  FAQ_CHECK_ARG(total >= 0 && total < (int64_t(1) << 31), "bad token count");
  FAQ_CHECK_ARG(heads > 0 && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  if (heads / kv_heads > MAX_GROUP) return fail(FAQ_ERR_UNSUPPORTED, "more than 128 query heads of a kv head");
  if (table_cols > MAX_COLUMNS) return fail(FAQ_ERR_UNSUPPORTED, "more than 32768 columns of the table");
  FAQ_CHECK_ARG(count > 0 && count < (int64_t(1) << 24) && first >= 0 && last >= 1 && first + last <= count,
                "count must hold the first pages and the last ones, of which there is at least one");
  if (total == 0) return FAQ_OK;
  FAQ_CHECK_ARG(q && selected, "null pointer");
  FAQ_CHECK_ARG(total * kv_heads < (int64_t(1) << 28), "too many tokens for one call");
  w.bounds = static_cast<const uint8_t*>(bounds);
  w.q = static_cast<const __nv_bfloat16*>(q);
  w.qt = q_token_stride;
  w.qh = q_head_stride;
  w.total = total;
  w.group = static_cast<int>(heads / kv_heads);
  w.count = static_cast<int>(count);
  w.first = static_cast<int>(first);
  w.last = static_cast<int>(last);
  w.out = selected;
  w.scores = scores;
  w.vec = aligned16(q) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
  const int64_t units = total * kv_heads;
  static std::atomic<uint64_t> set[4];  // devices on which the kernels' shared memory is set
  // Many rows, and room for the keys of a CTA's warps: a warp for the heads of 16 >> slots tokens, the more of them the later
  // (they are searched one after the other). A CTA each and a warp each, us, 32 of 512 pages where not said otherwise:
  //   512 tokens, 64 / 8 heads (4096 rows)  141   62;   128 tokens (1024)    41   47
  //   256 tokens, 32 / 8 heads (2048)        42   31;   128 tokens (1024)    23   29  (of 128 pages)
  //   800 tokens, 8 / 8 heads (6400)        100   62;   256 tokens (2048)    41   74  (of 125, 128)
  int slots = 0;
  while (slots < 3 && (1 << slots) < w.group) ++slots;
  const int64_t tokens = SELECT_WARPS * PRODUCTS * 8 >> slots, keys = tokens * table_cols;  // of a CTA
  if (units >= (8 + (16 >> slots)) * static_cast<int64_t>(num_sms()) && 4 * keys <= SELECT_KEY_BYTES) {
    w.slots = slots;
    w.key_ld = static_cast<int>(table_cols);
    auto kern = d == 64 ? select_pages_warp_kernel<1> : select_pages_warp_kernel<2>;
    const int rs = allow_smem(reinterpret_cast<const void*>(kern), SELECT_KEY_BYTES, set[d == 64 ? 0 : 1]);
    if (rs) return rs;
    FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>((total + tokens - 1) / tokens * kv_heads)), SELECT_THREADS,
                          4 * static_cast<size_t>(keys), stream, w));
    return launch_status("select_pages_warp_kernel");
  }
  // a CTA for every 128 columns (16 to a warp) as far as there are SMs
  int split = 1;
  while (split < 8 && 2 * split * units <= num_sms() && table_cols > 16 * SELECT_WARPS * split) split *= 2;
  w.slots = 3;
  w.key_ld = static_cast<int>(table_cols);
  auto kern = d == 64 ? select_pages_cta_kernel<1> : select_pages_cta_kernel<2>;
  const int rs = allow_smem(reinterpret_cast<const void*>(kern), 4 * MAX_COLUMNS, set[d == 64 ? 2 : 3]);
  if (rs) return rs;
  FAQ_CUDA(launch_clusters(kern, units * split, SELECT_THREADS, 4 * static_cast<size_t>(table_cols), split, stream, w, split));
  return launch_status("select_pages_cta_kernel");
}
