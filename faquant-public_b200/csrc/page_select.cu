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
// Measured (one B200): bounds of a step's pages 2.6 to 3.8 us. Selection for one token of 8 kv heads among 512 pages 7.1 us
// and for 32 sequences of 1 .. 1000 pages 13.0, both chains of loads that wait for one another (cu, lens, table,
// bounds), then the search; for 512 tokens of 64 query heads on 8 kv heads among 512 pages 41 us: rounding the queries 5, the
// scores 22 (about 160 instructions per 16 pages and two tokens, which wait for one another with 14 warps on an SM; the
// products and the loads of their operands take 9 each), the search 14. Dropped: bounds read by each warp (48 us, from
// L2), two sets of them in registers (61: they spill), one token's heads to a warp (76), two bits of the search at a time
// (43). With dp4a in place of the 8-bit products they took 17.6, 32 and 227.
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
  int key_ld;     // keys of a token in shared memory
  bool vec;       // q can be read 16 bytes at a time
};

constexpr int SELECT_WARPS = 8, SELECT_THREADS = 32 * SELECT_WARPS;
constexpr int MAX_COLUMNS = 32768;  // pages of a sequence whose keys fit in shared memory
constexpr int MAX_GROUP = 128;
constexpr int WARP_COLUMNS = 256;   // keys that one warp searches
constexpr int SELECT_KEY_BYTES = 90 << 10;  // of a CTA whose warps have tokens each: two to an SM
constexpr int HELD = 16;            // keys of a lane that it holds in registers while it searches

// The greatest-first order of fp32 as an order of whole numbers; 0 and 2^32 - 1 are no number's.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float number_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// c = a b, or c += a b where `add`.
__device__ __forceinline__ void mma_s8_16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1, bool add) {
  if (add)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}

// Four whole numbers of 8 bits in a word, the first in its lowest byte.
__device__ __forceinline__ uint32_t pack4_s8(const int (&n)[4]) {
  uint32_t high, word;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(high) : "r"(n[3]), "r"(n[2]), "r"(0));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(word) : "r"(n[1]), "r"(n[0]), "r"(high));
  return word;
}

// 255 in the bytes of x that hold negative numbers, 0 in the others.
__device__ __forceinline__ uint32_t signs4(uint32_t x) {
  uint32_t d;
  asm("prmt.b32 %0, %1, 0, 0xBA98;" : "=r"(d) : "r"(x));
  return d;
}

// Eight query heads in 8 bits, as the B operand of the products with the pages' bounds: column
// lane / 4, and per 64 bytes of the bounds [lo | hi] the lane's 16 from 16 (lane % 4) on; lo meets
// the negative entries, hi the others. (The order of the channels in a product is free.)
template <int NG>
struct Query {
  uint4 b[2 * NG];
  int e;  // the exponent of the lane's column
  // The greatest finite magnitude of the lane's part of `row`, its column's query.
  __device__ __forceinline__ float top_of(const __nv_bfloat16* row, int lane, bool vec) const {
    uint32_t top2 = 0;
#pragma unroll
    for (int j = 0; j < 2 * NG; ++j) {
      Raw<__nv_bfloat16> r;
      r.load(row + 64 * (j >> 1) + 16 * (lane & 3) + 8 * (j & 1), vec);
#pragma unroll
      for (int i = 0; i < 4; ++i) top2 = max2_bf16(top2, r.w[i] & 0x7FFF7FFFu);  // passes over what is not a number
    }
    float top = fmaxf(__uint_as_float(top2 << 16), __uint_as_float(top2 & 0xFFFF0000u));
    if (top == INFINITY) {
      top = 0.0f;
#pragma unroll 1
      for (int i = 0; i < 16 * NG; ++i) {
        const float v = fabsf(__bfloat162float(row[64 * (i >> 4) + 16 * (lane & 3) + (i & 15)]));
        if (v < INFINITY) top = fmaxf(top, v);
      }
    }
    return top;
  }
  __device__ __forceinline__ void round(const __nv_bfloat16* row, int lane, bool vec) {
    const float f0 = pow2f(-(e / 2)), f1 = pow2f(e / 2 - e);  // 2^-e passes fp32's range
    const float2 u0 = make_float2(f0, f0), u1 = make_float2(f1, f1), minus = make_float2(-1.0f, -1.0f);
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
          int n[4];
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float2 x = __fmul2_rn(__fmul2_rn(make_float2(v[4 * w + i], v[4 * w + i + 1]), u0), u1);
            const float2 y = __fadd2_rn(x, __ffma2_rn(x, minus, x));  // NaN, which becomes 0, for what is not finite
            n[i] = __float2int_rn(y.x);
            n[i + 1] = __float2int_rn(y.y);
          }
          const uint32_t x = pack4_s8(n), below = signs4(x);
          neg[2 * h + w] = x & below;
          pos[2 * h + w] = x & ~below;
        }
      }
      b[j] = make_uint4(neg[0], neg[1], neg[2], neg[3]);
      b[NG + j] = make_uint4(pos[0], pos[1], pos[2], pos[3]);
    }
  }
};

// Where a warp finds the bounds of its kv head.
struct BoundsOf {
  const uint8_t* base;   // of page 0, the lane's 16 bytes of every 64
  uint32_t stride, num;  // bytes to the next page's, pages
  int to_exponent;
  template <int NG>
  static __device__ __forceinline__ BoundsOf of(const SelectParams& w, int head, int lane) {
    constexpr int bytes = bounds_bytes(64 * NG);
    return {w.bounds + static_cast<int64_t>(head) * bytes + 16 * (lane & 3), static_cast<uint32_t>(w.p.kv_heads * bytes),
            static_cast<uint32_t>(w.p.num_pages), 128 * NG - 16 * (lane & 3)};
  }
};

// Bytes from a page's bounds in shared memory to the next page's: a row's 64 bytes and its neighbour's lie in different banks.
__host__ __device__ constexpr int staged_pitch(int d) { return 2 * d + 64; }
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The bounds of 16 pages from column c0 on as the A operand: rows lane / 4 and 8 further.
template <int NG>
struct PageRows {
  uint4 a[2][2 * NG];
  int e[2];
  bool ok[2];
  // entry: the table's entry of column c0 + lane % 16 (page 0 from `columns` on), loaded ahead
  static __device__ __forceinline__ int entry(const int32_t* row, int c0, int columns, int lane) {
    const int c = c0 + (lane & 15);
    return c < columns ? row[c] : 0;
  }
  // missing: whether the lane has seen an entry that is no page
  __device__ __forceinline__ void load(const BoundsOf& w, int entry, int lane, bool& missing) {
    missing = missing || static_cast<uint32_t>(entry) >= w.num;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t page = static_cast<uint32_t>(__shfl_sync(0xffffffffu, entry, (lane >> 2) + 8 * h));
      ok[h] = page < w.num;
      const uint8_t* src = w.base + static_cast<uint64_t>(ok[h] ? page : 0u) * w.stride;
#pragma unroll
      for (int j = 0; j < 2 * NG; ++j) a[h][j] = *reinterpret_cast<const uint4*>(src + 64 * j);
      e[h] = static_cast<int8_t>(src[w.to_exponent]);
    }
  }
  // the same from shared memory, `there` telling which pages are
  __device__ __forceinline__ void load(const unsigned char* staged, const uint8_t* there, int lane) {
    constexpr int D = 64 * NG, PITCH = staged_pitch(D);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned char* src = staged + ((lane >> 2) + 8 * h) * PITCH;
      ok[h] = there[(lane >> 2) + 8 * h];
#pragma unroll
      for (int j = 0; j < 2 * NG; ++j) a[h][j] = *reinterpret_cast<const uint4*>(src + 64 * j + 16 * (lane & 3));
      e[h] = static_cast<int8_t>(src[2 * D]);
    }
  }
  // key(k, slot, c, value) is called, by one lane each, for the columns below `columns` and the tokens' slots
  // (0 .. 7 >> SLOTS) of q[k] with the greatest score of the token's heads, 0 for a page that is not there.
  // Two sums per product, so that its steps do not all wait for one another; the lanes of a page that hold a
  // token's columns halve what they hold at each exchange of their maxima.
  template <int SLOTS, int K, typename F>
  __device__ __forceinline__ void score(const Query<NG> (&q)[K], int c0, int columns, int lane, F&& key) const {
    const int g = lane >> 2, t = lane & 3;
    int v[K][2][2];  // [product][row lane / 4 or 8 further][column 2 t or the next]
#pragma unroll
    for (int k = 0; k < K; ++k) {
      int acc[2][4];
#pragma unroll
      for (int j = 0; j < 2 * NG; ++j) {
        mma_s8_16832(acc[0], a[0][j].x, a[1][j].x, a[0][j].y, a[1][j].y, q[k].b[j].x, q[k].b[j].y, j > 0);
        mma_s8_16832(acc[1], a[0][j].z, a[1][j].z, a[0][j].w, a[1][j].w, q[k].b[j].z, q[k].b[j].w, j > 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[k][i >> 1][i & 1] = acc[0][i] + acc[1][i];
    }
    auto give = [&](int k, int slot, int h, int value) {
      const int c = c0 + g + 8 * h;
      const float unit = pow2f(min(max(h ? e[1] : e[0], -100), 100));
      if (c < columns) key(k, slot, c, (h ? ok[1] : ok[0]) ? order_key(static_cast<float>(value) * unit) : 0u);
    };
    if constexpr (SLOTS == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) give(k, 2 * t + (i & 1), i >> 1, v[k][i >> 1][i & 1]);
    } else {
      int x[K][2];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) x[k][h] = max(v[k][h][0], v[k][h][1]);
      if constexpr (SLOTS == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) give(k, t, h, x[k][h]);
      } else {
        const int h = t & 1;  // the lane keeps this row
        int y[K];
#pragma unroll
        for (int k = 0; k < K; ++k) y[k] = max(h ? x[k][1] : x[k][0], __shfl_xor_sync(0xffffffffu, h ? x[k][0] : x[k][1], 1));
        if constexpr (SLOTS == 2) {
#pragma unroll
          for (int k = 0; k < K; ++k) give(k, t >> 1, h, y[k]);
        } else if constexpr (K == 2) {
          const int k = t >> 1;  // and this product
          give(k, 0, h, max(k ? y[1] : y[0], __shfl_xor_sync(0xffffffffu, k ? y[0] : y[1], 2)));
        } else {
          const int z = max(y[0], __shfl_xor_sync(0xffffffffu, y[0], 2));
          if (t < 2) give(0, 0, h, z);
        }
      }
    }
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
  const float u0 = pow2f(eq / 2), u1 = pow2f(eq - eq / 2);  // the product with 2^eq is rounded where it leaves fp32 only
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
      if (scores != nullptr) scores[mine] = number_of(key) * u0 * u1;
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
template <int SLOTS, int NG>
__device__ __forceinline__ int query_exponent(const Query<NG>& q, const SelectParams& w, const __nv_bfloat16* heads, int first,
                                              int lane) {
  float top = 0.0f;
  for (int h = first; h < w.group; h += 8) top = fmaxf(top, q.top_of(heads + h * w.qh, lane, w.vec));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
#pragma unroll
  for (int o = 0; o < SLOTS; ++o) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4 << o));
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
  const BoundsOf bounds = BoundsOf::of<NG>(w, head, lane);
  bool missing = false;
  PageRows<NG> rows;  // the first pages' loads fly while q is rounded
  rows.load(bounds, PageRows<NG>::entry(row, begin, want.columns, lane), lane, missing);
  int entry = PageRows<NG>::entry(row, begin + step, want.columns, lane);
  Query<NG> q[1];
  q[0].e = query_exponent<3>(q[0], w, heads, min(lane >> 2, w.group - 1), lane);
  for (int h = 0; h < w.group; h += 8) {
    q[0].round(heads + min(h + (lane >> 2), w.group - 1) * w.qh, lane, w.vec);
    if (h > 0) {
      rows.load(bounds, PageRows<NG>::entry(row, begin, want.columns, lane), lane, missing);
      entry = PageRows<NG>::entry(row, begin + step, want.columns, lane);
    }
    for (int c0 = begin; c0 < want.columns; c0 += step) {
      const PageRows<NG> now = rows;
      if (c0 + step < want.columns) rows.load(bounds, entry, lane, missing);
      entry = PageRows<NG>::entry(row, c0 + 2 * step, want.columns, lane);
      now.template score<3>(q, c0, want.columns, lane, [&](int, int, int c, uint32_t key) {
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
  if (missing) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
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

// Many rows: a warp per kv head and two products' columns, 16 >> SLOTS tokens: the heads of several tokens
// share a product, and two products a page's bounds. Where the tokens of a CTA are of one sequence (a
// prompt), its warps share the bounds too, through shared memory, STAGE pages at a time, the next on their way
// meanwhile: read by each warp for itself they are 34 bytes per cycle of an SM from L2, which then bounds the kernel.
constexpr int PRODUCTS = 2, STAGE = SELECT_THREADS / 8;  // eight threads copy a page's bounds
__host__ __device__ constexpr int staged_bytes(int d) { return 2 * STAGE * staged_pitch(d); }
template <int NG, int SLOTS>
__global__ void __launch_bounds__(SELECT_THREADS, 2) select_pages_warp_kernel(SelectParams w) {
  constexpr int D = 64 * NG, PITCH = staged_pitch(D);
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ uint8_t s_there[2 * STAGE];
  const Pages& p = w.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_wait();
  allow_dependent_launch();
  if (blockIdx.x == 0) check_batch(p, w.total, tid, SELECT_THREADS);
  constexpr int each = 8 >> SLOTS, tokens = PRODUCTS * each;
  const int64_t block = blockIdx.x / p.kv_heads, cta0 = block * SELECT_WARPS * tokens, token0 = cta0 + warp * tokens;
  const int head = static_cast<int>(blockIdx.x - block * p.kv_heads);
  uint32_t* keys = s_keys + warp * tokens * w.key_ld;
  const int column = (lane >> 2) & ((1 << SLOTS) - 1);  // the lane's head of a pass
  bool missing = false;
  const __nv_bfloat16* heads[PRODUCTS];
  Query<NG> q[PRODUCTS];
  // the queries of the tokens from `first` to `last`; columns of others repeat one of them
  auto queries = [&](int64_t first, int64_t last) {
#pragma unroll
    for (int k = 0; k < PRODUCTS; ++k) {
      const int64_t token = std::min(std::max(token0 + k * each + (lane >> 2 >> SLOTS), first), last);
      heads[k] = w.q + token * w.qt + static_cast<int64_t>(head) * w.group * w.qh;
      q[k].e = query_exponent<SLOTS>(q[k], w, heads[k], min(column, w.group - 1), lane);
    }
  };
  auto round = [&](int h) {
#pragma unroll
    for (int k = 0; k < PRODUCTS; ++k) q[k].round(heads[k] + min(h + column, w.group - 1) * w.qh, lane, w.vec);
  };
  auto score = [&](const PageRows<NG>& rows, int h, int c0, int columns) {
    rows.template score<SLOTS>(q, c0, columns, lane, [&](int k, int slot, int c, uint32_t key) {
      uint32_t* at = keys + (k * each + slot) * w.key_ld + c;
      *at = h > 0 ? max(key, *at) : key;
    });
  };
  auto columns_of = [&](int64_t pos) {  // visible pages
    return pos < 0 ? 0 : static_cast<int>(std::min<int64_t>((pos >> p.page_shift) + 1, p.table_cols));
  };
  // the lists of the tokens done .. of the warp's, which begin at position pos
  auto search = [&](int done, int run, int64_t pos) {
    __syncwarp();
    for (int i = done; i < done + run; ++i) {
      const int64_t list = ((token0 + i) * p.kv_heads + head) * w.count;
      const Wanted want = {columns_of(pos + i - done), w.count, w.first, w.last};
      const int k = i / each, e = __shfl_sync(0xffffffffu, k == 0 ? q[0].e : q[1].e, (i - k * each) << SLOTS << 2);
      take<1>(keys + i * w.key_ld, want, e, w.out + list, w.scores == nullptr ? nullptr : w.scores + list, nullptr);
    }
    __syncwarp();
  };
  auto beyond = [&](int64_t last) {
    if (lane == 0 && last >= 0 && (last >> p.page_shift) >= p.table_cols) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
  };
  const int64_t cta_end = std::min<int64_t>(cta0 + SELECT_WARPS * tokens, w.total);
  int b;
  int64_t pos;
  if (find_token(p, cta0, w.total, b, pos) && p.cu[b + 1] >= cta_end) {
    const int64_t last = pos + (cta_end - 1 - cta0);
    const int columns = columns_of(last);
    beyond(last);
    const int32_t* row = p.table + b * p.table_ld;
    unsigned char* stages = reinterpret_cast<unsigned char*>(s_keys + SELECT_WARPS * tokens * w.key_ld);
    const int who = tid >> 3, part = tid & 7;
    const uint8_t* base = w.bounds + static_cast<int64_t>(head) * bounds_bytes(D) + 16 * part;
    const uint32_t stride = static_cast<uint32_t>(p.kv_heads * bounds_bytes(D)), num = static_cast<uint32_t>(p.num_pages);
    auto entry_of = [&](int i) {  // of the page of stage i that the thread copies
      const int c = STAGE * i + who;
      return static_cast<uint32_t>(c < columns ? row[c] : 0);
    };
    auto copy = [&](int i, uint32_t entry) {
      const int at = (i & 1) * STAGE + who;
      const bool there = entry < num;
      missing = missing || !there;
      const uint8_t* src = base + static_cast<uint64_t>(there ? entry : 0u) * stride;
      const uint32_t dst = smem_addr(stages + at * PITCH) + 16 * part;
#pragma unroll
      for (int x = 0; x < bounds_bytes(D) / 16; x += 8)
        if (part + x < bounds_bytes(D) / 16) copy16_async(dst + 16 * x, src + 16 * x);
      if (part == 0) s_there[at] = there;
      copies_commit();
    };
    queries(cta0, cta_end - 1);
    for (int h = 0; h < w.group; h += 8) {
      if (h > 0) __syncthreads();  // the stages are free
      copy(0, entry_of(0));
      uint32_t entry = entry_of(1);
      round(h);
      for (int i = 0; STAGE * i < columns; ++i) {
        copies_wait();
        __syncthreads();  // stage i is there, the other one free
        if (STAGE * (i + 1) < columns) {
          copy(i + 1, entry);
          entry = entry_of(i + 2);
        }
#pragma unroll 1
        for (int c0 = STAGE * i; c0 < min(STAGE * (i + 1), columns); c0 += 16) {
          PageRows<NG> rows;
          const int at = (i & 1) * STAGE + (c0 & (STAGE - 1));
          rows.load(stages + at * PITCH, s_there + at, lane);
          score(rows, h, c0, columns);
        }
      }
      copies_wait();
    }
    if (token0 < cta_end) search(0, static_cast<int>(std::min<int64_t>(tokens, cta_end - token0)), pos + (token0 - cta0));
  } else {
    const BoundsOf bounds = BoundsOf::of<NG>(w, head, lane);
    int done = 0;  // tokens of the group that have been looked at
    while (done < tokens && token0 + done < w.total) {
      // a run of tokens of one sequence
      if (!find_token(p, token0 + done, w.total, b, pos)) {
        ++done;
        continue;
      }
      const int run = static_cast<int>(std::min<int64_t>(p.cu[b + 1] - (token0 + done), tokens - done));
      const int64_t last = pos + run - 1;
      const int columns = columns_of(last);
      beyond(last);
      const int32_t* row = p.table + b * p.table_ld;
      queries(token0 + done, token0 + done + run - 1);
      for (int h = 0; h < w.group; h += 8) {
        round(h);
        int entry = PageRows<NG>::entry(row, 0, columns, lane);
        for (int c0 = 0; c0 < columns; c0 += 16) {
          PageRows<NG> rows;
          rows.load(bounds, entry, lane, missing);
          entry = PageRows<NG>::entry(row, c0 + 16, columns, lane);
          score(rows, h, c0, columns);
        }
      }
      search(done, run, pos);
      done += run;
    }
  }
  if (missing) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
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
  static std::atomic<uint64_t> set[10];  // devices on which the kernels' shared memory is set
  // Many rows, and room for the keys of a CTA's warps: a warp for the heads of 16 >> slots tokens, the more of them the later
  // (they are searched one after the other), later still where its tokens are of several sequences, each of which it
  // takes for itself, and not at all where there are more than four of these. A CTA each and a warp each, us, 32 of 512 pages
  // where not said otherwise:
  //   512 tokens, 64 / 8 heads (4096 rows)  130   42;   128 tokens (1024)   39   30;   64 tokens (512)    22   30
  //   256 tokens, 32 / 8 heads (2048)        69   41;   128 tokens (1024)   39   41
  //   64 sequences, 4 tokens, 32 / 8 heads, of 128 pages (2048)             37   24;   32 of them (1024)  20   23
  //   512 of one token, of 63 pages (4096)   61   35;   256 of them (2048)  30   34
  //   800 tokens, 8 / 8 heads, of 125 (6400) 96   55;   400 tokens (3200)   50   55
  //   800 sequences, one token, of 63 (6400) 100  177
  int slots = 0;
  while (slots < 3 && (1 << slots) < w.group) ++slots;
  const int64_t per_warp = 16 >> slots, tokens = SELECT_WARPS * per_warp, keys = tokens * table_cols;  // of a CTA
  const int64_t many = (4 + (20 >> slots)) * static_cast<int64_t>(num_sms()) * (total < batch * per_warp ? 2 : 1);
  if (units >= many && 4 * total >= batch * per_warp && 4 * keys <= SELECT_KEY_BYTES) {
    w.key_ld = static_cast<int>(table_cols);
    using Kernel = void (*)(SelectParams);
    static constexpr Kernel kernels[2][4] = {
        {select_pages_warp_kernel<1, 0>, select_pages_warp_kernel<1, 1>, select_pages_warp_kernel<1, 2>, select_pages_warp_kernel<1, 3>},
        {select_pages_warp_kernel<2, 0>, select_pages_warp_kernel<2, 1>, select_pages_warp_kernel<2, 2>, select_pages_warp_kernel<2, 3>}};
    const int wide = d == 64 ? 0 : 1;
    const Kernel kern = kernels[wide][slots];
    const int rs = allow_smem(reinterpret_cast<const void*>(kern), SELECT_KEY_BYTES + staged_bytes(d), set[4 * wide + slots]);
    if (rs) return rs;
    FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>((total + tokens - 1) / tokens * kv_heads)), SELECT_THREADS,
                          4 * static_cast<size_t>(keys) + staged_bytes(d), stream, w));
    return launch_status("select_pages_warp_kernel");
  }
  // a CTA for every 128 columns (16 to a warp) as far as there are SMs
  int split = 1;
  while (split < 8 && 2 * split * units <= num_sms() && table_cols > 16 * SELECT_WARPS * split) split *= 2;
  w.key_ld = static_cast<int>(table_cols);
  auto kern = d == 64 ? select_pages_cta_kernel<1> : select_pages_cta_kernel<2>;
  const int rs = allow_smem(reinterpret_cast<const void*>(kern), 4 * MAX_COLUMNS, set[d == 64 ? 8 : 9]);
  if (rs) return rs;
  FAQ_CUDA(launch_clusters(kern, units * split, SELECT_THREADS, 4 * static_cast<size_t>(table_cols), split, stream, w, split));
  return launch_status("select_pages_cta_kernel");
}
