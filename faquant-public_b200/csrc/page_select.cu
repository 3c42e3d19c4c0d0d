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
  int lo = 0, hi = p.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_page_slot(p, mid) <= slot) lo = mid; else hi = mid;
  }
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
constexpr int WARP_COLUMNS = 1024;  // keys that one warp searches
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

// The keys of 16 pages from column c0 on (of `columns`) for the eight columns of `q`: key(slot, c,
// value) is called for column c and the tokens' slots (0 .. 7 >> slots) with each its greatest score, or 0
// for a page that is not there.
template <int NG, typename F>
__device__ __forceinline__ void score_pages(const SelectParams& w, const int32_t* row, int head, const Query<NG>& q, int c0,
                                            int columns, int lane, F&& key) {
  constexpr int D = 64 * NG;
  const int g = lane >> 2, t = lane & 3;
  uint4 a[2][2 * NG];
  bool ok[2];
  int e[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = c0 + g + 8 * h, page = c < columns ? row[c] : -1;
    ok[h] = page >= 0 && page < w.p.num_pages;
    if (c < columns && !ok[h]) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
    const uint8_t* src = w.bounds + (static_cast<int64_t>(ok[h] ? page : 0) * w.p.kv_heads + head) * bounds_bytes(D);
#pragma unroll
    for (int j = 0; j < 2 * NG; ++j) a[h][j] = *reinterpret_cast<const uint4*>(src + 64 * j + 16 * t);
    e[h] = static_cast<int8_t>(src[2 * D]);
  }
  int acc[4] = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 2 * NG; ++j) {
    mma_s8_16832(acc, a[0][j].x, a[1][j].x, a[0][j].y, a[1][j].y, q.b[j].x, q.b[j].y);
    mma_s8_16832(acc, a[0][j].z, a[1][j].z, a[0][j].w, a[1][j].w, q.b[j].z, q.b[j].w);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = c0 + g + 8 * h;
    const float unit = pow2f(min(max(e[h], -100), 100));
    int v0 = acc[2 * h], v1 = acc[2 * h + 1];
    if (w.slots > 0) v0 = max(v0, v1);
    if (w.slots > 1) v0 = max(v0, __shfl_xor_sync(0xffffffffu, v0, 1));
    if (w.slots > 2) v0 = max(v0, __shfl_xor_sync(0xffffffffu, v0, 2));
    if (c >= columns) continue;
    if (w.slots == 0) {
      key(2 * t, c, ok[h] ? order_key(static_cast<float>(v0) * unit) : 0u);
      key(2 * t + 1, c, ok[h] ? order_key(static_cast<float>(v1) * unit) : 0u);
    } else if ((t & ((1 << (w.slots - 1)) - 1)) == 0) {
      key(t >> (w.slots - 1), c, ok[h] ? order_key(static_cast<float>(v0) * unit) : 0u);
    }
  }
}

// What a token's search knows.
struct Wanted {
  int columns;  // visible pages
  int count, first, last;
  __device__ __forceinline__ bool forced(int c) const { return c < first || c >= columns - last; }
};

// One warp: the count-th greatest of the keys bit by bit, then one pass in order. The keys of
// pages that are always taken do not take part in the search.
__device__ __forceinline__ void take_by_warp(const uint32_t* keys, const Wanted& w, int eq, int32_t* out, float* scores,
                                             int lane) {
  uint32_t held[HELD];
  const bool few = w.columns <= 32 * HELD;
  uint32_t top = 0, low = 0xFFFFFFFFu;
  int always = 0, others = 0;
  auto look = [&](int c) -> uint32_t {  // 0: not a choice
    const uint32_t key = c < w.columns ? keys[c] : 0;
    const bool f = w.forced(c);
    always += key != 0 && f;
    others += key != 0 && !f;
    return f ? 0 : key;
  };
  if (few) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      held[i] = look(32 * i + lane);
      top = max(top, held[i]);
      if (held[i]) low = min(low, held[i]);
    }
  } else {
    for (int c = lane; c < w.columns; c += 32) {
      const uint32_t key = look(c);
      top = max(top, key);
      if (key) low = min(low, key);
    }
  }
  always = __reduce_add_sync(0xffffffffu, always);
  others = __reduce_add_sync(0xffffffffu, others);
  const int need = max(w.count - always, 0);
  // taken are the keys above the limit and the first `ties` of those equal to it
  uint32_t limit = 0;
  int ties = 0;
  if (need == 0) {
    limit = 0xFFFFFFFFu;
  } else if (others > need) {
    top = __reduce_max_sync(0xffffffffu, top);
    low = __reduce_min_sync(0xffffffffu, low);
    int bit = 31 - __clz(top ^ low);  // the keys agree above it; -1: they are one
    uint32_t found = bit < 0 ? top : top & ~((2u << bit) - 1);
    int above = 0;
    bool exact = false;
    for (; bit >= 0; --bit) {
      const uint32_t at = found | (1u << bit);
      int n = 0;
      if (few) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) n += held[i] >= at;
      } else {
        for (int c = lane; c < w.columns; c += 32) n += !w.forced(c) && keys[c] >= at;
      }
      n = __reduce_add_sync(0xffffffffu, n);
      if (n >= need) found = at; else above = n;
      if (n == need) {
        exact = true;
        break;
      }
    }
    limit = exact ? found - 1 : found;
    ties = exact ? 0 : need - above;
  }
  int at = 0, equal = 0;
  const uint32_t below = (1u << lane) - 1;
  for (int c0 = 0; c0 < w.columns; c0 += 32) {
    const int c = c0 + lane;
    const uint32_t key = c < w.columns ? keys[c] : 0;
    const bool f = w.forced(c), same = key != 0 && !f && key == limit;
    const uint32_t vs = __ballot_sync(0xffffffffu, same);
    const bool take = key != 0 && (f || key > limit || (same && equal + __popc(vs & below) < ties));
    const uint32_t vt = __ballot_sync(0xffffffffu, take);
    const int mine = at + __popc(vt & below);
    if (take && mine < w.count) {
      out[mine] = c;
      if (scores != nullptr) scores[mine] = ldexpf(number_of(key), eq);
    }
    at += __popc(vt);
    equal += __popc(vs);
  }
  for (int i = min(at, w.count) + lane; i < w.count; i += 32) {
    out[i] = -1;
    if (scores != nullptr) scores[i] = -INFINITY;
  }
}

// The same by a CTA, byte by byte.
__device__ void take_by_cta(const uint32_t* keys, const Wanted& w, int eq, int32_t* out, float* scores) {
  __shared__ int s_hist[256], s_part[2][SELECT_WARPS], s_found[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto rank = [&](int c) -> uint32_t {
    const uint32_t key = keys[c];
    return key != 0 && w.forced(c) ? 0xFFFFFFFFu : key;
  };
  if (tid == 0) s_found[0] = 0;
  __syncthreads();
  int have = 0;
  for (int c = tid; c < w.columns; c += SELECT_THREADS) have += keys[c] != 0;
  have = __reduce_add_sync(0xffffffffu, have);
  if (lane == 0) atomicAdd(&s_found[0], have);
  __syncthreads();
  uint32_t limit = 0;  // taken are the keys above it and the first `ties` of its equals
  int ties = 0;
  const bool search = s_found[0] > w.count;
  if (search) {
    int need = w.count;
    for (int shift = 24; shift >= 0; shift -= 8) {
      s_hist[tid] = 0;
      __syncthreads();
      for (int c = tid; c < w.columns; c += SELECT_THREADS) {
        const uint32_t key = rank(c);
        if (shift == 24 || (key >> (shift + 8)) == (limit >> (shift + 8))) atomicAdd(&s_hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      if (warp == 0) {  // lane l: the bins 255 - 8 l .. 248 - 8 l, from the greatest down
        int n[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          n[i] = s_hist[255 - 8 * lane - i];
          sum += n[i];
        }
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += y;
        }
        before -= sum;
        if (before < need && need <= before + sum) {  // one lane's
          int bin = -1;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (bin < 0 && before + n[i] >= need) bin = i;
            if (bin < 0) before += n[i];
          }
          s_found[0] = 255 - 8 * lane - bin;
          s_found[1] = need - before;
        }
      }
      __syncthreads();
      limit |= static_cast<uint32_t>(s_found[0]) << shift;
      need = s_found[1];
      __syncthreads();
    }
    ties = need;
  }
  int done = 0, equal = 0;
  for (int c0 = 0; c0 < w.columns; c0 += SELECT_THREADS) {
    const int c = c0 + tid;
    const uint32_t key = c < w.columns ? rank(c) : 0;
    const bool above = key > limit, same = search && key == limit;
    const uint32_t va = __ballot_sync(0xffffffffu, above), vs = __ballot_sync(0xffffffffu, same);
    if (lane == 0) {
      s_part[0][warp] = __popc(va);
      s_part[1][warp] = __popc(vs);
    }
    __syncthreads();
    int a = done, s = equal;
    for (int k = 0; k < SELECT_WARPS; ++k) {
      if (k < warp) {
        a += s_part[0][k];
        s += s_part[1][k];
      }
      done += s_part[0][k];
      equal += s_part[1][k];
    }
    const uint32_t below = (1u << lane) - 1;
    a += __popc(va & below);
    s += __popc(vs & below);
    const int at = a + min(s, ties);
    if ((above || (same && s < ties)) && at < w.count) {
      out[at] = c;
      if (scores != nullptr) scores[at] = ldexpf(number_of(keys[c]), eq);
    }
    __syncthreads();
  }
  for (int i = min(done + min(equal, ties), w.count) + tid; i < w.count; i += SELECT_THREADS) {
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
__global__ void __launch_bounds__(SELECT_THREADS) select_pages_cta_kernel(SelectParams w, int split) {
  extern __shared__ __align__(16) uint32_t s_keys[];
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
  Query<NG> q;
  q.e = query_exponent(q, w, heads, min(lane >> 2, w.group - 1), lane);
  for (int h = 0; h < w.group; h += 8) {
    q.round(heads + min(h + (lane >> 2), w.group - 1) * w.qh, lane, w.vec);
    for (int c0 = 16 * (warp + SELECT_WARPS * rank); c0 < want.columns; c0 += 16 * SELECT_WARPS * split)
      score_pages(w, row, head, q, c0, want.columns, lane, [&](int, int c, uint32_t key) {
        const uint32_t at = dst + 4 * c;  // a column's passes are one warp's
        if (h > 0) {
          uint32_t old;
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(old) : "r"(at) : "memory");
          key = max(key, old);
        }
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(key) : "memory");
      });
  }
  if (split > 1) cluster_sync(); else __syncthreads();
  if (rank > 0) return;
  const int64_t list = unit * w.count;
  int32_t* out = w.out + list;
  float* scores = w.scores == nullptr ? nullptr : w.scores + list;
  if (want.columns > WARP_COLUMNS)
    take_by_cta(s_keys, want, q.e, out, scores);
  else if (warp == 0)
    take_by_warp(s_keys, want, q.e, out, scores, lane);
}

// Many rows: a warp per kv head and (8 >> slots) tokens, whose heads share the products with a page.
template <int NG>
__global__ void __launch_bounds__(SELECT_THREADS) select_pages_warp_kernel(SelectParams w) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  const Pages& p = w.p;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_wait();
  allow_dependent_launch();
  if (blockIdx.x == 0) check_batch(p, w.total, tid, SELECT_THREADS);
  const int tokens = 8 >> w.slots;
  const int64_t block = blockIdx.x / p.kv_heads, token0 = (block * SELECT_WARPS + warp) * tokens;
  const int head = static_cast<int>(blockIdx.x - block * p.kv_heads);
  uint32_t* keys = s_keys + static_cast<int64_t>(warp) * tokens * w.key_ld;
  const int mine = lane >> 2 >> w.slots;  // the token of the lane's column
  int done = 0;  // tokens of the group that have been looked at
  while (done < tokens && token0 + done < w.total) {
    // a run of tokens of one sequence
    int b;
    int64_t pos;
    const bool placed = find_token(p, token0 + done, w.total, b, pos);
    if (!placed) {
      ++done;
      continue;
    }
    const int run = static_cast<int>(std::min<int64_t>(p.cu[b + 1] - (token0 + done), tokens - done));
    const int64_t last = pos + run - 1;
    const int columns = last < 0 ? 0 : static_cast<int>(std::min<int64_t>((last >> p.page_shift) + 1, p.table_cols));
    if (lane == 0 && last >= 0 && (last >> p.page_shift) >= p.table_cols) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
    const int64_t token = token0 + min(max(mine, done), done + run - 1);  // columns of other tokens repeat one of the run
    const __nv_bfloat16* heads = w.q + token * w.qt + static_cast<int64_t>(head) * w.group * w.qh;
    const int32_t* row = p.table + b * p.table_ld;
    Query<NG> q;
    const int column = (lane >> 2) & ((1 << w.slots) - 1);
    q.e = query_exponent(q, w, heads, min(column, w.group - 1), lane);
    for (int h = 0; h < w.group; h += 8) {
      q.round(heads + min(h + column, w.group - 1) * w.qh, lane, w.vec);
      for (int c0 = 0; c0 < columns; c0 += 16)
        score_pages(w, row, head, q, c0, columns, lane, [&](int slot, int c, uint32_t key) {
          uint32_t* at = keys + static_cast<int64_t>(slot) * w.key_ld + c;
          *at = h > 0 ? max(key, *at) : key;
        });
    }
    __syncwarp();
    for (int i = done; i < done + run; ++i) {
      const int64_t at = pos + i - done, list = ((token0 + i) * p.kv_heads + head) * w.count;
      const Wanted want = {at < 0 ? 0 : static_cast<int>(std::min<int64_t>((at >> p.page_shift) + 1, p.table_cols)), w.count,
                           w.first, w.last};
      take_by_warp(keys + static_cast<int64_t>(i) * w.key_ld, want, __shfl_sync(0xffffffffu, q.e, i << w.slots << 2),
                   w.out + list, w.scores == nullptr ? nullptr : w.scores + list, lane);
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
  // Many rows, and room for the keys of a CTA's warps: a warp each, whose heads of several tokens share a
  // product.
  int slots = 0;
  while (slots < 3 && (1 << slots) < w.group) ++slots;
  const int64_t keys = (SELECT_WARPS * 8 >> slots) * table_cols;
  if (units << slots >= 64 * static_cast<int64_t>(num_sms()) && 4 * keys <= SELECT_KEY_BYTES) {
    w.slots = slots;
    w.key_ld = static_cast<int>(table_cols);
    const int64_t tokens = SELECT_WARPS * 8 >> slots;
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
