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
// Selection. The first pages and the token's last ones, then the greatest scores, ties to the
// lowest column: a search for the count-th greatest key byte by byte, then one pass in order.
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
};

constexpr int SELECT_THREADS = 256;
constexpr int MAX_COLUMNS = 32768;  // pages of a sequence whose keys fit in shared memory
constexpr int MAX_GROUP = 128;

// The greatest-first order of fp32 as an order of whole numbers; 0 and 2^32 - 1 are no number's.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float number_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// One CTA per token and kv head.
template <int NG>
__global__ void __launch_bounds__(SELECT_THREADS) select_pages_kernel(SelectParams w) {
  constexpr int D = 64 * NG, LANES = D / 16;  // lanes of a page: 16 channels each
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int s_hist[256], s_part[2][SELECT_THREADS / 32], s_found[2];
  __shared__ float s_top[SELECT_THREADS / 32];
  const Pages& p = w.p;
  int8_t* s_q = reinterpret_cast<int8_t*>(smem);  // [group][positive, negative][D]
  uint32_t* s_key = reinterpret_cast<uint32_t*>(smem + 2 * w.group * D);
  grid_dependency_wait();
  allow_dependent_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t token = blockIdx.x / p.kv_heads;
  const int head = static_cast<int>(blockIdx.x - token * p.kv_heads);
  int b;
  int64_t pos;
  if (blockIdx.x == 0) check_batch(p, w.total, tid, SELECT_THREADS);
  if (!find_token(p, token, w.total, b, pos)) return;
  const int64_t list = (token * p.kv_heads + head) * w.count;
  int32_t* out = w.out + list;
  float* scores = w.scores == nullptr ? nullptr : w.scores + list;
  int columns = 0;
  if (pos >= 0) {
    columns = static_cast<int>(std::min<int64_t>((pos >> p.page_shift) + 1, p.table_cols));
    if (tid == 0 && (pos >> p.page_shift) >= p.table_cols) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
  }

  // ---- q of the group in 8 bits
  const __nv_bfloat16* q = w.q + token * w.qt + static_cast<int64_t>(head) * w.group * w.qh;
  float top = 0.0f;
  for (int i = tid; i < w.group * D; i += SELECT_THREADS) {
    const float a = fabsf(__bfloat162float(q[(i / D) * w.qh + i % D]));
    if (a < INFINITY) top = fmaxf(top, a);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_top[warp] = top;
  if (tid < 2) s_found[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < SELECT_THREADS / 32; ++k) top = fmaxf(top, s_top[k]);
  const int eq = shared_exponent(top);
  for (int i = tid; i < w.group * D; i += SELECT_THREADS) {
    float a = __bfloat162float(q[(i / D) * w.qh + i % D]);
    if (!(fabsf(a) < INFINITY)) a = 0.0f;  // what is not finite does not count
    const int n = __float2int_rn(ldexpf(a, -eq));
    s_q[(i / D) * 2 * D + i % D] = static_cast<int8_t>(max(n, 0));
    s_q[(i / D) * 2 * D + D + i % D] = static_cast<int8_t>(min(n, 0));
  }
  __syncthreads();

  // ---- the pages' keys
  const int32_t* row = p.table + b * p.table_ld;
  int have = 0;  // pages that can be taken, of this thread's lane groups
  const int sub = lane % LANES;
  for (int c0 = warp * (32 / LANES); c0 < columns; c0 += SELECT_THREADS / LANES) {  // warp-uniform
    const int c = c0 + lane / LANES;
    const int page = c < columns ? row[c] : -1;
    const bool ok = page >= 0 && page < p.num_pages;
    if (c < columns && !ok) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
    const uint8_t* src = w.bounds + (static_cast<int64_t>(ok ? page : 0) * p.kv_heads + head) * bounds_bytes(D);
    const int4 lo = *reinterpret_cast<const int4*>(src + 16 * sub), hi = *reinterpret_cast<const int4*>(src + D + 16 * sub);
    const int e = static_cast<int8_t>(src[2 * D]);
    int best = INT32_MIN;
    for (int g = 0; g < w.group; ++g) {
      const int4 a = *reinterpret_cast<const int4*>(s_q + g * 2 * D + 16 * sub);
      const int4 n = *reinterpret_cast<const int4*>(s_q + g * 2 * D + D + 16 * sub);
      int sum = __dp4a(a.x, hi.x, __dp4a(n.x, lo.x, 0));
      sum = __dp4a(a.y, hi.y, __dp4a(n.y, lo.y, sum));
      sum = __dp4a(a.z, hi.z, __dp4a(n.z, lo.z, sum));
      sum = __dp4a(a.w, hi.w, __dp4a(n.w, lo.w, sum));
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      best = max(best, sum);
    }
    if (sub == 0 && c < columns) {
      s_key[c] = ok ? order_key(static_cast<float>(best) * pow2f(min(max(e, -100), 100))) : 0;
      have += ok;
    }
  }
  atomicAdd(&s_found[0], have);
  __syncthreads();

  auto rank = [&](int c) -> uint32_t {
    const uint32_t key = s_key[c];
    return key != 0 && (c < w.first || c >= columns - w.last) ? 0xFFFFFFFFu : key;
  };
  // ---- the count-th greatest key, and how many of its equals are taken
  uint32_t limit = 1;  // every page that is there
  int ties = s_found[0];
  if (s_found[0] > w.count) {
    int need = w.count;
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      s_hist[tid] = 0;
      __syncthreads();
      for (int c = tid; c < columns; c += SELECT_THREADS) {
        const uint32_t key = rank(c);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      if (warp == 0) {  // lane l: the bins 255 - 8 l .. 248 - 8 l, from the greatest down
        int n[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          n[i] = s_hist[255 - 8 * lane - i];
          sum += n[i];
        }
        int upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        int before = upto - sum;
        if (before < need && need <= upto) {  // one lane's
          int i = 0;
          while (before + n[i] < need) before += n[i++];
          s_found[0] = 255 - 8 * lane - i;
          s_found[1] = need - before;
        }
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(s_found[0]) << shift;
      need = s_found[1];
      __syncthreads();
    }
    limit = prefix;
    ties = need;
  }

  // ---- one pass in order: those above the limit, and the first of its equals
  int done = 0, equal = 0;
  for (int c0 = 0; c0 < columns; c0 += SELECT_THREADS) {
    const int c = c0 + tid;
    const uint32_t key = c < columns ? rank(c) : 0;
    const bool above = limit == 1 ? key != 0 : key > limit, same = limit != 1 && key == limit;
    const uint32_t va = __ballot_sync(0xffffffffu, above), vs = __ballot_sync(0xffffffffu, same);
    if (lane == 0) {
      s_part[0][warp] = __popc(va);
      s_part[1][warp] = __popc(vs);
    }
    __syncthreads();
    int a = done, s = equal;
    for (int k = 0; k < warp; ++k) {
      a += s_part[0][k];
      s += s_part[1][k];
    }
    const uint32_t below = (1u << lane) - 1;
    a += __popc(va & below);
    s += __popc(vs & below);
    if (above || (same && s < ties)) {
      const int at = a + min(s, ties);
      if (at < w.count) {
        out[at] = c;
        if (scores != nullptr) scores[at] = ldexpf(number_of(s_key[c]), eq);
      }
    }
    for (int k = 0; k < SELECT_THREADS / 32; ++k) {
      done += s_part[0][k];
      equal += s_part[1][k];
    }
    __syncthreads();
  }
  for (int i = min(done + min(equal, ties), w.count) + tid; i < w.count; i += SELECT_THREADS) {
    out[i] = -1;
    if (scores != nullptr) scores[i] = -INFINITY;
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
  FAQ_CHECK_ARG(total * kv_heads < (int64_t(1) << 31), "too many tokens for one call");
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
  const int bytes = 2 * w.group * d + 4 * static_cast<int>(table_cols);
  auto kern = d == 64 ? select_pages_kernel<1> : select_pages_kernel<2>;
  static std::atomic<uint64_t> set[2];
  const int most = 2 * MAX_GROUP * d + 4 * MAX_COLUMNS;
  const int rs = allow_smem(reinterpret_cast<const void*>(kern), most, set[d == 64 ? 0 : 1]);
  if (rs) return rs;
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(total * kv_heads)), SELECT_THREADS, bytes, stream, w));
  return launch_status("select_pages_kernel");
}
