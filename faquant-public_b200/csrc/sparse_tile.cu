// K13 for chunks of tokens: a tile of up to 128 rows (tokens x query heads of a kv head) over the
// union of its tokens' lists.
//
// Neighbouring tokens mostly list the same pages. Expanding a page's codes for each token apart is
// what the kernel of single tokens (sparse_attention.cu) spends its time on; here a page is expanded
// once for all rows of a tile, on the tensor cores as in paged_chunk.cu (the same operands), and a row's scores with pages that its token does not list are masked. At the start
// the CTA marks, per column, which of its tokens list it (one bit each, up to 32 tokens), and writes the
// marked columns in order: page, column, tokens. A column counts once, however often it is listed.
// Key tiles are 8 blocks of 16 tokens, as they come in that order.
//
// One CTA per (sequence, kv head, tile of tokens), or a cluster of 2, 4 or 8 that share the union's key tiles
// and add up their rows through distributed shared memory.
//
// Measured (one B200): 512 tokens of 32768 with 64 query heads on 8 kv heads of 128 and 32 pages of 64
// tokens each, 164 us (329 with the kernel of single tokens): 9000 key tiles (the lists of 16 neighbours
// hold some 75 pages) at 4300 cycles, two waves of CTAs. The expansion is what the others wait for: a warp
// takes 960 cycles for its block of K and 880 for one of V, 460 for the next block's address, 290 for its loads' issue, then come
// waits for its slots. P is rounded to bf16, as in the kernel of single tokens.
// Dropped: eight softmax warps with 64 keys a thread (186 us; read twice from
// tensor memory, with sixteen expanding warps, 173: then the softmax is), two tiles of rows to a CTA that share the
// expansion (173: their sixteen softmax warps move in step, and the exponentials' unit idles between),
// twelve expanding warps (175, with 64 registers and loads one block ahead), two places for S and a warp of their
// own for the products with V (167).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_pages.cuh"
#include "tma.h"

namespace faq {
namespace spa {

using namespace kvp;

constexpr int RB = 8;  // rows (query heads) of a unit of single tokens

struct Params {
  Pages p;
  const __nv_bfloat16* q;
  int64_t qt, qh;  // token, head strides
  __nv_bfloat16* out;
  int64_t ot, oh;
  int64_t total;   // rows of q and out
  int group, passes;  // query heads per kv head, units of a token and kv head
  const int32_t* list;  // [total, kv_heads, count]
  int count;
  float scale_log2;
};

__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float cluster_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int cluster_load_int(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

}  // namespace spa

namespace spt {

using namespace kvp;
using pat::ex2;
using pat::LOWEST;
using pat::pack_bf16;
using pre::block_scan;
using pre::CHUNK;
using pre::commit;
using pre::IDESC_QK;
using pre::idesc_pv;
using pre::mma_ss;
using pre::o_col;
using pre::s_col;
using pre::TILE;
using pre::TMEM_COLS;
using spa::cluster_load;
using spa::cluster_load4;
using spa::cluster_load_int;
using spa::Params;

constexpr int SOFTMAX_WARPS = 16, EXPAND_WARPS = 8;
constexpr int THREADS = 32 * (SOFTMAX_WARPS + EXPAND_WARPS + 4);  // and a warpgroup for Q and the products
constexpr int PRODUCTS = SOFTMAX_WARPS + EXPAND_WARPS;  // the warp that issues them
constexpr int MAX_UNION = 1536;  // columns of a tile's union
// the table's columns whose marks fit where K and V will be
__host__ __device__ constexpr int columns(int d) { return d / 64 * 4 * CHUNK / 4; }
__host__ __device__ constexpr int tile_tokens(int group) { return TILE / group < 32 ? TILE / group : 32; }

template <int NG>
struct Smem {
  static constexpr int tile = NG * CHUNK;
  static constexpr int q = 0;
  static constexpr int k = q + tile;
  static constexpr int v = k + 2 * tile;
  static constexpr int p = v + 2 * tile;
  static constexpr int page = p + 2 * CHUNK;          // [MAX_UNION]
  static constexpr int entry = page + 8 * MAX_UNION;  // [MAX_UNION + 8], the last ones' tokens none
  static constexpr int scratch = entry + 8 * (MAX_UNION + 8);  // [4][TILE]
  static constexpr int bar = scratch + 16 * TILE;
  static constexpr int bytes = 1024 + bar + 256;
  // at the end, where K and V were: O [TILE][D], m and l [TILE]
  static constexpr int o = k;
};
static_assert(Smem<2>::bytes <= 227 * 1024, "shared memory");

// As the slots of blocks (kv_cache.cu): n tokens are at most n / T + 1 tiles of T, so sequence b's
// tiles get the slots from cu[b] / T + b on.
__host__ __device__ inline int64_t slots_of(int64_t total, int64_t batch, int tokens) { return total / tokens + batch; }

template <int N>
__device__ __forceinline__ void tmem_stf(uint32_t taddr, const float* v) {
  if constexpr (N == 32) {
    tmem_st32f(taddr, v);
  } else {
    static_assert(N == 16, "16 or 32 columns");
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
            taddr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
  }
}

// The softmax of a tile's rows, of which each sees some of a key tile's blocks only, by sixteen warps.
// TMEM lets a warp read the lanes of its own quarter (warp % 4), so the four warps of a quarter share
// its 32 rows: part warp / 4 has the keys 32 part .. of every key tile and that quarter of O's channels.
// Eight warps with 64 keys a thread spilled their registers.
template <int D>
struct Softmax {
  static constexpr int KEYS = TILE / 4, BLOCKS = KEYS / BLOCK, CHANNELS = D / 4;
  int lane, quarter, part, row;
  uint32_t s_addr, o_addr, p_row;
  float* scratch;  // [4][TILE]
  uint32_t s_full, s_free, p_full, pv_done;
  float scale_log2, m, l;  // the reference maximum (log2) and, after run(), the row's sum

  __device__ __forceinline__ Softmax(uint32_t tmem, int warp, int lane_, uint8_t* p, float* x, uint64_t* full, uint64_t* free_,
                                     uint64_t* pfull, uint64_t* pv, float scale)
      : lane(lane_), quarter(warp & 3), part(warp >> 2), scratch(x), s_full(smem_addr(full)), s_free(smem_addr(free_)),
        p_full(smem_addr(pfull)), pv_done(smem_addr(pv)), scale_log2(scale) {
    row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    s_addr = tmem + lanes + s_col(0) + part * KEYS;
    o_addr = tmem + lanes + o_col(0) + part * CHANNELS;
    p_row = smem_addr(p) + (part >> 1) * CHUNK + row * 128;
  }

  // The values of a row's parts, among its four warps. They come here together, whatever happened
  // before: `ok` tells whether all are well.
  __device__ __forceinline__ bool exchange(bool ok, float mine, float (&all)[4]) {
    scratch[part * TILE + row] = mine;
    const bool well = pre::bar_and(1 + quarter, 128, ok);
#pragma unroll
    for (int i = 0; i < 4; ++i) all[i] = scratch[i * TILE + row];
    return pre::bar_and(1 + quarter, 128, well);  // read: it may be written again
  }

  // `count` key tiles; keys(j, block) is how many keys of block `block` (0 .. 7) of key tile j the row
  // sees. A block that none of the warp's rows sees costs nothing but its zeros. False: a wait ran out.
  template <typename F>
  __device__ __forceinline__ bool run(int count, bool there, F&& keys) {
    m = there ? LOWEST : INFINITY;  // rows that are not there never raise the others' maxima
    l = 0.0f;
    bool ok = true;
    for (int j = 0; j < count; ++j) {
      int seen[BLOCKS];
#pragma unroll
      for (int c = 0; c < BLOCKS; ++c) seen[c] = keys(j, part * BLOCKS + c);
      ok = ok && mbar_wait_warp(s_full, j & 1, 98, j);
      tc_fence_after();
      float f[KEYS];
      tmem_ld32f(s_addr, f);
      tc_wait_ld();
      reg_fence32f(f);
      // S is in registers: the tensor core may write the next one
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      float mine = -INFINITY;
#pragma unroll
      for (int c = 0; c < BLOCKS; ++c) {
        float* x = f + BLOCK * c;
        if (__any_sync(0xffffffffu, seen[c] > 0 && seen[c] < BLOCK)) {  // the token's own place
#pragma unroll
          for (int k = 0; k < BLOCK; ++k)
            if (k >= seen[c]) x[k] = -INFINITY;
        }
        float top = pre::max3(x[0], x[1], x[2]);
#pragma unroll
        for (int k = 3; k < 15; k += 2) top = pre::max3(top, x[k], x[k + 1]);
        top = fmaxf(top, x[15]);
        mine = fmaxf(mine, seen[c] > 0 ? top : -INFINITY);
      }
      // raise the rows' maxima when a part has a score far above them (or has to give up)
      float a = 1.0f;
      const bool raise = pre::bar_or(1 + quarter, 128, __fmul_rn(mine, scale_log2) > m + pat::RAISE || !ok);
      if (raise) {
        if (j > 0) ok = ok && mbar_wait_warp(pv_done, (j - 1) & 1, 99, j);
        float all[4];
        if (!exchange(ok, mine, all)) return false;
        const float top = fmaxf(fmaxf(all[0], all[1]), fmaxf(all[2], all[3]));
        const float next = fmaxf(__fmul_rn(top, scale_log2) - pat::LIFT, m);
        a = ex2(0.5f * (m - next));
        m = next;
        l = l * a * a;
      }
      const float2 c2 = make_float2(scale_log2, scale_log2), mneg = make_float2(-m, -m);
      uint32_t w[KEYS / 2];
#pragma unroll
      for (int c = 0; c < BLOCKS; ++c) {
        if (__any_sync(0xffffffffu, seen[c] > 0)) {
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int x = 0; x < BLOCK / 2; ++x) {
            const float2 d = __ffma2_rn(make_float2(f[BLOCK * c + 2 * x], f[BLOCK * c + 2 * x + 1]), c2, mneg);
            const float2 e = make_float2(ex2(d.x), ex2(d.y));
            sum[x & 1] = __fadd2_rn(sum[x & 1], e);
            const uint32_t pair = pack_bf16(e.x, e.y);
            w[BLOCK / 2 * c + x] = seen[c] > 0 ? pair : 0u;  // whatever the score was
          }
          const float2 s2 = __fadd2_rn(sum[0], sum[1]);
          if (seen[c] > 0) l += s2.x + s2.y;
        } else {
#pragma unroll
          for (int x = 0; x < BLOCK / 2; ++x) w[BLOCK / 2 * c + x] = 0u;
        }
      }
      // the product of the step before has read P, and O is its
      if (j > 0) ok = mbar_wait_warp(pv_done, (j - 1) & 1, 99, j);
#pragma unroll
      for (int u = 0; u < KEYS / 8; ++u)  // key chunk, row, unit at unit ^ (row % 8), as TMA would lay it out
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p_row + ((((part & 1) * 4 + u) ^ (row & 7)) << 4)),
                     "r"(w[4 * u]), "r"(w[4 * u + 1]), "r"(w[4 * u + 2]), "r"(w[4 * u + 3])
                     : "memory");
      fence_proxy_async_smem();  // the tensor core reads P through the async proxy
      tc_fence_after();
      if (raise && j > 0) {
        float o[CHANNELS];
        pre::tmem_ldf<CHANNELS>(o_addr, o);
        tc_wait_ld();
        pre::reg_fencef<CHANNELS>(o);
#pragma unroll
        for (int x = 0; x < CHANNELS; ++x) o[x] = o[x] * a * a;
        tmem_stf<CHANNELS>(o_addr, o);
        tc_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    ok = ok && mbar_wait_warp(pv_done, (count - 1) & 1, 99, count);
    tc_fence_after();
    float all[4];
    if (!exchange(ok, l, all)) return false;
    l = (all[0] + all[1]) + (all[2] + all[3]);
    return true;
  }

  // O of the row: to dst (bf16, normalized) or, unnormalized with m and l, to the rows `o` of a
  // partial. Whole warps take part; only live ones store.
  __device__ __forceinline__ void store(bool live, float* o, __nv_bfloat16* dst) {
    const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);  // NaN stays
    float v[CHANNELS];
    pre::tmem_ldf<CHANNELS>(o_addr, v);
    tc_wait_ld();
    pre::reg_fencef<CHANNELS>(v);
    if (live && o) {
      float4* d4 = reinterpret_cast<float4*>(o + row * D + part * CHANNELS);
#pragma unroll
      for (int x = 0; x < CHANNELS / 4; ++x) d4[x] = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
      if (part == 0) {
        o[TILE * D + row] = m;
        o[TILE * D + TILE + row] = l;
      }
    } else if (live) {
      uint4* d4 = reinterpret_cast<uint4*>(dst + part * CHANNELS);
#pragma unroll
      for (int x = 0; x < CHANNELS / 8; ++x)
        d4[x] = make_uint4(pack_bf16(v[8 * x] * inv, v[8 * x + 1] * inv), pack_bf16(v[8 * x + 2] * inv, v[8 * x + 3] * inv),
                           pack_bf16(v[8 * x + 4] * inv, v[8 * x + 5] * inv), pack_bf16(v[8 * x + 6] * inv, v[8 * x + 7] * inv));
    }
    tc_fence_before();
  }
};

template <int NG>
__global__ void __launch_bounds__(THREADS, 1) sparse_tile_kernel(const __grid_constant__ CUtensorMap map_q, Params P, int split) {
  using L = Smem<NG>;
  constexpr int D = 64 * NG, WARPS = THREADS / 32;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::bar);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 2;  // [2 stages]
  uint64_t* k_empty = bars + 4;
  uint64_t* v_full = bars + 6;
  uint64_t* v_empty = bars + 8;
  uint64_t* s_full = bars + 10;
  uint64_t* s_free = bars + 11;
  uint64_t* p_full = bars + 12;
  uint64_t* pv_done = bars + 13;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);
  int64_t* s_page = reinterpret_cast<int64_t*>(base + L::page);  // offset of a page's K of this head
  int2* s_entry = reinterpret_cast<int2*>(base + L::entry);  // a page's first block in the sequence, its tokens
  __shared__ int64_t s_scan[WARPS];
  __shared__ int s_well;  // softmax warps that came to their end
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Pages& p = P.p;
  grid_dependency_wait();

  // ---- the unit
  const int T = tile_tokens(P.group);
  const int rank = static_cast<int>(blockIdx.x % split);
  const int64_t unit = blockIdx.x / split, slot = unit / p.kv_heads;
  const int head = static_cast<int>(unit - slot * p.kv_heads);
  if (blockIdx.x == 0) check_batch(p, P.total, tid, THREADS);
  const int b = last_of(p.batch, [&](int i) { return p.cu[i] / T + static_cast<int64_t>(i) <= slot; });
  const int64_t c0 = p.cu[b], n = p.cu[b + 1] - c0;
  const int64_t u = slot - (c0 / T + b);
  if (c0 < 0 || n <= 0 || c0 + n > P.total || u < 0 || u * T >= n) return;  // the whole cluster
  const int64_t tok0 = u * T;
  const int tokens = static_cast<int>(std::min<int64_t>(T, n - tok0));
  const int64_t pos0 = p.lens[b] - n + tok0;  // of the tile's first token
  const int64_t last_pos = pos0 + tokens - 1;

  // ---- which of the tokens list a column
  uint32_t* marks = reinterpret_cast<uint32_t*>(base + L::k);
  const int seen = last_pos < 0 ? 0 : static_cast<int>(std::min<int64_t>((last_pos >> p.page_shift) + 1, p.table_cols));
  for (int c = tid; c < seen; c += THREADS) marks[c] = 0;
  if (tid == 0) {
    s_well = 0;
    mbar_init(smem_addr(q_full), 1);
    mbar_init(smem_addr(s_full), 1);
    mbar_init(smem_addr(s_free), SOFTMAX_WARPS);
    mbar_init(smem_addr(p_full), SOFTMAX_WARPS);
    mbar_init(smem_addr(pv_done), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&k_full[i]), EXPAND_WARPS);
      mbar_init(smem_addr(&k_empty[i]), 1);
      mbar_init(smem_addr(&v_full[i]), EXPAND_WARPS);
      mbar_init(smem_addr(&v_empty[i]), 1);
    }
    fence_barrier_init();
    tma_prefetch_desc(&map_q);
  }
  if (warp == PRODUCTS) {
    tmem_alloc(smem_addr(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  allow_dependent_launch();  // not before: a CTA of the next kernel that took this SM's columns would wait for this one's end
  for (int i = tid; i < tokens * P.count; i += THREADS) {
    const int tok = i / P.count;
    const int col = P.list[((c0 + tok0 + tok) * p.kv_heads + head) * P.count + (i - tok * P.count)];
    if (col >= 0 && static_cast<int64_t>(col) << p.page_shift <= pos0 + tok) {
      if (col < seen)
        atomicOr(&marks[col], 1u << tok);
      else
        atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);  // beyond the table
    }
  }
  __syncthreads();
  int found;
  {
    const int per = (seen + THREADS - 1) / THREADS, begin = tid * per, end = min(begin + per, seen);
    int64_t mine = 0, all;
    for (int c = begin; c < end; ++c)
      if (marks[c]) {
        const int page = p.table[b * p.table_ld + c];
        if (page < 0 || page >= p.num_pages) {
          atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
          marks[c] = 0;
        } else {
          ++mine;
        }
      }
    int i = static_cast<int>(block_scan<WARPS>(mine, s_scan, &all));
    found = static_cast<int>(all);
    for (int c = begin; c < end; ++c)
      if (marks[c]) {
        s_page[i] = p.table[b * p.table_ld + c] * p.page_stride + block_in_page<NG>(p, 0, head, 0);
        s_entry[i++] = make_int2(c << (p.page_shift - 4), static_cast<int>(marks[c]));
      }
    if (tid < 8) s_entry[found + tid] = make_int2(0, 0);
  }
  __syncthreads();
  const int block_shift = p.page_shift - 4, in_page = (1 << block_shift) - 1;
  // blocks of the union; of the last token's own page those up to it
  const bool own = found > 0 && s_entry[found - 1].x >> block_shift == last_pos >> p.page_shift;
  const int blocks = own ? ((found - 1) << block_shift) + (static_cast<int>(last_pos & ((1 << p.page_shift) - 1)) >> 4) + 1
                         : found << block_shift;
  const int tiles = (blocks + 7) >> 3;
  const int k0 = static_cast<int>(static_cast<int64_t>(tiles) * rank / split);
  const int count = static_cast<int>(static_cast<int64_t>(tiles) * (rank + 1) / split) - k0;

  // Registers: 896 x 72 at launch = 512 x 72 + 256 x 80 + 128 x 56.
  if (warp >= SOFTMAX_WARPS + EXPAND_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n" ::: "memory");
    if (warp == PRODUCTS + 1) {
      if (lane == 0 && count > 0) {
        mbar_arrive_expect_tx(smem_addr(q_full), static_cast<uint32_t>(T * P.group) * 128 * NG);
        for (int c = 0; c < NG; ++c)
          tma_load_3d(smem_addr(base + L::q + c * CHUNK), &map_q, smem_addr(q_full), c * 64, head * P.group,
                      static_cast<int>(c0 + tok0));
        mbar_wait_site(smem_addr(q_full), 0, 90, 0);  // (bounded) it is there before the CTA's end
      }
    } else if (warp == PRODUCTS) {
      // the whole warp walks the steps, one elected lane issues (paged_prefill.cu)
      const uint32_t q_desc = sw128_desc_lo(smem_addr(base + L::q), 16);
      const uint32_t k_desc = sw128_desc_lo(smem_addr(base + L::k), 16);
      const uint32_t v_desc = sw128_desc_lo(smem_addr(base + L::v), CHUNK);
      const uint32_t p_desc = sw128_desc_lo(smem_addr(base + L::p), 16);
      constexpr uint32_t TILE_D = L::tile >> 4;
      auto wait = [&](uint64_t* bar, uint32_t parity, int site, int step) {
        return mbar_wait_warp(smem_addr(bar), parity & 1, site, step);
      };
      auto issue_qk = [&](auto stage) {
        constexpr int st = decltype(stage)::value;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = static_cast<uint32_t>((kk >> 2) * CHUNK + (kk & 3) * 32) >> 4;
          mma_ss(tmem + s_col(0), q_desc + off, k_desc + st * TILE_D + off, IDESC_QK, kk != 0);
        }
        commit(smem_addr(s_full));
        commit(smem_addr(&k_empty[st]));
      };
      auto issue_pv = [&](auto stage, bool add) {
        constexpr int st = decltype(stage)::value;
#pragma unroll
        for (int kk = 0; kk < TILE / 16; ++kk) {
          const uint32_t off = static_cast<uint32_t>((kk >> 2) * CHUNK + (kk & 3) * 32) >> 4;
          mma_ss(tmem + o_col(0), p_desc + off, v_desc + st * TILE_D + ((kk * 2048) >> 4), idesc_pv(D), add || kk != 0);
        }
        commit(smem_addr(pv_done));
        commit(smem_addr(&v_empty[st]));
      };
      const std::integral_constant<int, 0> st0;
      const std::integral_constant<int, 1> st1;
      auto scores = [&](uint32_t step) {
        if (!wait(&k_full[step & 1], step >> 1, 91, step)) return false;
        if (step > 0 && !wait(s_free, step - 1, 92, step)) return false;
        tc_fence_after();
        if (step & 1) issue_qk(st1); else issue_qk(st0);
        return true;
      };
      const bool ok = count > 0 && wait(q_full, 0, 93, 0) && scores(0);
      for (int j = 0; j < count && ok; ++j) {
        if (j + 1 < count && !scores(j + 1)) break;
        if (!wait(&v_full[j & 1], j >> 1, 94, j) || !wait(p_full, j, 95, j)) break;
        tc_fence_after();
        if (j & 1) issue_pv(st1, j != 0); else issue_pv(st0, j != 0);
      }
    }
    __syncwarp();
  } else if (warp >= SOFTMAX_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 80;\n" ::: "memory");
    // ------------------------------------------------------------ expansion: block ew of each key tile
    const int ew = warp - SOFTMAX_WARPS;
    const int64_t v_off = (static_cast<int64_t>(p.kv_heads) << block_shift) * block_bytes(NG);  // from a page's K to its V
    // where block ew of tile j is (null: past the end; the softmax leaves such keys out, and the
    // registers' last block stands in for them, whose values are finite)
    auto block_of = [&](int j) -> const uint8_t* {
      const int i = (k0 + j) * 8 + ew;
      if (i >= blocks) return nullptr;
      return p.base + s_page[i >> block_shift] + (i & in_page) * block_bytes(NG);
    };
    const Expand expand;
    KBlock<NG> kb = {};
    VBlock<NG> vb = {};
    const uint8_t* src = count > 0 ? block_of(0) : nullptr;
    if (src) {
      kb.load(src, lane);
      vb.load(src + v_off, lane);
    }
    for (int step = 0; step < count; ++step) {
      src = step + 1 < count ? block_of(step + 1) : nullptr;  // of the next step
      const int st = step & 1;
      // rows of 128 bytes per group, token ew * 16 + i, unit at unit ^ (token % 8)
      auto write = [&](uint8_t* tile) {
        return [=](int token, int g, int at, const uint32_t (&x)[4]) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_addr(tile) + g * CHUNK +
                                                                         (ew * BLOCK + token) * 128 + ((at ^ (token & 7)) << 4)),
                       "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                       : "memory");
        };
      };
      if (!mbar_wait_warp(smem_addr(&k_empty[st]), ((step >> 1) & 1) ^ 1, 96, step)) break;
      kb.template each<2>(expand, lane, write(base + L::k + st * L::tile));
      fence_proxy_async_smem();  // the tensor core reads it through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&k_full[st]));
      if (src) kb.load(src, lane);
      if (!mbar_wait_warp(smem_addr(&v_empty[st]), ((step >> 1) & 1) ^ 1, 97, step)) break;
      vb.template each<2>(expand, lane, write(base + L::v + st * L::tile));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&v_full[st]));
      if (src) vb.load(src + v_off, lane);
    }
  } else {
    Softmax<D> sm(tmem, warp, lane, base + L::p, reinterpret_cast<float*>(base + L::scratch), s_full, s_free, p_full, pv_done,
                  P.scale_log2);
    const int row = sm.row, tok = row / P.group;
    const bool live = tok < tokens;
    const int sees = static_cast<int>(pos0) + tok + 1;  // keys, of the pages its token lists
    const uint32_t bit = live ? 1u << tok : 0u;
    const int block0 = k0 * 8;
    auto keys = [&](int j, int block) {
      const int i = block0 + j * 8 + block;
      const int2 e = s_entry[i >> block_shift];
      const int left = min(max(sees - ((e.x + (i & in_page)) << 4), 0), BLOCK);
      return e.y & bit ? left : 0;
    };
    const bool ok = count == 0 || sm.run(count, live, keys);
    if (ok && lane == 0) atomicAdd(&s_well, 1);
    if (ok && count > 0) {
      const int row_head = row - tok * P.group;
      sm.store(live, split == 1 ? nullptr : reinterpret_cast<float*>(base + L::o),
               P.out + (c0 + tok0 + (live ? tok : 0)) * P.ot + (static_cast<int64_t>(head) * P.group + row_head) * P.oh);
    }
  }
  __syncthreads();
  if (warp == PRODUCTS) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
  const int rows = tokens * P.group;
  auto place = [&](int row) {
    const int tok = row / P.group;
    return P.out + (c0 + tok0 + tok) * P.ot + (static_cast<int64_t>(head) * P.group + row - tok * P.group) * P.oh;
  };
  if (split == 1) {
    if (tiles == 0)  // rows without a key are zero
      for (int i = tid; i < rows * (D / 8); i += THREADS)
        *reinterpret_cast<uint4*>(place(i / (D / 8)) + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
    return;
  }
  // ---- the CTAs' rows meet, each takes a part of them
  cluster_sync();
  const uint32_t o_addr = smem_addr(base + L::o), m_addr = o_addr + TILE * D * 4, l_addr = m_addr + TILE * 4;
  bool all = true;
  int parts = 0;  // bit k: CTA k had key tiles
  for (int k = 0; k < split; ++k) {
    all = all && cluster_load_int(mapa_shared(smem_addr(&s_well), k)) == SOFTMAX_WARPS;
    if (static_cast<int64_t>(tiles) * (k + 1) / split > static_cast<int64_t>(tiles) * k / split) parts |= 1 << k;
  }
  for (int i = tid + THREADS * rank; i < rows * (D / 4); i += THREADS * split) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float top = LOWEST;
    for (int k = 0; k < split; ++k)
      if (parts >> k & 1) top = fmaxf(top, cluster_load(mapa_shared(m_addr + 4 * r, k)));
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float den = 0.0f;
    for (int k = 0; k < split; ++k) {
      if (!(parts >> k & 1)) continue;
      const float f = ex2(0.5f * (cluster_load(mapa_shared(m_addr + 4 * r, k)) - top));
      const float4 v = cluster_load4(mapa_shared(o_addr + (r * D + c) * 4, k));
      sum.x += f * v.x * f;
      sum.y += f * v.y * f;
      sum.z += f * v.z * f;
      sum.w += f * v.w * f;
      den += f * cluster_load(mapa_shared(l_addr + 4 * r, k)) * f;
    }
    const float inv = den > 0.0f ? __fdiv_rn(1.0f, den) : (den == 0.0f ? 0.0f : den);  // NaN stays
    if (all)
      *reinterpret_cast<uint2*>(place(r) + c) =
          make_uint2(pack_bf16(sum.x * inv, sum.y * inv), pack_bf16(sum.z * inv, sum.w * inv));
  }
  cluster_sync();  // the others have read this CTA's rows
}

template <int NG>
static int launch(const Params& P, int64_t heads, void* stream) {
  constexpr int D = 64 * NG;
  CUtensorMap map_q;
  const uint64_t dims[3] = {D, static_cast<uint64_t>(heads), static_cast<uint64_t>(P.total)};
  const uint64_t str[2] = {static_cast<uint64_t>(P.qh) * 2, static_cast<uint64_t>(P.qt) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(P.group), static_cast<uint32_t>(tile_tokens(P.group))};
  int rc = make_tmap(&map_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, P.q, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  auto kern = sparse_tile_kernel<NG>;
  static std::atomic<uint64_t> set{0};  // devices on which the kernel's shared memory is set
  rc = allow_smem(reinterpret_cast<const void*>(kern), Smem<NG>::bytes, set);
  if (rc) return rc;
  const int64_t units = slots_of(P.total, P.p.batch, tile_tokens(P.group)) * P.p.kv_heads;
  // as many CTAs as fill the SMs once, of some key tiles each
  const int64_t tiles = (static_cast<int64_t>(P.count) << (P.p.page_shift - 4)) / 8;
  int split = 1;
  while (split < 8 && units * split * 2 <= num_sms() && tiles >= 4 * split) split *= 2;
  FAQ_CHECK_ARG(units * split < (int64_t(1) << 31), "too many tokens for one call");
  FAQ_CUDA(launch_clusters(kern, units * split, THREADS, Smem<NG>::bytes, split, stream, map_q, P, split));
  return launch_status("sparse_tile_kernel");
}

}  // namespace spt
}  // namespace faq
