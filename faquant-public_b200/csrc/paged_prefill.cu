// K9 for chunks of many new tokens: the prompt kernel on tcgen05 tensor cores.
//
// Same operation as paged_attention.cu. With hundreds of rows per kv head the products bound
// the time (4 d FLOPs per visible key and row), and expanding the codes once costs little
// beside them, so a chunk takes three kernels:
//   expand   the long sequences' K and V, page by page, to bf16 [tokens][kv heads][d] in the
//            workspace (each sequence from a multiple of 128 tokens, zeros to its end), and the
//            plan of the next kernel's work (one CTA);
//   prefill  a persistent kernel, one CTA per SM. A unit is (sequence, kv head, 2 x T tokens, T =
//            128 / group whole tokens): two tiles A and B of 128 rows, row = token * group + query
//            head, so the keys are read once for the group. Key tiles of 128. The key tiles
//            of all units are cut into equal runs, one per CTA, as in paged_attention.cu;
//   combine  joins the partials of units that lie in several runs.
// In the prefill kernel (640 threads): warps 0-7 the softmax of tile A, 8-15 of tile B, a row's
// 128 keys split over two threads (each reads the other's scores too, for the maximum); warp
// 16 loads Q and K by TMA, warp 17 V; warp 18 issues the MMAs. S_t = Q_t K^T and O_t take 128
// columns of tensor memory each, all there is at d = 128. The softmax warps release S_t as
// soon as it is in their registers, so the next S_t is computed under their exponentials, and
// write P_t (bf16) to shared memory as the A operand of O_t += P_t V. (P_t in tensor memory,
// over S_t, saves shared-memory traffic but chains the next S_t behind this product: 4700
// cycles per pair of 128 x 128 tiles against 4000.)
// Softmax: a row's reference maximum is raised only when a score passes it by more than 2^8
// (then O is rescaled in tensor memory), so a step mostly has no rescaling.
//
// Measured (one B200, d = 128): the last 512 of 32768 tokens with 64 query heads on 8 kv heads
// in 531 us, 1027 TFLOP/s counting the visible pairs (592 to 604 us and some 915 TFLOP/s in a long
// series, where the power limit lowers the clocks); all of a 16384-token prompt with 32 heads 1078
// TFLOP/s. The expansion takes 32 us of the first. A key tile takes about 3900 cycles where the
// products alone need 2048. What bounds it is shared memory: the operands of the four products
// (2048 cycles at 128 bytes each), P's writes and the arriving K and V (512 each) fill 3072;
// leaving all exponentials out gains only 30 us, taking them in turns (one tile's under the other's
// waits) 4. At d = 64 it is the softmax's own chain.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_pages.cuh"
#include "tma.h"

namespace faq {
namespace pre {

using namespace kvp;
using pat::ex2;
using pat::LIFT;
using pat::LOWEST;
using pat::pack_bf16;
using pat::RAISE;

constexpr int TILE = 128;            // rows of a tile, keys of a key tile
constexpr int CHUNK = TILE * 128;    // 128 rows of 64 channels
constexpr int THREADS = 640;
constexpr int COST = 3;              // of a unit beyond its key tiles (filling, joining), in key tiles
constexpr int ROWS = 2 * TILE;
constexpr int NO_ROW = 0x7fffffff;   // the last visible key of a row that is not there: it sees all
constexpr int EXPAND_WARPS = 4;      // of a CTA of the expansion

struct Segment {  // a run's part of one unit
  int c0, head, tok0;       // first token of the sequence in q; kv head; first token of the unit
  int n, len;               // of the sequence
  int key_row;              // of the sequence's first key in the workspace
  int k0, count;            // key tiles
  int slot;                 // -1: the whole unit; else where its partial goes
  int b;                    // the sequence
  int pad[6];
};
struct Join {  // the unit that ends in a run and began in an earlier one
  int first;  // run, -1: none
  int c0, head, tok0, n;
  int pad[3];
};

struct Params {
  Pages p;
  int64_t total;
  int group, tile_tokens;  // query heads per kv head, whole tokens of a tile
  int min_rows;            // sequences with fewer rows are not ours
  float scale_log2;
  __nv_bfloat16* out;
  int64_t ot, oh;
  __nv_bfloat16 *k, *v;    // [cap][kv_heads][d]
  int64_t cap;             // tokens
  Segment* segments;       // [runs + units]
  int2* run;               // [runs]: first segment, segments
  Join* joins;             // [runs]
  float* parts;            // [2 runs][ROWS x d + 2 ROWS]
  int runs;
  int64_t max_units;
};

struct Seq {
  int n, len;  // n = 0: not ours
};
__device__ __forceinline__ Seq sequence(const Params& P, int b) {
  const int c0 = P.p.cu[b], c1 = P.p.cu[b + 1];
  Seq s;
  s.n = (c0 >= 0 && c1 > c0 && c1 <= P.total) ? c1 - c0 : 0;
  s.len = length_of(P.p, b);
  if (static_cast<int64_t>(s.n) * P.group < P.min_rows) s.n = 0;
  return s;
}
__device__ __forceinline__ int padded(const Seq& s) { return s.n ? (s.len + TILE - 1) / TILE * TILE : 0; }
// key tiles that unit u of a sequence sees
__device__ __forceinline__ int key_tiles(const Params& P, const Seq& s, int u) {
  const int last = min(s.n, (u + 1) * 2 * P.tile_tokens) - 1;
  const int seen = s.len - s.n + last + 1;
  return seen <= 0 ? 0 : (seen + TILE - 1) / TILE;
}
__device__ __forceinline__ int units_of(const Params& P, const Seq& s) {
  return (s.n + 2 * P.tile_tokens - 1) / (2 * P.tile_tokens);
}

// Exclusive prefix of `mine` over the CTA's threads; *sum receives the total.
template <int WARPS>
__device__ __forceinline__ int64_t block_scan(int64_t mine, int64_t* scratch, int64_t* sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  int64_t before = x - mine, all = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += scratch[w];
    all += scratch[w];
  }
  *sum = all;
  return before;
}

// Whether a key of the key tiles k0 .. k0 + count - 1 of sequence b has no page; asked by a whole warp.
__device__ __forceinline__ bool any_without_page(const Pages& p, int b, int len, int k0, int count, int lane) {
  const int64_t to = std::min<int64_t>(static_cast<int64_t>(k0 + count) * TILE, len);
  bool hole = false;
#pragma unroll 8
  for (int64_t col = (static_cast<int64_t>(k0) * TILE >> p.page_shift) + lane; col << p.page_shift < to; col += 32)
    hole |= no_page(p, b, static_cast<int>(col));
  return __any_sync(0xffffffffu, hole);
}

// ---------------------------------------------------------------- plan
// One CTA: the segments of every run. Units in the order (sequence, token block, kv head);
// segment of unit u in run c at index c + u.
__device__ void make_plan(const Params& P) {
  constexpr int N = 32 * EXPAND_WARPS;
  __shared__ int64_t s_scratch[EXPAND_WARPS];
  __shared__ int64_t s_cost, s_units, s_keys;  // before the sequence (and round of units) at hand
  const int tid = threadIdx.x;
  const int h = P.p.kv_heads;
  for (int c = tid; c < P.runs; c += N) {
    P.run[c] = make_int2(0x7fffffff, 0);
    P.joins[c].first = -1;
  }
  // totals
  int64_t cost = 0;
  for (int b = tid; b < P.p.batch; b += N) {
    const Seq s = sequence(P, b);
    if (s.n == 0) check_rows(P.p, b, P.total);
    for (int u = 0; u < (s.n ? units_of(P, s) : 0); ++u) {
      const int kt = key_tiles(P, s, u);
      cost += kt ? static_cast<int64_t>(kt + COST) * h : 0;
    }
  }
  int64_t total;
  block_scan<EXPAND_WARPS>(cost, s_scratch, &total);
  const int64_t per = std::max<int64_t>((total + P.runs - 1) / P.runs, COST + 2);
  if (tid == 0) s_cost = s_units = s_keys = 0;
  __syncthreads();
  for (int b = 0; b < P.p.batch; ++b) {  // every thread the same sequence, units over the threads
    const Seq s = sequence(P, b);
    if (s.n == 0) continue;
    const int nu = units_of(P, s);
    const int64_t key_row = s_keys;
    const bool fits = key_row + padded(s) <= P.cap && s_units + static_cast<int64_t>(nu) * h <= P.max_units;
    if (!fits && tid == 0) atomicOr(&g_status, FAQ_STATUS_BAD_BOUND);
    for (int u0 = 0; u0 < nu; u0 += N) {
      const int u = u0 + tid;
      const int kt = u < nu && fits ? key_tiles(P, s, u) : 0;
      int64_t cost_sum, unit_sum;
      const int64_t at0 = s_cost + block_scan<EXPAND_WARPS>(kt ? static_cast<int64_t>(kt + COST) * h : 0, s_scratch, &cost_sum);
      const int64_t id0 = s_units + block_scan<EXPAND_WARPS>(kt ? h : 0, s_scratch, &unit_sum);
      for (int hk = 0; kt && hk < h; ++hk) {
        const int64_t at = at0 + static_cast<int64_t>(hk) * (kt + COST), first = at + COST, end = first + kt;
        const int64_t id = id0 + hk;
        const int r0 = static_cast<int>(first / per), r1 = static_cast<int>((end - 1) / per);
        for (int c = r0; c <= r1; ++c) {
          Segment g;
          g.c0 = P.p.cu[b];
          g.head = hk;
          g.tok0 = u * 2 * P.tile_tokens;
          g.n = s.n;
          g.len = s.len;
          g.key_row = static_cast<int>(key_row);
          g.k0 = static_cast<int>(std::max<int64_t>(c * per - first, 0));
          g.count = static_cast<int>(std::min<int64_t>((c + 1) * per - first, kt)) - g.k0;
          g.slot = r0 == r1 ? -1 : 2 * c + (c == r0);
          g.b = b;
          P.segments[c + id] = g;
          atomicMin(&P.run[c].x, static_cast<int>(c + id));  // a run's segments have consecutive indexes
          atomicAdd(&P.run[c].y, 1);
        }
        if (r1 > r0) {
          Join j;
          j.first = r0;
          j.c0 = P.p.cu[b];
          j.head = hk;
          j.tok0 = u * 2 * P.tile_tokens;
          j.n = s.n;
          P.joins[r1] = j;
        }
      }
      __syncthreads();
      if (tid == 0) {
        s_cost += cost_sum;
        s_units += unit_sum;
      }
      __syncthreads();
    }
    if (tid == 0) s_keys += padded(s);
    __syncthreads();
  }
}

// ---------------------------------------------------------------- expand
// A warp takes a block of K or of V; it finds its sequence by a prefix over the sequences' key
// tiles, 32 sequences at a time. The first CTA makes the plan.
template <int NG>
__global__ void __launch_bounds__(32 * EXPAND_WARPS) paged_expand_kernel(Params P) {
  constexpr int D = 64 * NG;
  grid_dependency_wait();
  allow_dependent_launch();
  if (blockIdx.x == 0) {
    make_plan(P);
    return;
  }
  const int lane = threadIdx.x & 31, h = P.p.kv_heads;
  // rows that see no key are zero
  for (int b = blockIdx.x - 1; b < P.p.batch; b += gridDim.x - 1) {
    const Seq s = sequence(P, b);
    const int none = min(s.n, s.n - s.len), heads = P.group * h;
    for (int64_t x = threadIdx.x; x < static_cast<int64_t>(none) * heads * (D / 8); x += blockDim.x) {
      const int64_t r = x / (D / 8);
      *reinterpret_cast<uint4*>(P.out + (P.p.cu[b] + r / heads) * P.ot + (r % heads) * P.oh + x % (D / 8) * 8) =
          make_uint4(0, 0, 0, 0);
    }
  }
  const int64_t item = static_cast<int64_t>(blockIdx.x - 1) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int which = static_cast<int>(item & 1), head = static_cast<int>((item >> 1) % h);
  const int64_t block = (item >> 1) / h, row = block * BLOCK;  // of the workspace
  if (row + BLOCK > P.cap) return;
  int64_t before = 0;  // rows of the sequences before
  int b = -1, pos = 0, len = 0;
  for (int b0 = 0; b0 < P.p.batch; b0 += 32) {
    Seq s = {0, 0};
    if (b0 + lane < P.p.batch) s = sequence(P, b0 + lane);
    const int64_t mine = padded(s);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, row < before + upto);
    if (past) {
      const int who = __ffs(past) - 1;
      b = b0 + who;
      pos = static_cast<int>(row - before - __shfl_sync(0xffffffffu, upto - mine, who));
      len = __shfl_sync(0xffffffffu, s.len, who);
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (b < 0) return;
  const int64_t page = pos < len ? page_of(P.p, b, pos) : -1;
  const int have = page < 0 ? 0 : min(BLOCK, len - pos);
  const int64_t stride = static_cast<int64_t>(h) * D;
  __nv_bfloat16* dst = (which ? P.v : P.k) + row * stride + head * D;
  if (have) {
    const uint8_t* src = P.p.base + page * P.p.page_stride + block_in_page<NG>(P.p, which, head, pos);
    if (which)
      expand_block<__nv_bfloat16, VBlock, NG>(src, dst, stride, 0, have, lane);
    else
      expand_block<__nv_bfloat16, KBlock, NG>(src, dst, stride, 0, have, lane);
  }
  for (int i = have * (D / 8) + lane; i < BLOCK * (D / 8); i += 32)  // zeros behind the end
    *reinterpret_cast<uint4*>(dst + i / (D / 8) * stride + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
}

// ---------------------------------------------------------------- attention
template <int NG>
struct Smem {
  static constexpr int tile = NG * CHUNK;  // bytes of a Q, K or V tile
  static constexpr int q = 0;
  static constexpr int k = q + 2 * tile;
  static constexpr int v = k + 2 * tile;     // one stage
  static constexpr int p = v + tile;         // P of both tiles
  static constexpr int bar = p + 4 * CHUNK;
  static constexpr int bytes = 1024 + bar + 256;
};
constexpr int TMEM_COLS = 512;
__device__ __forceinline__ uint32_t s_col(int t) { return 128u * t; }
__device__ __forceinline__ uint32_t o_col(int t) { return 256u + 128u * t; }
constexpr uint32_t IDESC_QK = idesc_bf16_f32(TILE, TILE, false, false);
constexpr uint32_t idesc_pv(int d) { return idesc_bf16_f32(TILE, d, false, true); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// MMAs and commits by one elected lane of a warp that executes them as a whole.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p, e; .reg .b64 ad, bd; setp.ne.b32 p, %4, 0;\n"
      "mov.b64 ad, {%1, %5}; mov.b64 bd, {%2, %5};\n"
      "elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %3, p; }" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"(SW128_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "{ .reg .pred e; elect.sync _|e, 0xffffffff;\n"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar)
      : "memory");
}

// Named barriers over `count` threads that also AND or OR a predicate across them.
__device__ __forceinline__ bool bar_and(int id, int count, bool v) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v)), "r"(id), "r"(count)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ bool bar_or(int id, int count, bool v) { return !bar_and(id, count, !v); }

// `n` columns of this thread's lane of tensor memory
template <int N>
__device__ __forceinline__ void tmem_ldf(uint32_t taddr, float* f) {
  if constexpr (N >= 32) {
#pragma unroll
    for (int c = 0; c < N; c += 32) tmem_ld32f(taddr + c, f + c);
  } else {
    static_assert(N == 16, "16 or whole 32s");
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]),
          "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15])
        : "r"(taddr));
  }
}
template <int N>
__device__ __forceinline__ void reg_fencef(float* f) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(f[i]));
}

// The softmax of a tile of 128 rows by eight warps. TMEM lets a warp read the lanes of its own
// quarter (warp % 4) only, so a row's keys are shared by the two warps of its quarter: warps
// 0-3 of them take keys 0..63 of every key tile and the lower half of O's channels, warps 4-7
// the others. Units of at most 64 (32) rows stand two (four) times in the tile, one copy of the
// rows per half (quarter) of the lanes: PARTS = 4 (8) warps then share a row's keys, all
// write their P to its first copy's row, and the other copies' rows of O mean nothing.
template <int D>
struct Softmax {
  int quarter, half, lane, site, tile_barrier;
  uint32_t s_addr, o_addr;
  uint8_t* p_tile;
  uint32_t s_full, s_free, p_full, pv_done;
  float scale_log2;
  uint32_t done = 0;  // steps so far
  float m, l;         // the unit's reference maximum (log2) and, after run(), the row's sum

  __device__ __forceinline__ Softmax(uint32_t tmem, int t, int warp, int lane_, uint8_t* p, uint64_t* full,
                                     uint64_t* free_, uint64_t* pfull, uint64_t* pv, float scale)
      : lane(lane_), site(57 + t), p_tile(p), s_full(smem_addr(full)), s_free(smem_addr(free_)), p_full(smem_addr(pfull)),
        pv_done(smem_addr(pv)), scale_log2(scale) {
    quarter = warp & 3;
    half = (warp >> 2) & 1;
    tile_barrier = 1 + t * 4;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    s_addr = tmem + lanes + s_col(t);
    o_addr = tmem + lanes + o_col(t) + D / 2 * half;  // this half's channels
  }

  // quarters of the lanes that a copy of the rows takes
  template <int PARTS>
  static constexpr int QUARTERS = 8 / PARTS;
  // the thread's row, and whether it is its first copy, whose O counts
  template <int PARTS>
  __device__ __forceinline__ int row() const { return (quarter % QUARTERS<PARTS>)*32 + lane; }
  template <int PARTS>
  __device__ __forceinline__ bool first_copy() const { return quarter < QUARTERS<PARTS>; }

  // Part i's place in P_t's row, as TMA would lay out a tile: key chunk, row, unit u at u ^ (row % 8)
  template <int PARTS>
  __device__ __forceinline__ uint8_t* place(int row, int i) const {
    const int key = i * (TILE / PARTS);
    return p_tile + (key >> 6) * CHUNK + row * 128 + ((((key & 63) >> 3) ^ (row & 7)) << 4);
  }

  // The values of the row's parts, among their warps, through P_t's place (no product may be
  // reading it). They come here together, whatever happened before: `ok` tells whether all
  // are well, so that none is left waiting.
  template <int PARTS>
  __device__ __forceinline__ bool exchange(bool ok, int barrier, int row, int part, float mine, float (&all)[PARTS]) {
    *reinterpret_cast<float*>(place<PARTS>(row, part)) = mine;
    const bool well = bar_and(barrier, 32 * PARTS, ok);
#pragma unroll
    for (int i = 0; i < PARTS; ++i) all[i] = *reinterpret_cast<const float*>(place<PARTS>(row, i));
    return bar_and(barrier, 32 * PARTS, well);  // read: P_t may be written
  }

  // Key tiles k0 .. k0 + count - 1 of sequence b of `len` tokens for a row whose last visible key
  // is lim (NO_ROW: there is none in its place). False: a wait ran out. HOLES: some of these keys
  // have no page and are left out, tile by tile as the table has it. That is code of its own: a
  // test of it in the loop of all units took the drafted tokens of 16 sequences from 33.0 us to 34.1, this
  // to 33.4. meanwhile() is called while the last product runs: the prompt kernel sees there whether the
  // next unit has holes (at that unit's start: 560 us instead of 535 for 512 tokens on 32768). (Warps
  // whose rows are all dead work like the others: leaving their exponentials out gained nothing,
  // the live ones are bound by their own latency.)
  template <int PARTS, bool HOLES, typename F>
  __device__ __forceinline__ bool run(const Pages& pages, int b, int len, int k0, int count, int lim, F&& meanwhile) {
    constexpr int KEYS = TILE / PARTS;
    const int row = this->row<PARTS>(), part = quarter / QUARTERS<PARTS> * 2 + half;
    const int barrier = tile_barrier + quarter % QUARTERS<PARTS>;
    const uint32_t p_row = smem_addr(p_tile + (part * KEYS >> 6) * CHUNK + row * 128);
    const int unit0 = (part * KEYS & 63) >> 3;
    const float2 c2 = make_float2(scale_log2, scale_log2);
    // Rows that are not there hold another sequence's queries, or what shared memory held: no score
    // of theirs is above +inf, so they never raise the live rows' maxima, whose roundings would
    // else depend on them.
    m = lim == NO_ROW ? INFINITY : LOWEST;
    l = 0.0f;
    bool ok = true;
    for (int j = 0; j < count; ++j, ++done) {
      ok = ok && mbar_wait_warp(s_full, done & 1, site, j);
      tc_fence_after();
      float f[KEYS];
      tmem_ldf<KEYS>(s_addr + part * KEYS, f);
      tc_wait_ld();
      reg_fencef<KEYS>(f);
      // S_t is in registers: the tensor core may write the next one
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      const int rel = lim - (k0 + j) * TILE - part * KEYS;
      if (__any_sync(0xffffffffu, rel < KEYS - 1)) {
#pragma unroll
        for (int x = 0; x < KEYS; ++x)
          if (x > rel) f[x] = -INFINITY;
      }
      if constexpr (HOLES) {
#pragma unroll
        for (int x = 0; x < KEYS; x += BLOCK) {
          const int key = (k0 + j) * TILE + part * KEYS + x;
          const bool none = key < len && no_page(pages, b, key >> pages.page_shift);
#pragma unroll
          for (int i = 0; i < BLOCK; ++i)
            if (none) f[x + i] = -INFINITY;
        }
      }
      float mx[KEYS / 16];
#pragma unroll
      for (int c = 0; c < KEYS / 16; ++c) {
        mx[c] = max3(f[16 * c], f[16 * c + 1], f[16 * c + 2]);
#pragma unroll
        for (int x = 3; x < 15; x += 2) mx[c] = max3(mx[c], f[16 * c + x], f[16 * c + x + 1]);
      }
      float mine = fmaxf(mx[0], f[15]);
#pragma unroll
      for (int c = 1; c < KEYS / 16; ++c) mine = max3(mine, mx[c], f[16 * c + 15]);
      // raise the rows' maxima when a part has a score far above them (or has to give up)
      float a = 1.0f;
      const bool raise = bar_or(barrier, 32 * PARTS, __fmul_rn(mine, scale_log2) > m + RAISE || !ok);
      if (raise) {
        if (j > 0) ok = ok && mbar_wait_warp(pv_done, (done - 1) & 1, site + 2, j);
        float all[PARTS];
        if (!exchange<PARTS>(ok, barrier, row, part, mine, all)) return false;
        float top = all[0];
#pragma unroll
        for (int i = 1; i < PARTS; ++i) top = fmaxf(top, all[i]);
        const float next = fmaxf(__fmul_rn(top, scale_log2) - LIFT, m);
        a = ex2(0.5f * (m - next));
        m = next;
        l = l * a * a;
      }
      const float2 mneg = make_float2(-m, -m);
      float2 sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t w[KEYS / 2];
#pragma unroll
      for (int x = 0; x < KEYS / 2; ++x) {
        const float2 d = __ffma2_rn(make_float2(f[2 * x], f[2 * x + 1]), c2, mneg);
        const float2 e = make_float2(ex2(d.x), ex2(d.y));
        sum[x & 3] = __fadd2_rn(sum[x & 3], e);
        w[x] = pack_bf16(e.x, e.y);
      }
      const float2 s4 = __fadd2_rn(__fadd2_rn(sum[0], sum[1]), __fadd2_rn(sum[2], sum[3]));
      l += s4.x + s4.y;
      // the product of the step before has read P_t, and O_t is its
      if (j > 0) ok = mbar_wait_warp(pv_done, (done - 1) & 1, site + 2, j);
#pragma unroll
      for (int u = 0; u < KEYS / 8; ++u)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p_row + (((unit0 + u) ^ (row & 7)) << 4)),
                     "r"(w[4 * u]), "r"(w[4 * u + 1]), "r"(w[4 * u + 2]), "r"(w[4 * u + 3])
                     : "memory");
      fence_proxy_async_smem();  // the tensor core reads P through the async proxy
      tc_fence_after();
      if (raise && j > 0 && first_copy<PARTS>()) {
        const float2 a2 = make_float2(a, a);
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          float o[32];
          tmem_ld32f(o_addr + 32 * c, o);
          tc_wait_ld();
          reg_fence32f(o);
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const float2 v = __fmul2_rn(__fmul2_rn(make_float2(o[2 * x], o[2 * x + 1]), a2), a2);
            o[2 * x] = v.x;
            o[2 * x + 1] = v.y;
          }
          tmem_st32f(o_addr + 32 * c, o);
        }
        tc_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    meanwhile();
    ok = ok && mbar_wait_warp(pv_done, (done - 1) & 1, site + 4, count);
    tc_fence_after();
    float all[PARTS];
    if (!exchange<PARTS>(ok, barrier, row, part, l, all)) return false;
    l = all[0];
#pragma unroll
    for (int i = 1; i < PARTS; ++i) l += all[i];  // the same sum in all parts
    return true;
  }

  // O of the row: to dst (bf16, normalized) or, unnormalized with m and l, to row `at` of a
  // partial of `rows` rows. Whole warps take part; only live ones store.
  __device__ __forceinline__ void store(bool live, float* part, int rows, int at, __nv_bfloat16* dst) {
    const float inv = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);  // NaN stays
#pragma unroll 1
    for (int c = 0; c < D / 64; ++c) {
      float o[32];
      tmem_ld32f(o_addr + 32 * c, o);
      tc_wait_ld();
      reg_fence32f(o);
      if (live && part) {
        float4* d4 = reinterpret_cast<float4*>(part + at * D + D / 2 * half + 32 * c);
#pragma unroll
        for (int x = 0; x < 8; ++x) d4[x] = make_float4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
      } else if (live) {
        uint4* d4 = reinterpret_cast<uint4*>(dst + D / 2 * half + 32 * c);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          d4[x] = make_uint4(pack_bf16(o[8 * x] * inv, o[8 * x + 1] * inv), pack_bf16(o[8 * x + 2] * inv, o[8 * x + 3] * inv),
                             pack_bf16(o[8 * x + 4] * inv, o[8 * x + 5] * inv), pack_bf16(o[8 * x + 6] * inv, o[8 * x + 7] * inv));
      }
      __syncwarp();  // the loads above are made by whole warps
    }
    if (live && part && half == 0) {
      part[rows * D + at] = m;
      part[rows * D + rows + at] = l;
    }
    tc_fence_before();
  }
};

template <int NG>
__global__ void __launch_bounds__(THREADS, 1)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                         const __grid_constant__ CUtensorMap tmap_v, Params P) {
  using L = Smem<NG>;
  constexpr int D = 64 * NG;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::bar);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;   // [2 stages]
  uint64_t* k_empty = bars + 4;
  uint64_t* v_full = bars + 6;
  uint64_t* v_empty = bars + 7;
  uint64_t* s_full = bars + 8;   // [2 tiles] S_t computed
  uint64_t* s_free = bars + 10;  // S_t in the registers of the tile's eight warps
  uint64_t* p_full = bars + 12;  // P_t written (and O_t rescaled) by them
  uint64_t* pv_done = bars + 14; // O_t += P_t V completed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(smem_addr(q_full), 1);
    mbar_init(smem_addr(q_empty), 1);
    mbar_init(smem_addr(v_full), 1);
    mbar_init(smem_addr(v_empty), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&k_full[i]), 1);
      mbar_init(smem_addr(&k_empty[i]), 1);
      mbar_init(smem_addr(&s_full[i]), 1);
      mbar_init(smem_addr(&s_free[i]), 8);
      mbar_init(smem_addr(&p_full[i]), 8);
      mbar_init(smem_addr(&pv_done[i]), 1);
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 18) {
    tmem_alloc(smem_addr(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();
  allow_dependent_launch();
  const int2 run = P.run[blockIdx.x];
  // A run's segments are taken last first. Units are mostly about as long as runs, so a run is the
  // end of one unit and the start of the next: with the start first, all CTAs are at about the
  // same key tile at the same time, and the tiles' readers meet in L2. (512 tokens on 32768 with
  // 64/8 heads in a long series, where DRAM's power comes out of the clocks: 588 us against 625.)
  const Segment* last = P.segments + run.x + run.y - 1;
  const int nseg = run.y;
  // whether tile B has rows
  auto two_tiles = [&](const Segment& g) { return g.tok0 + P.tile_tokens < g.n; };

  // Registers: 640 x 96 at launch = 512 x 104 + 128 x 64.
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::: "memory");
    if (warp == 16) {
      if (lane == 0) {
        bool ok = true;
        int step = 0;
        const uint32_t q_bytes = static_cast<uint32_t>(P.group * P.tile_tokens) * 128;
        for (int i = 0; i < nseg && ok; ++i) {
          const Segment g = last[-i];
          const int tiles = two_tiles(g) ? 2 : 1;
          if (i > 0 && !mbar_wait_site(smem_addr(q_empty), (i - 1) & 1, 50, i)) break;
          mbar_arrive_expect_tx(smem_addr(q_full), tiles * NG * q_bytes);
          for (int t = 0; t < tiles; ++t)
            for (int c = 0; c < NG; ++c)
              tma_load_3d(smem_addr(base + L::q + t * L::tile + c * CHUNK), &tmap_q, smem_addr(q_full), c * 64,
                          g.head * P.group, g.c0 + g.tok0 + t * P.tile_tokens);
          for (int j = 0; j < g.count; ++j, ++step) {
            const int st = step & 1;
            if (!mbar_wait_site(smem_addr(&k_empty[st]), ((step >> 1) & 1) ^ 1, 51, step)) { ok = false; break; }
            mbar_arrive_expect_tx(smem_addr(&k_full[st]), L::tile);
            for (int c = 0; c < NG; ++c)
              tma_load_3d(smem_addr(base + L::k + st * L::tile + c * CHUNK), &tmap_k, smem_addr(&k_full[st]), c * 64,
                          g.head, g.key_row + (g.k0 + j) * TILE);
          }
        }
        // drain (bounded): the last loads were consumed before the CTA exits
        for (int x = std::max(0, step - 2); x < step; ++x)
          if (!mbar_wait_site(smem_addr(&k_empty[x & 1]), (x >> 1) & 1, 53, x)) break;
      }
    } else if (warp == 17) {
      if (lane == 0) {
        bool ok = true;
        int step = 0;
        for (int i = 0; i < nseg && ok; ++i) {
          const Segment g = last[-i];
          for (int j = 0; j < g.count; ++j, ++step) {
            if (!mbar_wait_site(smem_addr(v_empty), (step & 1) ^ 1, 52, step)) { ok = false; break; }
            mbar_arrive_expect_tx(smem_addr(v_full), L::tile);
            for (int c = 0; c < NG; ++c)
              tma_load_3d(smem_addr(base + L::v + c * CHUNK), &tmap_v, smem_addr(v_full), c * 64, g.head,
                          g.key_row + (g.k0 + j) * TILE);
          }
        }
        if (step > 0) mbar_wait_site(smem_addr(v_empty), (step - 1) & 1, 54, step);
      }
    } else if (warp == 18) {
      // The whole warp walks this loop and one elected lane issues each instruction, so that
      // addresses and descriptors stay in uniform registers: with one lane in the loop an MMA
      // took 85 cycles to issue (64 to run), beside warps that want the same issue slots.
      const uint32_t q_desc = sw128_desc_lo(smem_addr(base + L::q), 16);
      const uint32_t k_desc = sw128_desc_lo(smem_addr(base + L::k), 16);
      const uint32_t v_desc = sw128_desc_lo(smem_addr(base + L::v), CHUNK);
      const uint32_t p_desc = sw128_desc_lo(smem_addr(base + L::p), 16);
      constexpr uint32_t TILE_D = L::tile >> 4;
      auto wait = [&](uint64_t* bar, uint32_t parity, int site, int step) {
        return mbar_wait_warp(smem_addr(bar), parity & 1, site, step);
      };
      // S_t = Q_t K^T with K in stage st; t and st are constants
      auto issue_qk = [&](auto tile, auto stage) {
        constexpr int t = decltype(tile)::value, st = decltype(stage)::value;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr uint32_t a0 = t * TILE_D, b0 = st * TILE_D;
          const uint32_t off = static_cast<uint32_t>((kk >> 2) * CHUNK + (kk & 3) * 32) >> 4;
          mma_ss(tmem + s_col(t), q_desc + a0 + off, k_desc + b0 + off, IDESC_QK, kk != 0);
        }
        commit(smem_addr(&s_full[t]));
      };
      // O_t += P_t V
      auto issue_pv = [&](auto tile, bool add) {
        constexpr int t = decltype(tile)::value;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < TILE / 16; ++kk) {
          const uint32_t off = static_cast<uint32_t>((kk >> 2) * CHUNK + (kk & 3) * 32) >> 4;
          mma_ss(tmem + o_col(t), p_desc + t * ((2 * CHUNK) >> 4) + off, v_desc + ((kk * 2048) >> 4), idesc_pv(D), add || kk != 0);
        }
        commit(smem_addr(&pv_done[t]));
      };
      const std::integral_constant<int, 0> c0;
      const std::integral_constant<int, 1> c1;
      uint32_t ring = 0;                // key tiles so far
      uint32_t s0 = 0, s1 = 0;          // S_t computed so far
      uint32_t p0 = 0, p1 = 0;          // O_t products so far
      bool ok = true;
      // both tiles' S with the key tile `step`, each when its last one has been read
      auto scores = [&](uint32_t step, bool two) {
        if (!wait(&k_full[step & 1], step >> 1, 67, step)) return false;
        if (s0 > 0 && !wait(&s_free[0], s0 - 1, 68, step)) return false;
        if (step & 1) issue_qk(c0, c1); else issue_qk(c0, c0);
        ++s0;
        if (two) {
          if (s1 > 0 && !wait(&s_free[1], s1 - 1, 69, step)) return false;
          if (step & 1) issue_qk(c1, c1); else issue_qk(c1, c0);
          ++s1;
        }
        commit(smem_addr(&k_empty[step & 1]));
        return true;
      };
      for (int i = 0; i < nseg && ok; ++i) {
        const int n = __shfl_sync(0xffffffffu, last[-i].count, 0);
        const bool two = __all_sync(0xffffffffu, two_tiles(last[-i]));
        if (!wait(q_full, i, 55, i)) break;
        ok = scores(ring, two);
        if (n == 1) commit(smem_addr(q_empty));
        for (int j = 0; j < n && ok; ++j, ++ring) {
          if (j + 1 < n) {
            if (!scores(ring + 1, two)) { ok = false; break; }
            if (j + 2 == n) commit(smem_addr(q_empty));  // the next unit's Q may come
          }
          if (!wait(v_full, ring, 70, ring) || !wait(&p_full[0], p0, 71, ring)) { ok = false; break; }
          issue_pv(c0, j != 0);
          ++p0;
          if (two) {
            if (!wait(&p_full[1], p1, 72, ring)) { ok = false; break; }
            issue_pv(c1, j != 0);
            ++p1;
          }
          commit(smem_addr(v_empty));
        }
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n" ::: "memory");
    const int t = warp >> 3;
    Softmax<D> sm(tmem, t, warp, lane, base + L::p + t * 2 * CHUNK, &s_full[t], &s_free[t], &p_full[t], &pv_done[t],
                  P.scale_log2);
    const int row = sm.template row<2>(), row_tok = row / P.group, row_head = row - row_tok * P.group;
    auto look = [&](int i) {
      return i < nseg && any_without_page(P.p, last[-i].b, last[-i].len, last[-i].k0, last[-i].count, lane);
    };
    bool holes = look(0), next_holes = false;
    for (int i = 0; i < nseg; ++i, holes = next_holes) {
      const Segment g = last[-i];
      auto look_ahead = [&]() { next_holes = look(i + 1); };
      if (t == 1 && !two_tiles(g)) {
        look_ahead();
        continue;
      }
      const int tok = g.tok0 + t * P.tile_tokens + row_tok;
      const bool live = row_tok < P.tile_tokens && tok < g.n;
      const int lim = live ? g.len - g.n + tok : NO_ROW;
      if (!(holes ? sm.template run<2, true>(P.p, g.b, g.len, g.k0, g.count, lim, look_ahead)
                  : sm.template run<2, false>(P.p, g.b, g.len, g.k0, g.count, lim, look_ahead)))
        break;
      float* part = g.slot < 0 ? nullptr : P.parts + static_cast<int64_t>(g.slot) * (ROWS * D + 2 * ROWS);
      sm.store(live, part, ROWS, t * TILE + row,
               P.out + static_cast<int64_t>(g.c0 + (live ? tok : 0)) * P.ot + (g.head * P.group + row_head) * P.oh);
    }
  }
  __syncthreads();
  if (warp == 18) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Joins the partials of the unit that ended in run blockIdx.x, a warp per row, in run order.
template <int D, int ROWS, typename Params>
__global__ void __launch_bounds__(256) prefill_combine_kernel(Params P) {
  constexpr int V = D / 32;
  constexpr int64_t SIZE = ROWS * D + 2 * ROWS;
  grid_dependency_wait();
  allow_dependent_launch();
  const Join j = P.joins[blockIdx.x];
  if (j.first < 0) return;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int t = r / TILE, in_tile = r % TILE, tok_in = in_tile / P.group;
  const int tok = j.tok0 + t * P.tile_tokens + tok_in;
  if (tok_in >= P.tile_tokens || tok >= j.n) return;
  // 32 partials at a time: their weights one per lane, then their rows, loads in flight
  float sum[V], den = 0.0f, top = LOWEST;
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.0f;
  for (int c0 = j.first; c0 <= static_cast<int>(blockIdx.x); c0 += 32) {
    const int c = c0 + lane, n = min(32, static_cast<int>(blockIdx.x) - c0 + 1);
    const float* src = P.parts + (2 * static_cast<int64_t>(c) + (c == j.first)) * SIZE;
    const float m = lane < n ? src[ROWS * D + r] : LOWEST, l = lane < n ? src[ROWS * D + ROWS + r] : 0.0f;
    float next = fmaxf(top, m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, o));
    const float f = ex2(0.5f * (top - next)), e = lane < n ? ex2(0.5f * (m - next)) : 0.0f;
    float dl = lane < n ? e * l * e : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dl += __shfl_xor_sync(0xffffffffu, dl, o);
    den = den * f * f + dl;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = sum[i] * f * f;
    top = next;
#pragma unroll 4
    for (int x = 0; x < n; ++x) {
      const float w = __shfl_sync(0xffffffffu, e, x);
      const float* row = P.parts + (2 * static_cast<int64_t>(c0 + x) + (c0 + x == j.first)) * SIZE + r * D + lane * V;
      if constexpr (V == 4) {
        const float4 u = *reinterpret_cast<const float4*>(row);
        sum[0] += u.x * w * w;
        sum[1] += u.y * w * w;
        sum[2] += u.z * w * w;
        sum[3] += u.w * w * w;
      } else {
        const float2 u = *reinterpret_cast<const float2*>(row);
        sum[0] += u.x * w * w;
        sum[1] += u.y * w * w;
      }
    }
  }
  const float inv = den > 0.0f ? __fdiv_rn(1.0f, den) : (den == 0.0f ? 0.0f : den);
  __nv_bfloat16* dst = P.out + static_cast<int64_t>(j.c0 + tok) * P.ot +
                       (j.head * P.group + in_tile - tok_in * P.group) * P.oh + lane * V;
#pragma unroll
  for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf16(sum[i] * inv, sum[i + 1] * inv);
}

// Sections of the workspace, each 256-byte aligned.
struct Layout {
  int64_t cap, max_units;
  size_t k, v, segments, run, joins, parts, bytes;
};
inline Layout layout(int64_t total, int64_t heads, int64_t kv_heads, int64_t batch, int64_t max_len, int64_t total_len,
                     int min_rows, int d) {
  const int64_t group = heads / kv_heads, tokens = TILE / group;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  Layout a;
  // sequences that can have min_rows rows, and the keys they can have
  const int64_t most = std::min<int64_t>(batch, total * group / min_rows);
  const int64_t len = (max_len + TILE - 1) / TILE * TILE;
  a.cap = std::min(most * len, total_len + most * TILE);
  a.cap = std::max<int64_t>((a.cap + TILE - 1) / TILE * TILE, TILE);
  a.max_units = kv_heads * (total / (2 * tokens) + most);
  const int runs = num_sms();
  a.k = 0;
  a.v = a.k + up(static_cast<size_t>(a.cap) * kv_heads * d * 2);
  a.segments = a.v + up(static_cast<size_t>(a.cap) * kv_heads * d * 2);
  a.run = a.segments + up(static_cast<size_t>(a.max_units + runs) * sizeof(Segment));
  a.joins = a.run + up(runs * sizeof(int2));
  a.parts = a.joins + up(runs * sizeof(Join));
  a.bytes = a.parts + up(static_cast<size_t>(2) * runs * (ROWS * d + 2 * ROWS) * 4);
  return a;
}

template <int NG>
static int launch(Params& P, const __nv_bfloat16* q, int64_t heads, int64_t qt, int64_t qh, const Layout& a, char* ws,
                  void* stream) {
  constexpr int D = 64 * NG;
  P.k = reinterpret_cast<__nv_bfloat16*>(ws + a.k);
  P.v = reinterpret_cast<__nv_bfloat16*>(ws + a.v);
  P.cap = a.cap;
  P.max_units = a.max_units;
  P.segments = reinterpret_cast<Segment*>(ws + a.segments);
  P.run = reinterpret_cast<int2*>(ws + a.run);
  P.joins = reinterpret_cast<Join*>(ws + a.joins);
  P.parts = reinterpret_cast<float*>(ws + a.parts);
  P.runs = num_sms();
  CUtensorMap mq, mk, mv;
  {
    const uint64_t dims[3] = {D, static_cast<uint64_t>(heads), static_cast<uint64_t>(P.total)};
    const uint64_t str[2] = {static_cast<uint64_t>(qh) * 2, static_cast<uint64_t>(qt) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(P.group), static_cast<uint32_t>(P.tile_tokens)};
    const int rc = make_tmap(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  const uint64_t dims[3] = {D, static_cast<uint64_t>(P.p.kv_heads), static_cast<uint64_t>(P.cap)};
  const uint64_t str[2] = {D * 2, static_cast<uint64_t>(P.p.kv_heads) * D * 2};
  const uint32_t box[3] = {64, 1, TILE};
  int rc = make_tmap(&mk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, P.k, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  rc = make_tmap(&mv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, P.v, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  auto kern = paged_prefill_kernel<NG>;
  static std::atomic<uint64_t> set{0};
  rc = allow_smem(reinterpret_cast<const void*>(kern), Smem<NG>::bytes, set);
  if (rc) return rc;
  const int64_t ctas = (P.cap / BLOCK * P.p.kv_heads * 2 + EXPAND_WARPS - 1) / EXPAND_WARPS + 1;
  FAQ_CHECK_ARG(ctas < (int64_t(1) << 31), "too many keys for one call");
  FAQ_CUDA(launch_early(paged_expand_kernel<NG>, dim3(static_cast<unsigned>(ctas)), 32 * EXPAND_WARPS, 0, stream, P));
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(P.runs)), THREADS, Smem<NG>::bytes, stream, mq, mk, mv, P));
  FAQ_CUDA(launch_early(prefill_combine_kernel<D, ROWS, Params>, dim3(static_cast<unsigned>(P.runs), ROWS / 8), 256, 0, stream, P));
  return FAQ_OK;
}

}  // namespace pre
}  // namespace faq
