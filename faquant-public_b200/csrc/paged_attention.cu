// K9 -- attention of a few new tokens per sequence over the paged HiF4 K/V cache.
//
//   O[i] = sum_k p_k V[k] / sum_k p_k,  p_k = exp(scale q_i . K[k]),  k <= len - n + i
//
// for the n new tokens (i = 0 .. n - 1) of each sequence of a ragged batch, the G = heads /
// kv_heads query heads of a kv head sharing its keys. A row of the problem is (token i, query
// head), r = i G + g; a unit is (sequence, kv head, 8 rows).
//
// The cache holds 4.6 bits per value, so per byte of HBM a lot is computed: each code becomes a
// bf16 register value (about two instructions per value), which feeds mma.sync m16n8k16
// directly. The page format is the fragments' layout: no transposition, no shuffle, no
// second copy in shared memory.
//   S^T = K Q^T   A = 16 keys x 16 channels, B = 16 channels x 8 rows. A lane (g = lane / 4,
//                 t = lane % 4) holds keys g and g + 8 and per 64-channel group the channels
//                 of code words 2t, 2t + 1 (a permutation of the channels that Q's
//                 fragments repeat). The group's scale multiplies the 64-channel sum.
//   O^T = V^T P^T A = 16 channels x 16 keys: the words of a token pair hold a quad of channels
//                 of both tokens, and pair j of a word is channel j at two neighbouring
//                 keys. P^T comes from S^T's registers by movmatrix; V's scale (per key and
//                 group) multiplies P before its bf16 rounding, once per group.
// Softmax: one reference maximum per row and warp, raised only when a score passes it by
// more than 2^8 (the sum and the accumulator are fp32, with room for that, so the result does
// not depend on when it is raised beyond fp32 rounding); raising it takes a warp reduction
// and rescales O. The denominator sums the fp32 p before its rounding to bf16.
//
// Work split: the key blocks of all units, in the order (sequence, kv head, rows), are cut
// into equal runs, one per CTA (a function of the device's cu / lens only, so the host
// needs no lengths). Within a run the CTA's warps take blocks in turn, each with its own ring
// of bulk copies and its own O; they meet in shared memory at the unit's end. A unit that lies
// in one run is written out at once; else each run writes a partial (O, m, l) -- at most two per
// CTA -- and paged_combine_kernel joins them in run order (the same bits on every call). Where
// no sequence is longer than WHOLE tokens, units are not split and nothing is joined.
//
// Measured (one B200, 32 query heads on 8 kv heads of 128, one new token): a context of 32768
// tokens in 20.4 us, 32 sequences of 1 .. 16000 tokens (76 MB of cache) in 35.8 us, 2.1 TB/s
// of the pages. No one resource is full: HBM runs at a third of its rate, 54 % of the issue slots
// and 49 % of the integer pipe are taken over a call. A block of 16 tokens takes a warp about
// 470 instructions (118 cycles per block and SM), 223 of them in the integer pipe at half rate (111
// cycles), where 150 to 170 cycles are measured; and each call has some 5 us of dependent loads
// before its first block (cu and lens, the table, the pages) and 4 of its end (the warps' join,
// the runs' join), which is where the issue slots stay empty ("barrier" is the first stall).
#include <algorithm>
#include <atomic>

#include "kv_pages.cuh"

namespace faq {
namespace pat {

using namespace kvp;

constexpr int RB = 8;       // rows of a unit
constexpr int W = 16;       // warps of a CTA, one CTA per SM: 128 registers a thread
constexpr int THREADS = 32 * W;
constexpr int S = 4;        // blocks in flight per warp, 2 x 1184 bytes each at d = 128
constexpr int COST = 2 * W; // of a unit beyond its blocks, see below
// Up to this length a unit is one CTA's: four rounds of its warps cost no more than splitting
// them and joining the parts in a second kernel, whose launch is saved (a sequence of 1000
// tokens with 8 kv heads: 10.7 us against 11.3, 16 such sequences: 11.7 against 15.7).
constexpr int64_t WHOLE = 4 * W * BLOCK;
// A row's exponentials are p = 2^(score - m): m is put LIFT below the greatest score when it is
// raised, and raised when a score lies RAISE above it. The lift costs nothing (fp32 and bf16 hold
// 2^72 as they hold 2^8) and keeps keys that far below the others: p is flushed to zero at
// 2^-126, 190 binary places below the greatest, where its value times the largest of the
// cache (2^18.4) is below the output's own least. So that the factors 2^(m - m') of rescaling
// and joining lose nothing above that either, their half powers are multiplied in twice.
constexpr float LIFT = 64.0f, RAISE = LIFT + 8.0f;
constexpr float LOWEST = -3.402823466e38f;  // where it starts: below every finite score

struct Params {
  Pages p;
  const __nv_bfloat16* q;
  int64_t qt, qh;  // token, head strides
  __nv_bfloat16* out;
  int64_t ot, oh;
  int64_t total;   // rows of q and out
  int group;       // query heads per kv head
  uint32_t group_magic;  // ceil(2^32 / group), see small_div
  float scale_log2;
  bool split;      // units may lie in several runs; else a unit is its first block's run's
  float* parts;    // [2 gridDim][rows x d + 2 rows]: O, m, l
  int32_t* joins;  // [gridDim][8]: the unit that began in an earlier run and ends in this one
};

// x / group for x < 2^32 / group (x is below group + 32 here); a group of 1 has no magic number
__device__ __forceinline__ int small_div(const Params& P, int x) {
  return P.group == 1 ? x : static_cast<int>(__umulhi(static_cast<uint32_t>(x), P.group_magic));
}

struct Seq {
  int n, len, nrb;  // new tokens, length, row blocks of RB rows
};
__device__ __forceinline__ Seq sequence(const Params& P, int b) {
  Seq s;
  const int c0 = P.p.cu[b], c1 = P.p.cu[b + 1];
  s.n = (c0 >= 0 && c1 > c0 && c1 <= P.total) ? c1 - c0 : 0;
  s.len = length_of(P.p, b);
  s.nrb = (s.n * P.group + RB - 1) / RB;
  return s;
}
__device__ __forceinline__ int key_blocks(const Params& P, const Seq& s, int rb) {
  // the row block's last token
  const int last = rb + 1 >= s.nrb ? s.n - 1 : ((rb + 1) * RB - 1) / P.group;
  const int seen = s.len - s.n + last + 1;
  return seen <= 0 ? 0 : (seen + BLOCK - 1) / BLOCK;
}
// cost of a sequence's units of one kv head; units without a key cost nothing
__device__ __forceinline__ int64_t head_cost(const Params& P, const Seq& s) {
  int64_t sum = 0;
  for (int rb = 0; rb < s.nrb; ++rb) {
    const int blocks = key_blocks(P, s, rb);
    sum += blocks ? blocks + COST : 0;
  }
  return sum;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// shared memory: the warps' rings | their O (rows padded) and (m, l) at a unit's end | Q
// fragments | mbarriers
template <int NG>
struct Smem {
  static constexpr int old = 64 * NG + 8;  // floats of an O row
  static constexpr int stage = 2 * block_bytes(NG);
  static constexpr int o = W * S * stage;
  static constexpr int m = o + W * RB * old * 4;
  static constexpr int l = m + W * RB * 4;
  static constexpr int q = l + W * RB * 4;
  static constexpr int bar = q + NG * 2 * 32 * 16;
  static constexpr int bytes = bar + W * S * 8;
};

// A unit costs COST blocks beyond its own (filling the rings, joining the warps), two rounds
// of the warps: the runs are cut in this measure. Without it a CTA whose run holds many short
// units works four times as long as the others (32 sequences of 1 .. 16000 tokens: 129 us
// without it, 57 with one round; after later steps 51.8 with one, 35.1 with two).
// A run's part of one unit, made by one thread for the CTA.
struct Segment {
  int b, head, rb;       // the unit
  int c0, n, len, nrb;   // of its sequence: first token in q, new tokens, length, row blocks
  int rows;              // rows of the unit
  int tok0, rem0;        // its first row is query head rem0 of token tok0
  int k0, count, blocks; // key blocks k0 .. k0 + count - 1 of `blocks`
  int64_t at;            // the unit's place in the order of all costs
};

template <int NG>
__global__ void __launch_bounds__(THREADS, 1) paged_attention_kernel(Params P) {
  using L = Smem<NG>;
  constexpr int D = 64 * NG, OLD = L::old, UNIT = block_bytes(NG), STAGE = L::stage;
  extern __shared__ __align__(128) unsigned char smem[];
  float* s_o = reinterpret_cast<float*>(smem + L::o);  // [W][RB][OLD]
  float* s_m = reinterpret_cast<float*>(smem + L::m);  // [W][RB]
  float* s_l = reinterpret_cast<float*>(smem + L::l);
  uint4* s_q = reinterpret_cast<uint4*>(smem + L::q);  // [NG][2 step pairs][32 lanes]
  uint64_t* s_bar = reinterpret_cast<uint64_t*>(smem + L::bar);  // [W][S]
  __shared__ int64_t s_scan[W], s_per, s_end;
  __shared__ Segment s_seg[3];  // this one, the next, the one after
  __shared__ int s_any, s_empty;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const Pages& p = P.p;
  if (tid < W * S) {
    mbar_init(smem_addr(&s_bar[tid]), 1);
    fence_barrier_init();
  }
  if (tid == 0) s_any = s_empty = 0;
  __syncthreads();  // the count below sets s_empty from any warp
  grid_dependency_wait();
  allow_dependent_launch();

  // Segment x's part in the run [begin, end) of costs, and its unit's rows. A unit's blocks
  // stand behind its fixed cost.
  auto fill = [&](Segment& x, const Seq& s, int64_t begin, int64_t end) {
    x.c0 = p.cu[x.b];
    x.n = s.n;
    x.len = s.len;
    x.nrb = s.nrb;
    const int64_t first = x.at + COST;
    x.k0 = P.split ? static_cast<int>(std::max<int64_t>(begin - first, 0)) : 0;
    x.count = static_cast<int>(std::max<int64_t>(std::min<int64_t>(end - first, x.blocks) - x.k0, 0));
    if (!P.split) x.count = first >= begin && first < end ? x.blocks : 0;
    x.rows = min(RB, s.n * P.group - x.rb * RB);
    x.tok0 = x.rb * RB / P.group;
    x.rem0 = x.rb * RB - x.tok0 * P.group;
  };
  // x becomes the next unit with keys in the run (count 0: there is none)
  auto next_unit = [&](Segment& x, int64_t begin, int64_t end) {
    x.at += x.blocks + COST;
    x.count = 0;
    if (x.at + COST >= end) return;
    Seq s = {x.n, x.len, x.nrb};
    do {
      if (++x.rb >= s.nrb) {
        x.rb = 0;
        if (++x.head >= p.kv_heads || s.nrb == 0) {
          x.head = 0;
          do {
            if (++x.b >= p.batch) return;
            s = sequence(P, x.b);
          } while (s.nrb == 0);
        }
      }
      x.blocks = key_blocks(P, s, x.rb);
    } while (x.blocks == 0);
    fill(x, s, begin, end);
  };

  // ---- this CTA's run of key blocks: a prefix sum over the sequences, one per thread (and
  // round, past THREADS sequences); the thread that holds the run's start makes its segment
  Seq sq = {0, 0, 0};
  int64_t per_head = 0, mine = 0, upto = 0;
  auto count_blocks = [&](int b) {  // warps without a sequence do nothing
    if (b - lane >= p.batch) return;
    sq = {0, 0, 0};
    if (b < p.batch) {
      sq = sequence(P, b);
      if (sq.n == 0) check_rows(p, b, P.total);
    }
    per_head = head_cost(P, sq);
    mine = per_head * p.kv_heads;
    if (sq.n > sq.len) s_empty = 1;
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (lane == 31) s_scan[warp] = upto;
  };
  const int rounds = (p.batch + THREADS - 1) / THREADS;
  int64_t total = 0;
  for (int r = 0; r < rounds; ++r) {
    if (r > 0) __syncthreads();
    count_blocks(r * THREADS + tid);
    __syncthreads();
    if (rounds > 1 || warp * 32 < p.batch)
      for (int w = 0; w < W && r * THREADS + w * 32 < p.batch; ++w) total += s_scan[w];
  }
  int64_t base = 0;
  for (int r = 0; r < rounds; ++r) {
    const int b = r * THREADS + tid;
    if (rounds > 1) {
      __syncthreads();
      count_blocks(b);
      __syncthreads();
    }
    if (b - lane < p.batch) {
      // at least a round of the warps beyond a unit's cost, so that short problems have few
      // partials to join
      const int64_t per = std::max<int64_t>(
          total < (int64_t(1) << 31) ? (static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x
                                     : (total + gridDim.x - 1) / gridDim.x, W + COST);
      const int64_t begin = blockIdx.x * per, end = std::min<int64_t>(total, begin + per);
      int64_t start = base;  // of this thread's sequence, in the order of all costs
      for (int w = 0; w < warp; ++w) start += s_scan[w];
      start += upto - mine;
      if (begin < end && begin >= start && begin < start + mine) {
        Segment x;
        x.b = b;
        const int64_t at = begin - start;
        x.head = static_cast<int>(mine < (int64_t(1) << 31) ? static_cast<uint32_t>(at) / static_cast<uint32_t>(per_head)
                                                            : at / per_head);
        x.at = start + x.head * per_head;
        x.rb = 0;
        x.blocks = key_blocks(P, sq, 0);
        while (begin >= x.at + (x.blocks ? x.blocks + COST : 0)) {
          x.at += x.blocks ? x.blocks + COST : 0;
          x.blocks = key_blocks(P, sq, ++x.rb);
        }
        s_per = per;
        s_end = end;
        fill(x, sq, begin, end);
        if (x.count == 0) next_unit(x, begin, end);  // the run starts behind the unit's last block
        s_seg[0] = x;
        s_any = x.count > 0;
      }
    }
    if (rounds > 1) {
      for (int w = 0; w < W && r * THREADS + w * 32 < p.batch; ++w) base += s_scan[w];
    }
  }
  int32_t* join = P.joins + blockIdx.x * 8;
  if (P.split && tid == 0) join[0] = 0;
  __syncthreads();
  if (s_empty) {  // rows that see no key are zero: tokens at positions below zero
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      const Seq e = sequence(P, b);
      const int none = min(e.n, e.n - e.len), heads = P.group * p.kv_heads;
      for (int64_t i = tid; i < static_cast<int64_t>(none) * heads * (D / 8); i += THREADS) {
        const int64_t row = i / (D / 8);
        *reinterpret_cast<uint4*>(P.out + (p.cu[b] + row / heads) * P.ot + (row % heads) * P.oh + i % (D / 8) * 8) =
            make_uint4(0, 0, 0, 0);
      }
    }
  }
  if (!s_any) return;

  unsigned char* ring = smem + warp * S * STAGE;
  uint64_t* bars = s_bar + warp * S;
  int issued = 0, used = 0;  // copies of this warp's ring
  uint32_t has_page = 0;     // bit of a ring slot: its block has a page
  int ahead = 0, ahead_blocks = 0;  // the next block to copy, of this warp's blocks of s_seg[ahead_seg]
  int ahead_seg = 0;
  const uint8_t* address = nullptr;  // lane l: where the l-th block of the window of 32 starts
  uint32_t valid = 0;                // which of the window's blocks have a page
  auto blocks_of = [&](const Segment& x) { return x.count > warp ? (x.count - warp + W - 1) / W : 0; };
  // A block without a page is copied from page 0 and left out of the softmax.
  auto look_up = [&](const Segment& x) {
    const int i = ahead + lane;
    bool has = false;
    address = p.base;
    if (i < ahead_blocks) {
      const int pos = (x.k0 + warp + i * W) * BLOCK;
      const int64_t page = page_of(p, x.b, pos);
      has = page >= 0;
      address = p.base + (has ? page : 0) * p.page_stride + block_in_page<NG>(p, 0, x.head, pos);
    }
    valid = __ballot_sync(0xffffffffu, has);
  };
  // from a page's K to its V, in units of 16 bytes: bytes pass 32 bits in pages of 8 GiB
  const uint32_t v_dist = static_cast<uint32_t>(p.kv_heads << (p.page_shift - 4)) * (UNIT / 16);
  auto copy_next = [&]() {  // into a free slot of the ring
    if ((ahead & 31) == 0) look_up(s_seg[ahead_seg]);
    const uint32_t slot = issued % S;
    if (lane == (ahead & 31)) {
      const uint32_t bar = smem_addr(&bars[slot]);
      const uint32_t dst = smem_addr(ring + slot * STAGE);
      mbar_arrive_expect_tx(bar, STAGE);
      bulk_copy(dst, address, UNIT, bar);
      bulk_copy(dst + UNIT, address + static_cast<uint64_t>(v_dist) * 16, UNIT, bar);
    }
    has_page = (has_page & ~(1u << slot)) | (((valid >> (ahead & 31)) & 1u) << slot);
    ++issued;
    ++ahead;
  };
  // The fragments of a unit's rows, by one warp: a B fragment's column is row
  // g, and lane t holds channels 16 t .. 16 t + 15 of each group; step ks takes channels
  // 16 t + ks and + 4 (pair ks of word 2 t), then + 8 and + 12 (of word 2 t + 1).
  auto make_q = [&](const Segment& x) {
    const int r = x.rem0 + g, tok = small_div(P, r);
    const bool live = g < x.rows;
    const __nv_bfloat16* row = P.q + static_cast<int64_t>(x.c0 + x.tok0 + (live ? tok : 0)) * P.qt +
                               (x.head * P.group + (live ? r - tok * P.group : 0)) * P.qh;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      const uint4* src = reinterpret_cast<const uint4*>(row + 64 * gr + 16 * t);
      const uint4 u0 = live ? src[0] : make_uint4(0, 0, 0, 0), u1 = live ? src[1] : make_uint4(0, 0, 0, 0);
      const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        s_q[(gr * 2 + i) * 32 + lane] =
            make_uint4(__byte_perm(w[i], w[2 + i], 0x5410), __byte_perm(w[4 + i], w[6 + i], 0x5410),
                       __byte_perm(w[i], w[2 + i], 0x7632), __byte_perm(w[4 + i], w[6 + i], 0x7632));
    }
  };
  // fills the ring's free slots, going on with the next unit's blocks when this one's are done
  auto top_up = [&](int cur, int next, bool more) {
    while (issued - used < S) {
      if (ahead < ahead_blocks) {
        copy_next();
      } else {
        if (!more || ahead_seg != cur) break;
        ahead_seg = next;
        ahead = 0;
        ahead_blocks = blocks_of(s_seg[next]);
      }
    }
  };
  const Expand expand;
  int cur = 0;
  bool ok = true;
  ahead_blocks = blocks_of(s_seg[0]);
  // the last warps have the fewest blocks: Q and the second segment are theirs to make
  if (warp == W - 1) make_q(s_seg[0]);
  if (tid == THREADS - 64) {
    Segment y = s_seg[0];
    next_unit(y, blockIdx.x * s_per, s_end);
    s_seg[1] = y;
  }
  top_up(0, 0, false);
  __syncthreads();

  while (true) {
    const Segment x = s_seg[cur];
    const int next = cur == 2 ? 0 : cur + 1;
    const bool more = s_seg[next].count > 0;
    const int mine_blocks = blocks_of(x);
    top_up(cur, next, more);
    uint4 q[NG * 2];
#pragma unroll
    for (int i = 0; i < NG * 2; ++i) q[i] = s_q[i * 32 + lane];
    // last visible key of the C fragments' columns (rows 2 t, 2 t + 1); the
    // rows past the unit's are not masked (their scores are 0) and not written
    const int lim0 = x.len - x.n + x.tok0;
    int lim[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) lim[h] = lim0 + small_div(P, x.rem0 + 2 * t + h);

    float o[NG * 4][4], m[2] = {LOWEST, LOWEST}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NG * 4; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][c] = 0.0f;

    for (int i = 0; i < mine_blocks; ++i) {
      if (!mbar_wait_warp(smem_addr(&bars[used % S]), (used / S) & 1, 42, used)) {
        ok = false;
        break;
      }
      const unsigned char* kb = ring + (used % S) * STAGE;
      const unsigned char* vb = kb + UNIT;
      const bool page = (has_page >> (used % S)) & 1;
      ++used;

      // ---- S^T = K Q^T
      float acc[NG][4];
#pragma unroll
      for (int gr = 0; gr < NG; ++gr)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[gr][c] = 0.0f;
      uint32_t kw[2][2 * NG];  // [key g / g + 8][group][word 2 t, 2 t + 1]
      uint32_t ke[2][NG];
      float ks[2][NG], vs[2][NG];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        if constexpr (NG == 2) {
          const uint4 u = *reinterpret_cast<const uint4*>(kb + 64 * r + 16 * t);
          kw[h][0] = u.x; kw[h][1] = u.y; kw[h][2] = u.z; kw[h][3] = u.w;
          const uint2 e = *reinterpret_cast<const uint2*>(kb + exp_offset(NG) + 8 * r);
          ke[h][0] = e.x; ke[h][1] = e.y;
          const uint32_t sk = *reinterpret_cast<const uint16_t*>(kb + scale_offset(NG) + 2 * r);
          const uint32_t sv = *reinterpret_cast<const uint16_t*>(vb + scale_offset(NG) + 2 * r);
          ks[h][0] = twice_scale(sk & 255); ks[h][1] = twice_scale(sk >> 8);
          vs[h][0] = twice_scale(sv & 255); vs[h][1] = twice_scale(sv >> 8);
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(kb + 32 * r + 8 * t);
          kw[h][0] = u.x; kw[h][1] = u.y;
          ke[h][0] = *reinterpret_cast<const uint32_t*>(kb + exp_offset(NG) + 4 * r);
          ks[h][0] = twice_scale(kb[scale_offset(NG) + r]);
          vs[h][0] = twice_scale(vb[scale_offset(NG) + r]);
        }
      }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        uint32_t a[2][2][4];  // [key half][word][pair]
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int wd = 0; wd < 2; ++wd)
            expand.word(kw[h][2 * gr + wd], expand.exponents(ke[h][gr], (7 - 4 * t - 2 * wd) & 31), a[h][wd]);
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const uint32_t f0[4] = {a[0][0][2 * i2], a[1][0][2 * i2], a[0][1][2 * i2], a[1][1][2 * i2]};
          const uint32_t f1[4] = {a[0][0][2 * i2 + 1], a[1][0][2 * i2 + 1], a[0][1][2 * i2 + 1], a[1][1][2 * i2 + 1]};
          mma_bf16_16816(acc[gr], f0, q[gr * 2 + i2].x, q[gr * 2 + i2].y);
          mma_bf16_16816(acc[gr], f1, q[gr * 2 + i2].z, q[gr * 2 + i2].w);
        }
      }
      // ---- softmax; c of the fragment: key g + 8 (c / 2), row 2 t + c % 2
      const int first_key = (x.k0 + warp + i * W) * BLOCK, key0 = first_key + g;
      const bool edge = first_key + BLOCK - 1 > lim0 || !page;  // lim0: the unit's first row's
      uint32_t pf[NG][2];
      float s[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[c] = __fmul_rn(acc[0][c], ks[c >> 1][0]);
        if constexpr (NG == 2) s[c] = __fmaf_rn(acc[1][c], ks[c >> 1][1], s[c]);
      }
      if (edge) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (key0 + 8 * (c >> 1) > lim[c & 1] || !page) s[c] = -INFINITY;
      }
      // log2 p against the reference maxima (finite from the start, so no case of its own)
      float e[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) e[c] = __fmaf_rn(s[c], P.scale_log2, -m[c & 1]);
      if (__any_sync(0xffffffffu, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])) > RAISE)) {
        float n0 = __fmul_rn(fmaxf(s[0], s[2]), P.scale_log2), n1 = __fmul_rn(fmaxf(s[1], s[3]), P.scale_log2);
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) {
          n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, y));
          n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, y));
        }
        n0 = fmaxf(n0 - LIFT, m[0]);
        n1 = fmaxf(n1 - LIFT, m[1]);
        const float a0 = ex2(0.5f * (m[0] - n0)), a1 = ex2(0.5f * (m[1] - n1));
        m[0] = n0;
        m[1] = n1;
        l[0] = l[0] * a0 * a0;
        l[1] = l[1] * a1 * a1;
#pragma unroll
        for (int j = 0; j < NG * 4; ++j) {
          o[j][0] = o[j][0] * a0 * a0;
          o[j][1] = o[j][1] * a1 * a1;
          o[j][2] = o[j][2] * a0 * a0;
          o[j][3] = o[j][3] * a1 * a1;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) e[c] = __fmaf_rn(s[c], P.scale_log2, -m[c & 1]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) e[c] = ex2(e[c]);
      l[0] += e[0] + e[2];
      l[1] += e[1] + e[3];
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        pf[gr][0] = transpose8x8(pack_bf16(e[0] * vs[0][gr], e[1] * vs[0][gr]));
        pf[gr][1] = transpose8x8(pack_bf16(e[2] * vs[1][gr], e[3] * vs[1][gr]));
      }
      // ---- O^T += V^T P^T: pairs t and t + 4, sub-block g of each group
      uint32_t vw[2][2 * NG], ve[2][2 * NG];  // [pair][group][quad]
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int pr = t + 4 * h;
        if constexpr (NG == 2) {
          const uint4 u = *reinterpret_cast<const uint4*>(vb + 128 * pr + 16 * (g ^ (2 * t)));
          vw[h][0] = u.x; vw[h][1] = u.y; vw[h][2] = u.z; vw[h][3] = u.w;
          const uint4 e = *reinterpret_cast<const uint4*>(vb + exp_offset(NG) + 16 * pr);
          ve[h][0] = e.x; ve[h][1] = e.y; ve[h][2] = e.z; ve[h][3] = e.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(vb + 64 * pr + 8 * (g ^ (2 * t)));
          vw[h][0] = u.x; vw[h][1] = u.y;
          const uint2 e = *reinterpret_cast<const uint2*>(vb + exp_offset(NG) + 8 * pr);
          ve[h][0] = e.x; ve[h][1] = e.y;
        }
      }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        uint32_t a[2][2][4];  // [pair][quad][channel]
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int qd = 0; qd < 2; ++qd)
            expand.word(vw[h][2 * gr + qd], expand.exponents(ve[h][2 * gr + qd], (7 - 2 * g) & 31), a[h][qd]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t fa[4] = {a[0][0][j], a[0][1][j], a[1][0][j], a[1][1][j]};
          mma_bf16_16816(o[gr * 4 + j], fa, pf[gr][0], pf[gr][1]);
        }
      }
      __syncwarp();  // the slot may be refilled: every lane has read it
      if (ahead < ahead_blocks) copy_next();
      else if (more && ahead_seg == cur) top_up(cur, next, more);
    }

    // ---- the warps' results meet
    if (warp < x.count) {  // warps without a block hold nothing
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], y);
        const int r = 2 * t + h;
        if (r < x.rows) {
          float* dst = s_o + (warp * RB + r) * OLD + 8 * g;
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            *reinterpret_cast<float4*>(dst + 64 * gr) =
                make_float4(o[4 * gr][h], o[4 * gr + 1][h], o[4 * gr + 2][h], o[4 * gr + 3][h]);
            *reinterpret_cast<float4*>(dst + 64 * gr + 4) =
                make_float4(o[4 * gr][2 + h], o[4 * gr + 1][2 + h], o[4 * gr + 2][2 + h], o[4 * gr + 3][2 + h]);
          }
          if (g == 0) {
            s_m[warp * RB + r] = m[h];
            s_l[warp * RB + r] = l[h];
          }
        }
      }
    }
    const bool whole = x.count == x.blocks;
    if (tid == 0) {
      if (x.k0 > 0 && x.k0 + x.count == x.blocks) {  // the unit ends here and began in an earlier run
        join[1] = x.c0 + x.tok0;
        join[2] = x.head;
        join[3] = x.rem0;
        join[4] = x.rows;
        join[5] = static_cast<int>((x.at + COST) / s_per);  // the run that holds the unit's first block
        join[0] = 1;
      }
      if (more) {  // the unit after the next one
        Segment y = s_seg[next];
        next_unit(y, blockIdx.x * s_per, s_end);
        s_seg[next == 2 ? 0 : next + 1] = y;
      }
    }
    if (!__syncthreads_and(ok)) break;  // a copy never landed: recorded; this unit is not written
    float* part = P.parts + (2 * static_cast<int64_t>(blockIdx.x) + (x.k0 == 0)) * (RB * D + 2 * RB);
    const int parts = min(W, x.count);
    for (int i = tid; i < x.rows * (D / 4); i += THREADS) {
      const int r = i / (D / 4), c = i % (D / 4) * 4;
      float top = LOWEST;
      for (int w = 0; w < parts; ++w) top = fmaxf(top, s_m[w * RB + r]);
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float den = 0.0f;
#pragma unroll 4
      for (int w = 0; w < parts; ++w) {
        const float f = ex2(0.5f * (s_m[w * RB + r] - top));
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * RB + r) * OLD + c);
        sum.x += f * v.x * f;
        sum.y += f * v.y * f;
        sum.z += f * v.z * f;
        sum.w += f * v.w * f;
        den += f * s_l[w * RB + r] * f;
      }
      if (whole) {
        const int tok = small_div(P, x.rem0 + r);
        const float inv = den > 0.0f ? __fdiv_rn(1.0f, den) : (den == 0.0f ? 0.0f : den);  // NaN stays
        uint2 w2;
        w2.x = pack_bf16(sum.x * inv, sum.y * inv);
        w2.y = pack_bf16(sum.z * inv, sum.w * inv);
        *reinterpret_cast<uint2*>(P.out + static_cast<int64_t>(x.c0 + x.tok0 + tok) * P.ot +
                                  (x.head * P.group + x.rem0 + r - tok * P.group) * P.oh + c) = w2;
      } else {
        *reinterpret_cast<float4*>(part + r * D + c) = sum;
        if (c == 0) {
          part[RB * D + r] = top;
          part[RB * D + RB + r] = den;
        }
      }
    }
    if (!more) break;
    cur = next;
    if (warp == 0) make_q(s_seg[cur]);
    __syncthreads();  // s_o has been read, Q is there
  }
  // a timeout leaves copies in flight: wait for them (bounded) before the CTA's memory goes
  if (lane == 0)
    for (; used < issued; ++used)
      if (!mbar_wait(smem_addr(&bars[used % S]), (used / S) & 1)) break;
}

// Joins the partials of the unit that ended in run blockIdx.x: its first run's (slot 2 c + 1),
// then those of the runs up to this one (slot 2 c). One CTA per row: eight warps take the
// partials in turn, four channels (two at d = 64) per lane, and meet in shared memory.
template <int D>
__global__ void __launch_bounds__(256) paged_combine_kernel(Params P) {
  constexpr int V = D / 32;
  constexpr int64_t SIZE = RB * D + 2 * RB;
  __shared__ float s_sum[8][D], s_top[8], s_den[8];
  grid_dependency_wait();
  allow_dependent_launch();
  const int32_t* join = P.joins + blockIdx.x * 8;
  const int r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (join[0] == 0 || r >= join[4]) return;
  const int first = join[5], last = blockIdx.x;
  float sum[V], den = 0.0f, top = LOWEST;
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.0f;
#pragma unroll 4
  for (int c = first + warp; c <= last; c += 8) {
    const float* src = P.parts + (2 * static_cast<int64_t>(c) + (c == first)) * SIZE;
    float v[V];
    if constexpr (V == 4) {
      const float4 u = *reinterpret_cast<const float4*>(src + r * D + lane * 4);
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else {
      const float2 u = *reinterpret_cast<const float2*>(src + r * D + lane * 2);
      v[0] = u.x; v[1] = u.y;
    }
    const float m = src[RB * D + r], l = src[RB * D + RB + r];
    const float next = fmaxf(top, m);
    const float f = ex2(0.5f * (top - next)), e = ex2(0.5f * (m - next));
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = sum[i] * f * f + v[i] * e * e;
    den = den * f * f + l * e * e;
    top = next;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s_sum[warp][lane * V + i] = sum[i];
  if (lane == 0) {
    s_top[warp] = top;
    s_den[warp] = den;
  }
  __syncthreads();
  if (threadIdx.x >= D / 2) return;
  const int c = threadIdx.x * 2;
  float all = LOWEST, o0 = 0.0f, o1 = 0.0f, d = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) all = fmaxf(all, s_top[w]);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float f = ex2(0.5f * (s_top[w] - all));
    o0 += f * s_sum[w][c] * f;
    o1 += f * s_sum[w][c + 1] * f;
    d += f * s_den[w] * f;
  }
  const float inv = d > 0.0f ? __fdiv_rn(1.0f, d) : (d == 0.0f ? 0.0f : d);
  const int row = join[3] + r, tok = small_div(P, row);
  *reinterpret_cast<uint32_t*>(P.out + static_cast<int64_t>(join[1] + tok) * P.ot +
                               (join[2] * P.group + row - tok * P.group) * P.oh + c) = pack_bf16(o0 * inv, o1 * inv);
}

constexpr int JOIN_BYTES_PER_CTA = 32;
inline int ctas() { return num_sms(); }
inline size_t workspace(int d) { return static_cast<size_t>(ctas()) * (JOIN_BYTES_PER_CTA + 2 * (RB * d + 2 * RB) * 4); }

template <int NG>
static int launch(Params& P, void* ws, void* stream) {
  const int grid = ctas();
  P.joins = static_cast<int32_t*>(ws);
  P.parts = reinterpret_cast<float*>(static_cast<char*>(ws) + static_cast<size_t>(grid) * JOIN_BYTES_PER_CTA);
  constexpr int bytes = Smem<NG>::bytes;
  auto kern = paged_attention_kernel<NG>;
  static std::atomic<uint64_t> set{0};  // devices on which the kernel's shared memory is set
  int rc = allow_smem(reinterpret_cast<const void*>(kern), bytes, set);
  if (rc) return rc;
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(grid)), THREADS, bytes, stream, P));
  if (!P.split) return FAQ_OK;
  FAQ_CUDA(launch_early(paged_combine_kernel<64 * NG>, dim3(static_cast<unsigned>(grid), RB), 256, 0, stream, P));
  return FAQ_OK;
}

}  // namespace pat
}  // namespace faq

