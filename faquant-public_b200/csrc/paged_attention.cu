// K9 -- attention of a few new tokens per sequence over the paged HiF4 K/V cache.
//
//   O[i] = sum_k p_k V[k] / sum_k p_k,  p_k = exp(scale q_i . K[k]),  k <= len - n + i
//
// for the n new tokens (i = 0 .. n - 1) of each sequence of a ragged batch, the G = heads /
// kv_heads query heads of a kv head sharing its keys. A row of the problem is (token i, query
// head), r = i G + g; a unit is (sequence, kv head, 8 NB rows).
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
// more than 2^8 (p stays below 2^8, the sum and the accumulator are fp32, so the result does
// not depend on when it is raised beyond fp32 rounding); raising it takes a warp reduction
// and rescales O. The denominator sums the fp32 p before its rounding to bf16.
//
// Work split: the key blocks of all units, in the order (sequence, kv head, rows), are cut
// into equal runs, one per CTA (a function of the device's cu / lens only, so the host
// needs no lengths). Within a run the eight warps take blocks in turn, each with its own ring
// of bulk copies and its own O; they meet in shared memory at the unit's end. A unit that lies
// in one run is written out at once; else each run writes a partial (O, m, l) -- at most two per
// CTA -- and paged_combine_kernel joins them in run order (the same bits on every call).
#include <algorithm>

#include "kv_pages.cuh"

namespace faq {
namespace pat {

using namespace kvp;

constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr float RAISE = 8.0f;  // log2 headroom of a row's reference maximum

struct Params {
  Pages p;
  const __nv_bfloat16* q;
  int64_t qt, qh;  // token, head strides
  __nv_bfloat16* out;
  int64_t ot, oh;
  int64_t total;   // rows of q and out
  int group;       // query heads per kv head
  float scale_log2;
  float* parts;    // [2 gridDim][rows x d + 2 rows]: O, m, l
  int32_t* joins;  // [gridDim][8]: the unit that began in an earlier run and ends in this one
};

// rows r0 .. of a unit; number of key blocks they see
struct Seq {
  int n, len, rows, nrb;
};
template <int RB>
__device__ __forceinline__ Seq sequence(const Params& P, int b) {
  Seq s;
  const int c0 = P.p.cu[b], c1 = P.p.cu[b + 1];
  s.n = (c0 >= 0 && c1 > c0 && c1 <= P.total) ? c1 - c0 : 0;
  s.len = length_of(P.p, b);
  s.rows = s.n * P.group;
  s.nrb = (s.rows + RB - 1) / RB;
  return s;
}
template <int RB>
__device__ __forceinline__ int key_blocks(const Params& P, const Seq& s, int rb) {
  const int last = min(s.n - 1, ((rb + 1) * RB - 1) / P.group);  // the row block's last token
  const int seen = s.len - s.n + last + 1;
  return seen <= 0 ? 0 : (seen + BLOCK - 1) / BLOCK;
}
template <int RB>
__device__ __forceinline__ int64_t sequence_blocks(const Params& P, int b) {
  const Seq s = sequence<RB>(P, b);
  int64_t sum = 0;
  for (int rb = 0; rb < s.nrb; ++rb) sum += key_blocks<RB>(P, s, rb);
  return sum * P.p.kv_heads;
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

template <int NG>
__host__ __device__ constexpr int stage_bytes() { return 2 * block_bytes(NG); }
template <int NG, int NB>
__host__ __device__ constexpr int stages() { return NB == 2 ? 6 : 4; }
// shared memory: the warps' rings | their O and (m, l) at a unit's end | mbarriers
template <int NG, int NB>
__host__ __device__ constexpr int smem_bytes() {
  return WARPS * stages<NG, NB>() * stage_bytes<NG>() + WARPS * (8 * NB) * (64 * NG + 2) * 4 +
         WARPS * stages<NG, NB>() * 8;
}

template <int NG, int NB>
__global__ void __launch_bounds__(THREADS, NB == 1 ? 2 : 1) paged_attention_kernel(Params P) {
  constexpr int RB = 8 * NB, D = 64 * NG, S = stages<NG, NB>();
  constexpr int UNIT = block_bytes(NG), STAGE = stage_bytes<NG>();
  extern __shared__ __align__(128) unsigned char smem[];
  float* s_o = reinterpret_cast<float*>(smem + WARPS * S * STAGE);  // [WARPS][RB][D]
  float* s_m = s_o + WARPS * RB * D;                                // [WARPS][RB]
  float* s_l = s_m + WARPS * RB;
  uint64_t* s_bar = reinterpret_cast<uint64_t*>(s_l + WARPS * RB);  // [WARPS][S]
  __shared__ int64_t s_scan[WARPS + 1];
  __shared__ int s_start_b;
  __shared__ int64_t s_start_at;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const Pages& p = P.p;
  if (tid < WARPS * S) {
    mbar_init(smem_addr(&s_bar[tid]), 1);
    fence_barrier_init();
  }
  grid_dependency_wait();
  allow_dependent_launch();

  // ---- this CTA's run of key blocks
  auto scan = [&](int64_t mine, int64_t& before) {  // exclusive prefix over the CTA's threads; returns the sum
    int64_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    int64_t base = 0, all = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) base += s_scan[w];
      all += s_scan[w];
    }
    before = base + x - mine;
    return all;
  };
  int64_t total = 0, mine = 0, before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
    mine = b0 + tid < p.batch ? sequence_blocks<RB>(P, b0 + tid) : 0;
    total += scan(mine, before);
  }
  // at least one block per warp, so that short problems have few partials to join
  const int64_t per = std::max<int64_t>((total + gridDim.x - 1) / gridDim.x, WARPS);
  const int64_t begin = blockIdx.x * per, end = std::min<int64_t>(total, begin + per);
  if (tid == 0) s_start_b = -1;
  int64_t base = 0;
  for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
    if (p.batch > THREADS) mine = b0 + tid < p.batch ? sequence_blocks<RB>(P, b0 + tid) : 0;
    const int64_t sum = p.batch > THREADS ? scan(mine, before) : total;
    if (begin < end && begin >= base + before && begin < base + before + mine) {
      s_start_b = b0 + tid;
      s_start_at = base + before;
    }
    base += sum;
  }
  int32_t* join = P.joins + blockIdx.x * 8;
  if (tid == 0) join[0] = 0;
  // rows that see no key are zero
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const Seq s = sequence<RB>(P, b);
    const int none = min(s.n, s.n - s.len);  // tokens at positions below zero
    for (int64_t i = tid; i < static_cast<int64_t>(std::max(none, 0)) * P.group * p.kv_heads * D; i += THREADS) {
      const int c = i % D;
      const int64_t row = i / D;
      const int head = row % (P.group * p.kv_heads);
      P.out[(p.cu[b] + row / (P.group * p.kv_heads)) * P.ot + head * P.oh + c] = __float2bfloat16_rn(0.0f);
    }
  }
  __syncthreads();
  if (begin >= end || s_start_b < 0) return;

  // ---- the run's segments, one per unit
  int b = s_start_b, head, rb;
  Seq sq = sequence<RB>(P, b);
  int64_t at = begin - s_start_at;  // within the sequence, then within the unit
  {
    int64_t per_head = 0;
    for (int i = 0; i < sq.nrb; ++i) per_head += key_blocks<RB>(P, sq, i);
    head = static_cast<int>(at / per_head);
    at -= head * per_head;
    rb = 0;
    while (at >= key_blocks<RB>(P, sq, rb)) at -= key_blocks<RB>(P, sq, rb++);
  }
  int64_t left = end - begin;
  unsigned char* ring = smem + warp * S * STAGE;
  uint64_t* bars = s_bar + warp * S;
  int issued = 0, used = 0;  // copies of this warp's ring
  int64_t first_at = begin - at;  // the current unit's first block, in the order of all blocks
  bool ok = true;

  while (left > 0) {
    const int unit_blocks = key_blocks<RB>(P, sq, rb);
    const int k0 = static_cast<int>(at), count = static_cast<int>(std::min<int64_t>(left, unit_blocks - at));
    const int kend = k0 + count;
    // this warp's blocks: k0 + warp, + WARPS, ...; lane l looks up the page of the l-th (of 32 at a time)
    const int mine_blocks = count > warp ? (count - warp + WARPS - 1) / WARPS : 0;
    int64_t page_off = -1;
    auto look_up = [&](int from) {
      const int i = from + lane;
      page_off = -1;
      if (i < mine_blocks) {
        const int pos = (k0 + warp + i * WARPS) * BLOCK;
        const int64_t page = page_of(p, b, pos);
        if (page >= 0) page_off = page * p.page_stride + block_in_page<NG>(p, 0, head, pos);
      }
    };
    const int64_t v_off = static_cast<int64_t>(p.kv_heads) * (1 << (p.page_shift - 4)) * UNIT;
    auto issue = [&](int64_t off) {  // warp-uniform off
      if (off < 0) return;
      if (lane == 0) {
        const uint32_t bar = smem_addr(&bars[issued % S]);
        const uint32_t dst = smem_addr(ring + (issued % S) * STAGE);
        mbar_arrive_expect_tx(bar, STAGE);
        bulk_copy(dst, p.base + off, UNIT, bar);
        bulk_copy(dst + UNIT, p.base + off + v_off, UNIT, bar);
      }
      ++issued;
    };
    look_up(0);
    int64_t next_off = -1;  // pages of the window after this one are looked up when it starts
    // the fragments of this unit's rows: query head head * G + r % G of token r / G
    uint32_t qf[NB][NG][4][2];
    int lim[NB][2];
    const int rows = min(RB, sq.rows - rb * RB);
    const int nbs = (rows + 7) / 8;
    const int c0 = p.cu[b];
    for (int i = 0; i < min(mine_blocks, S - 1); ++i) issue(__shfl_sync(0xffffffffu, page_off, i));
    int lim_min = 0x7fffffff;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = rb * RB + nb * 8 + g;  // the B fragment's column
      const bool live = nb * 8 + g < rows;
      const __nv_bfloat16* row =
          P.q + static_cast<int64_t>(c0 + (live ? r / P.group : 0)) * P.qt + (head * P.group + (live ? r % P.group : 0)) * P.qh;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        uint32_t w[8];  // channels 16 t .. 16 t + 15 of the group
        const uint4* src = reinterpret_cast<const uint4*>(row + 64 * gr + 16 * t);
        const uint4 u0 = live ? src[0] : make_uint4(0, 0, 0, 0), u1 = live ? src[1] : make_uint4(0, 0, 0, 0);
        w[0] = u0.x; w[1] = u0.y; w[2] = u0.z; w[3] = u0.w;
        w[4] = u1.x; w[5] = u1.y; w[6] = u1.z; w[7] = u1.w;
        // step ks: channels 16 t + ks and + 4 (word 2 t's pair ks), then + 8 and + 12
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const uint32_t sel = (ks & 1) ? 0x7632 : 0x5410;
          qf[nb][gr][ks][0] = __byte_perm(w[ks >> 1], w[2 + (ks >> 1)], sel);
          qf[nb][gr][ks][1] = __byte_perm(w[4 + (ks >> 1)], w[6 + (ks >> 1)], sel);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // the C fragments' columns: row 2 t + h
        const int rr = nb * 8 + 2 * t + h;
        lim[nb][h] = rr < rows ? sq.len - sq.n + (rb * RB + rr) / P.group : 0x7fffffff;
        lim_min = min(lim_min, lim[nb][h]);
      }
    }
    lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 1));
    lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, 2));

    float o[NB][NG * 4][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < NG * 4; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nb][i][c] = 0.0f;
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.0f;
    }

    for (int i = 0; i < mine_blocks; ++i) {
      if ((i & 31) == 0 && i > 0) look_up(i);  // this window's pages
      const int64_t off = __shfl_sync(0xffffffffu, page_off, i & 31);
      // the block S - 1 ahead: its page is in this window or read here for the next one
      const int ahead = i + S - 1;
      if (ahead < mine_blocks) {
        if ((ahead >> 5) == (i >> 5)) {
          next_off = __shfl_sync(0xffffffffu, page_off, ahead & 31);
        } else {
          const int pos = (k0 + warp + ahead * WARPS) * BLOCK;
          const int64_t page = page_of(p, b, pos);
          next_off = page < 0 ? -1 : page * p.page_stride + block_in_page<NG>(p, 0, head, pos);
        }
        issue(next_off);
      }
      if (off < 0) continue;  // no such page: its keys are left out
      if (!mbar_wait_warp(smem_addr(&bars[used % S]), (used / S) & 1, 42, used)) {
        ok = false;
        break;
      }
      const unsigned char* kb = ring + (used % S) * STAGE;
      const unsigned char* vb = kb + UNIT;
      ++used;

      // ---- S^T = K Q^T
      float acc[NB][NG][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[nb][gr][c] = 0.0f;
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
            expand_word(kw[h][2 * gr + wd], exponent_pair(ke[h][gr], (7 - 4 * t - 2 * wd) & 31), a[h][wd]);
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const uint32_t fa[4] = {a[0][0][st], a[1][0][st], a[0][1][st], a[1][1][st]};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            if (nb < nbs) mma_bf16_16816(acc[nb][gr], fa, qf[nb][gr][st][0], qf[nb][gr][st][1]);
        }
      }
      // ---- softmax; c of the fragment: key g + 8 (c / 2), row 2 t + c % 2
      const int key0 = (k0 + warp + i * WARPS) * BLOCK + g;
      const bool edge = key0 - g + BLOCK - 1 > lim_min;
      uint32_t pf[NB][NG][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (nb >= nbs) continue;
        float s[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[c] = __fmul_rn(acc[nb][0][c], ks[c >> 1][0]);
          if constexpr (NG == 2) s[c] = __fmaf_rn(acc[nb][1][c], ks[c >> 1][1], s[c]);
          if (edge && key0 + 8 * (c >> 1) > lim[nb][c & 1]) s[c] = -INFINITY;
        }
        const float top0 = __fmul_rn(fmaxf(s[0], s[2]), P.scale_log2), top1 = __fmul_rn(fmaxf(s[1], s[3]), P.scale_log2);
        if (__any_sync(0xffffffffu, top0 > m[nb][0] + RAISE || top1 > m[nb][1] + RAISE)) {
          float n0 = top0, n1 = top1;
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
          }
          n0 = fmaxf(n0, m[nb][0]);
          n1 = fmaxf(n1, m[nb][1]);
          const float a0 = m[nb][0] == -INFINITY ? 0.0f : ex2(m[nb][0] - n0);
          const float a1 = m[nb][1] == -INFINITY ? 0.0f : ex2(m[nb][1] - n1);
          m[nb][0] = n0;
          m[nb][1] = n1;
          l[nb][0] *= a0;
          l[nb][1] *= a1;
#pragma unroll
          for (int j = 0; j < NG * 4; ++j) {
            o[nb][j][0] *= a0;
            o[nb][j][1] *= a1;
            o[nb][j][2] *= a0;
            o[nb][j][3] *= a1;
          }
        }
        const float u0 = m[nb][0] == -INFINITY ? 0.0f : m[nb][0], u1 = m[nb][1] == -INFINITY ? 0.0f : m[nb][1];
        float e[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) e[c] = ex2(__fmaf_rn(s[c], P.scale_log2, (c & 1) ? -u1 : -u0));
        l[nb][0] += e[0] + e[2];
        l[nb][1] += e[1] + e[3];
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          pf[nb][gr][0] = transpose8x8(pack_bf16(e[0] * vs[0][gr], e[1] * vs[0][gr]));
          pf[nb][gr][1] = transpose8x8(pack_bf16(e[2] * vs[1][gr], e[3] * vs[1][gr]));
        }
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
            expand_word(vw[h][2 * gr + qd], exponent_pair(ve[h][2 * gr + qd], (7 - 2 * g) & 31), a[h][qd]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t fa[4] = {a[0][0][j], a[0][1][j], a[1][0][j], a[1][1][j]};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
            if (nb < nbs) mma_bf16_16816(o[nb][gr * 4 + j], fa, pf[nb][gr][0], pf[nb][gr][1]);
        }
      }
      __syncwarp();  // the stage may be refilled: every lane has read it
    }

    // ---- the warps' results meet
    __syncthreads();  // the previous unit's s_o has been read
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if (nb >= nbs) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nb][h] += __shfl_xor_sync(0xffffffffu, l[nb][h], x);
        const int r = nb * 8 + 2 * t + h;
        float* dst = s_o + (warp * RB + r) * D + 8 * g;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          *reinterpret_cast<float4*>(dst + 64 * gr) =
              make_float4(o[nb][4 * gr][h], o[nb][4 * gr + 1][h], o[nb][4 * gr + 2][h], o[nb][4 * gr + 3][h]);
          *reinterpret_cast<float4*>(dst + 64 * gr + 4) =
              make_float4(o[nb][4 * gr][2 + h], o[nb][4 * gr + 1][2 + h], o[nb][4 * gr + 2][2 + h], o[nb][4 * gr + 3][2 + h]);
        }
        if (g == 0) {
          s_m[warp * RB + r] = m[nb][h];
          s_l[warp * RB + r] = l[nb][h];
        }
      }
    }
    const bool whole = k0 == 0 && kend == unit_blocks;
    if (!__syncthreads_and(ok)) break;  // a copy never landed: recorded; this unit is not written
    float* part = P.parts + (2 * static_cast<int64_t>(blockIdx.x) + (kend < unit_blocks && k0 == 0)) * (RB * D + 2 * RB);
    for (int i = tid; i < rows * (D / 4); i += THREADS) {
      const int r = i / (D / 4), c = i % (D / 4) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_m[w * RB + r]);
      const float use = top == -INFINITY ? 0.0f : top;
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float den = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = ex2(s_m[w * RB + r] - use);
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * RB + r) * D + c);
        sum.x += f * v.x;
        sum.y += f * v.y;
        sum.z += f * v.z;
        sum.w += f * v.w;
        den += f * s_l[w * RB + r];
      }
      if (whole) {
        const int row = rb * RB + r;
        const float inv = den > 0.0f ? __fdiv_rn(1.0f, den) : (den == 0.0f ? 0.0f : den);  // NaN stays
        uint2 w2;
        w2.x = pack_bf16(sum.x * inv, sum.y * inv);
        w2.y = pack_bf16(sum.z * inv, sum.w * inv);
        *reinterpret_cast<uint2*>(P.out + static_cast<int64_t>(c0 + row / P.group) * P.ot +
                                  (head * P.group + row % P.group) * P.oh + c) = w2;
      } else {
        *reinterpret_cast<float4*>(part + r * D + c) = sum;
        if (c == 0) {
          part[RB * D + r] = top;
          part[RB * D + RB + r] = den;
        }
      }
    }
    if (!whole && k0 > 0 && kend == unit_blocks && tid == 0) {
      join[1] = c0;
      join[2] = head;
      join[3] = rb;
      join[4] = rows;
      join[5] = static_cast<int>(first_at / per);  // the run that holds the unit's first block
      join[0] = 1;
    }
    // ---- the next unit with keys
    left -= count;
    if (left > 0) {
      first_at += unit_blocks;
      at = 0;
      do {
        if (++rb >= sq.nrb) {
          rb = 0;
          if (++head >= p.kv_heads || sq.nrb == 0) {
            head = 0;
            do sq = sequence<RB>(P, ++b);
            while (sq.nrb == 0 && b + 1 < p.batch);
          }
        }
      } while (key_blocks<RB>(P, sq, rb) == 0);
    }
  }
  // a timeout leaves copies in flight: wait for them (bounded) before the CTA's memory goes
  if (lane == 0)
    for (; used < issued; ++used)
      if (!mbar_wait(smem_addr(&bars[used % S]), (used / S) & 1)) break;
}

// Joins the partials of the unit that ended in run blockIdx.x: its first run's (slot 2 c + 1),
// then those of the runs up to this one (slot 2 c). One warp per row.
template <int D, int RB>
__global__ void __launch_bounds__(128) paged_combine_kernel(Params P) {
  grid_dependency_wait();
  allow_dependent_launch();
  const int32_t* join = P.joins + blockIdx.x * 8;
  if (join[0] == 0) return;
  const int r = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= join[4]) return;
  const int first = join[5], last = blockIdx.x;
  constexpr int64_t SIZE = RB * D + 2 * RB;
  auto part = [&](int c) { return P.parts + (2 * static_cast<int64_t>(c) + (c == first)) * SIZE; };
  float top = -INFINITY;
  for (int c = first + lane; c <= last; c += 32) top = fmaxf(top, part(c)[RB * D + r]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  const float use = top == -INFINITY ? 0.0f : top;
  constexpr int W = D / 32;  // channels per lane
  float sum[W], den = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) sum[i] = 0.0f;
#pragma unroll 4
  for (int c = first; c <= last; ++c) {
    const float* src = part(c);
    const float f = ex2(src[RB * D + r] - use);
    den += f * src[RB * D + RB + r];
#pragma unroll
    for (int i = 0; i < W; ++i) sum[i] += f * src[r * D + lane * W + i];
  }
  const float inv = den > 0.0f ? __fdiv_rn(1.0f, den) : (den == 0.0f ? 0.0f : den);
  const int row = join[3] * RB + r;
  __nv_bfloat16* dst = P.out + static_cast<int64_t>(join[1] + row / P.group) * P.ot +
                       (join[2] * P.group + row % P.group) * P.oh + lane * W;
#pragma unroll
  for (int i = 0; i < W; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf16(sum[i] * inv, sum[i + 1] * inv);
}

constexpr int JOIN_BYTES_PER_CTA = 32;
inline int ctas(int nb) { return num_sms() * (nb == 1 ? 2 : 1); }
inline int n_blocks(int64_t max_rows) { return max_rows <= 8 ? 1 : max_rows <= 16 ? 2 : 4; }
inline size_t workspace(int nb, int d) {
  const int64_t rows = 8 * nb;
  return static_cast<size_t>(ctas(nb)) * (JOIN_BYTES_PER_CTA + 2 * (rows * d + 2 * rows) * 4);
}

template <int NG, int NB>
static int launch(Params& P, void* ws, void* stream) {
  const int grid = ctas(NB);
  P.joins = static_cast<int32_t*>(ws);
  P.parts = reinterpret_cast<float*>(static_cast<char*>(ws) + static_cast<size_t>(grid) * JOIN_BYTES_PER_CTA);
  constexpr int bytes = smem_bytes<NG, NB>();
  auto kern = paged_attention_kernel<NG, NB>;
  FAQ_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(grid)), THREADS, bytes, stream, P));
  FAQ_CUDA(launch_early(paged_combine_kernel<64 * NG, 8 * NB>, dim3(static_cast<unsigned>(grid), 2 * NB), 128, 0, stream, P));
  return launch_status("paged attention kernels");
}

}  // namespace pat
}  // namespace faq

extern "C" size_t faq_hif4_paged_attention_workspace_bytes(int64_t heads, int64_t kv_heads, int64_t max_new, int d) {
  using namespace faq::pat;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_new < 0 || (d != 64 && d != 128)) return 0;
  return workspace(n_blocks(heads / kv_heads * max_new), d);
}

extern "C" int faq_hif4_paged_attention(const void* q, int64_t total, int64_t heads, int64_t q_token_stride,
                                        int64_t q_head_stride, const void* pages, int64_t num_pages,
                                        int64_t page_stride, int page_size, int64_t kv_heads, int d,
                                        const int32_t* table, int64_t table_ld, int64_t table_cols, const int32_t* cu,
                                        const int32_t* lens, int64_t batch, int64_t max_new, int64_t max_len, float scale,
                                        void* out, int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  using namespace faq;
  using namespace faq::pat;
  Params P;
  const int rc = make_pages(P.p, pages, num_pages, page_stride, page_size, kv_heads, d, table, table_ld, table_cols, cu,
                            lens, batch);
  if (rc) return rc;
  FAQ_CHECK_ARG(heads > 0 && heads % kv_heads == 0, "query heads must be divisible by key/value heads");
  FAQ_CHECK_ARG(total >= 0 && max_new >= 0 && max_len >= 0 && total * heads < (int64_t(1) << 31), "bad token count");
  if (total == 0) return FAQ_OK;
  FAQ_CHECK_ARG(q && out, "null pointer");
  FAQ_CHECK_ARG(scale > 0.0f && scale < 3.0e38f, "scale must be positive and finite");
  FAQ_CHECK_ARG(aligned16(q) && aligned16(out) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0 &&
                    out_token_stride % 8 == 0 && out_head_stride % 8 == 0,
                "q and out must be 16-byte aligned with strides multiple of 8");
  const int nb = n_blocks(heads / kv_heads * max_new);
  FAQ_CHECK_ARG(workspace != nullptr && aligned16(workspace), "workspace must be a 16-byte aligned device buffer");
  FAQ_CHECK_ARG(workspace_bytes >= pat::workspace(nb, d),
                "workspace too small: faq_hif4_paged_attention_workspace_bytes() bytes needed");
  P.q = static_cast<const __nv_bfloat16*>(q);
  P.qt = q_token_stride;
  P.qh = q_head_stride;
  P.out = static_cast<__nv_bfloat16*>(out);
  P.ot = out_token_stride;
  P.oh = out_head_stride;
  P.total = total;
  P.group = static_cast<int>(heads / kv_heads);
  P.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  if (d == 64) return nb == 1 ? launch<1, 1>(P, workspace, stream) : nb == 2 ? launch<1, 2>(P, workspace, stream) : launch<1, 4>(P, workspace, stream);
  return nb == 1 ? launch<2, 1>(P, workspace, stream) : nb == 2 ? launch<2, 2>(P, workspace, stream) : launch<2, 4>(P, workspace, stream);
}
