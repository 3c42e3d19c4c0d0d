// K13 -- attention of each new token over the pages listed for it:
//
//   O = sum_k p_k V[k] / sum_k p_k,  p_k = exp(scale q . K[k]),  k in the listed pages, k <= position
//
// per token, kv head and its G = heads / kv_heads query heads, which share a list. A unit is
// (token, kv head, 8 query heads). The arithmetic of a block of 16 tokens is K9's kernel of few rows
// (paged_attention.cu): codes to bf16 fragments in registers, S^T = K Q^T and O^T = V^T P^T on
// mma.sync, one reference maximum per row and warp, P rounded to bf16, the type of the products with V, after its product
// with V's scale: at most 2^-8 of a term, as in the dense kernels. Sums are fp32; that rounding and the output's own put
// the output 0.001 to 0.003 of its norm from one whose P stays in fp32. What differs is where the blocks come from: a warp
// looks up 32 of its blocks at once (list entry, table entry, address), drops those that are not there or lie behind the
// token, and streams the rest through a ring of bulk copies.
//
// A column counts once: where a list is not ascending, a warp first goes through it once, 32 entries at a time, with a
// bit per column and one per entry that is the first of its column (hence a list's most entries). 32 entries cost 0.8 us,
// 1024 (pages of 16) 13.5 beside 27, 32768 420 beside 650.
//
// Work split: a unit's blocks are dealt out to the warps of a cluster of 1, 2, 4 or 8 CTAs, as many as fill the
// SMs once; the CTAs' results meet through distributed shared memory, so there is no second
// kernel and no workspace. The order of every sum is fixed by the list and the cluster's size.
//
// Measured (one B200, 32 query heads on 8 kv heads of 128, one new token): 32 pages of 64 of a context
// of 32768 in 8.3 us, 64 pages of 16 of 32 sequences of 1 .. 16000 tokens in 16.6 us. The first is a chain of
// loads (cu and lens, the list, the table, the pages), two blocks per warp and the two joins; the second
// some 10700 blocks at 190 cycles of an SM each (see paged_attention.cu: 118 of issue), as 256 CTAs
// of unequal length in one wave; clusters of two there took 20.3 us, of four 31.2. 128 such sequences of 2000 tokens
// take 54 us, with four warps to a unit.
#include "kv_pages.cuh"

namespace faq {
namespace spa {

using namespace kvp;
using pat::ex2;
using pat::LIFT;
using pat::LOWEST;
using pat::pack_bf16;
using pat::RAISE;
using pat::transpose8x8;

constexpr int SM_WARPS = 16;  // in CTAs of 4 or 8: 128 registers a thread
constexpr int S = 4;   // blocks in flight per warp
constexpr int MAX_COUNT = 32768;  // entries of a list, as many as the selection has columns
constexpr int RANGE = 131072;     // columns whose bits are held at once, where the rings will be

// shared memory: the warps' rings, then in their place the warps' O (rows padded) | the CTA's O | (m, l) of
// warps and CTA | the ring slots' first keys | mbarriers | the entries that count, a bit each
template <int NG, int W>
struct Smem {
  static constexpr int old = 64 * NG + 8;  // floats of an O row
  static constexpr int stage = 2 * block_bytes(NG);
  static constexpr int rings = W * S * stage;
  static constexpr int warp_o = W * RB * old * 4;
  static constexpr int o = rings > warp_o ? rings : warp_o;
  static constexpr int m = o + RB * 64 * NG * 4;
  static constexpr int l = m + (W + 1) * RB * 4;
  static constexpr int key = l + (W + 1) * RB * 4;
  static constexpr int bar = key + W * S * 4;
  static constexpr int counts = bar + W * S * 8;
  static constexpr int bytes(int entries) { return counts + (entries + 31) / 32 * 4; }
  static_assert(rings >= RANGE / 8, "the columns' bits");
};

template <int NG, int W>
__global__ void __launch_bounds__(32 * W, SM_WARPS / W) sparse_attention_kernel(Params P, int split) {
  using L = Smem<NG, W>;
  constexpr int THREADS = 32 * W, D = 64 * NG, OLD = L::old, UNIT = block_bytes(NG), STAGE = L::stage;
  extern __shared__ __align__(128) unsigned char smem[];
  float* s_o = reinterpret_cast<float*>(smem);            // [W][RB][OLD], over the rings
  float* s_part = reinterpret_cast<float*>(smem + L::o);  // [RB][D]
  float* s_m = reinterpret_cast<float*>(smem + L::m);     // [W + 1][RB], the CTA's last
  float* s_l = reinterpret_cast<float*>(smem + L::l);
  int* s_key = reinterpret_cast<int*>(smem + L::key);     // [W][S]
  uint64_t* s_bar = reinterpret_cast<uint64_t*>(smem + L::bar);
  uint32_t* s_counts = reinterpret_cast<uint32_t*>(smem + L::counts);
  __shared__ int s_ok;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const Pages& p = P.p;
  if (tid < W * S) {
    mbar_init(smem_addr(&s_bar[tid]), 1);
    fence_barrier_init();
  }
  __syncthreads();
  grid_dependency_wait();
  allow_dependent_launch();

  const int rank = static_cast<int>(blockIdx.x % split);
  int64_t unit = blockIdx.x / split;
  const int pass = static_cast<int>(unit % P.passes);
  unit /= P.passes;
  const int head = static_cast<int>(unit % p.kv_heads);
  const int64_t token = unit / p.kv_heads;
  const int32_t* list = P.list + (token * p.kv_heads + head) * P.count;
  // whether the columns of the list are in ascending order, hence none is there twice
  bool ascending = true;
  for (int j = lane; j < P.count; j += 32) {
    const int before = j > 0 ? list[j - 1] : 0, col = list[j];
    ascending = ascending && (col < 0 || j == 0 || (before >= 0 && before < col));
  }
  ascending = __all_sync(0xffffffffu, ascending);  // in every warp alike
  int b;
  int64_t place;
  if (blockIdx.x == 0) check_batch(p, P.total, tid, THREADS);
  if (!find_token(p, token, P.total, b, place)) return;  // the whole cluster
  const int pos = static_cast<int>(max(place, static_cast<int64_t>(-1)));  // below a length
  const int rows = min(RB, P.group - pass * RB);
  if (!ascending) {  // the entries that count: of each column the first
    const int columns = pos < 0 ? 0 : min((pos >> p.page_shift) + 1, p.table_cols);
    uint32_t* seen = reinterpret_cast<uint32_t*>(smem);
    for (int c0 = 0; c0 < columns; c0 += RANGE) {
      const int n = min(RANGE, columns - c0);
      for (int i = tid; i < (n + 31) / 32; i += THREADS) seen[i] = 0;
      __syncthreads();
      if (warp == 0) {
        for (int j0 = 0; j0 < P.count; j0 += 32) {
          const int col = j0 + lane < P.count ? list[j0 + lane] : -1;
          const bool in = col >= c0 && col < c0 + n;
          const int at = in ? col - c0 : 0;
          const uint32_t alike = __match_any_sync(0xffffffffu, in ? col : -1);
          const bool fresh = in && __ffs(alike) - 1 == lane && !(seen[at >> 5] >> (at & 31) & 1);
          __syncwarp();
          if (fresh) atomicOr(&seen[at >> 5], 1u << (at & 31));
          const uint32_t bits = __ballot_sync(0xffffffffu, fresh || col >= p.table_cols);  // those are looked up, to be reported
          if (lane == 0) s_counts[j0 >> 5] = c0 > 0 ? s_counts[j0 >> 5] | bits : bits;
          __syncwarp();
        }
      }
      __syncthreads();
    }
    fence_proxy_async_smem();  // the rings' copies come through the async proxy
    __syncthreads();
  }

  // ---- the warp's blocks: numbers warp + W rank + W split i of the count << block_shift listed ones
  const int block_shift = p.page_shift - 4;
  const int blocks = P.count << block_shift;
  const int stride = W * split, begin = warp + W * rank;
  const int mine = blocks > begin ? (blocks - begin + stride - 1) / stride : 0;
  unsigned char* ring = smem + warp * S * STAGE;
  uint64_t* bars = s_bar + warp * S;
  int* keys = s_key + warp * S;
  int issued = 0, used = 0;
  int window = 0;   // the next blocks to look up
  uint32_t found = 0;   // those of the window looked up last that are still to be copied
  const uint8_t* address = nullptr;
  int first_of = 0;     // lane l: the first key of the window's l-th block
  const int64_t v_dist = (static_cast<int64_t>(p.kv_heads) << block_shift) * UNIT;  // from a page's K to its V
  auto look_up = [&]() {
    const int i = window + lane;
    bool has = false;
    if (i < mine) {
      const int block = begin + i * stride;
      const int entry = block >> block_shift, col = list[entry];
      const int64_t key = (static_cast<int64_t>(col) << p.page_shift) + ((block & ((1 << block_shift) - 1)) << 4);
      if (col >= 0 && key <= pos && (ascending || (s_counts[entry >> 5] >> (entry & 31) & 1))) {
        const int64_t page = page_of(p, b, static_cast<int>(key));
        has = page >= 0;
        first_of = static_cast<int>(key);
        address = p.base + (has ? page : 0) * p.page_stride + block_in_page<NG>(p, 0, head, first_of);
      }
    }
    found = __ballot_sync(0xffffffffu, has);
    window += 32;
  };
  auto copy_next = [&]() -> bool {
    while (found == 0 && window < mine) look_up();
    if (found == 0) return false;
    const int src = __ffs(found) - 1;
    found &= found - 1;
    const int slot = issued % S;
    if (lane == src) {
      keys[slot] = first_of;
      const uint32_t bar = smem_addr(&bars[slot]), dst = smem_addr(ring + slot * STAGE);
      mbar_arrive_expect_tx(bar, STAGE);
      pat::bulk_copy(dst, address, UNIT, bar);
      pat::bulk_copy(dst + UNIT, address + v_dist, UNIT, bar);
    }
    ++issued;
    return true;
  };
#pragma unroll 1
  for (int i = 0; i < S; ++i)
    if (!copy_next()) break;

  // ---- Q's fragments: column g is query head g of the unit, lane t holds channels 16 t .. of each group
  uint4 q[NG * 2];
  {
    const bool live = g < rows;
    const __nv_bfloat16* row = P.q + token * P.qt + (static_cast<int64_t>(head) * P.group + pass * RB + (live ? g : 0)) * P.qh;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      const uint4* src = reinterpret_cast<const uint4*>(row + 64 * gr + 16 * t);
      const uint4 u0 = live ? src[0] : make_uint4(0, 0, 0, 0), u1 = live ? src[1] : make_uint4(0, 0, 0, 0);
      const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        q[gr * 2 + i] = make_uint4(__byte_perm(w[i], w[2 + i], 0x5410), __byte_perm(w[4 + i], w[6 + i], 0x5410),
                                   __byte_perm(w[i], w[2 + i], 0x7632), __byte_perm(w[4 + i], w[6 + i], 0x7632));
    }
  }
  const Expand expand;
  float o[NG * 4][4], m[2] = {LOWEST, LOWEST}, l[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < NG * 4; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[i][c] = 0.0f;
  bool ok = true;
  while (used < issued) {
    const int slot = used % S;
    if (!mbar_wait_warp(smem_addr(&bars[slot]), (used / S) & 1, 43, used)) {
      ok = false;
      break;
    }
    const unsigned char* kb = ring + slot * STAGE;
    const unsigned char* vb = kb + UNIT;
    const int first_key = keys[slot];
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
    float s[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      s[c] = __fmul_rn(acc[0][c], ks[c >> 1][0]);
      if constexpr (NG == 2) s[c] = __fmaf_rn(acc[1][c], ks[c >> 1][1], s[c]);
    }
    if (first_key + BLOCK - 1 > pos) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (first_key + g + 8 * (c >> 1) > pos) s[c] = -INFINITY;
    }
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
    uint32_t pf[NG][2];
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
        const uint4 x = *reinterpret_cast<const uint4*>(vb + exp_offset(NG) + 16 * pr);
        ve[h][0] = x.x; ve[h][1] = x.y; ve[h][2] = x.z; ve[h][3] = x.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(vb + 64 * pr + 8 * (g ^ (2 * t)));
        vw[h][0] = u.x; vw[h][1] = u.y;
        const uint2 x = *reinterpret_cast<const uint2*>(vb + exp_offset(NG) + 8 * pr);
        ve[h][0] = x.x; ve[h][1] = x.y;
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
    copy_next();
  }
  // a timeout leaves copies in flight: wait for them (bounded) before their memory is used again
  if (lane == 0)
    for (; used < issued; ++used)
      if (!mbar_wait(smem_addr(&bars[used % S]), (used / S) & 1)) break;

  // ---- the warps' results meet
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int y = 4; y < 32; y <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], y);
  const bool cta_ok = __syncthreads_and(ok);  // the rings are free
  if (tid == 0) s_ok = cta_ok;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = 2 * t + h;
    if (r < rows) {
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
  __syncthreads();
  auto write = [&](int r, int c, const float4& sum, float den) {
    const float inv = den > 0.0f ? __fdiv_rn(1.0f, den) : (den == 0.0f ? 0.0f : den);  // NaN stays
    uint2 w2;
    w2.x = pack_bf16(sum.x * inv, sum.y * inv);
    w2.y = pack_bf16(sum.z * inv, sum.w * inv);
    *reinterpret_cast<uint2*>(P.out + token * P.ot + (static_cast<int64_t>(head) * P.group + pass * RB + r) * P.oh + c) = w2;
  };
  for (int i = tid; i < rows * (D / 4); i += THREADS) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float top = LOWEST;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w * RB + r]);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float den = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = ex2(0.5f * (s_m[w * RB + r] - top));
      const float4 v = *reinterpret_cast<const float4*>(s_o + (w * RB + r) * OLD + c);
      sum.x += f * v.x * f;
      sum.y += f * v.y * f;
      sum.z += f * v.z * f;
      sum.w += f * v.w * f;
      den += f * s_l[w * RB + r] * f;
    }
    if (split == 1) {
      if (cta_ok) write(r, c, sum, den);
    } else {
      *reinterpret_cast<float4*>(s_part + r * D + c) = sum;
      if (c == 0) {
        s_m[W * RB + r] = top;
        s_l[W * RB + r] = den;
      }
    }
  }
  if (split == 1) return;

  // ---- the CTAs' results meet: each takes its share of the unit's values
  cluster_sync();
  bool all = true;
  for (int k = 0; k < split; ++k) {
    all = all && cluster_load_int(mapa_shared(smem_addr(&s_ok), k)) != 0;
  }
  for (int i = tid + THREADS * rank; i < rows * (D / 4); i += THREADS * split) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float top = LOWEST;
    for (int k = 0; k < split; ++k) top = fmaxf(top, cluster_load(mapa_shared(smem_addr(s_m + W * RB + r), k)));
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float den = 0.0f;
    for (int k = 0; k < split; ++k) {
      const float f = ex2(0.5f * (cluster_load(mapa_shared(smem_addr(s_m + W * RB + r), k)) - top));
      const float4 v = cluster_load4(mapa_shared(smem_addr(s_part + r * D + c), k));
      sum.x += f * v.x * f;
      sum.y += f * v.y * f;
      sum.z += f * v.z * f;
      sum.w += f * v.w * f;
      den += f * cluster_load(mapa_shared(smem_addr(s_l + W * RB + r), k)) * f;
    }
    if (all) write(r, c, sum, den);
  }
  cluster_sync();  // the others have read this CTA's part
}

template <int NG, int W>
static int launch(const Params& P, int split, void* stream) {
  auto kern = sparse_attention_kernel<NG, W>;
  static std::atomic<uint64_t> set{0};  // devices on which the kernel's shared memory is set
  const int rc = allow_smem(reinterpret_cast<const void*>(kern), Smem<NG, W>::bytes(MAX_COUNT), set);
  if (rc) return rc;
  FAQ_CUDA(launch_clusters(kern, P.total * P.p.kv_heads * P.passes * split, 32 * W, Smem<NG, W>::bytes(P.count), split, stream, P,
                           split));
  return launch_status("sparse_attention_kernel");
}

}  // namespace spa
}  // namespace faq

extern "C" int faq_hif4_sparse_attention(const void* q, int64_t total, int64_t heads, int64_t q_token_stride,
                                         int64_t q_head_stride, const void* pages, int64_t num_pages, int64_t page_stride,
                                         int page_size, int64_t kv_heads, int d, const int32_t* table, int64_t table_ld,
                                         int64_t table_cols, const int32_t* cu, const int32_t* lens, int64_t batch,
                                         const int32_t* selected, int64_t count, float scale, void* out,
                                         int64_t out_token_stride, int64_t out_head_stride, void* stream) {
  using namespace faq;
  using namespace faq::spa;
  Params P;
  const int rc = make_pages(P.p, pages, num_pages, page_stride, page_size, kv_heads, d, table, table_ld, table_cols, cu,
                            lens, batch);
  if (rc) return rc;
  FAQ_CHECK_ARG(total >= 0 && total < (int64_t(1) << 31), "bad token count");
  FAQ_CHECK_ARG(heads > 0 && heads < (int64_t(1) << 24) && heads % kv_heads == 0,
                "query heads must be divisible by key/value heads");
  FAQ_CHECK_ARG(total * heads < (int64_t(1) << 31), "too many tokens for one call");
  FAQ_CHECK_ARG(count > 0, "bad page count");
  if (count > MAX_COUNT) return fail(FAQ_ERR_UNSUPPORTED, "more than 32768 listed pages");
  FAQ_CHECK_ARG(scale > 0.0f && scale < 1e30f, "scale must be positive");
  if (total == 0) return FAQ_OK;
  FAQ_CHECK_ARG(q && out && selected, "null pointer");
  FAQ_CHECK_ARG(aligned16(q) && aligned16(out), "q and out must be 16-byte aligned");
  for (const int64_t st : {q_token_stride, q_head_stride, out_token_stride, out_head_stride})
    FAQ_CHECK_ARG(st % 8 == 0, "strides must be multiples of 8 elements");
  P.q = static_cast<const __nv_bfloat16*>(q);
  P.qt = q_token_stride;
  P.qh = q_head_stride;
  P.out = static_cast<__nv_bfloat16*>(out);
  P.ot = out_token_stride;
  P.oh = out_head_stride;
  P.total = total;
  P.group = static_cast<int>(heads / kv_heads);
  P.passes = (P.group + RB - 1) / RB;
  P.list = selected;
  P.count = static_cast<int>(count);
  P.scale_log2 = scale * 1.4426950408889634f;
  const int64_t units = total * kv_heads * P.passes, blocks = std::min(count, table_cols) << (P.p.page_shift - 4);
  // Tokens of a sequence mostly want the same pages. Tiles of them (sparse_tile.cu) take a call where a sequence has
  // eight tokens, or blocks of eight query heads of them, on average, and the kernel of single tokens would
  // expand 440 blocks or more per SM, some 50 us. Both kernels, us, where neighbours' lists differ in about a third
  // of the pages (the tiles' also where they are the same, and have nothing in common), 32 pages of 64, heads of 128:
  //   16 sequences, 4 tokens, 32 / 8 heads (443 blocks per SM)  52   59 (48, 104)
  //   the same, 8 tokens (886)                                  88   65 (52, 134)
  //   1 sequence, 8 tokens, 64 / 8 heads (55)                   13   26 (23, 41)
  //   4 sequences, 8 tokens, 8 / 8 heads (221)                  28   40 (32, 70)
  //   the same, 32 tokens (886)                                 87   46 (36, 77)
  //   1 sequence, 512 tokens, 64 / 8 heads (3542)              329  164 (110, 598)
  const int tokens = P.group <= pre::TILE ? spt::tile_tokens(P.group) : 0;
  if (tokens && total * P.passes >= 8 * batch && units * blocks >= 440 * static_cast<int64_t>(num_sms()) &&
      std::min(tokens * count, table_cols) <= spt::MAX_UNION && table_cols <= spt::columns(d) && q_token_stride >= 8 &&
      q_head_stride >= 8)
    return d == 64 ? spt::launch<1>(P, heads, stream) : spt::launch<2>(P, heads, stream);
  // Units that fill the SMs more than once take four warps each: the waits at a unit's beginning and end are then those of
  // half as many waves. Eight and four warps, us, 64 pages of 16, one token, 32 / 8 heads of 128:
  //   32 sequences (256 units)  17.1  18.5;   40 (320)  25.8  28.3;   64 (512)  33.2  29.7;   128 (1024)  60.7  53.3
  //   128 sequences, heads of 64 42.1  34.8;   64, 8 pages of 64  20.5  16.8
  int split = 1, warps = 8;
  if (units > 3 * static_cast<int64_t>(num_sms()))
    warps = 4;
  else
    while (split < 8 && units * split * 2 <= 2 * num_sms() && blocks > warps * split) split *= 2;
  FAQ_CHECK_ARG(units * split < (int64_t(1) << 31), "too many tokens for one call");
  if (warps == 4) return d == 64 ? launch<1, 4>(P, split, stream) : launch<2, 4>(P, split, stream);
  return d == 64 ? launch<1, 8>(P, split, stream) : launch<2, 8>(P, split, stream);
}
