// K9 for chunks of tens of rows (drafted tokens, short prompt chunks): one tile of up to 128
// rows per (sequence, kv head) on the tensor cores of paged_prefill.cu, its keys expanded
// on the way.
//
// With so few rows the bf16 keys would be read once or twice, so they are not written to memory
// first: eight warps load a key tile's blocks from the pages (the next tile's while this one
// is expanded), and write K and V to shared memory as TMA would have laid them out. The
// products take the whole tile whatever its rows (a quarter of the tensor cores' time), so
// units of at most 64 or 32 rows stand in it two or four times: each copy's scores give it a
// half or a quarter of the keys, and the softmax has no work on rows that mean nothing.
// Work is cut into equal runs of key tiles, one per CTA, as in paged_attention.cu, and
// paged_prefill.cu's join adds up the units of several runs.
//
// Measured (one B200): 8 new tokens for each of 16 sequences of 1 .. 8192 tokens, 32 query heads
// on 8 kv heads of 128, in 33.5 us (without the copies 3.8 more). A key tile takes an SM about 3000
// cycles, of which a warp's expansion of its block of K and of V is 1900, at one instruction in
// more than four cycles. The warps wait for loads first (2.7 cycles per issue: the table's entry,
// then the block, both one tile ahead only), then at barriers (2.5), then for instructions (1.6):
// the roles' code together is more than the instruction caches hold. Hence the rolled loops; 16
// expanding warps, K and V apart, were slower (92 us against 58 for 16 sequences of 4096 tokens, 77
// with rolled loops), "no instruction" standing at 5.7 per issue there.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_pages.cuh"
#include "tma.h"

namespace faq {
namespace chk {

using namespace kvp;
using pre::CHUNK;
using pre::commit;
using pre::IDESC_QK;
using pre::idesc_pv;
using pre::Join;
using pre::mma_ss;
using pre::o_col;
using pre::s_col;
using pre::Softmax;
using pre::THREADS;
using pre::TILE;
using pre::TMEM_COLS;

constexpr int COST = 2;  // of a unit beyond its key tiles, in key tiles

struct Params {
  Pages p;
  int64_t total;
  int group, tile_tokens;  // query heads per kv head, whole tokens of a tile
  int max_rows;            // sequences with more rows are the prompt kernel's
  bool alone;              // which does not run, as max_new excludes them
  float scale_log2;
  __nv_bfloat16* out;
  int64_t ot, oh;
  Join* joins;   // [runs]
  float* parts;  // [2 runs][TILE x d + 2 TILE]
};

// A place in the order of all units (sequence, kv head, tile_tokens tokens), and the part of
// the unit that lies in this CTA's run [begin, end) of costs.
struct Walk {
  int b, head, u;
  int c0, n, len, units;  // of the sequence: first token in q, new tokens (0: not ours), length, units
  int tiles, k0, count;   // key tiles of the unit; of the run: k0 .. k0 + count - 1
  int64_t at;             // the unit's place: a fixed cost, then its tiles
};
__device__ __forceinline__ void enter(const Params& P, Walk& w, int b) {
  const int c0 = P.p.cu[b], c1 = P.p.cu[b + 1];
  w.b = b;
  w.c0 = c0;
  w.n = (c0 >= 0 && c1 > c0 && c1 <= P.total) ? c1 - c0 : 0;
  if (static_cast<int64_t>(w.n) * P.group > P.max_rows) {
    if (P.alone) atomicOr(&g_status, FAQ_STATUS_BAD_BOUND);
    w.n = 0;
  }
  w.len = length_of(P.p, b);
  w.units = (w.n + P.tile_tokens - 1) / P.tile_tokens;
}
// Copies of the unit's rows in the tile, see Softmax.
__device__ __forceinline__ int copies_of(const Params& P, const Walk& w) {
  const int rows = min(P.tile_tokens, w.n - w.u * P.tile_tokens) * P.group;
  return rows <= 32 ? 4 : rows <= 64 ? 2 : 1;
}
struct QMaps {
  CUtensorMap q[3];  // boxes of whole tokens, at most 128, 64, 32 rows
};
__device__ __forceinline__ int key_tiles(const Params& P, const Walk& w, int u) {
  const int seen = w.len - w.n + min(w.n, (u + 1) * P.tile_tokens);
  return seen <= 0 ? 0 : (seen + TILE - 1) / TILE;
}
__device__ __forceinline__ int64_t head_cost(const Params& P, const Walk& w) {
  int64_t sum = 0;
  for (int u = 0; u < w.units; ++u) {
    const int kt = key_tiles(P, w, u);
    sum += kt ? kt + COST : 0;
  }
  return sum;
}
__device__ __forceinline__ void clip(Walk& w, int64_t begin, int64_t end) {
  const int64_t first = w.at + COST;
  w.k0 = static_cast<int>(std::max<int64_t>(begin - first, 0));
  w.count = static_cast<int>(std::max<int64_t>(std::min<int64_t>(end - first, w.tiles) - w.k0, 0));
}
// The next unit with keys in the run (count 0: there is none).
__device__ __forceinline__ void next_unit(const Params& P, Walk& w, int64_t begin, int64_t end) {
  w.at += w.tiles + COST;
  w.count = 0;
  if (w.at + COST >= end) return;
  do {
    if (++w.u >= w.units) {
      w.u = 0;
      if (++w.head >= P.p.kv_heads || w.units == 0) {
        w.head = 0;
        do {
          if (w.b + 1 >= P.p.batch) return;
          enter(P, w, w.b + 1);
        } while (w.units == 0);
      }
    }
    w.tiles = key_tiles(P, w, w.u);
  } while (w.tiles == 0);
  clip(w, begin, end);
}

template <int NG>
struct Smem {
  static constexpr int tile = NG * CHUNK;
  static constexpr int q = 0;
  static constexpr int k = q + tile;
  static constexpr int v = k + 2 * tile;
  static constexpr int p = v + 2 * tile;
  static constexpr int bar = p + 2 * CHUNK;
  static constexpr int bytes = 1024 + bar + 256;
};

template <int NG>
__global__ void __launch_bounds__(THREADS, 1) paged_chunk_kernel(const __grid_constant__ QMaps maps, Params P) {
  using L = Smem<NG>;
  constexpr int D = 64 * NG, WARPS = THREADS / 32;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + L::bar);
  uint64_t* q_full = bars + 0;
  uint64_t* q_empty = bars + 1;
  uint64_t* k_full = bars + 2;   // [2 stages]
  uint64_t* k_empty = bars + 4;
  uint64_t* v_full = bars + 6;
  uint64_t* v_empty = bars + 8;
  uint64_t* s_full = bars + 10;
  uint64_t* s_free = bars + 11;
  uint64_t* p_full = bars + 12;
  uint64_t* pv_done = bars + 13;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);
  __shared__ int64_t s_scan[WARPS], s_begin, s_end, s_per;
  __shared__ Walk s_walk;
  __shared__ int s_empty;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Pages& p = P.p;
  if (tid == 0) {
    mbar_init(smem_addr(q_full), 1);
    mbar_init(smem_addr(q_empty), 1);
    mbar_init(smem_addr(s_full), 1);
    mbar_init(smem_addr(s_free), 8);
    mbar_init(smem_addr(p_full), 8);
    mbar_init(smem_addr(pv_done), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&k_full[i]), 8);  // the eight expanding warps
      mbar_init(smem_addr(&k_empty[i]), 1);
      mbar_init(smem_addr(&v_full[i]), 8);
      mbar_init(smem_addr(&v_empty[i]), 1);
    }
    fence_barrier_init();
    for (int i = 0; i < 3; ++i) tma_prefetch_desc(&maps.q[i]);
    s_walk.count = 0;
    s_empty = 0;
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

  // ---- this CTA's run: a prefix sum over the sequences, one per thread and round
  {
    const int rounds = (p.batch + THREADS - 1) / THREADS;
    Walk w;
    int64_t mine = 0, before = 0, total = 0, sum = 0;
    auto count = [&](int r) {
      const int b = r * THREADS + tid;
      w.n = w.units = 0;
      if (b < p.batch) {
        enter(P, w, b);
        if (w.n == 0) check_rows(p, b, P.total);
      }
      if (w.n > 0 && w.n > w.len) s_empty = 1;
      mine = head_cost(P, w) * p.kv_heads;
      before = pre::block_scan<WARPS>(mine, s_scan, &sum);
    };
    for (int r = 0; r < rounds; ++r) {
      count(r);
      total += sum;
    }
    const int64_t per = std::max<int64_t>(
        total < (int64_t(1) << 31) ? (static_cast<uint32_t>(total) + gridDim.x - 1) / gridDim.x
                                   : (total + gridDim.x - 1) / gridDim.x, COST + 1);
    const int64_t begin = blockIdx.x * per, end = std::min<int64_t>(total, begin + per);
    int64_t start = 0;
    for (int r = 0; r < rounds; ++r) {
      if (rounds > 1) count(r);
      if (begin < end && begin >= start + before && begin < start + before + mine) {
        const int64_t per_head = mine / p.kv_heads, at = begin - start - before;
        w.head = static_cast<int>(mine < (int64_t(1) << 31) ? static_cast<uint32_t>(at) / static_cast<uint32_t>(per_head)
                                                            : at / per_head);
        w.at = start + before + w.head * per_head;
        w.u = 0;
        w.tiles = key_tiles(P, w, 0);
        while (begin >= w.at + (w.tiles ? w.tiles + COST : 0)) {
          w.at += w.tiles ? w.tiles + COST : 0;
          w.tiles = key_tiles(P, w, ++w.u);
        }
        clip(w, begin, end);
        if (w.count == 0) next_unit(P, w, begin, end);
        s_begin = begin;
        s_end = end;
        s_per = per;
        s_walk = w;
      }
      start += sum;
    }
    if (tid == 0) P.joins[blockIdx.x].first = -1;
  }
  __syncthreads();
  if (s_empty) {  // rows that see no key are zero
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
      Walk e;
      enter(P, e, b);
      const int none = min(e.n, e.n - e.len), heads = P.group * p.kv_heads;
      for (int64_t i = tid; i < static_cast<int64_t>(none) * heads * (D / 8); i += THREADS) {
        const int64_t r = i / (D / 8);
        *reinterpret_cast<uint4*>(P.out + (e.c0 + r / heads) * P.ot + (r % heads) * P.oh + i % (D / 8) * 8) =
            make_uint4(0, 0, 0, 0);
      }
    }
  }
  const int64_t begin = s_begin, end = s_end;

  // Registers: 640 x 96 at launch = 512 x 104 + 128 x 64.
  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::: "memory");
    if (warp == 16) {
      if (lane == 0) {  // Q, and the record of a unit that other runs began
        int i = 0;
        for (Walk w = s_walk; w.count > 0; next_unit(P, w, begin, end), ++i) {
          if (w.k0 > 0 && w.k0 + w.count == w.tiles) {
            Join j;
            j.first = static_cast<int>((w.at + COST) / s_per);
            j.c0 = w.c0;
            j.head = w.head;
            j.tok0 = w.u * P.tile_tokens;
            j.n = w.n;
            P.joins[blockIdx.x] = j;
          }
          if (i > 0 && !mbar_wait_site(smem_addr(q_empty), (i - 1) & 1, 80, i)) break;
          const int copies = copies_of(P, w), rows = TILE / copies;
          const int map = copies >> 1;  // the box of 128, 64 or 32 rows
          mbar_arrive_expect_tx(smem_addr(q_full), static_cast<uint32_t>(copies * (rows / P.group) * P.group) * 128 * NG);
          for (int c = 0; c < NG * copies; ++c)
            tma_load_3d(smem_addr(base + L::q + (c / copies) * CHUNK + c % copies * rows * 128), &maps.q[map],
                        smem_addr(q_full), c / copies * 64, w.head * P.group, w.c0 + w.u * P.tile_tokens);
        }
        // drain (bounded): the last Q was read before the CTA exits
        if (i > 0) mbar_wait_site(smem_addr(q_empty), (i - 1) & 1, 81, i);
      }
    } else if (warp == 18) {
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
      const std::integral_constant<int, 0> c0;
      const std::integral_constant<int, 1> c1;
      uint32_t ring = 0;
      auto scores = [&](uint32_t step) {
        if (!wait(&k_full[step & 1], step >> 1, 82, step)) return false;
        if (step > 0 && !wait(s_free, step - 1, 83, step)) return false;
        tc_fence_after();
        if (step & 1) issue_qk(c1); else issue_qk(c0);
        return true;
      };
      int i = 0;
      bool ok = true;
      for (Walk w = s_walk; ok; next_unit(P, w, begin, end), ++i) {
        const int n = __shfl_sync(0xffffffffu, w.count, 0);
        if (n == 0 || !wait(q_full, i, 84, i)) break;
        ok = scores(ring);
        if (n == 1) commit(smem_addr(q_empty));
        for (int j = 0; j < n && ok; ++j, ++ring) {
          if (j + 1 < n) {
            if (!scores(ring + 1)) { ok = false; break; }
            if (j + 2 == n) commit(smem_addr(q_empty));  // the next unit's Q may come
          }
          if (!wait(&v_full[ring & 1], ring >> 1, 85, ring) || !wait(p_full, ring, 86, ring)) { ok = false; break; }
          tc_fence_after();
          if (ring & 1) issue_pv(c1, j != 0); else issue_pv(c0, j != 0);
        }
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n" ::: "memory");
    // ------------------------------------------------------------ expansion: block ew of each key tile
    const int ew = warp - 8;
    // from a page's K to its V (64 bits here: 34.1 us instead of 33.5 for 16 sequences' drafted tokens)
    const uint32_t v_off = static_cast<uint32_t>(p.kv_heads << (p.page_shift - 4)) * block_bytes(NG);
    // where block ew of tile j is (null: past the end, or no page; the softmax leaves such keys out,
    // and the registers' last block stands in for them, whose values are finite)
    auto block_of = [&](const Walk& w, int j) -> const uint8_t* {
      const int pos = (w.k0 + j) * TILE + ew * BLOCK;
      if (pos >= w.len) return nullptr;
      const int64_t page = page_of(p, w.b, pos);
      return page < 0 ? nullptr : p.base + page * p.page_stride + block_in_page<NG>(p, 0, w.head, pos);
    };
    const Expand expand;
    KBlock<NG> kb = {};
    VBlock<NG> vb = {};
    Walk w = s_walk;
    int j = 0;
    if (w.count > 0) {
      const uint8_t* src = block_of(w, 0);
      if (src) {
        kb.load(src, lane);
        vb.load(src + v_off, lane);
      }
    }
    for (int step = 0; w.count > 0; ++step) {
      if (++j == w.count) {
        next_unit(P, w, begin, end);
        j = 0;
      }
      const uint8_t* src = w.count > 0 ? block_of(w, j) : nullptr;  // of the next step
      const int st = step & 1;
      // rows of 128 bytes per group, token ew * 16 + i, unit u at u ^ (token % 8)
      auto write = [&](uint8_t* tile) {
        return [=](int token, int g, int unit, const uint32_t (&x)[4]) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(smem_addr(tile) + g * CHUNK +
                                                                         (ew * BLOCK + token) * 128 + ((unit ^ (token & 7)) << 4)),
                       "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                       : "memory");
        };
      };
      if (!mbar_wait_warp(smem_addr(&k_empty[st]), ((step >> 1) & 1) ^ 1, 87, step)) break;
      kb.template each<1>(expand, lane, write(base + L::k + st * L::tile));
      fence_proxy_async_smem();  // the tensor core reads it through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&k_full[st]));
      if (src) kb.load(src, lane);
      if (!mbar_wait_warp(smem_addr(&v_empty[st]), ((step >> 1) & 1) ^ 1, 88, step)) break;
      vb.template each<1>(expand, lane, write(base + L::v + st * L::tile));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&v_full[st]));
      if (src) vb.load(src + v_off, lane);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;\n" ::: "memory");
    Softmax<D> sm(tmem, 0, warp, lane, base + L::p, s_full, s_free, p_full, pv_done, P.scale_log2);
    auto unit = [&](const Walk& w, auto parts) {
      constexpr int PARTS = decltype(parts)::value;
      const int row = sm.template row<PARTS>(), row_tok = row / P.group, row_head = row - row_tok * P.group;
      const int tok = w.u * P.tile_tokens + row_tok;
      const bool live = row_tok < P.tile_tokens && tok < w.n;
      const int lim = live ? w.len - w.n + tok : pre::NO_ROW;
      if (!(pre::any_without_page(p, w.b, w.len, w.k0, w.count, lane)
                ? sm.template run<PARTS, true>(p, w.b, w.len, w.k0, w.count, lim, [] {})
                : sm.template run<PARTS, false>(p, w.b, w.len, w.k0, w.count, lim, [] {})))
        return false;
      if (!sm.template first_copy<PARTS>()) return true;
      float* part = w.count == w.tiles ? nullptr
                                       : P.parts + (2 * static_cast<int64_t>(blockIdx.x) + (w.k0 == 0)) * (TILE * D + 2 * TILE);
      sm.store(live, part, TILE, row,
               P.out + static_cast<int64_t>(w.c0 + (live ? tok : 0)) * P.ot + (w.head * P.group + row_head) * P.oh);
      return true;
    };
    for (Walk w = s_walk; w.count > 0; next_unit(P, w, begin, end)) {
      const int copies = copies_of(P, w);
      const bool ok = copies == 4   ? unit(w, std::integral_constant<int, 8>())
                      : copies == 2 ? unit(w, std::integral_constant<int, 4>())
                                    : unit(w, std::integral_constant<int, 2>());
      if (!ok) break;
    }
  }
  __syncthreads();
  if (warp == 18) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

inline size_t workspace(int d) {
  return static_cast<size_t>(num_sms()) * (sizeof(Join) + 2 * (TILE * d + 2 * TILE) * 4);
}

template <int NG>
static int launch(Params& P, const __nv_bfloat16* q, int64_t heads, int64_t qt, int64_t qh, char* ws, void* stream) {
  constexpr int D = 64 * NG;
  const int runs = num_sms();
  P.joins = reinterpret_cast<Join*>(ws);
  P.parts = reinterpret_cast<float*>(ws + runs * sizeof(Join));
  QMaps maps;
  const uint64_t dims[3] = {D, static_cast<uint64_t>(heads), static_cast<uint64_t>(P.total)};
  const uint64_t str[2] = {static_cast<uint64_t>(qh) * 2, static_cast<uint64_t>(qt) * 2};
  int rc = FAQ_OK;
  for (int i = 0; i < 3; ++i) {
    const uint32_t box[3] = {64, static_cast<uint32_t>(P.group), static_cast<uint32_t>(std::max((TILE >> i) / P.group, 1))};
    rc = make_tmap(&maps.q[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
  }
  auto kern = paged_chunk_kernel<NG>;
  static std::atomic<uint64_t> set{0};
  rc = allow_smem(reinterpret_cast<const void*>(kern), Smem<NG>::bytes, set);
  if (rc) return rc;
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(runs)), THREADS, Smem<NG>::bytes, stream, maps, P));
  FAQ_CUDA(launch_early(pre::prefill_combine_kernel<D, TILE, Params>, dim3(static_cast<unsigned>(runs), TILE / 8), 256, 0,
                        stream, P));
  return FAQ_OK;
}

}  // namespace chk
}  // namespace faq

// Which kernel takes a sequence, by its rows (new tokens x query heads of a kv head):
// - up to FEW_ROWS in every sequence of the call, paged_attention.cu's, in units of eight: 16
//   sequences of 4096 tokens (32 query heads on 8 kv heads of 128) take 54.5 us with 12 or 16
//   rows against 57.8 in paged_chunk.cu, with 24 rows 77 against 58. Also when no unit is split
//   and each can have an SM: 32 rows of 4 sequences of 1000 tokens 12.5 against 15.8, but of 32
//   such sequences 64 against 37.5;
// - else up to CHUNK_ROWS, one tile of paged_chunk.cu: 128 rows of those 16 sequences take 78 us
//   against 164 in the prompt kernel, whose expansion writes the keys to memory;
// - beyond them the prompt kernel's. That is not where the two cross: with a limit of 512 rows
//   units of several tiles in paged_chunk.cu took 130 us against 175 here for 144 rows, 135 against
//   200 for 256, 194 against 261 for 384 (with heads of 64: 100 / 160, 114 / 166, 163 / 224; 4 sequences
//   of 16384 tokens, heads of 128: 132 / 139, 128 / 153, 183 / 209). The limit is still
//   one tile: raising it is a change to measure and test by itself.
// More than 128 query heads to a kv head do not fit a tile of whole tokens: paged_attention.cu
// takes those.
namespace faq {
namespace pag {
constexpr int FEW_ROWS = 16, CHUNK_ROWS = 128, ALL_PROMPT_TILES = 600;
struct Kinds {
  bool few, chunks, prompts;
  int min_rows() const { return chunks ? CHUNK_ROWS + 1 : 1; }  // of a sequence of the prompt kernel
};
inline Kinds kinds(int64_t group, int64_t kv_heads, int64_t max_new, int64_t max_len, int64_t total_len, int64_t total,
                   int64_t batch) {
  const int64_t rows = group * std::min(max_new, total);
  if (rows <= FEW_ROWS || group > pre::TILE) return {true, false, false};
  if (max_len <= pat::WHOLE && (rows + pat::RB - 1) / pat::RB * kv_heads * batch <= num_sms()) return {true, false, false};
  const bool prompts = rows > CHUNK_ROWS;
  // The prompt kernel takes the shorter sequences too when there are none (all have max_new
  // tokens as they add up to that; rows of q may lie beyond cu's end) and when their keys are
  // few: a key tile costs it more, the other kernel and its join cost 10 us at the least. 256 tokens
  // on 2048 (32 query heads on 8 kv heads of 128) beside one token on 500: 55.0 us with both
  // kernels, 44.3 with one; beside two on 4096 (512 key tiles of all heads): 58.0 and 59.9; four:
  // 64.4 and 81.2. What is known of those keys is a bound: of all sequences' lengths, and of
  // the sequences there can be beside one of max_new tokens. Mostly they are fewer, so it may lie
  // a little above the lengths at which the two ways take the same time.
  const int64_t beside = std::max<int64_t>(std::min(batch - 1, total - max_new), 0);
  const int64_t keys = std::min(total_len - max_new, beside * max_len);
  const bool alone = total == batch * max_new || kv_heads * keys <= ALL_PROMPT_TILES * pre::TILE;
  return {false, !(prompts && alone), prompts};
}
}  // namespace pag
}  // namespace faq

extern "C" size_t faq_hif4_paged_attention_workspace_bytes(int64_t total, int64_t heads, int64_t kv_heads, int64_t batch,
                                                           int64_t max_new, int64_t max_len, int64_t total_len, int d) {
  using namespace faq;
  if (total < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || batch <= 0 || max_new < 0 || max_len < 0 ||
      total_len < 0 || (d != 64 && d != 128))
    return 0;
  const int64_t group = heads / kv_heads;
  const pag::Kinds kinds = pag::kinds(group, kv_heads, max_new, max_len, total_len, total, batch);
  size_t bytes = kinds.few && max_len > pat::WHOLE ? pat::workspace(d) : 0;  // units that are not split need none
  if (kinds.chunks) bytes = std::max(bytes, chk::workspace(d));
  if (kinds.prompts)
    bytes = std::max(bytes, pre::layout(total, heads, kv_heads, batch, max_len, total_len, kinds.min_rows(), d).bytes);
  return bytes;
}

extern "C" int faq_hif4_paged_attention(const void* q, int64_t total, int64_t heads, int64_t q_token_stride,
                                        int64_t q_head_stride, const void* pages, int64_t num_pages,
                                        int64_t page_stride, int page_size, int64_t kv_heads, int d,
                                        const int32_t* table, int64_t table_ld, int64_t table_cols, const int32_t* cu,
                                        const int32_t* lens, int64_t batch, int64_t max_new, int64_t max_len,
                                        int64_t total_len, float scale, void* out, int64_t out_token_stride,
                                        int64_t out_head_stride, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace faq;
  kvp::Pages pages_;
  int rc = kvp::make_pages(pages_, pages, num_pages, page_stride, page_size, kv_heads, d, table, table_ld, table_cols, cu,
                           lens, batch);
  if (rc) return rc;
  FAQ_CHECK_ARG(heads > 0 && heads % kv_heads == 0, "query heads must be divisible by key/value heads");
  const int64_t group = heads / kv_heads;
  FAQ_CHECK_ARG(group < 4096, "more than 4095 query heads per key/value head");
  FAQ_CHECK_ARG(total >= 0 && max_new >= 0 && max_len >= 0 && total_len >= 0 && total * heads < (int64_t(1) << 31) &&
                    max_len < (int64_t(1) << 31) && total_len < (int64_t(1) << 40), "bad token count");
  if (total == 0) return FAQ_OK;
  FAQ_CHECK_ARG(q && out, "null pointer");
  FAQ_CHECK_ARG(scale > 0.0f && scale < 3.0e38f, "scale must be positive and finite");
  FAQ_CHECK_ARG(aligned16(q) && aligned16(out) && q_token_stride % 8 == 0 && q_head_stride % 8 == 0 &&
                    out_token_stride % 8 == 0 && out_head_stride % 8 == 0,
                "q and out must be 16-byte aligned with strides multiple of 8");
  const size_t need =
      faq_hif4_paged_attention_workspace_bytes(total, heads, kv_heads, batch, max_new, max_len, total_len, d);
  FAQ_CHECK_ARG(need == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
                "workspace must be a 256-byte aligned device buffer");
  FAQ_CHECK_ARG(workspace_bytes >= need,
                "workspace too small: faq_hif4_paged_attention_workspace_bytes() bytes needed");
  const float scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  const __nv_bfloat16* query = static_cast<const __nv_bfloat16*>(q);
  __nv_bfloat16* output = static_cast<__nv_bfloat16*>(out);
  char* ws = static_cast<char*>(workspace);
  pag::Kinds kinds = pag::kinds(group, kv_heads, max_new, max_len, total_len, total, batch);
  // pages of 8 GiB and more: V is further behind K than the chunk kernel's 32 bits reach; the kernel of
  // few rows takes the batch (its workspace is the smaller one)
  if (kinds.chunks && kv_heads * (page_size / 16) * kvp::block_bytes(d / 64) >= (int64_t(1) << 32))
    kinds = {true, false, false};
  if (kinds.few) {
    pat::Params P;
    P.p = pages_;
    P.q = query;
    P.qt = q_token_stride;
    P.qh = q_head_stride;
    P.out = output;
    P.ot = out_token_stride;
    P.oh = out_head_stride;
    P.total = total;
    P.group = static_cast<int>(group);
    P.split = max_len > pat::WHOLE;
    P.group_magic = static_cast<uint32_t>(((uint64_t(1) << 32) + group - 1) / group);
    P.scale_log2 = scale_log2;
    return d == 64 ? pat::launch<1>(P, ws, stream) : pat::launch<2>(P, ws, stream);
  }
  if (kinds.chunks) {
    chk::Params P;
    P.p = pages_;
    P.total = total;
    P.group = static_cast<int>(group);
    P.tile_tokens = static_cast<int>(pre::TILE / group);
    P.max_rows = pag::CHUNK_ROWS;
    P.alone = !kinds.prompts;
    P.scale_log2 = scale_log2;
    P.out = output;
    P.ot = out_token_stride;
    P.oh = out_head_stride;
    rc = d == 64 ? chk::launch<1>(P, query, heads, q_token_stride, q_head_stride, ws, stream)
                 : chk::launch<2>(P, query, heads, q_token_stride, q_head_stride, ws, stream);
    if (rc || !kinds.prompts) return rc;
  }
  pre::Params P;
  P.p = pages_;
  P.total = total;
  P.group = static_cast<int>(group);
  P.tile_tokens = static_cast<int>(pre::TILE / group);
  P.min_rows = kinds.min_rows();
  P.scale_log2 = scale_log2;
  P.out = output;
  P.ot = out_token_stride;
  P.oh = out_head_stride;
  const pre::Layout a = pre::layout(total, heads, kv_heads, batch, max_len, total_len, P.min_rows, d);
  return d == 64 ? pre::launch<1>(P, query, heads, q_token_stride, q_head_stride, a, ws, stream)
                 : pre::launch<2>(P, query, heads, q_token_stride, q_head_stride, a, ws, stream);
}
