// Pages of the HiF4 K/V cache: addressing, the page format (include/faquant_b200.h) and
// the expansion of its codes to bf16 register pairs.
#pragma once

#include "common.cuh"
#include "hif4.cuh"

namespace faq {
namespace kvp {

constexpr int BLOCK = 16;  // tokens of a block, the unit of the format
// bytes of a block of one head's K or V with NG = d / 64 groups, and its sections
__host__ __device__ constexpr int block_bytes(int ng) { return 592 * ng; }
__host__ __device__ constexpr int exp_offset(int ng) { return 512 * ng; }
__host__ __device__ constexpr int scale_offset(int ng) { return 576 * ng; }

struct Pages {
  uint8_t* base;
  int64_t page_stride;  // bytes
  int64_t num_pages;
  const int32_t* table;  // [batch, table_ld], the first table_cols columns valid
  int64_t table_ld;
  int table_cols;
  int kv_heads;
  int page_shift;        // log2(page_size)
  const int32_t* cu;     // [batch + 1]
  const int32_t* lens;   // [batch]
  int batch;
};

// byte offset of the block of token `pos` within its page, which = 0 K, 1 V
template <int NG>
__device__ __forceinline__ int64_t block_in_page(const Pages& p, int which, int head, int pos) {
  const int blocks = 1 << (p.page_shift - 4);
  const int blk = (pos >> 4) & (blocks - 1);
  return (static_cast<int64_t>(which * p.kv_heads + head) * blocks + blk) * block_bytes(NG);
}

// The page of token `pos` of sequence b, or -1 (recorded in the status word) when the
// table has no valid entry for it.
__device__ __forceinline__ int64_t page_of(const Pages& p, int b, int pos) {
  const int col = pos >> p.page_shift;
  int64_t page = -1;
  if (col < p.table_cols) page = p.table[b * p.table_ld + col];
  if (page < 0 || page >= p.num_pages) {
    atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
    return -1;
  }
  return page;
}

// Whether column `col` of sequence b's table row holds no page.
__device__ __forceinline__ bool no_page(const Pages& p, int b, int col) {
  if (col >= p.table_cols) return true;
  const int page = p.table[b * p.table_ld + col];
  return page < 0 || page >= p.num_pages;
}

// Records a sequence whose new tokens do not lie in the `total` given rows (it is left out).
__device__ __forceinline__ void check_rows(const Pages& p, int b, int64_t total) {
  const int c0 = p.cu[b], c1 = p.cu[b + 1];
  if (c0 < 0 || c1 < c0 || c1 > total) atomicOr(&g_status, FAQ_STATUS_BAD_BOUND);
}

// Length of sequence b, at most what its table row can hold (a longer one is recorded).
__device__ __forceinline__ int length_of(const Pages& p, int b) {
  const int len = p.lens[b], most = p.table_cols << p.page_shift;
  if (len > most) atomicOr(&g_status, FAQ_STATUS_BAD_PAGE);
  return min(max(len, 0), most);
}

// twice the scale of a scale byte: the expansion below yields half the value over it
__device__ __forceinline__ float twice_scale(uint32_t code) { return __uint_as_float((code << 21) + (80u << 23)); }

__device__ __forceinline__ uint32_t hmul2_bf16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// The constants of the expansion, in registers whose values the compiler does not know: it
// would else split (x & mask) | bits with two constants into two instructions, or make the
// constants anew at each use (the integer pipe, which bounds the expansion, then does 40 %
// more).
struct Expand {
  uint32_t magic, base, shift;
  __device__ __forceinline__ Expand() {
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(magic));  // bf16 128, twice
    asm volatile("mov.b32 %0, 0x3E003E00;" : "=r"(base));   // 2^-3
    asm volatile("mov.b32 %0, 0xC308C308;" : "=r"(shift));  // -136
  }
  // (2^(e - 3), 2^(e' - 3)) as bf16, from the exponent word's two halves: e is bits 2 s,
  // 2 s + 1 of the half of sub-block s, rotated into the low bits of the exponent field
  // (rot = 7 - 2 s modulo 32; the bits it wraps are masked off; 2^-3's field ends in 00).
  __device__ __forceinline__ uint32_t exponents(uint32_t ew, int rot) const {
    uint32_t d;
    asm("lop3.b32 %0, %1, 0x01800180, %2, 0xEA;" : "=r"(d) : "r"(__funnelshift_l(ew, ew, rot)), "r"(base));
    return d;
  }
  // The eight nibbles of a code word as four bf16 pairs (n - 8) 2^(e - 3): pair j holds
  // nibble j of the word's low and high halves. 0x4300 | n is 128 + n exactly, and one
  // FMA with (E, -136 E) gives (n - 8) E exactly (at most 4 significant bits).
  __device__ __forceinline__ void word(uint32_t w, uint32_t e, uint32_t (&out)[4]) const {
    const uint32_t n = hmul2_bf16(e, shift);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t x;
      asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(x) : "r"(w >> (4 * j)), "r"(magic));
      out[j] = hfma2_bf16(x, e, n);
    }
  }
};

}  // namespace kvp
}  // namespace faq
