// K8 -- the HiF4 K/V cache in pages: quantizing tokens as they are written, reading them
// back as bf16 or fp32.
//
// Write: per token, kv head and 64-channel group the HiF4 fit of K1 and K4 (hif4.cuh, the same
// bits), eight channels per lane, eight lanes per group; the codes and exponents go to the
// places of the page format (include/faquant_b200.h). Every byte of the cache belongs to one
// token, so tokens are written without reading what is there.
// Read: the inverse, value = (n - 8) / 4 * 2^e * scale, exact in bf16.
// Both give a warp a block of 16 tokens of one head, so that a lane holds both tokens of a pair
// (V's words interleave them) and stores 8 or 16 bytes. The packed tokens of a ragged batch
// are found without a prefix sum over its blocks: sequence b's blocks get the slots from
// cu[b] / 16 + 2 b on, always enough of them (n tokens touch at most n / 16 + 2 blocks).
//
// Measured (one B200, 8 kv heads of 128): writing 8192 tokens and reading them back 26.0 us for
// 86 MB, 3.3 TB/s: the write takes 18.8 us of it (cold), three times its bytes' time, with 63 % of the
// issue slots and 64 % of the integer pipe taken by the fit and the rest lost to its loads'
// latency; reading whole contexts of 8 sequences back (156 MB) 36.4 us, 4.3 TB/s, waiting for loads (7.7
// cycles per issue): a warp has one block, behind a chain of dependent ones (cu, lens, the
// table, the block). A decode step's tokens take the 8 us of two launches.
#include <algorithm>
#include <atomic>

#include "kv_pages.cuh"

namespace faq {
namespace kvp {

struct WriteParams {
  Pages p;
  const void *k, *v;
  int64_t total, kt, kh, vt, vh;  // tokens; token and head strides (elements)
  int k_levels, v_levels;
};

// HiF4 of eight values: the code word (nibble i = 8 + signed code of value i), the two
// quarters' exponents and the group's scale byte. All lanes of the warp take part. The
// arithmetic of hif4.cuh on FP32x2 pairs: t = min(fl(fl(|x| 4qm) + 0.5), 7.5), whose floor is
// t + 2^23 rounded toward zero; with the sign of x put back, the four codes of a quarter are
// digits of base 16 that three exact FMAs add up (2^23 + 0x8888 makes them n = 8 + code, and
// the sum's low 16 bits are the quarter's nibbles).
__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], int levels, uint32_t& ea, uint32_t& eb,
                                              uint32_t& scale) {
  const float ma = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
  const float mb = fmaxf(fmaxf(fabsf(v[4]), fabsf(v[5])), fmaxf(fabsf(v[6]), fabsf(v[7])));
  float m1 = fmaxf(ma, mb);
  m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 1));
  m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 2));
  m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, 4));
  const Hif4Scale sc = hif4_scale(m1, levels);
  scale = sc.code;
  hif4_level_shifts(__fmul_rn(ma, sc.rec), __fmul_rn(mb, sc.rec), levels, ea, eb);
  const uint32_t rec_q = __float_as_uint(sc.rec) + (2u << 23);
  const float qa = __uint_as_float(rec_q - ea), qb = __uint_as_float(rec_q - eb);  // 4 qm
  ea >>= 23;
  eb >>= 23;
  uint32_t quarter[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float c[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x0 = v[4 * h + 2 * i], x1 = v[4 * h + 2 * i + 1], q = h ? qb : qa;
      float2 t = __fadd2_rn(__fmul2_rn(make_float2(fabsf(x0), fabsf(x1)), make_float2(q, q)), make_float2(0.5f, 0.5f));
      t = make_float2(fminf(t.x, 7.5f), fminf(t.y, 7.5f));
      const float2 r = __fadd2_rn(__fadd2_rz(t, make_float2(8388608.0f, 8388608.0f)), make_float2(-8388608.0f, -8388608.0f));
      c[2 * i] = __uint_as_float(__float_as_uint(r.x) | (__float_as_uint(x0) & 0x80000000u));
      c[2 * i + 1] = __uint_as_float(__float_as_uint(r.y) | (__float_as_uint(x1) & 0x80000000u));
    }
    const float n = __fmaf_rn(c[3], 4096.0f, __fmaf_rn(c[2], 256.0f, __fmaf_rn(c[1], 16.0f, __fadd_rn(c[0], 8423560.0f))));
    quarter[h] = __float_as_uint(n);
  }
  return __byte_perm(quarter[0], quarter[1], 0x5410);
}

// Eight consecutive values as loaded, so that a lane's loads are all in flight before the
// first of them is quantized.
template <typename T>
struct Raw;
template <>
struct Raw<__nv_bfloat16> {
  uint32_t w[4];
  __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
  __device__ __forceinline__ void load(const __nv_bfloat16* src, bool vec) {
    if (vec) {
      const uint4 u = *reinterpret_cast<const uint4*>(src);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};
template <>
struct Raw<float> {
  float f[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.0f;
  }
  __device__ __forceinline__ void load(const float* src, bool vec) {
    if (vec) {
      const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
      f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = src[i];
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i];
  }
};

// Slot -> (sequence, first position of a block, the live tokens [from, to) of the block, the
// packed token of the block's first position, the number of new tokens at positions below
// zero); false if the slot holds nothing. A sequence whose new tokens all have no position
// has its first slot, with to = 0.
struct Slot {
  int b, pos, from, to;
  int64_t token, none;
};
__device__ __forceinline__ int64_t first_slot(const Pages& p, int b) { return (p.cu[b] >> 4) + 2 * static_cast<int64_t>(b); }
__host__ __device__ inline int64_t slots_of(int64_t total, int64_t batch) { return total / 16 + 2 * batch; }
__device__ __forceinline__ bool find_slot(const Pages& p, int64_t slot, int64_t total, Slot& s) {
  int lo = 0, hi = p.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_slot(p, mid) <= slot) lo = mid; else hi = mid;
  }
  s.b = lo;
  const int c0 = p.cu[lo], c1 = p.cu[lo + 1];
  if (c0 < 0 || c1 <= c0 || c1 > total || slot < first_slot(p, lo)) {
    check_rows(p, lo, total);
    return false;
  }
  const int64_t first = static_cast<int64_t>(p.lens[lo]) - (c1 - c0);  // position of the first new token
  // positions below zero have no block; the first block is that of position max(first, 0)
  const int64_t block = (first > 0 ? first >> 4 : 0) + (slot - first_slot(p, lo));
  const int64_t pos = block * BLOCK;
  s.none = first < 0 ? std::min<int64_t>(-first, c1 - c0) : 0;
  if (pos >= p.lens[lo] && !(pos == 0 && s.none)) return false;
  s.pos = static_cast<int>(pos);
  s.from = static_cast<int>(first > pos ? first - pos : 0);
  s.to = static_cast<int>(std::max<int64_t>(std::min<int64_t>(p.lens[lo] - pos, BLOCK), 0));
  s.token = c0 + (pos - first);
  return true;
}

// A warp takes half a block (8 tokens): its loads are then all in flight at once.
constexpr int WRITE_WARPS = 4;
template <typename T, int NG>
__global__ void __launch_bounds__(32 * WRITE_WARPS, sizeof(T) == 2 ? 8 : 4) kv_write_kernel(WriteParams w, bool vec) {
  grid_dependency_wait();
  allow_dependent_launch();
  const Pages& p = w.p;
  const int lane = threadIdx.x & 31, s = lane & 7;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * WRITE_WARPS + (threadIdx.x >> 5);
  const int h = static_cast<int>(item & 1);
  const int64_t slot = (item >> 1) / p.kv_heads;
  const int head = static_cast<int>((item >> 1) - slot * p.kv_heads);
  Slot x;
  if (slot >= slots_of(w.total, p.batch) || !find_slot(p, slot, w.total, x)) return;  // warp-uniform
  if (x.from >= 8 * (h + 1) || x.to <= 8 * h) return;
  const int64_t page = page_of(p, x.b, x.pos);
  if (page < 0) return;
  uint8_t* kdst = p.base + page * p.page_stride + block_in_page<NG>(p, 0, head, x.pos);
  uint8_t* vdst = p.base + page * p.page_stride + block_in_page<NG>(p, 1, head, x.pos);
  const T* ksrc = static_cast<const T*>(w.k) + x.token * w.kt + head * w.kh + 8 * s;
  const T* vsrc = static_cast<const T*>(w.v) + x.token * w.vt + head * w.vh + 8 * s;
  const int pr = (lane >> 3) + 4 * h;  // tokens 2 pr, 2 pr + 1 of the block
  const bool live[2] = {2 * pr >= x.from && 2 * pr < x.to, 2 * pr + 1 >= x.from && 2 * pr + 1 < x.to};
  Raw<T> rk[2][NG], rv[2][NG];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (live[k]) {
        rk[k][g].load(ksrc + (2 * pr + k) * w.kt + 64 * g, vec);
        rv[k][g].load(vsrc + (2 * pr + k) * w.vt + 64 * g, vec);
      } else {
        rk[k][g].zero();
        rv[k][g].zero();
      }
    }
  uint32_t vw[2][NG], ve[2][NG];  // [token]; the exponents of all sub-blocks, (a, b) halves
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = 2 * pr + k;
    if (!__any_sync(0xffffffffu, live[k])) continue;  // a step of one token per sequence
    uint32_t kw[NG], kx[NG], kscale = 0, vscale = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float v[8];
      uint32_t ea, eb, sc;
      rk[k][g].values(v);
      kw[g] = quantize8(v, w.k_levels, ea, eb, sc);
      kx[g] = (ea | (eb << 16)) << (2 * s);
      kscale |= sc << (8 * g);
      rv[k][g].values(v);
      vw[k][g] = quantize8(v, w.v_levels, ea, eb, sc);
      ve[k][g] = (ea | (eb << 16)) << (2 * s);
      vscale |= sc << (8 * g);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        kx[g] |= __shfl_xor_sync(0xffffffffu, kx[g], o);
        ve[k][g] |= __shfl_xor_sync(0xffffffffu, ve[k][g], o);
      }
    }
    // K: the even lane of two stores both lanes' words of group 0, the odd one of group 1
    uint8_t* krow = kdst + 32 * NG * r + (s >> 1) * 8 * NG;
    if constexpr (NG == 2) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, (s & 1) ? kw[0] : kw[1], 1);
      if (live[k]) {
        *reinterpret_cast<uint2*>(krow + 8 * (s & 1)) = (s & 1) ? make_uint2(other, kw[1]) : make_uint2(kw[0], other);
        if (s == 0) *reinterpret_cast<uint2*>(kdst + exp_offset(NG) + r * 8) = make_uint2(kx[0], kx[1]);
        if (s == 1) *reinterpret_cast<uint16_t*>(kdst + scale_offset(NG) + r * 2) = static_cast<uint16_t>(kscale);
        if (s == 2) *reinterpret_cast<uint16_t*>(vdst + scale_offset(NG) + r * 2) = static_cast<uint16_t>(vscale);
      }
    } else if (live[k]) {
      *reinterpret_cast<uint32_t*>(krow + 4 * (s & 1)) = kw[0];
      if (s == 0) *reinterpret_cast<uint32_t*>(kdst + exp_offset(NG) + r * 4) = kx[0];
      if (s == 1) kdst[scale_offset(NG) + r] = static_cast<uint8_t>(kscale);
      if (s == 2) vdst[scale_offset(NG) + r] = static_cast<uint8_t>(vscale);
    }
  }
  // V: words of a quad's halves (token 2 pr, 2 pr + 1)
  uint8_t* vrow = vdst + 64 * NG * pr + (s ^ (2 * (pr & 3))) * 8 * NG;
  uint8_t* vexp = vdst + exp_offset(NG) + pr * NG * 8;
  if (live[0] && live[1]) {
    uint32_t q[2 * NG], e[2 * NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      q[2 * g] = __byte_perm(vw[0][g], vw[1][g], 0x5410);
      q[2 * g + 1] = __byte_perm(vw[0][g], vw[1][g], 0x7632);
      e[2 * g] = __byte_perm(ve[0][g], ve[1][g], 0x5410);
      e[2 * g + 1] = __byte_perm(ve[0][g], ve[1][g], 0x7632);
    }
    if constexpr (NG == 2) {
      *reinterpret_cast<uint4*>(vrow) = make_uint4(q[0], q[1], q[2], q[3]);
      if (s == 3) *reinterpret_cast<uint4*>(vexp) = make_uint4(e[0], e[1], e[2], e[3]);
    } else {
      *reinterpret_cast<uint2*>(vrow) = make_uint2(q[0], q[1]);
      if (s == 3) *reinterpret_cast<uint2*>(vexp) = make_uint2(e[0], e[1]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!live[k]) continue;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint16_t* q = reinterpret_cast<uint16_t*>(vrow + 8 * g + 2 * k);
        q[0] = static_cast<uint16_t>(vw[k][g]);
        q[2] = static_cast<uint16_t>(vw[k][g] >> 16);
        if (s == 0) {
          uint16_t* e = reinterpret_cast<uint16_t*>(vexp + 8 * g + 2 * k);
          e[0] = static_cast<uint16_t>(ve[k][g]);
          e[2] = static_cast<uint16_t>(ve[k][g] >> 16);
        }
      }
    }
  }
}

struct ReadParams {
  Pages p;
  void *k, *v;
  int64_t total, kt, kh, vt, vh;
};

// Eight consecutive channels as four bf16 pairs, to bf16 or fp32.
__device__ __forceinline__ void store_pairs(__nv_bfloat16* dst, bool vec, const uint32_t (&w)[4]) {
  if (vec) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) reinterpret_cast<uint16_t*>(dst)[i] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
  }
}
__device__ __forceinline__ void store_pairs(float* dst, bool vec, const uint32_t (&w)[4]) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float((i & 1) ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
  if (vec) {
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = v[i];
  }
}

// A block of one head's K or V, as a warp loads it and hands it out: for K a lane has sixteen
// channels of each group of two tokens, for V a sub-block of both tokens of two pairs.
// each(expand, lane, f) calls f(token, group, unit, four bf16 pairs) for every eight channels 8
// unit .. of a group. y = (n - 8) 2^(e - 3) times twice the scale is exact in bf16 (six
// significant bits), so a pair costs one packed product.
__device__ __forceinline__ uint32_t scale_pair(uint32_t code) {
  const uint32_t s = (code << 5) + (80u << 7);  // bf16 bits of twice the scale
  return s | (s << 16);
}
// each<UNROLL>: 1 keeps the loop over the lane's two tokens (of V: token pairs), half the code.
template <int NG>
struct KBlock {
  uint32_t w[2][2 * NG], e[2][NG], sc[2];
  __device__ __forceinline__ void load(const uint8_t* src, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (lane >> 2) + 8 * h;
      if constexpr (NG == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(src + 64 * r + 16 * t);
        w[h][0] = u.x; w[h][1] = u.y; w[h][2] = u.z; w[h][3] = u.w;
        const uint2 x = *reinterpret_cast<const uint2*>(src + exp_offset(NG) + 8 * r);
        e[h][0] = x.x; e[h][1] = x.y;
        sc[h] = *reinterpret_cast<const uint16_t*>(src + scale_offset(NG) + 2 * r);
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(src + 32 * r + 8 * t);
        w[h][0] = u.x; w[h][1] = u.y;
        e[h][0] = *reinterpret_cast<const uint32_t*>(src + exp_offset(NG) + 4 * r);
        sc[h] = src[scale_offset(NG) + r];
      }
    }
  }
  template <int UNROLL = 2, typename F>
  __device__ __forceinline__ void each(const Expand& expand, int lane, F&& f) const {
    const int t = lane & 3;
#pragma unroll UNROLL
    for (int h = 0; h < 2; ++h) {
      const int r = (lane >> 2) + 8 * h;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t s = scale_pair(((h ? sc[1] : sc[0]) >> (8 * g)) & 255), eg = h ? e[1][g] : e[0][g];
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // pair j: channels j and 4 + j of sub-block 2 t + i
          uint32_t y[4];
          expand.word(h ? w[1][2 * g + i] : w[0][2 * g + i], expand.exponents(eg, (7 - 4 * t - 2 * i) & 31), y);
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = hmul2_bf16(y[j], s);
          const uint32_t row[4] = {__byte_perm(y[0], y[1], 0x5410), __byte_perm(y[2], y[3], 0x5410),
                                   __byte_perm(y[0], y[1], 0x7632), __byte_perm(y[2], y[3], 0x7632)};
          f(r, g, 2 * t + i, row);
        }
      }
    }
  }
};
template <int NG>
struct VBlock {
  uint32_t w[2][2 * NG], e[2][2 * NG], sc[2];
  __device__ __forceinline__ void load(const uint8_t* src, int lane) {
    const int s = lane & 7;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p = (lane >> 3) + 4 * h;  // tokens 2 p, 2 p + 1
      if constexpr (NG == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(src + 128 * p + 16 * (s ^ (2 * (p & 3))));
        w[h][0] = u.x; w[h][1] = u.y; w[h][2] = u.z; w[h][3] = u.w;
        const uint4 x = *reinterpret_cast<const uint4*>(src + exp_offset(NG) + 16 * p);
        e[h][0] = x.x; e[h][1] = x.y; e[h][2] = x.z; e[h][3] = x.w;
        sc[h] = *reinterpret_cast<const uint32_t*>(src + scale_offset(NG) + 4 * p);  // [token][group]
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(src + 64 * p + 8 * (s ^ (2 * (p & 3))));
        w[h][0] = u.x; w[h][1] = u.y;
        const uint2 x = *reinterpret_cast<const uint2*>(src + exp_offset(NG) + 8 * p);
        e[h][0] = x.x; e[h][1] = x.y;
        sc[h] = *reinterpret_cast<const uint16_t*>(src + scale_offset(NG) + 2 * p);
      }
    }
  }
  template <int UNROLL = 2, typename F>
  __device__ __forceinline__ void each(const Expand& expand, int lane, F&& f) const {
    const int s = lane & 7;
#pragma unroll UNROLL
    for (int h = 0; h < 2; ++h) {
      const int p = (lane >> 3) + 4 * h;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t c = h ? sc[1] : sc[0];
        const uint32_t pair = __byte_perm(scale_pair((c >> (8 * g)) & 255), scale_pair((c >> (8 * (NG + g))) & 255), 0x5410);
        uint32_t y[2][4];  // [quad]: pair j is channel j of both tokens
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          expand.word(h ? w[1][2 * g + q] : w[0][2 * g + q], expand.exponents(h ? e[1][2 * g + q] : e[0][2 * g + q], (7 - 2 * s) & 31),
                      y[q]);
#pragma unroll
          for (int j = 0; j < 4; ++j) y[q][j] = hmul2_bf16(y[q][j], pair);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t sel = k ? 0x7632 : 0x5410;
          const uint32_t row[4] = {__byte_perm(y[0][0], y[0][1], sel), __byte_perm(y[0][2], y[0][3], sel),
                                   __byte_perm(y[1][0], y[1][1], sel), __byte_perm(y[1][2], y[1][3], sel)};
          f(2 * p + k, g, s, row);
        }
      }
    }
  }
};

// The tokens [from, to) of a block as rows of `stride` elements from dst (the block's first token).
template <typename T, template <int> class Block, int NG>
__device__ __forceinline__ void expand_block(const uint8_t* src, T* dst, int64_t stride, int from, int to, int lane,
                                             bool vec = true) {
  const Expand expand;
  Block<NG> x;
  x.load(src, lane);
  x.each(expand, lane, [&](int token, int g, int unit, const uint32_t (&w)[4]) {
    if (token >= from && token < to) store_pairs(dst + token * stride + 64 * g + 8 * unit, vec, w);
  });
}

// Zeros for `count` tokens' rows, which have no place in the cache.
template <typename T>
__device__ __forceinline__ void zero_rows(T* rows, int64_t stride, int64_t count, int d, int lane) {
  for (int64_t i = 0; i < count; ++i)
    for (int c = lane; c < d; c += 32) rows[i * stride + c] = T(0.0f);
}

// A warp takes a block of K or of V.
constexpr int READ_WARPS = 4;
template <typename T, int NG>
__global__ void __launch_bounds__(32 * READ_WARPS) kv_read_kernel(ReadParams w, bool vec) {
  grid_dependency_wait();
  allow_dependent_launch();
  const Pages& p = w.p;
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * READ_WARPS + (threadIdx.x >> 5);
  const int which = static_cast<int>(item & 1);
  const int64_t slot = (item >> 1) / p.kv_heads;
  const int head = static_cast<int>((item >> 1) - slot * p.kv_heads);
  Slot x;
  if (slot >= slots_of(w.total, p.batch) || !find_slot(p, slot, w.total, x)) return;
  const int64_t stride = which ? w.vt : w.kt;
  T* rows = which ? static_cast<T*>(w.v) + head * w.vh : static_cast<T*>(w.k) + head * w.kh;
  const int64_t page = x.to ? page_of(p, x.b, x.pos) : -1;
  if (page >= 0) {
    const uint8_t* src = p.base + page * p.page_stride + block_in_page<NG>(p, which, head, x.pos);
    if (which)
      expand_block<T, VBlock, NG>(src, rows + x.token * stride, stride, x.from, x.to, lane, vec);
    else
      expand_block<T, KBlock, NG>(src, rows + x.token * stride, stride, x.from, x.to, lane, vec);
  } else {
    zero_rows<T>(rows + (x.token + x.from) * stride, stride, x.to - x.from, 64 * NG, lane);
  }
  if (x.pos == 0) zero_rows<T>(rows + p.cu[x.b] * stride, stride, x.none, 64 * NG, lane);
}

// The checks every entry point over pages makes; fills `p`.
static int make_pages(Pages& p, const void* pages, int64_t num_pages, int64_t page_stride, int page_size,
                      int64_t kv_heads, int d, const int32_t* table, int64_t table_ld, int64_t table_cols,
                      const int32_t* cu, const int32_t* lens, int64_t batch) {
  FAQ_CHECK_ARG(pages && table && cu && lens, "null pointer");
  if (d != 64 && d != 128) return fail(FAQ_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (page_size < 16 || page_size > 4096 || (page_size & (page_size - 1)))
    return fail(FAQ_ERR_UNSUPPORTED, "page_size must be a power of two, 16 to 4096");
  FAQ_CHECK_ARG(kv_heads > 0 && kv_heads <= 65535 && num_pages > 0 && num_pages < (int64_t(1) << 31), "bad pool shape");
  FAQ_CHECK_ARG(batch > 0 && batch < (int64_t(1) << 24) && table_cols > 0 && table_ld >= table_cols, "bad table shape");
  FAQ_CHECK_ARG(table_cols * page_size < (int64_t(1) << 31), "sequences must be shorter than 2^31 tokens");
  FAQ_CHECK_ARG(aligned16(pages) && page_stride % 16 == 0, "pages must be 16-byte aligned, their stride too");
  FAQ_CHECK_ARG(page_stride >= 2 * kv_heads * (page_size / 16) * block_bytes(d / 64), "page stride below a page's bytes");
  p.base = static_cast<uint8_t*>(const_cast<void*>(pages));
  p.page_stride = page_stride;
  p.num_pages = num_pages;
  p.table = table;
  p.table_ld = table_ld;
  p.table_cols = static_cast<int>(table_cols);
  p.kv_heads = static_cast<int>(kv_heads);
  p.page_shift = 0;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.cu = cu;
  p.lens = lens;
  p.batch = static_cast<int>(batch);
  return FAQ_OK;
}

// Lets `kernel` use `bytes` of dynamic shared memory on the current device, once per device
// (`set` holds a bit per device).
static int allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& set) {
  int dev = 0;
  FAQ_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev < 64 && (set.load(std::memory_order_acquire) & bit)) return FAQ_OK;
  FAQ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) set.fetch_or(bit, std::memory_order_release);
  return FAQ_OK;
}

// A launch that may start while the kernel before it drains (its first statement waits).
template <typename... Args, typename... Given>
static cudaError_t launch_early(void (*kernel)(Args...), dim3 grid, int threads, size_t smem, void* stream,
                                Given... given) {
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, given...);
}

}  // namespace kvp
}  // namespace faq

extern "C" int faq_hif4_kv_write(const void* k, const void* v, int dtype, int64_t total, int64_t kv_heads, int d,
                                 int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                 int64_t v_head_stride, void* pages, int64_t num_pages, int64_t page_stride,
                                 int page_size, const int32_t* table, int64_t table_ld, int64_t table_cols,
                                 const int32_t* cu, const int32_t* lens, int64_t batch, int k_levels, int v_levels,
                                 void* stream) {
  using namespace faq;
  using namespace faq::kvp;
  WriteParams w;
  const int rc = make_pages(w.p, pages, num_pages, page_stride, page_size, kv_heads, d, table, table_ld, table_cols, cu,
                            lens, batch);
  if (rc) return rc;
  FAQ_CHECK_ARG(total >= 0 && total < (int64_t(1) << 31), "bad token count");
  if (total == 0) return FAQ_OK;
  FAQ_CHECK_ARG(k && v, "null pointer");
  FAQ_CHECK_ARG(dtype == FAQ_BF16 || dtype == FAQ_F32, "dtype must be FAQ_BF16 or FAQ_F32");
  for (const int lv : {k_levels, v_levels})
    FAQ_CHECK_ARG(lv == 123 || lv == 12 || lv == 13, "levels must be 123/12/13");
  w.k = k;
  w.v = v;
  w.total = total;
  w.kt = k_token_stride;
  w.kh = k_head_stride;
  w.vt = v_token_stride;
  w.vh = v_head_stride;
  w.k_levels = k_levels;
  w.v_levels = v_levels;
  const int unit = dtype == FAQ_BF16 ? 8 : 4;  // elements of 16 bytes
  const bool vec = aligned16(k) && aligned16(v) && k_token_stride % unit == 0 && k_head_stride % unit == 0 &&
                   v_token_stride % unit == 0 && v_head_stride % unit == 0;
  const int ng = d / 64;
  const int64_t blocks = (2 * slots_of(total, batch) * kv_heads + WRITE_WARPS - 1) / WRITE_WARPS;
  FAQ_CHECK_ARG(blocks < (int64_t(1) << 31), "too many tokens for one call");
  auto kern = dtype == FAQ_BF16 ? (ng == 1 ? kv_write_kernel<__nv_bfloat16, 1> : kv_write_kernel<__nv_bfloat16, 2>)
                                : (ng == 1 ? kv_write_kernel<float, 1> : kv_write_kernel<float, 2>);
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(blocks)), 32 * WRITE_WARPS, 0, stream, w, vec));
  return launch_status("kv_write_kernel");
}

extern "C" int faq_hif4_kv_read(const void* pages, int64_t num_pages, int64_t page_stride, int page_size,
                                int64_t kv_heads, int d, const int32_t* table, int64_t table_ld, int64_t table_cols,
                                const int32_t* cu, const int32_t* lens, int64_t batch, void* k, void* v, int dtype,
                                int64_t total, int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                int64_t v_head_stride, void* stream) {
  using namespace faq;
  using namespace faq::kvp;
  ReadParams w;
  const int rc = make_pages(w.p, pages, num_pages, page_stride, page_size, kv_heads, d, table, table_ld, table_cols, cu,
                            lens, batch);
  if (rc) return rc;
  FAQ_CHECK_ARG(total >= 0 && total < (int64_t(1) << 31), "bad token count");
  if (total == 0) return FAQ_OK;
  FAQ_CHECK_ARG(k && v, "null pointer");
  FAQ_CHECK_ARG(dtype == FAQ_BF16 || dtype == FAQ_F32, "dtype must be FAQ_BF16 or FAQ_F32");
  w.k = k;
  w.v = v;
  w.total = total;
  w.kt = k_token_stride;
  w.kh = k_head_stride;
  w.vt = v_token_stride;
  w.vh = v_head_stride;
  const int unit = dtype == FAQ_BF16 ? 8 : 4;
  const bool vec = aligned16(k) && aligned16(v) && k_token_stride % unit == 0 && k_head_stride % unit == 0 &&
                   v_token_stride % unit == 0 && v_head_stride % unit == 0;
  const int ng = d / 64;
  const int64_t blocks = (2 * slots_of(total, batch) * kv_heads + READ_WARPS - 1) / READ_WARPS;
  FAQ_CHECK_ARG(blocks < (int64_t(1) << 31), "too many tokens for one call");
  auto kern = dtype == FAQ_BF16 ? (ng == 1 ? kv_read_kernel<__nv_bfloat16, 1> : kv_read_kernel<__nv_bfloat16, 2>)
                                : (ng == 1 ? kv_read_kernel<float, 1> : kv_read_kernel<float, 2>);
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(blocks)), 32 * READ_WARPS, 0, stream, w, vec));
  return launch_status("kv_read_kernel");
}
