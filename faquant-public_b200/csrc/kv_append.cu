// K11 -- appending to the HiF4 K/V cache with everything that stands between the projections and
// the cache: per new token at position p of its sequence
//
//   q' = bf16( had( rope_p( norm(q) ) * s ) ),   K = HiF4( had( (rope_p(norm(k)) - offset) / s ) ),   V = HiF4(v)
//
//   norm(x) = x / sqrt(mean x^2 + eps) * w over a head's d channels,
//   rope_p(x) = (a c - b t, b c + a t) for the halves (a, b) of x and row p of the tables (c, t),
//   had = the Hadamard transform over d (Sylvester's order) / sqrt(d),
//
// each step optional. The composition of faq_qk_norm_rope_prep and faq_hif4_kv_write rounds
// to bf16 after every step, as the modules it replaces do because they store there; here nothing is stored in
// between, so nothing is rounded: q is computed in fp32 and rounded once, and a key in fp64,
// rounded once to the fp32 that the fit of HiF4 takes. Codes jump where a value passes a border
// of the fit, so with fp32 sums a key's bits would depend on the order of their terms; from fp64
// they are those of the formula, whichever kernel writes them (drafts written again, a prompt in chunks).
//
// Mapping: eight lanes per row of a head, lane s with channels 8 s .. of each group of 64, as the
// fit wants them. The strides 1, 2, 4 of the transform are in a lane, 8, 16, 32 across lanes, 64 is
// between a lane's groups, and a half's partner is the other group's channel (d = 128) or four lanes
// away (d = 64). The first blocks of the grid take half a block of keys and values per warp as
// kv_write_kernel does, the others one token's rows of q, four at a time.
//
// Measured (one B200, 64 query heads on 8 kv heads of 128, norm, rotation, smoothing and transform):
// 8192 tokens in 99 us, 311 MB at 3.1 TB/s, half the issue slots active with 16 warps on an SM. Alone
// q takes 58 us (its bytes' time is 41) and the keys and values 44, of which fp64 some 25. Dropped: two
// launches, the queries' with fewer registers (101 to 113 us); blocks of keys spread among those of queries (105);
// 96 registers a thread (no gain, with spills). One token: 4.1 us, a launch and a chain of loads.
#include "kv_pages.cuh"

namespace faq {
namespace kvp {

struct TurnParams {
  const void *q_norm, *k_norm;  // [d] or null
  bool norm_f32;                // fp32, else bf16
  double eps;
  const void *cos, *sin;        // [rope_rows, >= d / 2] or null
  bool rope_f32;
  int64_t rope_ld, rope_rows;
  const float* offset;          // [kv_heads, d] or null
  const float* smooth;          // [d] or [kv_heads, d] or null
  int64_t smooth_head_stride;
  bool rotate;
};

struct AppendParams {
  WriteParams w;
  TurnParams t;
  const void* q;
  int64_t qt, qh;  // token, head strides
  __nv_bfloat16* out;
  int64_t ot, oh;
  int heads, group;  // query heads, per kv head
  int hpw;           // query heads of a warp's item
  int64_t kv_blocks; // blocks of the grid that write K and V
};

// Eight consecutive entries of a table, fp32 or bf16.
__device__ __forceinline__ void load8(const void* base, bool f32, int64_t at, float (&v)[8]) {
  if (f32) {
    const float* p = static_cast<const float*>(base) + at;
    Raw<float> r;
    r.load(p, (reinterpret_cast<uintptr_t>(p) & 15) == 0);
    r.values(v);
  } else {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(base) + at;
    Raw<__nv_bfloat16> r;
    r.load(p, (reinterpret_cast<uintptr_t>(p) & 15) == 0);
    r.values(v);
  }
}

// A row's position-dependent entries of one lane.
struct Angles {
  float c[8], s[8];
  __device__ __forceinline__ void load(const TurnParams& t, int64_t pos, int s_, int ng) {
    const int64_t at = pos * t.rope_ld + 8 * (ng == 2 ? s_ : s_ & 3);
    load8(t.cos, t.rope_f32, at, c);
    load8(t.sin, t.rope_f32, at, s);
  }
};

// 1 / w in fp64 to 2^-47, w a normal number: a Newton's step from the fp32 reciprocal (a key is rounded to 2^-24).
// The step is on the reciprocal, not on a quotient, so that an infinite key stays infinite.
__device__ __forceinline__ double reciprocal(float w) {
  const double r = __frcp_rn(w);
  return fma(fma(-static_cast<double>(w), r, 1.0), r, r);
}

// A key: norm, rotation, offset, smoothing and transform of the lane's part of a row in fp64; all
// lanes take part.
template <int NG>
__device__ __forceinline__ void turn_key(float (&v)[NG][8], const TurnParams& t, const Angles& a, int head, int s) {
  constexpr int D = 64 * NG;
  double x[NG][8], factor = 1.0;  // the norm's, which waits for the transform's: the steps between are linear
  if (t.k_norm != nullptr) {
    double sum = 0;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float w[8];
      load8(t.k_norm, t.norm_f32, 64 * g + 8 * s, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double y = v[g][i];
        sum = fma(y, y, sum);
        x[g][i] = y * w[i];  // in fp64 for bf16 too: the product of two may leave fp32's range, and the norm bring it back
      }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    factor = rsqrt(sum * (1.0 / D) + t.eps);
  } else {
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[g][i] = v[g][i];
  }
  if (t.cos != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double c = a.c[i], n = a.s[i];
      if constexpr (NG == 2) {
        const double u = x[0][i], v = x[1][i];
        x[0][i] = u * c - v * n;
        x[1][i] = v * c + u * n;
      } else {
        const double other = __shfl_xor_sync(0xffffffffu, x[0][i], 4);
        x[0][i] = x[0][i] * c + (s & 4 ? other : -other) * n;
      }
    }
  }
  if (t.offset != nullptr) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float w[8];
      load8(t.offset, true, head * D + 64 * g + 8 * s, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[g][i] = fma(x[g][i], factor, -static_cast<double>(w[i]));
    }
    factor = 1.0;
  }
  if (t.smooth != nullptr) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float w[8];
      load8(t.smooth, true, head * t.smooth_head_stride + 64 * g + 8 * s, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[g][i] *= reciprocal(w[i]);
    }
  }
  if (t.rotate) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int d = 1; d < 8; d <<= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if ((i & d) == 0) {
            const double u = x[g][i], v = x[g][i + d];
            x[g][i] = u + v;
            x[g][i + d] = u - v;
          }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const double sign = (s & o) ? -1.0 : 1.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[g][i] = fma(x[g][i], sign, __shfl_xor_sync(0xffffffffu, x[g][i], o));
      }
    }
    if constexpr (NG == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double u = x[0][i], w = x[1][i];
        x[0][i] = u + w;
        x[1][i] = u - w;
      }
    }
    factor *= NG == 2 ? 0.08838834764831843 : 0.125;  // 1 / sqrt(d)
  }
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[g][i] = __double2float_rn(x[g][i] * factor);
}

// A query: what a token's rows have in common is multiplied together once, weight times cosine or sine
// times smoothing (where that is one for all heads): out = x * own + partner * other, partner the same
// channel of the other half. The norm's factor waits for the transform's, both linear.
template <int NG>
struct QueryTurn {
  float2 own[NG][4], other[NG][4];
  __device__ __forceinline__ void make(const TurnParams& t, int64_t pos, int s) {
    Angles a;
    if (t.cos != nullptr) a.load(t, pos, s, NG);
    float w[NG][8], m[NG][8];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) w[g][i] = m[g][i] = 1.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if (t.q_norm != nullptr) load8(t.q_norm, t.norm_f32, 64 * g + 8 * s, w[g]);
      if (t.smooth != nullptr && t.smooth_head_stride == 0) load8(t.smooth, true, 64 * g + 8 * s, m[g]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool low = NG == 2 ? g == 0 : s < 4;
        float partner;  // its weight
        if constexpr (NG == 2) partner = w[1 - g][i]; else partner = __shfl_xor_sync(0xffffffffu, w[0][i], 4);
        const float c = t.cos != nullptr ? a.c[i] : 1.0f, n = t.cos != nullptr ? a.s[i] : 0.0f;
        const float x = w[g][i] * c * m[g][i], y = (low ? -partner : partner) * n * m[g][i];
        if (i & 1) {
          own[g][i >> 1].y = x;
          other[g][i >> 1].y = y;
        } else {
          own[g][i >> 1].x = x;
          other[g][i >> 1].x = y;
        }
      }
  }
  __device__ __forceinline__ void apply(float2 (&x)[NG][4], const TurnParams& t, int h, int group, int s) const {
    constexpr int D = 64 * NG;
    float r = 1.0f;
    if (t.q_norm != nullptr) {
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = __ffma2_rn(x[g][i], x[g][i], sum);
      float ss = sum.x + sum.y;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      r = rsqrtf(ss * (1.0f / D) + static_cast<float>(t.eps));
    }
    if (t.cos != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (NG == 2) {
          const float2 u = x[0][i], v = x[1][i];
          x[0][i] = __ffma2_rn(u, own[0][i], __fmul2_rn(v, other[0][i]));
          x[1][i] = __ffma2_rn(v, own[1][i], __fmul2_rn(u, other[1][i]));
        } else {
          const float2 v = make_float2(__shfl_xor_sync(0xffffffffu, x[0][i].x, 4), __shfl_xor_sync(0xffffffffu, x[0][i].y, 4));
          x[0][i] = __ffma2_rn(x[0][i], own[0][i], __fmul2_rn(v, other[0][i]));
        }
      }
    } else {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[g][i] = __fmul2_rn(x[g][i], own[g][i]);
    }
    if (t.smooth_head_stride != 0) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float m[8];
        load8(t.smooth, true, h / group * t.smooth_head_stride + 64 * g + 8 * s, m);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[g][i] = __fmul2_rn(x[g][i], make_float2(m[2 * i], m[2 * i + 1]));
      }
    }
    if (t.rotate) {
      const float2 minus = make_float2(-1.0f, -1.0f);
#pragma unroll
      for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[g][i] = make_float2(x[g][i].x + x[g][i].y, x[g][i].x - x[g][i].y);
#pragma unroll
        for (int d = 1; d < 4; d <<= 1)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((i & d) == 0) {
              const float2 u = x[g][i], v = x[g][i + d];
              x[g][i] = __fadd2_rn(u, v);
              x[g][i + d] = __ffma2_rn(v, minus, u);
            }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
          const float sign = (s & o) ? -1.0f : 1.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = make_float2(__shfl_xor_sync(0xffffffffu, x[g][i].x, o), __shfl_xor_sync(0xffffffffu, x[g][i].y, o));
            x[g][i] = __ffma2_rn(x[g][i], make_float2(sign, sign), v);
          }
        }
      }
      if constexpr (NG == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 u = x[0][i], v = x[1][i];
          x[0][i] = __fadd2_rn(u, v);
          x[1][i] = __ffma2_rn(v, minus, u);
        }
      }
      r *= NG == 2 ? 0.08838834764831843f : 0.125f;  // 1 / sqrt(d)
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[g][i] = __fmul2_rn(x[g][i], make_float2(r, r));
  }
};

template <typename T, int NG>
__global__ void __launch_bounds__(32 * WRITE_WARPS) kv_append_kernel(AppendParams a, bool vec, bool out_vec) {
  grid_dependency_wait();
  allow_dependent_launch();
  const WriteParams& w = a.w;
  const Pages& p = w.p;
  const TurnParams& t = a.t;
  const int lane = threadIdx.x & 31, s = lane & 7;
  if (blockIdx.x < a.kv_blocks) {
    const int64_t item = static_cast<int64_t>(blockIdx.x) * WRITE_WARPS + (threadIdx.x >> 5);
    const int h = static_cast<int>(item & 1);
    const int64_t slot = (item >> 1) / p.kv_heads;
    const int head = static_cast<int>((item >> 1) - slot * p.kv_heads);
    Slot x;
    if (slot >= slots_of(w.total, p.batch) || !find_slot(p, slot, w.total, x)) return;  // warp-uniform
    if (t.cos != nullptr && x.pos + x.to > t.rope_rows) {  // tokens beyond the tables are not written
      atomicOr(&g_status, FAQ_STATUS_BAD_BOUND);
      x.to = static_cast<int>(t.rope_rows > x.pos ? t.rope_rows - x.pos : 0);
    }
    if (x.from >= 8 * (h + 1) || x.to <= 8 * h || x.from >= x.to) return;
    const int64_t page = page_of(p, x.b, x.pos);
    if (page < 0) return;
    write_half_block<T, NG>(w, x, h, lane, static_cast<const T*>(w.k) + x.token * w.kt + head * w.kh + 8 * s,
                            static_cast<const T*>(w.v) + x.token * w.vt + head * w.vh + 8 * s,
                            p.base + page * p.page_stride + block_in_page<NG>(p, 0, head, x.pos),
                            p.base + page * p.page_stride + block_in_page<NG>(p, 1, head, x.pos), vec,
                            [&](float (&v)[NG][8], int r) {
                              if (t.k_norm == nullptr && t.cos == nullptr && t.offset == nullptr && t.smooth == nullptr && !t.rotate)
                                return;
                              Angles ang;
                              if (t.cos != nullptr) ang.load(t, x.pos + min(max(r, x.from), x.to - 1), s, NG);
                              turn_key<NG>(v, t, ang, head, s);
                            });
    return;
  }
  // ---- q: heads h0 .. of one token, four at a time
  const int64_t items = (a.heads + a.hpw - 1) / a.hpw;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) - a.kv_blocks) * WRITE_WARPS + (threadIdx.x >> 5);
  const int64_t token = item / items;
  if (token >= w.total) return;
  int b;
  int64_t pos;
  if (!find_token(p, token, w.total, b, pos)) return;  // reported where its keys would be written
  const int h_begin = static_cast<int>(item - token * items) * a.hpw, h_end = min(h_begin + a.hpw, a.heads);
  const bool placed = pos >= 0 && (t.cos == nullptr || pos < t.rope_rows);
  __nv_bfloat16* out_row = a.out + token * a.ot + 8 * s;
  if (!placed) {
    const uint32_t zero[4] = {0, 0, 0, 0};
    for (int h = h_begin + (lane >> 3); h < h_end; h += 4)
#pragma unroll
      for (int g = 0; g < NG; ++g) store_pairs(out_row + h * a.oh + 64 * g, out_vec, zero);
    return;
  }
  QueryTurn<NG> turn;
  turn.make(t, pos, s);
  const T* row = static_cast<const T*>(a.q) + token * a.qt + 8 * s;
  Raw<T> raw[NG];
  auto load = [&](int h0) {  // rows past the last head repeat it, unstored
    const T* src = row + min(h0 + (lane >> 3), h_end - 1) * a.qh;
#pragma unroll
    for (int g = 0; g < NG; ++g) raw[g].load(src + 64 * g, vec);
  };
  load(h_begin);
  for (int h0 = h_begin; h0 < h_end; h0 += 4) {
    const int h = min(h0 + (lane >> 3), h_end - 1);
    float2 x[NG][4];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float v[8];
      raw[g].values(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[g][i] = make_float2(v[2 * i], v[2 * i + 1]);
    }
    if (h0 + 4 < h_end) load(h0 + 4);
    turn.apply(x, t, h, a.group, s);
    if (h0 + (lane >> 3) >= h_end) continue;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[g][i].x, x[g][i].y);
        o[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
      store_pairs(out_row + h * a.oh + 64 * g, out_vec, o);
    }
  }
}

}  // namespace kvp
}  // namespace faq

extern "C" int faq_hif4_kv_append(const void* q, const void* k, const void* v, int dtype, int64_t total, int64_t heads,
                                  int64_t kv_heads, int d, int64_t q_token_stride, int64_t q_head_stride,
                                  int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                  int64_t v_head_stride, const void* q_norm, const void* k_norm, int norm_dtype,
                                  double eps, const void* cos, const void* sin, int rope_dtype, int64_t rope_ld,
                                  int64_t rope_rows, const float* key_offset, const float* smooth,
                                  int64_t smooth_head_stride, int rotate, void* out, int64_t out_token_stride,
                                  int64_t out_head_stride, void* pages, int64_t num_pages, int64_t page_stride,
                                  int page_size, const int32_t* table, int64_t table_ld, int64_t table_cols,
                                  const int32_t* cu, const int32_t* lens, int64_t batch, int k_levels, int v_levels,
                                  void* stream) {
  using namespace faq;
  using namespace faq::kvp;
  AppendParams a;
  WriteParams& w = a.w;
  const int rc = make_pages(w.p, pages, num_pages, page_stride, page_size, kv_heads, d, table, table_ld, table_cols, cu,
                            lens, batch);
  if (rc) return rc;
  FAQ_CHECK_ARG(total >= 0 && total < (int64_t(1) << 31), "bad token count");
  FAQ_CHECK_ARG(heads > 0 && heads < (int64_t(1) << 24) && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  if (total == 0) return FAQ_OK;
  FAQ_CHECK_ARG(q && k && v && out, "null pointer");
  FAQ_CHECK_ARG(dtype == FAQ_BF16 || dtype == FAQ_F32, "dtype must be FAQ_BF16 or FAQ_F32");
  FAQ_CHECK_ARG((norm_dtype == FAQ_BF16 || norm_dtype == FAQ_F32) && (rope_dtype == FAQ_BF16 || rope_dtype == FAQ_F32),
                "dtype of a table must be FAQ_BF16 or FAQ_F32");
  FAQ_CHECK_ARG((cos == nullptr) == (sin == nullptr), "cos and sin go together");
  FAQ_CHECK_ARG(cos == nullptr || (rope_ld >= d / 2 && rope_rows > 0), "cos and sin must be [positions, >= d / 2]");
  FAQ_CHECK_ARG((q_norm == nullptr && k_norm == nullptr) || (eps >= 0.0 && eps < 1e30), "eps must not be negative");
  FAQ_CHECK_ARG(smooth_head_stride == 0 || smooth_head_stride == d, "smooth is [d] or [kv_heads, d]");
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
  a.t = {q_norm, k_norm, norm_dtype == FAQ_F32, eps, cos, sin, rope_dtype == FAQ_F32, rope_ld, rope_rows,
         key_offset, smooth, smooth ? smooth_head_stride : 0, rotate != 0};
  a.q = q;
  a.qt = q_token_stride;
  a.qh = q_head_stride;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ot = out_token_stride;
  a.oh = out_head_stride;
  a.heads = static_cast<int>(heads);
  a.group = static_cast<int>(heads / kv_heads);
  const int unit = dtype == FAQ_BF16 ? 8 : 4;  // elements of 16 bytes
  bool vec = aligned16(q) && aligned16(k) && aligned16(v);
  for (const int64_t st : {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride})
    vec = vec && st % unit == 0;
  const bool out_vec = aligned16(out) && out_token_stride % 8 == 0 && out_head_stride % 8 == 0;
  const int ng = d / 64;
  a.kv_blocks = (2 * slots_of(total, batch) * kv_heads + WRITE_WARPS - 1) / WRITE_WARPS;
  // a warp takes more of a token's heads where there are more items than the SMs hold at once
  const int64_t iters = (heads + 3) / 4, resident = static_cast<int64_t>(num_sms()) * 32;
  a.hpw = 4 * static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(iters, total * iters / resident)));
  const int64_t q_blocks = (total * ((heads + a.hpw - 1) / a.hpw) + WRITE_WARPS - 1) / WRITE_WARPS;
  FAQ_CHECK_ARG(a.kv_blocks + q_blocks < (int64_t(1) << 31), "too many tokens for one call");
  auto kern = dtype == FAQ_BF16 ? (ng == 1 ? kv_append_kernel<__nv_bfloat16, 1> : kv_append_kernel<__nv_bfloat16, 2>)
                                : (ng == 1 ? kv_append_kernel<float, 1> : kv_append_kernel<float, 2>);
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(a.kv_blocks + q_blocks)), 32 * WRITE_WARPS, 0, stream, a, vec,
                        out_vec));
  return launch_status("kv_append_kernel");
}
