// K8 -- the HiF4 K/V cache in pages: quantizing tokens as they are written, reading them
// back as bf16 or fp32.
//
// Write: per token, kv head and 64-channel group the HiF4 fit of K1 and K4 (hif4.cuh, the same
// bits), eight channels per lane, eight lanes per group; the codes and exponents go to the
// places of the page format (include/faquant_b200.h). Every byte of the cache belongs to one
// token, so tokens are written without reading what is there.
// Read: the inverse, value = (n - 8) / 4 * 2^e * scale, exact in bf16.
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
// quarters' exponents and the group's scale byte. All lanes of the warp take part.
__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], int levels, uint32_t& ea, uint32_t& eb,
                                              uint32_t& scale) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = fabsf(v[i]);
  const float ma = fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
  const float mb = fmaxf(fmaxf(a[4], a[5]), fmaxf(a[6], a[7]));
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
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float m = hif4_code4(a[i], i < 4 ? qa : qb);
    const float n = __fadd_rn(v[i] < 0.0f ? -m : m, 8388616.0f);  // 2^23 + 8 + signed code
    word |= (__float_as_uint(n) & 15u) << (4 * i);
  }
  return word;
}

template <typename T>
__device__ __forceinline__ void load8(const T* src, bool vec, float (&v)[8]);
template <>
__device__ __forceinline__ void load8(const __nv_bfloat16* src, bool vec, float (&v)[8]) {
  if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(src[i]);
  }
}
template <>
__device__ __forceinline__ void load8(const float* src, bool vec, float (&v)[8]) {
  if (vec) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = src[i];
  }
}

template <typename T, int NG>
__global__ void __launch_bounds__(256) kv_write_kernel(WriteParams w, bool vec) {
  grid_dependency_wait();
  allow_dependent_launch();
  const Pages& p = w.p;
  constexpr int LANES = 8 * NG;  // of a token's row of one head
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = idx / LANES;
  const int64_t t = row / p.kv_heads;
  const int head = static_cast<int>(row - t * p.kv_heads);
  const int c = static_cast<int>(idx % LANES), g = c >> 3, s = c & 7;
  bool live = t < w.total;
  int pos = -1;
  int64_t page = -1;
  if (live) {
    const int b = sequence_of(p, t);
    if (b >= 0) pos = p.lens[b] - p.cu[b + 1] + static_cast<int>(t);
    if (pos >= 0) page = page_of(p, b, pos);
  }
  live = page >= 0;
  float vk[8], vv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) vk[i] = vv[i] = 0.0f;
  if (live) {
    load8<T>(static_cast<const T*>(w.k) + t * w.kt + head * w.kh + 8 * c, vec, vk);
    load8<T>(static_cast<const T*>(w.v) + t * w.vt + head * w.vh + 8 * c, vec, vv);
  }
  uint32_t ka, kb, ks, va, vb, vs;
  const uint32_t kw = quantize8(vk, w.k_levels, ka, kb, ks);
  const uint32_t vw = quantize8(vv, w.v_levels, va, vb, vs);
  // the group's exponent words: quarter a in the low half, b in the high half
  uint32_t ke = (ka | (kb << 16)) << (2 * s), ve = (va | (vb << 16)) << (2 * s);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    ke |= __shfl_xor_sync(0xffffffffu, ke, o);
    ve |= __shfl_xor_sync(0xffffffffu, ve, o);
  }
  if (!live) return;
  const int r = pos & 15, pair = r >> 1, par = r & 1;
  uint8_t* kdst = p.base + page * p.page_stride + block_in_page<NG>(p, 0, head, pos);
  uint8_t* vdst = p.base + page * p.page_stride + block_in_page<NG>(p, 1, head, pos);
  *reinterpret_cast<uint32_t*>(kdst + 32 * NG * r + (s >> 1) * 8 * NG + 8 * g + 4 * (s & 1)) = kw;
  uint16_t* vq = reinterpret_cast<uint16_t*>(vdst + 64 * NG * pair + (s ^ (2 * (pair & 3))) * 8 * NG + 8 * g + 2 * par);
  vq[0] = static_cast<uint16_t>(vw);
  vq[2] = static_cast<uint16_t>(vw >> 16);
  if (s == 0) {
    *reinterpret_cast<uint32_t*>(kdst + exp_offset(NG) + (r * NG + g) * 4) = ke;
    kdst[scale_offset(NG) + r * NG + g] = static_cast<uint8_t>(ks);
  } else if (s == 1) {
    uint16_t* vx = reinterpret_cast<uint16_t*>(vdst + exp_offset(NG) + (pair * NG + g) * 8 + 2 * par);
    vx[0] = static_cast<uint16_t>(ve);
    vx[2] = static_cast<uint16_t>(ve >> 16);
    vdst[scale_offset(NG) + r * NG + g] = static_cast<uint8_t>(vs);
  }
}

struct ReadParams {
  Pages p;
  void *k, *v;
  int64_t total, kt, kh, vt, vh;
};

template <typename T>
__device__ __forceinline__ void store8(T* dst, bool vec, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8(__nv_bfloat16* dst, bool vec, const float (&v)[8]) {
  if (vec) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = exact_bf16_bits(v[2 * i]) | (__float_as_uint(v[2 * i + 1]) & 0xFFFF0000u);
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = __float2bfloat16_rn(v[i]);
  }
}
template <>
__device__ __forceinline__ void store8(float* dst, bool vec, const float (&v)[8]) {
  if (vec) {
    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = v[i];
  }
}

template <typename T, int NG>
__global__ void __launch_bounds__(256) kv_read_kernel(ReadParams w, bool vec) {
  grid_dependency_wait();
  allow_dependent_launch();
  const Pages& p = w.p;
  constexpr int LANES = 8 * NG;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = idx / LANES;
  const int64_t t = row / p.kv_heads;
  if (t >= w.total) return;
  const int head = static_cast<int>(row - t * p.kv_heads);
  const int c = static_cast<int>(idx % LANES), g = c >> 3, s = c & 7;
  int pos = -1;
  int64_t page = -1;
  const int b = sequence_of(p, t);
  if (b >= 0) pos = p.lens[b] - p.cu[b + 1] + static_cast<int>(t);
  if (pos >= 0) page = page_of(p, b, pos);
  float vk[8], vv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) vk[i] = vv[i] = 0.0f;  // a token without a place reads as zeros
  if (page >= 0) {
    const int r = pos & 15, pair = r >> 1, par = r & 1;
    const uint8_t* ksrc = p.base + page * p.page_stride + block_in_page<NG>(p, 0, head, pos);
    const uint8_t* vsrc = p.base + page * p.page_stride + block_in_page<NG>(p, 1, head, pos);
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(ksrc + 32 * NG * r + (s >> 1) * 8 * NG + 8 * g + 4 * (s & 1));
    const uint16_t* vq =
        reinterpret_cast<const uint16_t*>(vsrc + 64 * NG * pair + (s ^ (2 * (pair & 3))) * 8 * NG + 8 * g + 2 * par);
    const uint32_t vw = vq[0] | (static_cast<uint32_t>(vq[2]) << 16);
    const uint32_t ke = *reinterpret_cast<const uint32_t*>(ksrc + exp_offset(NG) + (r * NG + g) * 4);
    const uint16_t* vx = reinterpret_cast<const uint16_t*>(vsrc + exp_offset(NG) + (pair * NG + g) * 8 + 2 * par);
    const uint32_t ve = vx[0] | (static_cast<uint32_t>(vx[2]) << 16);
    const float ks = twice_scale(ksrc[scale_offset(NG) + r * NG + g]);
    const float vs = twice_scale(vsrc[scale_offset(NG) + r * NG + g]);
    const Expand expand;
    uint32_t y[4];
    expand.word(kw, expand.exponents(ke, (7 - 2 * s) & 31), y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      vk[j] = __fmul_rn(__uint_as_float(y[j] << 16), ks);
      vk[4 + j] = __fmul_rn(__uint_as_float(y[j] & 0xFFFF0000u), ks);
    }
    expand.word(vw, expand.exponents(ve, (7 - 2 * s) & 31), y);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      vv[j] = __fmul_rn(__uint_as_float(y[j] << 16), vs);
      vv[4 + j] = __fmul_rn(__uint_as_float(y[j] & 0xFFFF0000u), vs);
    }
  }
  store8<T>(static_cast<T*>(w.k) + t * w.kt + head * w.kh + 8 * c, vec, vk);
  store8<T>(static_cast<T*>(w.v) + t * w.vt + head * w.vh + 8 * c, vec, vv);
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
  const int64_t blocks = (total * kv_heads * 8 * ng + 255) / 256;
  FAQ_CHECK_ARG(blocks < (int64_t(1) << 31), "too many tokens for one call");
  auto kern = dtype == FAQ_BF16 ? (ng == 1 ? kv_write_kernel<__nv_bfloat16, 1> : kv_write_kernel<__nv_bfloat16, 2>)
                                : (ng == 1 ? kv_write_kernel<float, 1> : kv_write_kernel<float, 2>);
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(blocks)), 256, 0, stream, w, vec));
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
  const int64_t blocks = (total * kv_heads * 8 * ng + 255) / 256;
  FAQ_CHECK_ARG(blocks < (int64_t(1) << 31), "too many tokens for one call");
  auto kern = dtype == FAQ_BF16 ? (ng == 1 ? kv_read_kernel<__nv_bfloat16, 1> : kv_read_kernel<__nv_bfloat16, 2>)
                                : (ng == 1 ? kv_read_kernel<float, 1> : kv_read_kernel<float, 2>);
  FAQ_CUDA(launch_early(kern, dim3(static_cast<unsigned>(blocks)), 256, 0, stream, w, vec));
  return launch_status("kv_read_kernel");
}
