// K10 -- verification of drafted tokens (speculative sampling): draft i of a sequence is
// accepted while u_i q_i(x_i) < p_i(x_i); at the first rejection the next token is drawn from
// max(p - q, 0) (from p without the drafted token when there is no draft distribution), after
// the last acceptance from p. The drawn token is the first j with sum_{i <= j} w_i > u sum w.
//
// The sums run over whole numbers, w = rint(2^40 min(r, 1)) of the fp32 weight r, so they do
// not depend on the order of the additions: the same token on every call, for every split of
// the vocabulary. 2^-40 is far below fp32's own step for a weight that matters, and 2^22
// weights fit 64 bits. The threshold u sum w is one fp64 product.
//
// Bound by reading one row of p and q per sequence; a small batch by its round trips. A
// cluster of one to eight CTAs takes a sequence: every warp sums its own contiguous piece (the loads
// of four steps in flight), the CTAs' sums meet through distributed shared memory, and the CTA
// whose part holds the threshold reads that warp's piece again (from L2), a step per warp,
// to find the token. The target's own weights are summed only when nothing is left over.
#include "common.cuh"

namespace faq {
namespace ver {

constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int STEP = 128;  // weights a warp takes at a time, four per lane

struct Params {
  const int64_t* draft;  // [batch, k]
  const void *target, *drafter;  // [batch, k + 1, vocab], [batch, k, vocab] or null
  int64_t tb, ts, qb, qs;        // batch and step strides (elements)
  const float *accept_u, *sample_u;
  const int32_t* count;  // [batch] or null
  int64_t* tokens;       // [batch, k + 1]
  int32_t* accepted;     // [batch]
  int k;
  int64_t vocab;
  bool vec;
  int cluster;  // CTAs per sequence
};

// CTAs per sequence: as many (up to 8) as fill the GPU's two CTAs per SM once. More than that
// run in waves whose gathers and joins leave the memory idle: 128 sequences of 151936 fp32
// weights and their draft distributions took 43 us with clusters of 8, 28.8 with 2.
inline int cluster_of(int64_t batch) {
  int c = 8;
  while (c > 1 && batch * c > 2 * num_sms()) c /= 2;
  return c;
}

__device__ __forceinline__ float load1(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float load1(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xFFFF0000u);
  v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xFFFF0000u);
}

// rint(2^40 min(max(r, 0), 1)) as hi 2^20 + lo (0 for NaN): x = 2^20 r; x + 2^23 rounded
// toward zero is 2^23 + floor(x), the rest is exact, and 2^20 times it rounds to the nearest
// whole number (ties to even, as hi 2^20 is even) when 2^23 is added.
struct Weight {
  uint32_t hi, lo;
};
__device__ __forceinline__ Weight weight(float r) {
  const float x = __fmul_rn(fminf(fmaxf(r, 0.0f), 1.0f), 1048576.0f);
  const float f = __fadd_rz(x, 8388608.0f);
  const float rest = __fsub_rn(x, __fsub_rn(f, 8388608.0f));
  const float g = __fadd_rn(__fmul_rn(rest, 1048576.0f), 8388608.0f);
  return {__float_as_uint(f) - 0x4B000000u, __float_as_uint(g) - 0x4B000000u};
}
__device__ __forceinline__ uint64_t join(Weight w) { return (static_cast<uint64_t>(w.hi) << 20) + w.lo; }

template <typename T>
struct Rows {
  const T *p, *q;  // q null: no subtraction
  int64_t vocab, dropped;  // the token whose weight is 0 (-1: none)
  bool vec;
  // the weights of entries at .. at + 3
  __device__ __forceinline__ void get(int64_t at, float (&r)[4]) const {
    float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (vec && at + 4 <= vocab) {
      load4(p + at, r);
      if (q) load4(q + at, b);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r[i] = at + i < vocab ? load1(p, at + i) : 0.0f;
        if (q && at + i < vocab) b[i] = load1(q, at + i);
      }
    }
    take(at, r, b);
  }
  __device__ __forceinline__ void take(int64_t at, float (&r)[4], const float (&b)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = at + i == dropped ? 0.0f : __fsub_rn(r[i], b[i]);
  }
};

__device__ __forceinline__ uint64_t sum4(const float (&r)[4]) {
  uint32_t hi = 0, lo = 0;  // four weights of at most 2^20 each
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Weight w = weight(r[i]);
    hi += w.hi;
    lo += w.lo;
  }
  return join({hi, lo});
}

// This lane's part of the sum over steps s0 .. s1 - 1 of the row. Q: there is a draft row.
template <typename T, bool Q>
__device__ __forceinline__ uint64_t sum_steps(const Rows<T>& rows, int64_t s0, int64_t s1, int lane) {
  constexpr int AHEAD = 4;
  uint64_t sum = 0;
  int64_t s = s0;
  if (rows.vec) {
    for (; s + AHEAD <= s1 && (s + AHEAD) * STEP <= rows.vocab; s += AHEAD) {
      float r[AHEAD][4], b[AHEAD][4];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        load4(rows.p + (s + i) * STEP + lane * 4, r[i]);
        if constexpr (Q) load4(rows.q + (s + i) * STEP + lane * 4, b[i]);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if constexpr (!Q) b[i][0] = b[i][1] = b[i][2] = b[i][3] = 0.0f;
        rows.take((s + i) * STEP + lane * 4, r[i], b[i]);
        sum += sum4(r[i]);
      }
    }
  }
  for (; s < s1; ++s) {
    float r[4];
    rows.get(s * STEP + lane * 4, r);
    sum += sum4(r);
  }
  return sum;
}

__device__ __forceinline__ uint64_t warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) verify_kernel(Params P) {
  __shared__ uint64_t s_warp[WARPS], s_step[WARPS];
  __shared__ uint64_t s_cta[2];  // of the residual, then of the target's row
  __shared__ int s_first;
  grid_dependency_wait();
  allow_dependent_launch();
  const int b = blockIdx.x / P.cluster, rank = blockIdx.x % P.cluster;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* target = static_cast<const T*>(P.target) + b * P.tb;
  const T* drafter = P.drafter ? static_cast<const T*>(P.drafter) + b * P.qb : nullptr;
  const int64_t* draft = P.draft + static_cast<int64_t>(b) * P.k;
  const int count = P.count ? min(max(P.count[b], 0), P.k) : P.k;
  if (tid == 0) s_first = count;
  __syncthreads();
  for (int i = tid; i < count; i += THREADS) {
    const int64_t x = draft[i];
    bool good = false;
    if (x >= 0 && x < P.vocab) {
      const float q = drafter ? load1(drafter + i * P.qs, x) : 1.0f;
      good = __fmul_rn(P.accept_u[static_cast<int64_t>(b) * P.k + i], q) < load1(target + i * P.ts, x);
    }
    if (!good) atomicMin(&s_first, i);
  }
  __syncthreads();
  const int n = s_first;  // accepted drafts
  Rows<T> rows;
  rows.p = target + n * P.ts;
  rows.q = n < count && drafter ? drafter + n * P.qs : nullptr;
  rows.dropped = n < count && !drafter ? draft[n] : -1;
  rows.vocab = P.vocab;
  rows.vec = P.vec;

  // each warp's piece: whole steps, in the order (rank, warp)
  const int64_t steps = (P.vocab + STEP - 1) / STEP;
  const int64_t each = (steps + P.cluster * WARPS - 1) / (P.cluster * WARPS);
  const int64_t s0 = (rank * WARPS + warp) * each, s1 = min(steps, s0 + each);
  uint64_t total = 0, before = 0;
  auto sum_row = [&](int use) {  // the row's total, and what stands before this CTA's part
    const uint64_t mine = warp_sum(rows.q ? sum_steps<T, true>(rows, s0, s1, lane) : sum_steps<T, false>(rows, s0, s1, lane));
    if (lane == 0) s_warp[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      uint64_t sum = 0;
      for (int w = 0; w < WARPS; ++w) sum += s_warp[w];
      s_cta[use] = sum;
    }
    __syncthreads();
    cluster_sync();
    total = before = 0;
#pragma unroll 1
    for (int r = 0; r < P.cluster; ++r) {
      uint64_t v;
      asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_addr(&s_cta[use]), r)));
      total += v;
      if (r < rank) before += v;
    }
  };
  sum_row(0);
  if (total == 0) {  // nothing left over: the target's own row
    rows.q = nullptr;
    rows.dropped = -1;
    sum_row(1);
  }
  cluster_sync();  // no CTA leaves while its sums are read
  int64_t* tokens = P.tokens + static_cast<int64_t>(b) * (P.k + 1);
  if (rank == 0) {
    for (int i = tid; i <= P.k; i += THREADS)
      if (i != n) tokens[i] = i < n ? draft[i] : -1;
    if (tid == 0) {
      P.accepted[b] = n;
      if (total == 0) tokens[n] = -1;  // no mass at all
    }
  }
  if (total == 0) return;
  // u in [0, 1): below it by construction; anything else is brought there (NaN to 0)
  const float u = fminf(fmaxf(P.sample_u[b], 0.0f), 0.99999994f);
  const double at = __dmul_rn(static_cast<double>(u), __ull2double_rn(total));
  auto past = [&](uint64_t sum) { return __ull2double_rn(sum) > at; };
  // the warp of this CTA whose piece passes the threshold (the same for all threads)
  uint64_t start = before;
  int owner = -1;
  if (!past(start)) {
    for (int w = 0; w < WARPS; ++w) {
      if (past(start + s_warp[w])) {
        owner = w;
        break;
      }
      start += s_warp[w];
    }
  }
  if (owner < 0) return;
  const int64_t f0 = (rank * WARPS + owner) * each, f1 = min(steps, f0 + each);
  for (int64_t s = f0; s < f1; s += WARPS) {  // a step per warp
    float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t at4 = (s + warp) * STEP + lane * 4;
    if (s + warp < f1) rows.get(at4, r);
    uint64_t v[4], mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine += v[i] = join(weight(r[i]));
    uint64_t x = mine;  // inclusive prefix over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_step[warp] = x;
    __syncthreads();
    uint64_t mine0 = start;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) mine0 += s_step[w];
      start += s_step[w];
    }
    // past() grows along the row: the first lane of the first warp that passes
    const uint32_t here = __ballot_sync(0xffffffffu, past(mine0 + x));
    if (!past(mine0) && here && lane == __ffs(here) - 1) {
      uint64_t c = mine0 + x - mine;
      int i = 0;
      for (; i < 3; ++i) {
        c += v[i];
        if (past(c)) break;
      }
      tokens[n] = at4 + i;
    }
    if (past(start)) return;  // CTA-uniform
    __syncthreads();
  }
}

}  // namespace ver
}  // namespace faq

extern "C" int faq_verify_drafts(const int64_t* draft_tokens, const void* target_probs, const void* draft_probs,
                                 int dtype, int64_t batch, int64_t k, int64_t vocab, int64_t target_batch_stride,
                                 int64_t target_step_stride, int64_t draft_batch_stride, int64_t draft_step_stride,
                                 const float* accept_u, const float* sample_u, const int32_t* num_drafts,
                                 int64_t* tokens, int32_t* accepted, void* stream) {
  using namespace faq;
  using namespace faq::ver;
  FAQ_CHECK_ARG(batch >= 0 && batch <= (int64_t(1) << 27) && k >= 0 && k <= 4096, "bad batch or draft count (at most 4096)");
  FAQ_CHECK_ARG(vocab > 0 && vocab <= (int64_t(1) << 22), "vocab must be 1 to 2^22");
  FAQ_CHECK_ARG(dtype == FAQ_BF16 || dtype == FAQ_F32, "dtype must be FAQ_BF16 or FAQ_F32");
  if (batch == 0) return FAQ_OK;
  FAQ_CHECK_ARG(target_probs && sample_u && tokens && accepted && (k == 0 || (draft_tokens && accept_u)), "null pointer");
  Params P;
  P.draft = draft_tokens;
  P.target = target_probs;
  P.drafter = draft_probs;
  P.tb = target_batch_stride;
  P.ts = target_step_stride;
  P.qb = draft_batch_stride;
  P.qs = draft_step_stride;
  P.accept_u = accept_u;
  P.sample_u = sample_u;
  P.count = num_drafts;
  P.tokens = tokens;
  P.accepted = accepted;
  P.k = static_cast<int>(k);
  P.vocab = vocab;
  P.vec = aligned16(target_probs) && aligned16(draft_probs) && target_batch_stride % 4 == 0 &&
          target_step_stride % 4 == 0 && draft_batch_stride % 4 == 0 && draft_step_stride % 4 == 0;
  P.cluster = cluster_of(batch);
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = static_cast<unsigned>(P.cluster);
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * P.cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attrs;
  cfg.numAttrs = 2;
  FAQ_CUDA(cudaLaunchKernelEx(&cfg, dtype == FAQ_BF16 ? verify_kernel<__nv_bfloat16> : verify_kernel<float>, P));
  return launch_status("verify_kernel");
}
