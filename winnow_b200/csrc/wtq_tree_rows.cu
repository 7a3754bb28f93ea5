// The two products with a rotation either side of a tree scan, on the tensor cores, head_dim 64 or 128:
// queries into the key basis (q_rot = q_scale * q Pi_K^T) and joined states out of the value basis
// (out = a Pi_V, a = sum_c w_c acc_c / sum_c w_c l_c).
//
// Up to 128 rows a block, one accumulator.  Both factors are split into fp16 high and low parts and three
// products summed in fp32, which leaves 2^-22 of the result as error, the class of an fp32 product
// (16-bit queries have no low part: two products; neither do states that leave as bf16, whose rounding is
// eight times that of the fp16 high part).  A row is scaled by a power of two to its largest
// element first, and Pi to 2^8 times its own, so that any matrix fits and low parts stay clear of fp16's subnormal range.  Pi is laid out
// as the operand once and serves both: read along its rows for the queries (K-major), across them for
// the states (MN-major).  A thread per row quarter converts and stores.  Bound by the reads of rows and of
// Pi from L2: 13 and 21 us from a cold cache at 16 384 rows, where the CUDA-core kernels of wtq_tree.cu
// take 187 and 70.
#include <algorithm>
#include <atomic>

#include "wtq_tree.cuh"
#include "wtq_umma.cuh"

namespace wtq {
namespace tree {
namespace rows {

using namespace umma;

constexpr int kThreads = 512, kRows = 128;
constexpr int kWaitTries = 1 << 20;
constexpr float kPiScale = 256.f;

template <int D> struct Map {
  static constexpr uint32_t kGroup = (uint32_t)D * 16u;     // eight rows of an operand
  static constexpr uint32_t kScales = 1024;                 // a row's power of two
  static constexpr uint32_t kBar = kScales + 4 * kRows, kSlot = kBar + 8, kMostPi = kSlot + 8, kPrefix = kMostPi + 4 * (kThreads / 32);
  static constexpr uint32_t kA = 10240, kABytes = kRows / 8 * kGroup, kBBytes = D / 8 * kGroup;
  static constexpr uint32_t kB = kA + kABytes, kALow = kB + 2 * kBBytes;     // the rows' low parts, where there are any
  static constexpr uint32_t kBytes = kALow + kABytes;
  static_assert(kPrefix + 4 * (kMaxBatch + 1) <= kA, "low region");
  static constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
};

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// Eight values as fp16 high parts at `at`, what they leave as low parts at `at` + `low` (0: dropped).
__device__ __forceinline__ void store_split(uint32_t at, uint32_t low, const float (&x)[8]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = half2_bits(x[2 * i], x[2 * i + 1]);
    const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
    l[i] = half2_bits(x[2 * i] - back.x, x[2 * i + 1] - back.y);
  }
  sts128(at, h[0], h[1], h[2], h[3]);
  if (low) sts128(at + low, l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ void sts_float(uint32_t a, float v) {
  asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ float lds_float(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(a));
  return v;
}
// The largest power of two not above |x|'s, and its inverse (1 for zeros and what is not finite).
__device__ __forceinline__ float power_of(float x, float &inverse) {
  const uint32_t e = __float_as_uint(x) >> 23 & 255u;
  const bool plain = e >= 2 && e <= 252;
  inverse = plain ? __uint_as_float((254u - e) << 23) : 1.f;
  return plain ? __uint_as_float(e << 23) : 1.f;
}

__device__ __forceinline__ void place(const Params &p, int64_t row_, int &b, int &i, int &h) {
  const uint32_t row = (uint32_t)row_, t = row / (uint32_t)p.Hq;       // (fewer than 2^31 rows)
  h = (int)(row - t * (uint32_t)p.Hq);
  b = (int)(t / (uint32_t)p.Q);
  i = (int)(t - (uint32_t)b * (uint32_t)p.Q);
}
// x / share of tile numbers, in 32 bits where they fit
__device__ __forceinline__ int run_of(long long x, long long share) {
  return ((x | share) >> 31) == 0 ? (int)((uint32_t)x / (uint32_t)share) : (int)(x / share);
}

template <bool JOIN, int D, bool WIDE>
__global__ void __launch_bounds__(kThreads, WIDE ? 1 : 2) product_kernel(Params p, int terms, int rows_per) {
  using M = Map<D>;
  extern __shared__ __align__(1024) uint8_t dyn_smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(dyn_smem);
  if (base > 1024u) {
    if (p.status && tid == 0) atomicOr(p.status, WTQ_STATUS_LAYOUT);
    return;
  }
  constexpr int kPieces = D / 8;
  const float *Pi = JOIN ? p.v.Pi : p.k.Pi;
  constexpr int kPi = D * kPieces / kThreads;              // pieces of Pi of a thread
  float4 pi[kPi][2];
  {
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < kPi; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float4 a = pi[k][h] = __ldg(reinterpret_cast<const float4 *>(Pi + 8 * (tid + k * kThreads)) + h);
        most = fmaxf(fmaxf(most, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(a.z), fabsf(a.w)));
      }
    const uint32_t of_warp = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    if (lane == 0) sts_float(M::kMostPi + 4u * warp, __uint_as_float(of_warp));
  }
  auto take_columns = [&] {
    if (warp == 0) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(M::kSlot), "r"((uint32_t)D)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
  };
  if constexpr (!JOIN) take_columns();
  if (tid == 0) {
    mbar_init(M::kBar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  int *prefix = reinterpret_cast<int *>(dyn_smem + (M::kPrefix - base));
  long long share = 1;
  if constexpr (JOIN) {
    tile_prefix(p, prefix);                                 // (ends with a block barrier)
  } else {
    __syncthreads();
    // Only now that this block has its tensor memory: a block of the scan that took all of it first would
    // wait for this kernel while this block waited for it.
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  }
  float most_pi = 0.f, inverse_pi;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) most_pi = fmaxf(most_pi, lds_float(M::kMostPi + 4u * w));
  const float power_pi = power_of(most_pi, inverse_pi);
#pragma unroll
  for (int k = 0; k < kPi; ++k) {
    const int row = (tid + k * kThreads) / kPieces, piece = (tid + k * kThreads) % kPieces;
    const float4 a = pi[k][0], b = pi[k][1];
    float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * inverse_pi * kPiScale;
    store_split(M::kB + (uint32_t)(row >> 3) * M::kGroup + (uint32_t)piece * 128u + (uint32_t)(row & 7) * 16u, M::kBBytes, x);
  }
  if constexpr (JOIN) {
    share = run_length(p, prefix);
    take_columns();                                         // (which the scan's blocks give back at their end)
    asm volatile("griddepcontrol.wait;\n" ::: "memory");   // the states
  }
  // ---- the rows: kPieces lanes a row, several rows of a warp at a time ------------------------------
  const int64_t row0 = (int64_t)blockIdx.x * rows_per, rows = min((int64_t)p.B * p.Q * p.Hq, row0 + rows_per);
  constexpr int kPerWarp = 32 / kPieces, kStep = kThreads / 32 * kPerWarp;
  const int piece = lane % kPieces, first = warp * kPerWarp + lane / kPieces;
  // all of a thread's loads of queries go out before the first is used
  uint4 raw[JOIN ? 1 : kRows / kStep][2];
  const bool wide = ((uintptr_t)p.q & 15) == 0 && (p.qb | p.qh | p.qt) % 8 == 0;
  if constexpr (!JOIN) {
#pragma unroll
    for (int k = 0; k < kRows / kStep; ++k) {
      const int64_t row = row0 + first + k * kStep;
      raw[k][0] = raw[k][1] = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows && wide) {
        int b, i, h;
        place(p, row, b, i, h);
        const int64_t at = b * p.qb + i * p.qt + h * p.qh + 8 * piece;
        const uint4 *from = reinterpret_cast<const uint4 *>((const char *)p.q + at * (p.dtype == WTQ_F32 ? 4 : 2));
        raw[k][0] = __ldg(from);
        if (p.dtype == WTQ_F32) raw[k][1] = __ldg(from + 1);
      }
    }
  }
  // Of joined states, first all that weights and addresses hang on, for several of a thread's rows at once: a row's
  // pieces, a lane each, with maximum and sum (a whole group is one piece); then the first accumulators.
  constexpr int kMine = !JOIN ? 1 : WIDE ? kRows / kStep : 2, kAhead = WIDE ? 2 : 1;
  int at_of[kMine] = {};                                         // state of its first piece; number e > 0 is (2 e - 1) * p.rows on
  int n_of[kMine] = {};
  float m_of[kMine], l_of[kMine];                           // of piece number `piece`
  float4 ahead[kMine][kAhead][2];
  auto fetch = [&](float4 (&to)[2], const float *from) {
    to[0] = __ldcg(reinterpret_cast<const float4 *>(from));
    to[1] = __ldcg(reinterpret_cast<const float4 *>(from) + 1);
  };
  auto state = [&](int k, int e) { return at_of[k] + (e ? (2 * e - 1) * p.rows : 0); };
  auto acc = [&](int k, int e) { return (n_of[k] == 1 ? p.acc : p.part_acc) + (int64_t)state(k, e) * D + 8 * piece; };
  auto read_ahead = [&](int from_row) {
#pragma unroll
    for (int k = 0; k < kMine; ++k) {
      const int64_t row = row0 + from_row + k * kStep;
      n_of[k] = 0;
      m_of[k] = -INFINITY;
      l_of[k] = 0.f;
      if (row >= rows) continue;
      int b, i, h;
      place(p, row, b, i, h);
      const int n = prefix[b + 1] - prefix[b];
      if (n == 0) continue;
      const int kvh = h / p.n_rep, qr = i * p.n_rep + h - kvh * p.n_rep, rb = qr / p.rows;
      const long long g0 = (long long)prefix[b] * p.row_blocks * p.Hkv + (long long)(rb * p.Hkv + kvh) * n;
      const int c0 = run_of(g0, share);
      n_of[k] = run_of(g0 + n - 1, share) - c0 + 1;
      at_of[k] = n_of[k] == 1 ? (int)row : (c0 * 2 + 1) * p.rows + qr - rb * p.rows;
      if (n_of[k] == 1) {
        if (piece == 0) {
          l_of[k] = __ldcg(p.l + row);
          m_of[k] = l_of[k] != 0.f ? 0.f : -INFINITY;
        }
      } else if (piece < n_of[k]) {
        m_of[k] = __ldcg(p.part_m + state(k, piece));
        l_of[k] = __ldcg(p.part_l + state(k, piece));
      }
    }
#pragma unroll
    for (int k = 0; k < kMine; ++k)
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        ahead[k][e][0] = ahead[k][e][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (e < n_of[k]) fetch(ahead[k][e], acc(k, e));
      }
  };
#pragma unroll
  for (int k = 0; k < kRows / kStep; ++k) {
    const int r = first + k * kStep;
    if (k > 0 && k * kStep >= rows_per) break;              // (the same for all)
    const int64_t row = row0 + r;
    if constexpr (JOIN)
      if (k % kMine == 0) read_ahead(r);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if constexpr (!JOIN) {
      if (row < rows && !wide) {
        int b, i, h;
        place(p, row, b, i, h);
        const int64_t at = b * p.qb + i * p.qt + h * p.qh + 8 * piece;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = load_as_float(p.q, at + e, p.dtype);
      } else {
        const uint32_t w[8] = {raw[k][0].x, raw[k][0].y, raw[k][0].z, raw[k][0].w,
                               raw[k][1].x, raw[k][1].y, raw[k][1].z, raw[k][1].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = p.dtype == WTQ_F16 ? __half22float2(*reinterpret_cast<const __half2 *>(&w[e]))
                                              : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[e]));
          x[2 * e] = v.x;
          x[2 * e + 1] = v.y;
        }
        if (p.dtype == WTQ_F32) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
        }
      }
    } else {
      const int at = k % kMine;
      auto add = [&](const float4 (&v)[2], float w) {
        x[0] = fmaf(w, v[0].x, x[0]); x[1] = fmaf(w, v[0].y, x[1]); x[2] = fmaf(w, v[0].z, x[2]); x[3] = fmaf(w, v[0].w, x[3]);
        x[4] = fmaf(w, v[1].x, x[4]); x[5] = fmaf(w, v[1].y, x[5]); x[6] = fmaf(w, v[1].z, x[6]); x[7] = fmaf(w, v[1].w, x[7]);
      };
      const uint32_t group = (kPieces == 32 ? 0xffffffffu : ((1u << kPieces) - 1u)) << (lane / kPieces * kPieces);
      const int n = n_of[at], lane0 = lane / kPieces * kPieces;
      // A row with nothing to see has sum 0, and what its accumulators hold (they may never have been written) is not
      // used; other rows' are all written.
      if (n > 0) {
        float top = m_of[at];
        for (int e = piece + kPieces; e < n; e += kPieces) top = fmaxf(top, __ldcg(p.part_m + state(at, e)));
#pragma unroll
        for (int o = kPieces / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(group, top, o));
        float m = m_of[at], l = l_of[at], sum = 0.f;
        for (int from = 0; from < n; from += kPieces) {
          if (from > 0) {
            const int e = from + piece;
            m = e < n ? __ldcg(p.part_m + state(at, e)) : -INFINITY;
            l = e < n ? __ldcg(p.part_l + state(at, e)) : 0.f;
          }
          const float w = m == -INFINITY ? 0.f : exp2f(m - top);
          if (m != -INFINITY) sum = fmaf(w, l, sum);        // (NaN counts whatever its weight)
          int e = from;
          if (from == 0) {
#pragma unroll
            for (; e < kAhead; ++e) add(ahead[at][e], __shfl_sync(group, w, lane0 + e));
          }
          const int last = min(n, from + kPieces);
#pragma unroll 4
          for (; e < last; ++e) {
            float4 v[2];
            fetch(v, acc(at, e));
            add(v, __shfl_sync(group, w, lane0 + e - from));
          }
        }
#pragma unroll
        for (int o = kPieces / 2; o; o >>= 1) sum += __shfl_xor_sync(group, sum, o);
        const float f = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = sum != 0.f ? x[e] * f : 0.f;
      }
    }
    float most = 0.f, inverse;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
#pragma unroll
    for (int o = kPieces / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float power = power_of(most, inverse);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= inverse;
    store_split(M::kA + (uint32_t)(r >> 3) * M::kGroup + (uint32_t)piece * 128u + (uint32_t)(r & 7) * 16u,
                terms > 2 ? M::kALow - M::kA : 0u, x);
    if (piece == 0) sts_float(M::kScales + 4u * r, power);
  }
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(tmem) : "r"(M::kSlot));
  if (warp == 0) {
    if (elect_one()) {
      constexpr uint32_t kIdesc = M::kIdesc | (JOIN ? 1u << 16 : 0u);       // states: Pi is MN-major
      for (int t = terms - 1; t >= 0; --t) {               // low x high, high x low, high x high: small sums first
        const uint64_t a = descriptor(t == 2 ? M::kALow : M::kA, 128u, M::kGroup);
        const uint32_t from = M::kB + (t == 1 ? M::kBBytes : 0u);
        const uint64_t b = JOIN ? descriptor(from, M::kGroup, 128u) : descriptor(from, 128u, M::kGroup);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          umma_ss(tmem, a + 16u * ks, b + (JOIN ? (uint64_t)(2 * M::kGroup / 16) * ks : 16u * ks), kIdesc, t < terms - 1 || ks > 0);
      }
      umma_commit(M::kBar);
    }
    __syncwarp();
  }
  bool done = false;
  for (int spin = 0; spin < kWaitTries && !done; ++spin) done = mbar_try(M::kBar, 0u);
  if (!__syncthreads_and(done)) {
    if (tid == 0 && p.status) atomicOr(p.status, WTQ_STATUS_SCAN_TIMEOUT);
  }
  fence_after();
  // ---- a thread per row and quarter of the columns ---------------------------------------------------
  const int r = 32 * (warp & 3) + lane;
  const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
  const int64_t row = row0 + r;
  const float f = lds_float(M::kScales + 4u * r) * (JOIN ? 1.f / kPiScale : p.q_scale / kPiScale);
#pragma unroll 1
  for (int c0 = (warp >> 2) * (D / 4); c0 < ((warp >> 2) + 1) * (D / 4); c0 += 16) {
    uint32_t o[16];
    __syncwarp();                                           // (lanes without a row are back from the last columns)
    tmem_load16(tmem + lanes + c0, o);
    tmem_wait_load();
    if (row >= rows || !done) continue;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f * power_pi);
    if constexpr (!JOIN) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<uint4 *>(p.q_rot + row * D + c0)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
    } else {
      int b, i, h;
      place(p, row, b, i, h);
      const int64_t at = b * p.ob + i * p.ot + h * p.oh + c0;
      char *dst = (char *)p.out + at * (p.dtype == WTQ_F32 ? 4 : 2);
      if (((uintptr_t)dst & 15) != 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e) store_from_float(p.out, at + e, __uint_as_float(o[e]), p.dtype);
      } else if (p.dtype == WTQ_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          reinterpret_cast<uint4 *>(dst)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      } else {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __uint_as_float(o[2 * e]), y = __uint_as_float(o[2 * e + 1]);
          const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
          w[e] = p.dtype == WTQ_F16 ? half2_bits(x, y) : *reinterpret_cast<const uint32_t *>(&v);
        }
        reinterpret_cast<uint4 *>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4 *>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 0) {
    // (after a wait that ran out the products end before their tensor memory goes to somebody else; bounded as well)
    for (int spin = 0; spin < kWaitTries && !done; ++spin) done = mbar_try(M::kBar, 0u);
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"((uint32_t)D) : "memory");
  }
}

template <bool JOIN, int D, bool WIDE> int launch_blocks(const Params &p, int rows_per, int blocks, cudaStream_t stream) {
  using M = Map<D>;
  static std::atomic<bool> opted_in[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !opted_in[dev & 63].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(product_kernel<JOIN, D, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)M::kBytes);
    if (e != cudaSuccess) return check_cuda(e, "wtq_tree: shared memory opt-in");
    opted_in[dev & 63].store(true, std::memory_order_release);
  }
  const int terms = p.dtype == WTQ_F32 || (JOIN && p.dtype == WTQ_F16) ? 3 : 2;
  const size_t bytes = terms > 2 ? M::kBytes : M::kALow;    // (two blocks a multiprocessor without low parts)
  if (JOIN)
    return launch_behind(product_kernel<JOIN, D, WIDE>, blocks, kThreads, bytes, stream, "wtq_tree join launch", p, terms, rows_per);
  product_kernel<JOIN, D, WIDE><<<blocks, kThreads, bytes, stream>>>(p, terms, rows_per);
  note_launches(1);
  return check_cuda(cudaGetLastError(), "wtq_tree rotate launch");
}
template <bool JOIN, int D> int launch(const Params &p, cudaStream_t stream) {
  const int64_t all = (int64_t)p.B * p.Q * p.Hq;
  // Few rows are spread over more blocks, as far as there are multiprocessors: a block's time is the
  // chain of reads that its rows' pieces make (2688 rows of 8 pieces: 26 us on 21 blocks).
  int rows_per = kRows;
  while (rows_per > 16 && (all + rows_per / 2 - 1) / (rows_per / 2) <= device_sms()) rows_per /= 2;
  const int blocks = (int)((all + rows_per - 1) / rows_per);
  // A join that has a multiprocessor for every block reads all of a thread's rows ahead, in up to 128 registers
  // (16 384 rows: call 151 -> 146 us); more blocks than that are better off two a multiprocessor (19 968 rows:
  // 320 -> 307 us).
  if constexpr (JOIN)
    if (blocks <= device_sms()) return launch_blocks<true, D, true>(p, rows_per, blocks, stream);
  return launch_blocks<JOIN, D, false>(p, rows_per, blocks, stream);
}

}  // namespace rows

bool rows_on_tensor_cores(const Params &p) {
  return (p.D == 64 || p.D == 128) && (((uintptr_t)p.k.Pi | (uintptr_t)p.v.Pi) & 15) == 0;
}
int launch_rotate(const Params &p, cudaStream_t stream) {
  return p.D == 128 ? rows::launch<false, 128>(p, stream) : rows::launch<false, 64>(p, stream);
}
int launch_join(const Params &p, cudaStream_t stream) {
  return p.D == 128 ? rows::launch<true, 128>(p, stream) : rows::launch<true, 64>(p, stream);
}

}  // namespace tree
}  // namespace wtq
