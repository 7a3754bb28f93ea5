// Attention of drafted trees over paged packed K/V: entry point, the fp32 scan, and the two small
// products either side of a scan (queries into the key basis, states out of the value basis).
//
//   s_ij = q_i Pi_K^T . c_j n_j * scale,   j in history or tree token j visible to i
//   out_i = (sum_j softmax(s_i)_j n_j c_j) Pi_V
//
// One pass over the pages per block of query rows with the running maximum and sum of the softmax;
// the schedule is in wtq_tree.cuh.  The fp32 scan serves fp32 queries, whose results would lose
// what they have over 16 bits in the tensor cores' operands, and every layout the tensor-core scan
// (wtq_tree_umma.cu) does not: any width, page size and head_dim up to 256.
#include <algorithm>
#include <atomic>

#include "wtq_tree.cuh"

namespace wtq {
namespace tree {

// ---- products of rows with a rotation ----------------------------------------------------------
// 32 rows of a block in shared memory, a thread per column (several row groups where D < 256):
// out[r][c] = sum_d a[r][d] m(d, c), summed in d order.
constexpr int kRowThreads = 256, kRowBlock = 32;
template <bool TRANSPOSED, typename Store>
__device__ __forceinline__ void rows_product(const float *a, int pitch, const float *Pi, int D, Store store) {
  const int sets = max(1, kRowThreads / D);              // row groups
  const int set = threadIdx.x / D, c = threadIdx.x - set * D;
  if (set >= sets) return;
  constexpr int kMost = 8;
  for (int r0 = set * kMost; r0 < kRowBlock; r0 += sets * kMost) {
    float acc[kMost];
#pragma unroll
    for (int r = 0; r < kMost; ++r) acc[r] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; ++d) {
      const float m = __ldg(TRANSPOSED ? Pi + (int64_t)c * D + d : Pi + (int64_t)d * D + c);
#pragma unroll
      for (int r = 0; r < kMost; ++r) acc[r] = fmaf(a[(r0 + r) * pitch + d], m, acc[r]);
    }
#pragma unroll
    for (int r = 0; r < kMost; ++r) store(r0 + r, c, acc[r]);
  }
}

// q_rot = q_scale * q Pi_K^T, rows (b, token, head).
__global__ void __launch_bounds__(kRowThreads) rotate_kernel(Params p) {
  extern __shared__ float a[];
  const int64_t rows = (int64_t)p.B * p.Q * p.Hq, row0 = (int64_t)blockIdx.x * kRowBlock;
  for (int e = threadIdx.x; e < kRowBlock * p.D; e += kRowThreads) {
    const int r = e / p.D, d = e - r * p.D;
    const int64_t row = row0 + r;
    float x = 0.f;
    if (row < rows) {
      const int h = (int)(row % p.Hq);
      const int64_t t = row / p.Hq;
      x = load_as_float(p.q, t / p.Q * p.qb + t % p.Q * p.qt + h * p.qh + d, p.dtype);
    }
    a[r * (p.D + 4) + d] = x * p.q_scale;
  }
  __syncthreads();
  rows_product<true>(a, p.D + 4, p.k.Pi, p.D, [&](int r, int c, float v) {
    if (row0 + r < rows) p.q_rot[(row0 + r) * p.D + c] = v;
  });
}

// States of a query row joined, normalised and turned back: out = (sum_c w_c acc_c / sum_c w_c l_c) Pi_V.
__global__ void __launch_bounds__(kRowThreads) join_kernel(Params p) {
  extern __shared__ float a[];
  __shared__ int prefix[kMaxBatch + 1];
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  tile_prefix(p, prefix);
  const long long share = run_length(p, prefix);
  const int64_t rows = (int64_t)p.B * p.Q * p.Hq, row0 = (int64_t)blockIdx.x * kRowBlock;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int r = warp; r < kRowBlock; r += kRowThreads / 32) {
    const int64_t row = row0 + r;
    float *to = a + r * (p.D + 4);
    const int h = (int)(row % p.Hq);
    const int64_t t = row / p.Hq;
    const int b = (int)(t / p.Q), i = (int)(t - (int64_t)b * p.Q);
    const int n = row < rows ? prefix[b + 1] - prefix[b] : 0;
    if (n == 0) {                                        // nothing stored: zeros
      for (int d = lane; d < p.D; d += 32) to[d] = 0.f;
      continue;
    }
    const int kvh = h / p.n_rep, qr = i * p.n_rep + h - kvh * p.n_rep, rb = qr / p.rows;
    const long long g0 = (long long)prefix[b] * p.row_blocks * p.Hkv + (long long)(rb * p.Hkv + kvh) * n;
    const int c0 = (int)(g0 / share), c1 = (int)((g0 + n - 1) / share);
    auto state = [&](int c) -> int64_t {                 // of the piece in run c, when there are several
      return ((int64_t)c * 2 + (c == c0 ? 1 : 0)) * p.rows + qr - rb * p.rows;
    };
    if (c0 == c1) {
      const float l = p.l[row];
      const float f = l != 0.f ? 1.f / l : 0.f;
      for (int d = lane; d < p.D; d += 32) to[d] = l != 0.f ? p.acc[row * p.D + d] * f : 0.f;
      continue;
    }
    float top = -INFINITY;
    for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, p.part_m[state(c)]);
    top = warp_max(top);
    float sum = 0.f;
    for (int c = c0 + lane; c <= c1; c += 32) {
      const int64_t s = state(c);
      if (p.part_m[s] != -INFINITY) sum += p.part_l[s] * exp2f(p.part_m[s] - top);
    }
    sum = warp_sum(sum);
    const float f = sum != 0.f ? 1.f / sum : 0.f;
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = 0.f;
    for (int c = c0; c <= c1; ++c) {
      const int64_t s = state(c);
      const float m = p.part_m[s];
      if (m == -INFINITY) continue;                      // (an empty state's accumulator is not read)
      const float w = exp2f(m - top);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (lane + 32 * k < p.D) x[k] = fmaf(w, p.part_acc[s * p.D + lane + 32 * k], x[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane + 32 * k < p.D) to[lane + 32 * k] = x[k] * f;
  }
  __syncthreads();
  rows_product<false>(a, p.D + 4, p.v.Pi, p.D, [&](int r, int c, float v) {
    const int64_t row = row0 + r;
    if (row >= rows) return;
    const int h = (int)(row % p.Hq);
    const int64_t t = row / p.Hq;
    store_from_float(p.out, t / p.Q * p.ob + t % p.Q * p.ot + h * p.oh + c, v, p.dtype);
  });
}

// ---- the fp32 scan -----------------------------------------------------------------------------
// 256 threads, 64 query rows by 32 tokens.  Scores: a thread has 4 rows x 2 tokens, operands from
// shared memory four coordinates at a time (6 loads for 32 products).  Softmax: a warp has 8 rows, a
// lane per token.  Values: a thread has 4 rows x 4 NJ coordinates (NJ + 1 loads for 16 NJ products a
// token).  Bound by shared-memory operands at long histories, by latency at short ones: a call of 8
// tokens over 1000, 8 heads on 2, takes 49 us with both products; 16 x 8192 tokens, 128 rows a kv head,
// 4.2 ms (16.5 TFLOP/s).
constexpr int kScanThreads = 256, kScanRows = 64, kScanTile = 32;

__host__ __device__ inline int scan_pitch(int D) { return (D + 3) / 4 * 4 + 4; }
inline size_t scan_bytes(int D) {
  return sizeof(float) * ((size_t)(kScanRows + 2 * kScanTile) * scan_pitch(D) + kScanRows * (kScanTile + 4) + kScanRows);
}

// Eight codes of `bw` bits, whole bytes whatever the width (`words`: 4- or 8-bit codes on 4-byte borders).
__device__ __forceinline__ uint64_t eight_codes(const uint8_t *src, int bw, bool words) {
  uint64_t w = 0;
  if (words) {
    w = __ldg(reinterpret_cast<const uint32_t *>(src));
    if (bw == 8) w |= (uint64_t)__ldg(reinterpret_cast<const uint32_t *>(src) + 1) << 32;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < bw) w |= (uint64_t)__ldg(src + i) << (8 * i);
  }
  return w;
}

// A tile's rows of both sides as centroid times norm; rows past the end and of pages outside the pool are
// zeros, and so are values whose norm is not finite, which the product would carry (0 x inf) to query rows
// that do not see them: their tokens' bits go to `bad`.  Eight threads a row; all of a thread's codes are read before the first is looked up.
__device__ __forceinline__ void decode_rows(const Params &p, const int32_t *table, int h, int tok0, int end, const float *cents,
                                            float *ks, float *vs, int pitch, int padded, uint32_t *bad) {
  constexpr int kPer = kScanThreads / kScanTile;
  const int r = threadIdx.x / kPer, tok = tok0 + r, d_first = 8 * (threadIdx.x % kPer);
  const uint8_t *row[2] = {nullptr, nullptr};
  float norm[2] = {0.f, 0.f};
  if (tok < end) {
    const int page = table[tok / p.S], slot = tok % p.S;
    if ((uint32_t)page < (uint32_t)p.P) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const DecodeSideDev &sd = s ? p.v : p.k;
        row[s] = sd.pages + (int64_t)page * sd.page_stride + h * sd.head_stride + (int64_t)slot * sd.nb;
        norm[s] = __half2float(sd.norms[(int64_t)page * sd.norm_page_stride + h * sd.norm_head_stride + slot]);
      }
      if (!(fabsf(norm[1]) < INFINITY)) {
        norm[1] = 0.f;
        if (threadIdx.x % kPer == 0) atomicOr(bad, 1u << r);
      }
    } else if (p.status && threadIdx.x % kPer == 0) {
      atomicOr(p.status, WTQ_STATUS_BAD_PAGE);
    }
  }
  constexpr int kMost = 256 / (8 * kPer);                     // groups of eight codes of a thread
  uint64_t w[2][kMost];
#pragma unroll
  for (int k = 0; k < kMost; ++k)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const DecodeSideDev &sd = s ? p.v : p.k;
      const int d0 = d_first + 8 * kPer * k;
      w[s][k] = 0;
      if (row[s] != nullptr && d0 + 8 <= p.D)
        w[s][k] = eight_codes(row[s] + d0 / 8 * sd.bw, sd.bw, sd.bw % 4 == 0 && ((uintptr_t)row[s] & 3) == 0);
    }
#pragma unroll
  for (int k = 0; k < kMost; ++k)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const DecodeSideDev &sd = s ? p.v : p.k;
      const int d0 = d_first + 8 * kPer * k;
      float *to = (s ? vs : ks) + r * pitch + d0;
      if (d0 >= padded) continue;
      uint64_t x = w[s][k];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int code = (int)(x & ((1u << sd.bw) - 1u));
        x >>= sd.bw;
        if (d0 + 8 <= p.D) to[i] = row[s] ? cents[256 * s + code] * norm[s] : 0.f;
        else if (d0 + i < padded)                             // the last, odd group
          to[i] = row[s] && d0 + i < p.D ? cents[256 * s + extract_code(row[s], d0 + i, sd.bw, sd.nb)] * norm[s] : 0.f;
      }
    }
}

template <int NJ>
__global__ void __launch_bounds__(kScanThreads) scan_kernel(Params p) {
  extern __shared__ __align__(16) float smem[];
  __shared__ int prefix[kMaxBatch + 1];
  __shared__ float cents[512];
  __shared__ uint32_t bad;                                // tokens of the tile whose value norm is not finite
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  for (int e = threadIdx.x; e < 512; e += kScanThreads) {
    const DecodeSideDev &sd = e < 256 ? p.k : p.v;
    cents[e] = (e & 255) < 1 << sd.bw ? __ldg(sd.centroids + (e & 255)) : 0.f;
  }
  const int pitch = scan_pitch(p.D), padded = (p.D + 3) / 4 * 4;
  float *qs = smem, *ks = qs + kScanRows * pitch, *vs = ks + kScanTile * pitch, *ps = vs + kScanTile * pitch;
  float *factor = ps + kScanRows * (kScanTile + 4);
  constexpr int kP = kScanTile + 4;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ty = tid >> 4, tx = tid & 15;                 // 4 rows from 4 ty; tokens tx, tx + 16
  tile_prefix(p, prefix);
  const long long share = run_length(p, prefix), all = (long long)prefix[p.B] * p.row_blocks * p.Hkv;
  const long long begin = share * blockIdx.x, end = min(all, begin + share);
  asm volatile("griddepcontrol.wait;\n" ::: "memory");       // the rotated queries
  for (long long x = begin; x < end;) {
    const Piece c = piece_at(p, prefix, x, begin, end);
    x += c.last - c.first;
    const int L = length_of(p, c.b), hist = history_of(p, c.b), places = places_of(p, c.b), row0 = c.rb * p.rows;
    const int32_t *table = p.page_table + (int64_t)c.b * p.table_stride;
    __syncthreads();
    {
      if (tid == 0) bad = 0u;
      const int r = tid >> 2, qr = row0 + r;                  // four threads a row
      const int i = qr / p.n_rep, head = c.h * p.n_rep + qr - i * p.n_rep;
      const float *from = p.q_rot + (((int64_t)c.b * p.Q + i) * p.Hq + head) * p.D;
      if (p.D % 4 == 0) {
#pragma unroll 4
        for (int d = 4 * (tid & 3); d < padded; d += 16)
          *reinterpret_cast<float4 *>(qs + r * pitch + d) =
              qr < p.R ? *reinterpret_cast<const float4 *>(from + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      } else {
        for (int d = tid & 3; d < padded; d += 4) qs[r * pitch + d] = qr < p.R && d < p.D ? from[d] : 0.f;
      }
    }
    const bool idle = row0 + 8 * warp >= p.R;             // a warp whose rows do not exist
    float m[8], l[8];                                     // of rows 8 warp .. 8 warp + 7
    bool dead[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      m[k] = -INFINITY;
      l[k] = 0.f;
      const int qr = row0 + 8 * warp + k;
      dead[k] = qr >= p.R || padding(p.mask + c.b * p.mask_b + qr / p.n_rep * p.mask_t, p.Q);
    }
    float acc[4][4 * NJ];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < 4 * NJ; ++j) acc[r][j] = 0.f;
    for (int tile = c.first; tile < c.last; ++tile) {
      const int tok0 = tile * kScanTile;
      __syncthreads();                                    // the last tile's rows have been used
      decode_rows(p, table, c.h, tok0, L, cents, ks, vs, pitch, padded, &bad);
      __syncthreads();
      float s[4][2] = {};
      for (int d = 0; d < (idle ? 0 : padded); d += 4) {
        float4 q4[4], k4[2];
#pragma unroll
        for (int r = 0; r < 4; ++r) q4[r] = *reinterpret_cast<const float4 *>(qs + (4 * ty + r) * pitch + d);
#pragma unroll
        for (int t = 0; t < 2; ++t) k4[t] = *reinterpret_cast<const float4 *>(ks + (tx + 16 * t) * pitch + d);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            s[r][t] = fmaf(q4[r].x, k4[t].x, s[r][t]);
            s[r][t] = fmaf(q4[r].y, k4[t].y, s[r][t]);
            s[r][t] = fmaf(q4[r].z, k4[t].z, s[r][t]);
            s[r][t] = fmaf(q4[r].w, k4[t].w, s[r][t]);
          }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < 2; ++t) ps[(4 * ty + r) * kP + tx + 16 * t] = s[r][t];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = 8 * warp + k;
        float w = 0.f, f = 1.f;
        if (!dead[k]) {
          const int32_t *words = p.mask + c.b * p.mask_b + (row0 + r) / p.n_rep * p.mask_t;
          const uint32_t seen = visible(words, places, tok0 - hist);
          const float v = (seen >> lane & 1u) != 0 && tok0 + lane < L ? ps[r * kP + lane] : -INFINITY;
          const float now = fmaxf(m[k], warp_max(v));
          if ((now == -INFINITY && __any_sync(0xffffffffu, v != v)) || (seen & bad) != 0u) l[k] = NAN;
          if (now != -INFINITY) {
            f = m[k] == -INFINITY ? 0.f : exp2f(m[k] - now);
            w = v == -INFINITY ? 0.f : exp2f(v - now);
            l[k] = l[k] * f + warp_sum(w);
            m[k] = now;
          }
        }
        ps[r * kP + lane] = w;
        if (lane == 0) factor[r] = f;
      }
      __syncthreads();
      if (tid == 0) bad = 0u;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = factor[4 * ty + r];
#pragma unroll
        for (int j = 0; j < 4 * NJ; ++j) acc[r][j] *= f;
      }
      for (int t0 = 0; t0 < (idle ? 0 : kScanTile); t0 += 4) {
        float4 w4[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w4[r] = *reinterpret_cast<const float4 *>(ps + (4 * ty + r) * kP + t0);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const int d = 4 * tx + 64 * j;
            if (d < padded) {
              const float4 v = *reinterpret_cast<const float4 *>(vs + (t0 + t) * pitch + d);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float w = t == 0 ? w4[r].x : t == 1 ? w4[r].y : t == 2 ? w4[r].z : w4[r].w;
                acc[r][4 * j + 0] = fmaf(w, v.x, acc[r][4 * j + 0]);
                acc[r][4 * j + 1] = fmaf(w, v.y, acc[r][4 * j + 1]);
                acc[r][4 * j + 2] = fmaf(w, v.z, acc[r][4 * j + 2]);
                acc[r][4 * j + 3] = fmaf(w, v.w, acc[r][4 * j + 3]);
              }
            }
          }
      }
    }
    // the rows' states
    auto place = [&](int r, float *&at, float *&at_m, float *&at_l) -> bool {
      const int qr = row0 + r;
      if (qr >= p.R) return false;
      int64_t s;
      if (c.slot < 0) {
        const int i = qr / p.n_rep, head = c.h * p.n_rep + qr - i * p.n_rep;
        s = ((int64_t)c.b * p.Q + i) * p.Hq + head;
        at = p.acc + s * p.D; at_m = p.m + s; at_l = p.l + s;
      } else {
        s = ((int64_t)blockIdx.x * 2 + c.slot) * p.rows + r;
        at = p.part_acc + s * p.D; at_m = p.part_m + s; at_l = p.part_l + s;
      }
      return true;
    };
    float *at, *at_m, *at_l;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane == 0 && place(8 * warp + k, at, at_m, at_l)) {
        *at_m = l[k] != l[k] ? 0.f : m[k];                // a query that is not a number: so is its result
        *at_l = l[k];
      }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (place(4 * ty + r, at, at_m, at_l)) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (4 * tx + 64 * j + e < p.D) at[4 * tx + 64 * j + e] = acc[r][4 * j + e];
      }
  }
}

template <int NJ> int launch_scan(const Params &p, cudaStream_t stream) {
  static std::atomic<bool> opted_in[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !opted_in[dev & 63].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(scan_kernel<NJ>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)scan_bytes(64 * NJ));
    if (e != cudaSuccess) return check_cuda(e, "wtq_tree: shared memory opt-in");
    opted_in[dev & 63].store(true, std::memory_order_release);
  }
  return launch_behind(scan_kernel<NJ>, p.blocks, kScanThreads, scan_bytes(p.D), stream, "wtq_tree scan launch", p);
}

size_t round_up(size_t x) { return (x + 255) / 256 * 256; }
// Blocks of a scan: as many as are resident at once.
int scan_blocks(bool umma, int D) { return device_sms() * (umma ? 1 : D <= 128 ? 2 : 1); }
size_t workspace_for(int B, int Hq, int Q, int D, int blocks, int rows) {
  const size_t all = (size_t)B * Q * Hq, parts = (size_t)blocks * 2 * rows;
  return 2 * round_up(all * D * 4) + 2 * round_up(all * 4) + round_up(parts * D * 4) + 2 * round_up(parts * 4);
}

}  // namespace tree
}  // namespace wtq

using namespace wtq;

extern "C" size_t wtq_tree_workspace_bytes(int B, int Hq, int Hkv, int Q, int D) {
  (void)Hkv;
  if (B < 1 || Hq < 1 || Q < 1 || D < 1) return 256;
  const int most = std::min(B, tree::kMaxBatch);
  return std::max(tree::workspace_for(most, Hq, Q, D, tree::scan_blocks(true, D), tree::kUmmaRows),
                  tree::workspace_for(most, Hq, Q, D, tree::scan_blocks(false, D), tree::kScanRows));
}

extern "C" int wtq_tree_on_tensor_cores(const wtq_side_t *k_side, const wtq_side_t *v_side, int dtype, int D, int S) {
  return k_side && v_side && tree::on_tensor_cores(*k_side, *v_side, dtype, D, S) ? 1 : 0;
}

extern "C" int wtq_tree(const void *q, int dtype, const int64_t q_strides[3], void *out, const int64_t out_strides[3],
                        const wtq_side_t *k_side, const wtq_side_t *v_side, const int32_t *page_table,
                        int64_t table_stride, const int32_t *seq_lens, const int32_t *mask,
                        const int64_t mask_strides[2], float scale, int B, int Hq, int Hkv, int Q, int D, int S, int P,
                        int max_pages, void *workspace, size_t workspace_bytes, int32_t *status, void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  if (Q < 1) return fail(WTQ_ERR_ARG, "wtq_tree: need Q >= 1");
  if (!mask_strides || (B > 0 && !mask)) return fail(WTQ_ERR_ARG, "wtq_tree: null mask");
  if (int rc = decode_validate(q, dtype, q_strides, out, out_strides, false, k_side, v_side, page_table, seq_lens, B,
                               Hq, Hkv, D, S, P, max_pages))
    return rc;
  if (B == 0) return WTQ_OK;
  if ((int64_t)B * Q > (int64_t)1 << 24 || (int64_t)B * Q * Hq > 0x7fffffff)
    return fail(WTQ_ERR_ARG, "wtq_tree: B * Q is limited to 2^24 query tokens, B * Q * Hq to 2^31 rows");
  if ((int64_t)max_pages * S > (int64_t)1 << 30 ||
      (((int64_t)max_pages * S + 31) / 32) * std::min(B, tree::kMaxBatch) > 0x7fffffff)
    return fail(WTQ_ERR_ARG, "wtq_tree: the table covers too many tokens");
  if (!workspace || ((uintptr_t)workspace & 255) != 0)
    return fail(WTQ_ERR_ARG, "wtq_tree: the workspace has to be aligned to 256 bytes");
  const size_t need = wtq_tree_workspace_bytes(B, Hq, Hkv, Q, D);
  if (workspace_bytes < need)
    return fail(WTQ_ERR_WORKSPACE, "wtq_tree: workspace %zu < %zu bytes", workspace_bytes, need);
  const bool umma = tree::on_tensor_cores(*k_side, *v_side, dtype, D, S);
  tree::Params p = {};
  auto fill = [&](DecodeSideDev &d, const wtq_side_t &s) {
    d.pages = (const uint8_t *)s.pages; d.norms = (const __half *)s.norms;
    d.page_stride = s.page_stride; d.head_stride = s.head_stride;
    d.norm_page_stride = s.norm_page_stride; d.norm_head_stride = s.norm_head_stride;
    d.Pi = s.Pi; d.centroids = s.centroids; d.bw = s.bw; d.nb = D * s.bw / 8;
  };
  fill(p.k, *k_side);
  fill(p.v, *v_side);
  p.dtype = dtype; p.q_scale = scale * 1.4426950408889634f;
  p.qb = q_strides[0]; p.qh = q_strides[1]; p.qt = q_strides[2];
  p.ob = out_strides[0]; p.oh = out_strides[1]; p.ot = out_strides[2];
  p.table_stride = table_stride; p.mask_b = mask_strides[0]; p.mask_t = mask_strides[1];
  p.Hq = Hq; p.Hkv = Hkv; p.n_rep = Hq / Hkv; p.Q = Q; p.R = Q * p.n_rep; p.D = D; p.S = S; p.P = P;
  p.max_tokens = max_pages * S; p.status = status;
  p.rows = umma ? tree::kUmmaRows : tree::kScanRows;
  p.tile = umma ? tree::kUmmaTile : tree::kScanTile;
  p.row_blocks = (p.R + p.rows - 1) / p.rows;
  p.blocks = tree::scan_blocks(umma, D);
  p.least = umma ? 2 : 1;
  const int el = dtype == WTQ_F32 ? 4 : 2;
  for (int b0 = 0; b0 < B; b0 += tree::kMaxBatch) {
    p.B = std::min(B - b0, tree::kMaxBatch);
    p.q = (const char *)q + (int64_t)b0 * p.qb * el;
    p.out = (char *)out + (int64_t)b0 * p.ob * el;
    p.page_table = page_table + b0 * table_stride;
    p.seq_lens = seq_lens + b0;
    p.mask = mask + b0 * p.mask_b;
    const size_t all = (size_t)p.B * Q * Hq, parts = (size_t)p.blocks * 2 * p.rows;
    char *ws = (char *)workspace;
    auto take = [&](size_t bytes) { float *at = (float *)ws; ws += tree::round_up(bytes); return at; };
    p.q_rot = take(all * D * 4);
    p.acc = take(all * D * 4);
    p.m = take(all * 4);
    p.l = take(all * 4);
    p.part_acc = take(parts * D * 4);
    p.part_m = take(parts * 4);
    p.part_l = take(parts * 4);
    const unsigned row_grid = (unsigned)((all + tree::kRowBlock - 1) / tree::kRowBlock);
    const size_t row_bytes = (size_t)tree::kRowBlock * (D + 4) * sizeof(float);
    const bool products = tree::rows_on_tensor_cores(p);
    int rc;
    if (products) {
      rc = tree::launch_rotate(p, stream);
    } else {
      tree::rotate_kernel<<<row_grid, tree::kRowThreads, row_bytes, stream>>>(p);
      note_launches(1);
      rc = check_cuda(cudaGetLastError(), "wtq_tree rotate launch");
    }
    if (rc) return rc;
    if (umma) rc = tree::launch_scan_umma(p, stream);
    else if (D <= 64) rc = tree::launch_scan<1>(p, stream);
    else if (D <= 128) rc = tree::launch_scan<2>(p, stream);
    else if (D <= 192) rc = tree::launch_scan<3>(p, stream);
    else rc = tree::launch_scan<4>(p, stream);
    if (rc) return rc;
    if (products) {
      rc = tree::launch_join(p, stream);
    } else {
      tree::join_kernel<<<row_grid, tree::kRowThreads, row_bytes, stream>>>(p);
      note_launches(1);
      rc = check_cuda(cudaGetLastError(), "wtq_tree join launch");
    }
    if (rc) return rc;
  }
  return WTQ_OK;
}
