// Norms of queries and keys for each head with the rotary position rotation, in one pass:
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (a side without weights is not normalised)
//   (a, b) -> (a cos - b sin, b cos + a sin)    over the first `rot` coordinates
//
// where a pair is (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved, and cos, sin come from a
// table row per position.  Every value is read once and rounded once, from fp32.  A token's
// values may be copied along (a serving step stages all three tensors).
//
// A group of threads holds a row of a head in registers: thread c of the group two pieces of 16
// bytes, piece c of the rotated part's first half and the piece of its second half that it turns
// with (an interleaved pair never leaves a piece; the unrotated tail is dealt two pieces to a
// thread too), so the rotation needs no exchange and the norm a few shuffles.  A block takes adjacent
// tokens and a run of heads, the same for all its groups: the table's rows and a side's weights stay in
// registers, sides change for the whole block at once, and rows of a head are written side by side.
// How many heads depends on the call: one with few tokens, which is the shortest chain, all of them
// with many, which reads the table once.  Arithmetic is on two values at a time (f32x2).
// Bound by HBM at prompts and by the launch at single tokens.  8191 tokens of 32 + 8 heads of 128 in bf16,
// 172 MB: 42 us (56 with scalar arithmetic and a group walking over a token's heads).
#include <algorithm>

#include "wtq_common.cuh"

namespace wtq {
namespace rope {

struct Side {                   // q, k or v of a call
  const void *x;
  void *out;
  int64_t xb, xh, xt, ob, oh, ot;   // element strides: batch, head, token
  const void *weight;           // (D), or null: no norm
  int heads;
  bool turned;                  // v is copied
};

struct Params {
  Side side[3];
  const int32_t *positions;     // (B, n)
  int64_t position_stride;
  const float *table;           // (rows, rot): cos of the pairs, then sin
  int64_t table_stride;
  int table_rows;
  int weight_dtype;
  float eps;
  int B, n, D, rot, heads;      // heads: of all sides
  int heads_per_group;
  int32_t *status;
};

template <int DT> struct Vec {
  static constexpr int kN = DT == WTQ_F32 ? 4 : 8;      // elements of 16 bytes
};
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 16 bytes as pairs of fp32 values and back.
template <int DT> __device__ __forceinline__ void unpack(const uint4 &v, uint64_t *x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (DT == WTQ_F32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == WTQ_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        x[i] = pair(f.x, f.y);
      } else {
        x[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      }
    }
  }
}
template <int DT> __device__ __forceinline__ uint4 packed(const uint64_t *x) {
  uint32_t w[4];
  if constexpr (DT == WTQ_F32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = halves(x[i]);
      w[2 * i] = __float_as_uint(f.x);
      w[2 * i + 1] = __float_as_uint(f.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = halves(x[i]);
      if constexpr (DT == WTQ_F16) {
        const __half2 h = __floats2half2_rn(f.x, f.y);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ const Side &side_of(const Params &p, int &head) {
  int s = 0;
  if (head >= p.side[0].heads) {
    head -= p.side[0].heads;
    s = 1;
    if (head >= p.side[1].heads) {
      head -= p.side[1].heads;
      s = 2;
    }
  }
  return p.side[s];
}
// A token's row of the table, or -1: padding (a negative position; the outputs are zeros) or a
// position that the table does not have (the same, and reported).
__device__ __forceinline__ int table_row(const Params &p, int b, int i, bool report) {
  const int pos = p.positions[(int64_t)b * p.position_stride + i];
  if (pos >= p.table_rows && report && p.status) atomicOr(p.status, WTQ_STATUS_BAD_POSITION);
  return pos < p.table_rows ? pos : -1;
}

// TPR threads a row (a power of two, at most 32); D, rot and D - rot are multiples of two pieces
// and every row is 16-byte aligned.  The pieces of kBatch heads are read before the first is worked on.
constexpr int kThreads = 128, kBatch = 2;
template <int DT, int TPR, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads, 5) rows_kernel(Params p) {
  constexpr int V = Vec<DT>::kN, N = V / 2;               // values and pairs of a piece
  constexpr int kEl = 16 / V;
  const int lane_in_row = threadIdx.x % TPR;
  const int64_t token = (int64_t)blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
  const int first = blockIdx.y * p.heads_per_group, last = min(first + p.heads_per_group, p.heads);
  // (threads of a warp stay together for the shuffles: a group past the end works on nothing)
  const bool real = token < (int64_t)p.B * p.n;
  const int b = real ? (int)((uint32_t)token / (uint32_t)p.n) : 0, i = real ? (int)(token - (int64_t)b * p.n) : 0;
  const int pairs = p.D / (2 * V), turned_pairs = p.rot / (2 * V);
  const bool work = real && lane_in_row < pairs, turns = lane_in_row < turned_pairs;
  // where this thread's two pieces start
  const int at0 = turns ? lane_in_row * V : p.rot + 2 * (lane_in_row - turned_pairs) * V;
  const int at1 = turns ? at0 + p.rot / 2 : at0 + V;
  // the side that the walk stands in: rows of this token, head by head
  int side = -1, left = 0;
  const char *src = nullptr;
  char *dst = nullptr;
  int64_t src_step = 0, dst_step = 0;
  auto enter = [&](int s, int head) {                     // the same for the whole block
    side = s;
    const Side &sd = p.side[s];
    left = sd.heads - head;
    src = (const char *)sd.x + (b * sd.xb + head * sd.xh + i * sd.xt) * kEl;
    dst = (char *)sd.out + (b * sd.ob + head * sd.oh + i * sd.ot) * kEl;
    src_step = sd.xh * kEl;
    dst_step = sd.oh * kEl;
  };
  {
    int head = first, s = 0;
    while (head >= p.side[s].heads) head -= p.side[s++].heads;
    enter(s, head);
  }
  const int row = real ? table_row(p, b, i, lane_in_row == 0 && blockIdx.y == 0) : -1;
  // cosines and sines: halves: of piece 0's values; interleaved: (c, c) and (-s, s) of both pieces' pairs
  uint64_t cs[INTERLEAVED ? 2 * N : N], sn[INTERLEAVED ? 2 * N : N], minus[INTERLEAVED ? 1 : N];
#pragma unroll
  for (int j = 0; j < (INTERLEAVED ? 2 * N : N); ++j) cs[j] = twice(1.f), sn[j] = 0;
#pragma unroll
  for (int j = 0; j < (INTERLEAVED ? 1 : N); ++j) minus[j] = 0;
  if (turns && row >= 0) {
    const float *t = p.table + (int64_t)row * p.table_stride, *u = t + p.rot / 2;
#pragma unroll
    for (int j = 0; j < (INTERLEAVED ? 2 * N : N); ++j) {
      if constexpr (INTERLEAVED) {
        const int k = j < N ? at0 / 2 + j : at1 / 2 + j - N;
        const float c = __ldg(t + k), s = __ldg(u + k);
        cs[j] = twice(c);
        sn[j] = pair(-s, s);
      } else {
        const int k = at0 + 2 * j;
        const float s0 = __ldg(u + k), s1 = __ldg(u + k + 1);
        cs[j] = pair(__ldg(t + k), __ldg(t + k + 1));
        sn[j] = pair(s0, s1);
        minus[j] = pair(-s0, -s1);
      }
    }
  }
  uint64_t weight[2 * N];
  int weighed = -1;                                       // the side whose weights these are
  for (int head = first; head < last; head += kBatch) {
    uint4 raw[kBatch][2];
    char *to[kBatch];
    int of[kBatch];
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      of[e] = -1;
      if (head + e >= last) continue;
      while (left == 0) enter(side + 1, 0);
      of[e] = side;
      to[e] = dst;
      if (work) {
        raw[e][0] = *reinterpret_cast<const uint4 *>(src + at0 * kEl);
        raw[e][1] = *reinterpret_cast<const uint4 *>(src + at1 * kEl);
      } else {
        raw[e][0] = raw[e][1] = make_uint4(0u, 0u, 0u, 0u);
      }
      src += src_step;
      dst += dst_step;
      --left;
    }
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      if (of[e] < 0) continue;                            // (the same for the whole block)
      const void *w = p.side[of[e]].weight;
      if (of[e] < 2) {
        uint64_t x[2 * N];
        unpack<DT>(raw[e][0], x);
        unpack<DT>(raw[e][1], x + N);
        if (w != nullptr) {
          if (weighed != of[e] && work) {
#pragma unroll
            for (int j = 0; j < 2 * N; ++j) {
              const int k = (j < N ? at0 : at1 - V) + 2 * j;
              weight[j] = pair(load_as_float(w, k, p.weight_dtype), load_as_float(w, k + 1, p.weight_dtype));
            }
          }
          weighed = of[e];
          uint64_t sums = 0;
#pragma unroll
          for (int j = 0; j < 2 * N; ++j) fma2(sums, x[j], x[j]);
          const float2 both = halves(sums);
          float sum = both.x + both.y;
#pragma unroll
          for (int o = TPR / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o, TPR);
          const uint64_t r = twice(rsqrtf(sum / (float)p.D + p.eps));
#pragma unroll
          for (int j = 0; j < 2 * N; ++j) x[j] = mul2(mul2(x[j], weight[j]), r);
        }
        if (row < 0) {
#pragma unroll
          for (int j = 0; j < 2 * N; ++j) x[j] = 0;
        } else if (INTERLEAVED && turns) {
#pragma unroll
          for (int j = 0; j < 2 * N; ++j) {
            const float2 v = halves(x[j]);
            constexpr int kTop = INTERLEAVED ? 2 * N - 1 : 0;
            uint64_t y = mul2(pair(v.y, v.x), sn[j < kTop ? j : kTop]);
            fma2(y, x[j], cs[j < kTop ? j : kTop]);
            x[j] = y;
          }
        } else if (!INTERLEAVED && turns) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            uint64_t y = mul2(x[N + j], minus[INTERLEAVED ? 0 : j]), z = mul2(x[j], sn[j]);
            fma2(y, x[j], cs[j]);
            fma2(z, x[N + j], cs[j]);
            x[j] = y;
            x[N + j] = z;
          }
        }
        raw[e][0] = packed<DT>(x);
        raw[e][1] = packed<DT>(x + N);
      }
      if (work) {
        *reinterpret_cast<uint4 *>(to[e] + at0 * kEl) = raw[e][0];
        *reinterpret_cast<uint4 *>(to[e] + at1 * kEl) = raw[e][1];
      }
    }
  }
}

// Any even rot, any D up to 256, any alignment: a warp per row, the row in shared memory.
__global__ void __launch_bounds__(128) any_kernel(Params p, int dtype, int interleaved) {
  __shared__ float rows[4][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *x = rows[warp];
  const int64_t count = (int64_t)p.B * p.n * p.heads;
  for (int64_t r = (int64_t)blockIdx.x * 4 + warp; r < count; r += (int64_t)gridDim.x * 4) {
    int head = (int)(r % p.heads);
    const int64_t token = r / p.heads;
    const int b = (int)(token / p.n), i = (int)(token - (int64_t)b * p.n);
    const int row = table_row(p, b, i, lane == 0 && head == 0);
    const Side &sd = side_of(p, head);
    const int64_t from = b * sd.xb + head * sd.xh + i * sd.xt, to = b * sd.ob + head * sd.oh + i * sd.ot;
    float sum = 0.f;
    for (int d = lane; d < p.D; d += 32) {
      const float v = load_as_float(sd.x, from + d, dtype);
      x[d] = v;
      sum = fmaf(v, v, sum);
    }
    const float r1 = 1.f / sqrtf(warp_sum(sum) / (float)p.D + p.eps);
    if (sd.weight != nullptr)
      for (int d = lane; d < p.D; d += 32) x[d] *= r1 * load_as_float(sd.weight, d, p.weight_dtype);
    __syncwarp();
    const int half = p.rot / 2;
    for (int d = lane; d < p.D; d += 32) {
      float v = x[d];
      if (sd.turned && row < 0) v = 0.f;
      else if (sd.turned && d < p.rot) {
        const int pair = interleaved ? d >> 1 : d % half;
        const bool second = interleaved ? d & 1 : d >= half;
        const float other = x[interleaved ? d ^ 1 : second ? d - half : d + half];
        const float *t = p.table + (int64_t)row * p.table_stride;
        const float c = __ldg(t + pair), s = __ldg(t + half + pair);
        v = second ? v * c + other * s : v * c - other * s;
      }
      store_from_float(sd.out, to + d, v, dtype);
    }
    __syncwarp();
  }
}

template <int DT, int TPR>
void launch(const Params &p, bool interleaved, cudaStream_t stream) {
  const int64_t tokens = (int64_t)p.B * p.n;
  const dim3 grid((unsigned)((tokens * TPR + kThreads - 1) / kThreads), (p.heads + p.heads_per_group - 1) / p.heads_per_group);
  if (interleaved) rows_kernel<DT, TPR, true><<<grid, kThreads, 0, stream>>>(p);
  else rows_kernel<DT, TPR, false><<<grid, kThreads, 0, stream>>>(p);
}
template <int DT>
void launch_width(const Params &p, int tpr, bool interleaved, cudaStream_t stream) {
  if (tpr <= 2) launch<DT, 2>(p, interleaved, stream);
  else if (tpr <= 4) launch<DT, 4>(p, interleaved, stream);
  else if (tpr <= 8) launch<DT, 8>(p, interleaved, stream);
  else if (tpr <= 16) launch<DT, 16>(p, interleaved, stream);
  else launch<DT, 32>(p, interleaved, stream);
}

}  // namespace rope
}  // namespace wtq

using namespace wtq;

extern "C" int wtq_qk_norm_rope(const wtq_rope_side_t sides[3], int dtype, int weight_dtype, float eps,
                                const int32_t *positions, int64_t position_stride, const float *table,
                                int64_t table_stride, int table_rows, int B, int n, int D, int rot,
                                int interleaved, int32_t *status, void *stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  if (!sides) return fail(WTQ_ERR_ARG, "wtq_qk_norm_rope: null sides");
  if (B < 0 || n < 0 || D < 1 || D > 256 || rot < 0 || rot > D || rot % 2)
    return fail(WTQ_ERR_ARG, "wtq_qk_norm_rope: need 1 <= head_dim <= 256 and an even rot up to it");
  if (dtype < WTQ_F32 || dtype > WTQ_BF16 || weight_dtype < WTQ_F32 || weight_dtype > WTQ_BF16)
    return fail(WTQ_ERR_ARG, "wtq_qk_norm_rope: bad dtype");
  if (table_rows < 0 || (int64_t)B * n > (int64_t)1 << 28)
    return fail(WTQ_ERR_ARG, "wtq_qk_norm_rope: bad sizes");
  rope::Params p = {};
  const int el = dtype == WTQ_F32 ? 4 : 2, V = 16 / el;
  bool vec = D % (2 * V) == 0 && rot % (2 * V) == 0;
  for (int s = 0; s < 3; ++s) {
    const wtq_rope_side_t &w = sides[s];
    if (w.heads < 0) return fail(WTQ_ERR_ARG, "wtq_qk_norm_rope: bad head count");
    rope::Side &d = p.side[s];
    d = {w.x, w.out, w.strides[0], w.strides[1], w.strides[2], w.out_strides[0], w.out_strides[1],
         w.out_strides[2], w.weight, w.heads, s < 2};
    p.heads += w.heads;
    if (p.heads > 65535) return fail(WTQ_ERR_ARG, "wtq_qk_norm_rope: too many heads");
    if (w.heads == 0 || B == 0 || n == 0) continue;
    if (!w.x || !w.out) return fail(WTQ_ERR_ARG, "wtq_qk_norm_rope: null input or output");
    vec = vec && ((uintptr_t)w.x % 16 | (uintptr_t)w.out % 16) == 0;
    for (int i = 0; i < 3; ++i) vec = vec && w.strides[i] % V == 0 && w.out_strides[i] % V == 0;
  }
  if (B == 0 || n == 0 || p.heads == 0) return WTQ_OK;
  if (!positions || (rot > 0 && !table)) return fail(WTQ_ERR_ARG, "wtq_qk_norm_rope: null positions or table");
  p.positions = positions; p.position_stride = position_stride;
  p.table = table; p.table_stride = table_stride; p.table_rows = table_rows;
  p.weight_dtype = weight_dtype; p.eps = eps;
  p.B = B; p.n = n; p.D = D; p.rot = rot; p.status = status;
  if (!vec) {
    const int64_t rows = (int64_t)B * n * p.heads;
    const int grid = (int)std::min<int64_t>((rows + 3) / 4, (int64_t)device_sms() * 16);
    rope::any_kernel<<<grid, 128, 0, stream>>>(p, dtype, interleaved);
  } else {
    const int tpr = D / (2 * V);
    // All of a token's heads to a group once that still leaves every multiprocessor its 2048
    // threads; a head to a group where there are few.
    const int64_t threads = (int64_t)B * n * std::max(tpr, 2);
    const int64_t room = (int64_t)device_sms() * 2048;
    const int64_t per_token = std::min<int64_t>(p.heads, std::max<int64_t>(1, (room + threads - 1) / threads));
    p.heads_per_group = (int)((p.heads + per_token - 1) / per_token);
    if (p.heads_per_group > rope::kBatch)                // whole batches
      p.heads_per_group = (p.heads_per_group + rope::kBatch - 1) / rope::kBatch * rope::kBatch;
    if (dtype == WTQ_F32) rope::launch_width<WTQ_F32>(p, tpr, interleaved, stream);
    else if (dtype == WTQ_F16) rope::launch_width<WTQ_F16>(p, tpr, interleaved, stream);
    else rope::launch_width<WTQ_BF16>(p, tpr, interleaved, stream);
  }
  note_launches(1);
  return check_cuda(cudaGetLastError(), "wtq_qk_norm_rope launch");
}
