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
// thread too), so the rotation needs no exchange and the norm a few shuffles.  A group keeps a
// token's table row in registers and walks over heads; how many depends on the call: with few
// tokens a head each, which is the shortest chain, with many all of a token's heads, which reads
// the table once.  Bound by HBM at prompts and by the launch at single tokens.
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
template <int DT> __device__ __forceinline__ void unpack(const uint4 &v, float *x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (DT == WTQ_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f;
      if constexpr (DT == WTQ_F16) f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <int DT> __device__ __forceinline__ uint4 packed(const float *x) {
  uint32_t w[4];
  if constexpr (DT == WTQ_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == WTQ_F16) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
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

// A thread's two pieces of a weight vector (ones without weights).
template <int V> __device__ __forceinline__ void load_weights(const void *w, int dtype, int at0, int at1, float (&x)[2 * V]) {
  const int el = dtype == WTQ_F32 ? 4 : 2;
  if (w == nullptr) {
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) x[j] = 1.f;
  } else if (16 / el == V && ((uintptr_t)w & 15) == 0) {
    const uint4 a = __ldg(reinterpret_cast<const uint4 *>((const char *)w + at0 * el));
    const uint4 c = __ldg(reinterpret_cast<const uint4 *>((const char *)w + at1 * el));
    if constexpr (V == 4) {
      unpack<WTQ_F32>(a, x);
      unpack<WTQ_F32>(c, x + V);
    } else if (dtype == WTQ_F16) {
      unpack<WTQ_F16>(a, x);
      unpack<WTQ_F16>(c, x + V);
    } else {
      unpack<WTQ_BF16>(a, x);
      unpack<WTQ_BF16>(c, x + V);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      x[j] = load_as_float(w, at0 + j, dtype);
      x[V + j] = load_as_float(w, at1 + j, dtype);
    }
  }
}

// TPR threads a row (a power of two, at most 32); D, rot and D - rot are multiples of two pieces
// and every row is 16-byte aligned.  The pieces of kBatch heads are read before the first is worked on.
constexpr int kBatch = 4;
template <int DT, int TPR, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rows_kernel(Params p) {
  constexpr int V = Vec<DT>::kN;
  const int lane_in_row = threadIdx.x % TPR;
  const int64_t group = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const int per_token = (p.heads + p.heads_per_group - 1) / p.heads_per_group;
  const int64_t token = group / per_token;
  // (threads of a warp stay together for the shuffles: a group past the end works on nothing)
  const bool real = token < (int64_t)p.B * p.n;
  const int first = real ? (int)(group - token * per_token) * p.heads_per_group : p.heads;
  const int last = min(first + p.heads_per_group, p.heads);
  const int b = real ? (int)(token / p.n) : 0, i = real ? (int)(token - (int64_t)b * p.n) : 0;
  const int pairs = p.D / (2 * V), turned_pairs = p.rot / (2 * V);
  const bool has = lane_in_row < pairs, turns = lane_in_row < turned_pairs;
  // where this thread's two pieces start
  const int at0 = turns ? lane_in_row * V : p.rot + 2 * (lane_in_row - turned_pairs) * V;
  const int at1 = turns ? at0 + p.rot / 2 : at0 + V;
  auto load = [&](int k, uint4 &a, uint4 &c) {
    int head = first + k;
    if (head >= last || !has) return;
    const Side &sd = side_of(p, head);
    const char *src = (const char *)sd.x + (b * sd.xb + head * sd.xh + i * sd.xt) * (16 / V);
    a = *reinterpret_cast<const uint4 *>(src + at0 * (16 / V));
    c = *reinterpret_cast<const uint4 *>(src + at1 * (16 / V));
  };
  uint4 raw[kBatch][2];
  auto load_batch = [&](int k) {
#pragma unroll
    for (int e = 0; e < kBatch; ++e) {
      raw[e][0] = raw[e][1] = make_uint4(0u, 0u, 0u, 0u);
      if (k + e < p.heads_per_group) load(k + e, raw[e][0], raw[e][1]);
    }
  };
  load_batch(0);
  const int row = real ? table_row(p, b, i, lane_in_row == 0 && first == 0) : -1;
  float c[V], s[V];               // of the pairs of both pieces (halves: of piece 0's elements)
#pragma unroll
  for (int j = 0; j < V; ++j) c[j] = 1.f, s[j] = 0.f;
  if (turns && row >= 0) {
    const float *t = p.table + (int64_t)row * p.table_stride;
    // interleaved: pairs at0 / 2 .. and at1 / 2 .. of V / 2 each
    const int half = p.rot / 2, from0 = INTERLEAVED ? at0 / 2 : at0, from1 = INTERLEAVED ? at1 / 2 : at0 + V / 2;
    if ((((uintptr_t)t | (uintptr_t)(half * 4)) & 15) == 0 && V / 2 % 4 == 0) {
      *reinterpret_cast<float4 *>(c) = __ldg(reinterpret_cast<const float4 *>(t + from0));
      *reinterpret_cast<float4 *>(s) = __ldg(reinterpret_cast<const float4 *>(t + half + from0));
      if constexpr (V == 8) {
        *reinterpret_cast<float4 *>(c + V / 2) = __ldg(reinterpret_cast<const float4 *>(t + from1));
        *reinterpret_cast<float4 *>(s + V / 2) = __ldg(reinterpret_cast<const float4 *>(t + half + from1));
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int pair = j < V / 2 ? from0 + j : from1 + j - V / 2;
        c[j] = __ldg(t + pair);
        s[j] = __ldg(t + half + pair);
      }
    }
  }
  float weight[2 * V];
  const void *held = nullptr;
  bool any_held = false;
  for (int k0 = 0; k0 < p.heads_per_group; k0 += kBatch) {
   if (k0 > 0) load_batch(k0);
#pragma unroll
   for (int e = 0; e < kBatch; ++e) {
    if (k0 + e >= p.heads_per_group) break;              // (the same for all)
    int head = first + k0 + e;
    const bool work = head < last && has;
    if (!work) head = 0;
    const Side &sd = side_of(p, head);
    float x[2 * V];
    unpack<DT>(raw[e][0], x);
    unpack<DT>(raw[e][1], x + V);
    if (work && (!any_held || held != sd.weight)) {
      load_weights<V>(sd.weight, p.weight_dtype, at0, at1, weight);
      held = sd.weight;
      any_held = true;
    }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) sum = fmaf(x[j], x[j], sum);
    if (!work) sum = 0.f;
#pragma unroll
    for (int o = TPR / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o, TPR);
    if (work) {
      if (sd.weight != nullptr) {
        const float r = 1.f / sqrtf(sum / (float)p.D + p.eps);
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) x[j] *= r * weight[j];
      }
      if (sd.turned) {
        if (row < 0) {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) x[j] = 0.f;
        } else if (INTERLEAVED) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = x[2 * j], d = x[2 * j + 1];
            x[2 * j] = a * c[j] - d * s[j];
            x[2 * j + 1] = d * c[j] + a * s[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = x[j], d = x[V + j];
            x[j] = a * c[j] - d * s[j];
            x[V + j] = d * c[j] + a * s[j];
          }
        }
      }
      char *dst = (char *)sd.out + (b * sd.ob + head * sd.oh + i * sd.ot) * (16 / V);
      *reinterpret_cast<uint4 *>(dst + at0 * (16 / V)) = packed<DT>(x);
      *reinterpret_cast<uint4 *>(dst + at1 * (16 / V)) = packed<DT>(x + V);
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
  const int per_token = (p.heads + p.heads_per_group - 1) / p.heads_per_group;
  const int64_t groups = (int64_t)p.B * p.n * per_token;
  const unsigned blocks = (unsigned)((groups + 256 / TPR - 1) / (256 / TPR));
  if (interleaved) rows_kernel<DT, TPR, true><<<blocks, 256, 0, stream>>>(p);
  else rows_kernel<DT, TPR, false><<<blocks, 256, 0, stream>>>(p);
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
