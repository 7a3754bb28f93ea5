// The accepted path of a drafted tree moves to the end of the kept history, in every layer: of the
// `drafted` tokens a sequence appended, token keep[i] becomes token i (i = 0 .. count - 1), as the
// codes and norms that it has, and the sequence ends there.  keep ascends, so keep[i] >= i.
//
// A warp takes four kv heads of one side of one (layer, sequence), sixteen-byte words of as many rows as
// fit at a time: it reads them all, then writes them.  A batch of rows may only write
// places up to its last row's, and every later source lies behind those, so the batches of a
// warp can follow one another and no two warps meet.  Where a row comes from and goes to is looked up
// once for the four: a warp per head spent its time in that chain of three dependent reads (64
// sequences, 28 layers, 7 tokens kept, 28 MB moved: 27 us, this form 20).
#include <algorithm>
#include <type_traits>

#include "wtq_common.cuh"

namespace wtq {
namespace keep {

struct Side {
  uint8_t *pages;
  __half *norms;
  int64_t layer_stride, page_stride, head_stride;                // bytes
  int64_t norm_layer_stride, norm_page_stride, norm_head_stride; // elements
  int nb;
};
struct Params {
  Side side[2];
  const int32_t *table, *seq_lens, *keep, *counts;
  int64_t table_stride, keep_stride;
  int B, Hkv, S, P, W, layers, A, drafted;
  const int32_t *granted;
  int32_t *out, *status;
};

constexpr int kThreads = 128;
constexpr int kMost = 32;                 // rows looked up at a time
constexpr int kHeads = 4;                 // kv heads of a warp

// The path of a sequence holds: 0 <= keep[0] < keep[1] < .. < drafted, and the drafted tokens exist.
// `mine`: entry `lane`, read beside the count that says whether it is one.
__device__ __forceinline__ bool path_holds(const Params &p, int b, int lane, int &count, int &base, int &mine) {
  const int32_t *path = p.keep + (int64_t)b * p.keep_stride;
  mine = lane < p.A ? path[lane] : -1;
  const int L = p.seq_lens[b];
  count = p.counts[b];
  base = L - p.drafted;
  bool ok = base >= 0 && (int64_t)L <= (int64_t)p.W * p.S && count >= 0 && count <= p.A && count <= p.drafted;
  const int before = __shfl_up_sync(0xffffffffu, mine, 1);
  if (ok && lane < count) ok = mine > (lane > 0 ? before : -1) && mine < p.drafted;
  for (int i = lane + 32; ok && i < count; i += 32) ok = path[i] > path[i - 1] && path[i] < p.drafted;
  return __all_sync(0xffffffffu, ok);
}

// WORD bytes a lane: rows are multiples of it and aligned to it.
template <int WORD>
__global__ void __launch_bounds__(kThreads, 8) keep_kernel(Params p) {
  using T = typename std::conditional<WORD == 16, uint4, typename std::conditional<WORD == 4, uint32_t, uint8_t>::type>::type;
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int groups = (p.Hkv + kHeads - 1) / kHeads;
  const int64_t units = (int64_t)p.layers * p.B * groups * 2;
  if (unit >= units) return;
  const int side = (int)(unit & 1);
  const int h0 = (int)((unit >> 1) % groups) * kHeads;
  const int b = (int)((unit >> 1) / groups % p.B);
  const int layer = (int)((unit >> 1) / groups / p.B);
  if (p.granted != nullptr && *p.granted == 0) {         // the trees were never appended
    if (layer == 0 && side == 0 && h0 == 0 && lane == 0) p.out[b] = p.seq_lens[b];
    return;
  }
  int count, base, mine;
  const bool ok = path_holds(p, b, lane, count, base, mine);
  if (layer == 0 && side == 0 && h0 == 0 && lane == 0) {
    // (a malformed path: nothing is kept of the tree; a sequence too short for it stays as it is)
    p.out[b] = ok ? base + count : base >= 0 ? base : p.seq_lens[b];
    if (!ok && p.status) atomicOr(p.status, WTQ_STATUS_BAD_POSITION);
  }
  if (!ok) return;
  const Side &sd = p.side[side];
  const int words = sd.nb / WORD;                        // of a row
  const int32_t *table = p.table + (int64_t)b * p.table_stride;
  uint8_t *pages = sd.pages + layer * sd.layer_stride;
  __half *norms = sd.norms + layer * sd.norm_layer_stride;
  for (int i0 = 0; i0 < count; i0 += kMost) {
    const int rows = min(kMost, count - i0);
    // lane r: where row i0 + r comes from and goes to (-1: it stays, or a page is not the pool's)
    int64_t from = -1, to = -1, norm_from = 0, norm_to = -1;
    if (lane < rows) {
      const int i = i0 + lane, k = i0 == 0 ? mine : p.keep[(int64_t)b * p.keep_stride + i];
      if (k != i) {
        const int src = base + k, dst = base + i;
        const int sp = table[src / p.S], dp = table[dst / p.S];
        if ((uint32_t)sp < (uint32_t)p.P && (uint32_t)dp < (uint32_t)p.P) {
          from = (int64_t)sp * sd.page_stride + (int64_t)(src % p.S) * sd.nb;
          to = (int64_t)dp * sd.page_stride + (int64_t)(dst % p.S) * sd.nb;
          norm_from = (int64_t)sp * sd.norm_page_stride + src % p.S;
          norm_to = (int64_t)dp * sd.norm_page_stride + dst % p.S;
        } else if (p.status) {
          atomicOr(p.status, WTQ_STATUS_BAD_PAGE);
        }
      }
    }
    {
      __half n[kHeads];
      __syncwarp();
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
        if (norm_to >= 0 && h0 + h < p.Hkv) n[h] = norms[norm_from + (h0 + h) * sd.norm_head_stride];
      __syncwarp();
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
        if (norm_to >= 0 && h0 + h < p.Hkv) norms[norm_to + (h0 + h) * sd.norm_head_stride] = n[h];
      // words of the rows in order, 32 at a time; row i's places lie at or before its source
      for (int w0 = 0; w0 < rows * words; w0 += 32) {
        const int w = w0 + lane, r = min(w / words, kMost - 1);
        const int64_t f = __shfl_sync(0xffffffffu, from, r), t = __shfl_sync(0xffffffffu, to, r);
        const bool moves = w < rows * words && f >= 0;
        const int64_t off = (int64_t)(w - r * words) * WORD;
        T v[kHeads];
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
          if (moves && h0 + h < p.Hkv) v[h] = *reinterpret_cast<const T *>(pages + f + off + (h0 + h) * sd.head_stride);
        __syncwarp();
#pragma unroll
        for (int h = 0; h < kHeads; ++h)
          if (moves && h0 + h < p.Hkv) *reinterpret_cast<T *>(pages + t + off + (h0 + h) * sd.head_stride) = v[h];
        __syncwarp();
      }
    }
  }
}

}  // namespace keep
}  // namespace wtq

using namespace wtq;

extern "C" int wtq_keep_tokens(const wtq_pool_side_t *k_side, const wtq_pool_side_t *v_side, const int32_t *page_table,
                               int64_t table_stride, const int32_t *seq_lens, const int32_t *keep, int64_t keep_stride,
                               const int32_t *counts, int layers, int B, int Hkv, int S, int P, int max_pages, int most,
                               int drafted, const int32_t *granted, int32_t *out, int32_t *status, void *stream_) {
  if (!k_side || !v_side) return fail(WTQ_ERR_ARG, "wtq_keep_tokens: null sides");
  if (layers < 1 || B < 0 || Hkv < 1 || S < 1 || P < 1 || max_pages < 1 || most < 0 || drafted < 0)
    return fail(WTQ_ERR_ARG, "wtq_keep_tokens: bad sizes");
  if (B == 0) return WTQ_OK;
  if (!page_table || !seq_lens || !counts || !out || (most > 0 && !keep))
    return fail(WTQ_ERR_ARG, "wtq_keep_tokens: null argument");
  // (one warp writes a sequence's result while those of its other layers, sides and heads read these)
  const Span result = {out, (int64_t)B * 4};
  const Span read[5] = {{seq_lens, (int64_t)B * 4}, {counts, (int64_t)B * 4}, {granted, 4},
                        {keep, most > 0 ? ((B - 1) * keep_stride + most) * 4 : 0},
                        {page_table, ((B - 1) * table_stride + max_pages) * 4}};
  for (const Span &r : read)
    if (meet(result, r)) return fail(WTQ_ERR_ARG, "wtq_keep_tokens: out must not share memory with what is read");
  keep::Params p = {};
  bool by16 = true, by4 = true;
  const wtq_pool_side_t *sides[2] = {k_side, v_side};
  for (int i = 0; i < 2; ++i) {
    const wtq_pool_side_t &w = *sides[i];
    if (!w.pages || !w.norms || w.row_bytes < 1) return fail(WTQ_ERR_ARG, "wtq_keep_tokens: null pages or norms");
    p.side[i] = {w.pages, (__half *)w.norms, w.layer_stride, w.page_stride, w.head_stride, w.norm_layer_stride,
                 w.norm_page_stride, w.norm_head_stride, w.row_bytes};
    const uint64_t all = (uint64_t)(uintptr_t)w.pages | (uint64_t)w.layer_stride | (uint64_t)w.page_stride |
                         (uint64_t)w.head_stride | (uint64_t)w.row_bytes;
    by16 = by16 && all % 16 == 0;
    by4 = by4 && all % 4 == 0;
  }
  p.table = page_table; p.seq_lens = seq_lens; p.keep = keep; p.counts = counts;
  p.table_stride = table_stride; p.keep_stride = keep_stride;
  p.B = B; p.Hkv = Hkv; p.S = S; p.P = P; p.W = max_pages; p.layers = layers; p.A = most; p.drafted = drafted;
  p.granted = granted; p.out = out; p.status = status;
  const int64_t units = (int64_t)layers * B * ((Hkv + keep::kHeads - 1) / keep::kHeads) * 2, blocks = (units + 3) / 4;
  if (blocks > 0x7fffffff) return fail(WTQ_ERR_ARG, "wtq_keep_tokens: too many rows");
  cudaStream_t stream = (cudaStream_t)stream_;
  if (by16) keep::keep_kernel<16><<<(unsigned)blocks, keep::kThreads, 0, stream>>>(p);
  else if (by4) keep::keep_kernel<4><<<(unsigned)blocks, keep::kThreads, 0, stream>>>(p);
  else keep::keep_kernel<1><<<(unsigned)blocks, keep::kThreads, 0, stream>>>(p);
  note_launches(1);
  return check_cuda(cudaGetLastError(), "wtq_keep_tokens launch");
}
