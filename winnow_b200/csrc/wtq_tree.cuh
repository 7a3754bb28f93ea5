// Parameter blocks and the schedule shared by the kernels of drafted trees' attention.
//
// A group is one (sequence, block of query rows, kv head); a kv head's query rows are (token, head)
// pairs in token-major order.  The tiles of all groups, laid end to end (sequence, row block, kv
// head), are cut into one equal run per block.  A group that lies inside one run leaves its state
// (reference maximum m in the log2 domain, sum l, un-normalised accumulator in the value basis) per
// query row; the pieces of a group that run boundaries cut go to two slots per block: slot 0 holds
// the piece a run begins with when its group began earlier, slot 1 a piece whose group goes on in
// the next run.  So the states take the same room whatever the lengths are.
#pragma once

#include "wtq_decode.cuh"

namespace wtq {
namespace tree {

constexpr int kMaxBatch = 1024;           // sequences of one launch (their tile prefix in shared memory)

struct Params {
  DecodeSideDev k, v;
  const void *q;
  int64_t qb, qh, qt;
  int dtype;
  float q_scale;                          // scale * log2(e)
  void *out;
  int64_t ob, oh, ot;
  const int32_t *page_table;
  int64_t table_stride;
  const int32_t *seq_lens;
  const int32_t *mask;
  int64_t mask_b, mask_t;
  int B, Hq, Hkv, n_rep, Q, R, D, S, P, max_tokens;   // R = Q * n_rep: rows of a kv head
  int rows, tile, row_blocks;             // query rows of a group, tokens of a tile
  int blocks, least;                      // blocks of the scan; fewest tiles of a run
  float *q_rot;                           // (B, Q, Hq, D) rotated queries times q_scale
  float *acc, *m, *l;                     // whole groups: (B, Q, Hq) states
  float *part_acc, *part_m, *part_l;      // cut groups: (blocks, 2, rows) states
  int32_t *status;
};

__device__ __forceinline__ int length_of(const Params &p, int b) {
  const int L = p.seq_lens[b];
  return L < 0 ? 0 : L > p.max_tokens ? p.max_tokens : L;
}
// Tokens before a sequence's tree.  Its length as it is says where the tree stands, also where the table has no room
// for all of it: tokens past the table do not exist then.
__device__ __forceinline__ int history_of(const Params &p, int b) { return p.seq_lens[b] - p.Q; }
__device__ __forceinline__ int tiles_of(const Params &p, int b) { return (length_of(p, b) + p.tile - 1) / p.tile; }

// Exclusive prefix (B + 1 entries) of the sequences' tiles, by the whole block.  Lengths past the table are reported.
__device__ __forceinline__ void tile_prefix(const Params &p, int *prefix) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int running = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int n = b0 + lane < p.B ? tiles_of(p, b0 + lane) : 0;
      if (blockIdx.x == 0 && b0 + lane < p.B && p.seq_lens[b0 + lane] > p.max_tokens && p.status)
        atomicOr(p.status, WTQ_STATUS_BAD_POSITION);
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      if (b0 + lane < p.B) prefix[b0 + lane] = running + incl - n;
      running += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) prefix[p.B] = running;
  }
  __syncthreads();
}
// Tiles of a run, from the prefix.
__device__ __forceinline__ long long run_length(const Params &p, const int *prefix) {
  const long long all = (long long)prefix[p.B] * p.row_blocks * p.Hkv;
  const long long share = (all + p.blocks - 1) / p.blocks;
  return share > p.least ? share : p.least;
}

// One piece of a run: tiles [first, last) of a group.
struct Piece {
  int b, rb, h, first, last;
  int slot;                               // -1: the whole group
};
// The piece that begins at tile x (of all groups') of the run that ends at `end`.
__device__ __forceinline__ Piece piece_at(const Params &p, const int *prefix, long long x, long long begin,
                                          long long end) {
  const int heads = p.row_blocks * p.Hkv;
  int lo = 0, hi = p.B - 1;
  while (lo < hi) {                       // last sequence that starts at or before x (empty ones start where the next does)
    const int mid = (lo + hi + 1) / 2;
    if ((long long)prefix[mid] * heads <= x) lo = mid;
    else hi = mid - 1;
  }
  Piece c;
  c.b = lo;
  const int n = prefix[lo + 1] - prefix[lo];
  const long long in = x - (long long)prefix[lo] * heads;
  const int g = (int)(in / n);
  c.rb = g / p.Hkv;
  c.h = g - c.rb * p.Hkv;
  c.first = (int)(in - (long long)g * n);
  const long long left = end - x;
  c.last = left < n - c.first ? c.first + (int)left : n;
  c.slot = c.first > 0 ? 0 : c.last < n ? 1 : -1;
  return c;
}

// Tree places of a sequence that the table has room for (negative: not even all of the history).
__device__ __forceinline__ int places_of(const Params &p, int b) {
  const int room = p.max_tokens - history_of(p, b);
  return room < p.Q ? room : p.Q;
}
// 32 tokens from tree place `j0` on as bits, of a row with the mask words at `words`: places before
// the tree are its history, those from `places` on do not exist.
__device__ __forceinline__ uint32_t visible(const int32_t *words, int places, int j0) {
  if (j0 <= -32 && places >= 0) return 0xffffffffu;
  const int k = j0 >> 5, r = j0 & 31;     // (floor)
  auto word = [&](int i) -> uint32_t {
    if (32 * i >= places) return 0u;
    const uint32_t w = i < 0 ? 0xffffffffu : (uint32_t)__ldg(words + i);
    return places - 32 * i >= 32 ? w : w & ((1u << (places - 32 * i)) - 1u);
  };
  return __funnelshift_r(word(k), word(k + 1), r);
}
// Whether a row's token is padding: no bit set.
__device__ __forceinline__ bool padding(const int32_t *words, int Q) {
  uint32_t any = 0;
  for (int i = 0; 32 * i < Q; ++i) {
    const uint32_t w = (uint32_t)__ldg(words + i);
    any |= Q - 32 * i >= 32 ? w : w & ((1u << (Q - 32 * i)) - 1u);
  }
  return any == 0;
}

// Launch behind the kernel ahead in the stream: its blocks may start, and set themselves up, while that
// one's last blocks run; what depends on it comes after griddepcontrol.wait.
template <typename... Kernel, typename... Args>
int launch_behind(void (*kernel)(Kernel...), int blocks, int threads, size_t bytes, cudaStream_t stream, const char *what,
                  Args... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  note_launches(1);
  return check_cuda(e, what);
}

bool on_tensor_cores(const wtq_side_t &k, const wtq_side_t &v, int dtype, int D, int S);
int launch_scan_umma(const Params &p, cudaStream_t stream);
bool rows_on_tensor_cores(const Params &p);
int launch_rotate(const Params &p, cudaStream_t stream);
int launch_join(const Params &p, cudaStream_t stream);
constexpr int kUmmaRows = 128, kUmmaTile = 64;

}  // namespace tree
}  // namespace wtq
