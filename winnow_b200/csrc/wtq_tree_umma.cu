// Tensor-core scan of drafted trees' attention: 16-bit queries, head_dim 64 or 128, packed widths 4, 6
// and 8.  The schedule is in wtq_tree.cuh; a group has 128 query rows, a tile 64 tokens.
//
// The query rows of a group lie in tensor memory as the fp16 A operand of all score products.  The
// group's tiles alternate between two streams, each with scores, probabilities, accumulator, running
// maximum and sum of its own, so that one stream's softmax runs under the other's products; the two
// states are joined when the piece ends.  Sixteen warps in four roles that meet at mbarriers only:
//
//   fetch     one warp: codes and norms of a tile as bulk copies into a ring of raw tiles, a lane per
//             16 tokens of codes or norms of a side;
//   decode    six warps: tasks of 16 tokens of one side through the per-lane lookup tables
//             (wtq_lut.cuh) into the canonical operand layout, three tiles deep.  Keys go as
//             centroids, their norms beside them in fp32 (the scores take them after the product,
//             unrounded); values as centroid times norm;
//   multiply  one warp, an elected lane issues: S = Q K^T (N 64) two tiles ahead of O += P V
//             (A = P from tensor memory, V read with tokens as the contraction);
//   softmax   a warpgroup per stream, a thread per query row: scores from tensor memory, handed back at
//             once; norms, tree mask, running maximum, probabilities as fp16.  O is rescaled only when
//             a row's maximum grows by 2^8.
//
// The roles walk the static schedule by themselves: fetch and decode work into the next piece while
// the softmax warps write the last one's states.  Every wait is bounded; one that runs out
// raises a flag that ends all others, and the status word says so.
//
// fp16 scores carry an error that grows with |q| |k|; a warp whose tile holds a row maximum beyond
// kPreciseAbove (log2 domain) recomputes that tile's scores in fp32 from the packed codes.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "wtq_lut.cuh"
#include "wtq_tree.cuh"
#include "wtq_umma.cuh"

namespace wtq {
namespace tree {
namespace um {

using namespace umma;

constexpr int kSoftWarps = 8, kDecodeWarps = 6, kFetchWarp = kSoftWarps + kDecodeWarps, kMmaWarp = kFetchWarp + 1;
constexpr int kThreads = 32 * (kMmaWarp + 1);
constexpr int kRows = kUmmaRows, kTile = kUmmaTile;
constexpr int kStages = 3;                      // decoded tiles of a side
constexpr int kNormRing = 8;                    // tiles whose key norms are kept
constexpr uint32_t kFull = 0xffffffffu;
// shared memory; dynamic shared memory is assumed to start at or below kBase
constexpr uint32_t kBase = 1024;
constexpr uint32_t kKFull = kBase, kVFull = kKFull + 8 * kStages, kKFree = kVFull + 8 * kStages,
                   kVFree = kKFree + 8 * kStages;                          // [stage]
constexpr uint32_t kSFull = kVFree + 8 * kStages, kSFree = kSFull + 16, kPFull = kSFree + 16,
                   kODone = kPFull + 16;                                   // [stream]
constexpr uint32_t kNFull = kODone + 16;                                   // [ring]: key norms are there
constexpr int kMostRaw = 5;                     // raw tiles: as many of these as fit
constexpr uint32_t kRawFull = kNFull + 8 * kNormRing, kRawFree = kRawFull + 8 * kMostRaw;   // [raw tile]
constexpr uint32_t kQFull = kRawFree + 8 * kMostRaw, kLast = kQFull + 8, kTmemSlot = kLast + 8, kAbort = kTmemSlot + 4;
constexpr uint32_t kValid = kAbort + 4;                                    // [raw tile]: tokens of it that exist
constexpr uint32_t kPrefix = kBase + 512;                                  // kMaxBatch + 1 words
constexpr uint32_t kNorms = kPrefix + 4 * (kMaxBatch + 4);                 // [ring][64] fp32
constexpr uint32_t kStates = kNorms + kNormRing * kTile * 4;               // [stream][m, l][row]
constexpr uint32_t kVTile = 16384;
static_assert(kValid + 4 * kMostRaw <= kPrefix && kStates + 4 * kRows * 4 <= kVTile, "low region");
static_assert(kVTile + kStages * kTile * 256 <= mma::kLutAddr, "value tiles end where the tables begin");
// tensor memory columns
constexpr uint32_t kColQ = 0, kColS = 64, kColP = 192, kColO = 256, kCols = 512;   // S + 64, P + 32, O + 128 per stream
constexpr float kPreciseAbove = 24.f;
constexpr float kSlack = 8.f;
constexpr int kWaitTries = 1 << 20;

template <int BWK, int BWV, int D> struct Map {
  static constexpr int kEntries = mma::lut_entries(BWK) > mma::lut_entries(BWV) ? mma::lut_entries(BWK)
                                                                                : mma::lut_entries(BWV);
  static constexpr uint32_t kGroup = (uint32_t)D * 16u;                    // eight rows of an operand tile
  static constexpr uint32_t kTileBytes = kTile / 8 * kGroup;
  static constexpr uint32_t kKTile = mma::kLutAddr + (uint32_t)kEntries * 256u;
  // a raw tile: codes of K and V as the pages have them, then norms
  static constexpr uint32_t kCodesK = kTile * D * BWK / 8, kCodesV = kTile * D * BWV / 8;
  static constexpr uint32_t kRawBytes = kCodesK + kCodesV + 4 * kTile;
  static constexpr uint32_t kRaw = kKTile + kStages * kTileBytes;
  static constexpr int kFit = (int)((227u * 1024u - kRaw) / kRawBytes);
  static constexpr int kRawTiles = kFit < kMostRaw ? kFit : kMostRaw;
  static constexpr uint32_t kDynamic = kRaw + kRawTiles * kRawBytes;
  static_assert(kRawTiles >= 2 && kDynamic <= 227u * 1024u, "shared memory budget");
  static constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
  static constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
};

__device__ __forceinline__ void bulk_copy(uint32_t to, const void *from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(to),
               "l"(from), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}

// Bounded wait for completion number `use` (0, 1, ..) of an mbarrier; false if it, or any
// other wait of the block, ran out.
__device__ __forceinline__ bool wait(uint32_t bar, int use) {
  for (int spin = 0; spin < kWaitTries; ++spin) {
    if (mbar_try(bar, (uint32_t)(use & 1))) return true;
    if ((spin & 255) == 255 && lds32(kAbort) != 0u) return false;
  }
  sts32(kAbort, 1u);
  return false;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// ---- decode ------------------------------------------------------------------------------------
// A lane's quarter of a packed row, D * BW / 32 bytes, is read by load_words of wtq_lut.cuh.
// Codes 2 I, 2 I + 1 of the quarter as fp16 centroids.
template <int BW, int I, int NW> __device__ __forceinline__ uint32_t two_codes(const uint32_t (&w)[NW], uint32_t sel) {
  if constexpr (BW == 4) return lut_byte<I % 4>(w[I / 4], sel);
  else return join(lut_code<BW, 2 * I>(w, sel), lut_code<BW, 2 * I + 1>(w, sel));
}
template <int BW, int NW, int... I>
__device__ __forceinline__ void quarter_codes(const uint32_t (&w)[NW], uint32_t sel, uint32_t *f,
                                              std::integer_sequence<int, I...>) {
  ((f[I] = two_codes<BW, I>(w, sel)), ...);
}
__device__ __forceinline__ uint32_t times(uint32_t c, __half2 n) {
  const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&c), n);
  return *reinterpret_cast<const uint32_t *>(&y);
}
// Rows g and g + 8 of tokens 16 u .. 16 u + 15, the quarter t of each, into an operand tile: all
// lookups of a row go out before its stores.
template <int BW, int D, bool SCALED, int NW>
__device__ __forceinline__ void decode_task(uint32_t tile, int u, int g, int t, uint32_t sel, const uint32_t (&w)[2][NW],
                                            const __half (&nrm)[2]) {
  constexpr int kPairs = D / 8;                       // code pairs of a quarter
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t f[kPairs];
    quarter_codes<BW>(w[h], sel, f, std::make_integer_sequence<int, kPairs>{});
    if constexpr (SCALED) {
      const __half2 n = __half2half2(nrm[h]);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) f[i] = times(f[i], n);
    }
    const uint32_t at = tile + (uint32_t)(2 * u + h) * (uint32_t)(D * 16) + (uint32_t)t * (D / 32 * 128) + (uint32_t)g * 16u;
#pragma unroll
    for (int i = 0; i < kPairs / 4; ++i) sts128(at + 128u * i, f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
  }
}

// fp32 products of this thread's query row with the 64 tokens' centroids, written over the tile's
// scores in tensor memory: the packed codes are read from the pages (the same address for the whole
// warp) and the row of `q` along with them.  Out of line: only for tiles whose scores came out large.
template <int BW, int D>
__device__ __noinline__ void precise_tile(const uint8_t *pages, int64_t page_stride, const float *centroids,
                                          const int32_t *table, int P, int S, int tok0, int end, const float *q,
                                          uint32_t s_addr) {
  constexpr int kRowBytes = D * BW / 8;
#pragma unroll 1
  for (int blk = 0; blk < kTile / 16; ++blk) {                // sixteen tokens of one page
    const int tok = tok0 + 16 * blk;
    const int page = tok < end ? table[tok / S] : -1;
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.f;
    if ((uint32_t)page < (uint32_t)P) {
      const uint8_t *row = pages + (int64_t)page * page_stride + (int64_t)(tok % S) * kRowBytes;
#pragma unroll 1
      for (int d = 0; d < D / 4; ++d) {                        // four coordinates: BW / 2 bytes of each row
        const float4 x = q ? __ldg(reinterpret_cast<const float4 *>(q) + d) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          uint32_t w = 0;
#pragma unroll
          for (int b = 0; b < BW / 2; ++b) w |= (uint32_t)__ldg(row + i * kRowBytes + d * (BW / 2) + b) << (8 * b);
          constexpr uint32_t kMask = (1u << BW) - 1u;
          acc[i] = fmaf(x.x, __ldg(centroids + (w & kMask)), acc[i]);
          acc[i] = fmaf(x.y, __ldg(centroids + ((w >> BW) & kMask)), acc[i]);
          acc[i] = fmaf(x.z, __ldg(centroids + ((w >> (2 * BW)) & kMask)), acc[i]);
          acc[i] = fmaf(x.w, __ldg(centroids + ((w >> (3 * BW)) & kMask)), acc[i]);
        }
      }
    }
    uint32_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(acc[i]);
    __syncwarp();
    tmem_store16(s_addr + 16 * blk, v);
  }
  tmem_wait_store();
}

// Scores times key norms, those of unseen tokens -inf (`masked`: the tile reaches into the tree);
// returns the row's maximum.
__device__ __forceinline__ float norms_and_maximum(uint32_t (&s)[64], uint32_t norms, bool masked, uint32_t lo, uint32_t hi) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint4 n = lds128(norms + 16 * i);
    const float2 a = halves(mul2(pair(__uint_as_float(s[4 * i]), __uint_as_float(s[4 * i + 1])),
                                 pair(__uint_as_float(n.x), __uint_as_float(n.y))));
    const float2 b = halves(mul2(pair(__uint_as_float(s[4 * i + 2]), __uint_as_float(s[4 * i + 3])),
                                 pair(__uint_as_float(n.z), __uint_as_float(n.w))));
    s[4 * i] = __float_as_uint(a.x); s[4 * i + 1] = __float_as_uint(a.y);
    s[4 * i + 2] = __float_as_uint(b.x); s[4 * i + 3] = __float_as_uint(b.y);
  }
  if (masked) {
#pragma unroll
    for (int i = 0; i < 64; ++i) s[i] = ((i < 32 ? lo >> i : hi >> (i - 32)) & 1u) ? s[i] : 0xff800000u;
  }
  float a = -INFINITY, c = -INFINITY;
#pragma unroll
  for (int i = 0; i < 64; i += 4) {
    a = max3(a, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    c = max3(c, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
  }
  return fmaxf(a, c);
}

template <int BWK, int BWV, int D>
__global__ void __launch_bounds__(kThreads, 1) scan_kernel(Params p) {
  using M = Map<BWK, BWV, D>;
  extern __shared__ __align__(128) uint8_t dyn_smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((uint32_t)__cvta_generic_to_shared(dyn_smem) > kBase) {   // layout assumption broken
    if (p.status && tid == 0) atomicOr(p.status, WTQ_STATUS_LAYOUT);
    return;
  }
  int *prefix = reinterpret_cast<int *>(dyn_smem + (kPrefix - (uint32_t)__cvta_generic_to_shared(dyn_smem)));
  for (int e = tid; e < M::kEntries * 64; e += kThreads)
    sts32(mma::kLutAddr + 4u * e, mma::lut_word(e, BWK, BWV, p.k.centroids, p.v.centroids));
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(kTmemSlot),
                 "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      mbar_init(kKFull + 8u * i, 4);                        // the four 16-token groups of a tile
      mbar_init(kVFull + 8u * i, 4);
      mbar_init(kKFree + 8u * i, 1);
      mbar_init(kVFree + 8u * i, 1);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(kSFull + 8u * i, 1);
      mbar_init(kSFree + 8u * i, 4);                        // the four warps of a stream
      mbar_init(kPFull + 8u * i, 4);
      mbar_init(kODone + 8u * i, 1);
    }
#pragma unroll
    for (int i = 0; i < kNormRing; ++i) mbar_init(kNFull + 8u * i, 4);
#pragma unroll
    for (int i = 0; i < kMostRaw; ++i) {
      mbar_init(kRawFull + 8u * i, 1);
      mbar_init(kRawFree + 8u * i, 8);                      // the eight tasks of a tile
    }
    mbar_init(kQFull, kSoftWarps);
    mbar_init(kLast, 1);
    sts32(kAbort, 0u);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  fence_before();
  tile_prefix(p, prefix);                                   // (ends with a block barrier)
  fence_after();
  const uint32_t tmem = lds32(kTmemSlot);
  const long long share = run_length(p, prefix), all = (long long)prefix[p.B] * p.row_blocks * p.Hkv;
  const long long begin = share * blockIdx.x, end = min(all, begin + share);

  // Registers go from the other warps to the softmax warps, which hold 64 scores a thread: 2 x 128 x
  // (168 + 88) are the 512 x 128 that the block was launched with.
  if (warp < kSoftWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;\n");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 88;\n");

  if (warp < kSoftWarps) {
    // ================= softmax: stream `st`, one query row per thread ====================
    const int st = warp >> 2, r = 32 * (warp & 3) + lane;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_addr = tmem + lanes + kColS + 64u * st, p_addr = tmem + lanes + kColP + 32u * st,
                   o_addr = tmem + lanes + kColO + 128u * st;
    int tiles = 0, units = 0;                               // tiles of the pieces before; units of this stream
    bool ok = true;
    for (long long x = begin; x < end;) {
      const Piece c = piece_at(p, prefix, x, begin, end);
      const int nt = c.last - c.first;
      x += nt;
      const int L = length_of(p, c.b), hist = L - p.Q, qr = c.rb * kRows + r;
      const int32_t *table = p.page_table + (int64_t)c.b * p.table_stride;
      const int i = qr / p.n_rep;
      const int32_t *words = p.mask + c.b * p.mask_b + i * p.mask_t;
      const bool live = qr < p.R && !padding(words, p.Q);
      const bool working = __any_sync(kFull, live);         // a warp without live rows only keeps step
      const int64_t row = ((int64_t)c.b * p.Q + i) * p.Hq + c.h * p.n_rep + qr - i * p.n_rep;
      const float *q = live ? p.q_rot + row * D : nullptr;
      // this warpgroup's half of the query rows into tensor memory (the products of the last piece are done)
      if constexpr (D == 128) {
        uint32_t v[32];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float4 y = q ? __ldg(reinterpret_cast<const float4 *>(q + 64 * st) + k) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[2 * k] = pack_half2(y.x, y.y);
          v[2 * k + 1] = pack_half2(y.z, y.w);
        }
        tmem_store32(tmem + lanes + kColQ + 32u * st, v);
      } else {
        uint32_t v[16];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float4 y = q ? __ldg(reinterpret_cast<const float4 *>(q + 32 * st) + k) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[2 * k] = pack_half2(y.x, y.y);
          v[2 * k + 1] = pack_half2(y.z, y.w);
        }
        tmem_store16(tmem + lanes + kColQ + 16u * st, v);
      }
      tmem_wait_store();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(kQFull);
      float ref = -INFINITY, sum = 0.f;
      const int mine = (nt + 1 - st) / 2;                   // units of this stream in the piece
      for (int k = 0; k < mine && ok; ++k) {
        const int j = 2 * k + st, T = tiles + j, n = units + k, tok0 = (c.first + j) * kTile;
        ok = wait(kSFull + 8u * st, n) && wait(kNFull + 8u * (T % kNormRing), T / kNormRing);
        if (!__all_sync(kFull, ok)) { ok = false; break; }
        fence_after();
        const uint32_t norms = kNorms + (uint32_t)(T % kNormRing) * (kTile * 4);
        const bool masked = tok0 + kTile > hist;
        uint32_t lo = kFull, hi = kFull;
        if (masked && live) {
          lo = visible(words, p.Q, tok0 - hist);
          hi = visible(words, p.Q, tok0 + 32 - hist);
        }
        if (!working) {
          if (lane == 0) mbar_arrive(kSFree + 8u * st);
          if (k > 0) {
            ok = __all_sync(kFull, wait(kODone + 8u * st, n - 1));
            if (!ok) break;
          }
          if (lane == 0) mbar_arrive(kPFull + 8u * st);
          continue;
        }
        uint32_t s[64];
        tmem_load32<0>(s_addr, s);
        tmem_load32<32>(s_addr + 32, s);
        tmem_wait_load();
        float mx = norms_and_maximum(s, norms, masked, lo, hi);
        if (__any_sync(kFull, !(fabsf(mx) <= kPreciseAbove) && mx != -INFINITY)) {
          precise_tile<BWK, D>(p.k.pages + (int64_t)c.h * p.k.head_stride, p.k.page_stride, p.k.centroids, table, p.P,
                               p.S, tok0, L, q, s_addr);
          tmem_load32<0>(s_addr, s);
          tmem_load32<32>(s_addr + 32, s);
          tmem_wait_load();
          mx = norms_and_maximum(s, norms, masked, lo, hi);
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(kSFree + 8u * st);       // the scores are in registers
        if (k > 0) {                                        // the stream's last products have ended
          ok = wait(kODone + 8u * st, n - 1);
          if (!__all_sync(kFull, ok)) { ok = false; break; }
          fence_after();
        }
        if (__any_sync(kFull, mx > ref + kSlack || (ref == -INFINITY && mx != -INFINITY))) {
          const float now = mx > ref + kSlack || ref == -INFINITY ? mx : ref;
          if (k > 0) {                                      // rescale what is accumulated
            const float scale = ref == now ? 1.f : ref == -INFINITY ? 0.f : ex2(ref - now);
            sum *= scale;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
              uint32_t o[32];
              tmem_load32<0>(o_addr + c0, o);
              tmem_wait_load();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale);
              tmem_store32(o_addr + c0, o);
            }
            tmem_wait_store();
          }
          ref = now;
        }
        const uint64_t base = twice(ref == -INFINITY ? 0.f : -ref);
        uint32_t pr[32];
        uint64_t sums = 0;                                  // (the bits of two zeros)
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 y = halves(add2(pair(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), base));
          const float a = ex2(y.x), b = ex2(y.y);
          sums = add2(sums, pair(a, b));
          pr[e] = pack_half2(a, b);
        }
        const float2 both = halves(sums);
        sum += both.x + both.y;
        tmem_store32(p_addr, pr);
        tmem_wait_store();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(kPFull + 8u * st);
      }
      // ---- the rows' states: the two streams joined, half the coordinates to each warpgroup ----
      if (ok && mine > 0) ok = wait(kODone + 8u * st, units + mine - 1);
      ok = __all_sync(kFull, ok);
      sts32(kStates + 4u * ((2 * st) * kRows + r), __float_as_uint(ref));
      sts32(kStates + 4u * ((2 * st + 1) * kRows + r), __float_as_uint(sum));
      fence_before();
      asm volatile("bar.sync 1, %0;\n" ::"r"(32 * kSoftWarps) : "memory");   // every softmax warp, whatever it gave up on
      fence_after();
      ok = ok && lds32(kAbort) == 0u;
      ok = __all_sync(kFull, ok);
      if (ok) {
        const float m0 = __uint_as_float(lds32(kStates + 4u * r)), l0 = __uint_as_float(lds32(kStates + 4u * (kRows + r)));
        const float m1 = __uint_as_float(lds32(kStates + 4u * (2 * kRows + r)));
        const float l1 = __uint_as_float(lds32(kStates + 4u * (3 * kRows + r)));
        const float top = fmaxf(m0, m1);
        const float w0 = m0 == -INFINITY ? 0.f : ex2(m0 - top), w1 = m1 == -INFINITY ? 0.f : ex2(m1 - top);
        float *acc;
        if (c.slot < 0) {
          acc = p.acc + row * D;
          if (st == 0 && qr < p.R) p.m[row] = live ? top : -INFINITY, p.l[row] = live ? w0 * l0 + w1 * l1 : 0.f;
        } else {
          const int64_t s = ((int64_t)blockIdx.x * 2 + c.slot) * kRows + r;
          acc = p.part_acc + s * D;
          if (st == 0) p.part_m[s] = live ? top : -INFINITY, p.part_l[s] = live ? w0 * l0 + w1 * l1 : 0.f;
        }
#pragma unroll 1
        for (int c0 = st * (D / 2); c0 < (st + 1) * (D / 2); c0 += 32) {
          uint32_t o[32], o1[32];
          tmem_load32<0>(tmem + lanes + kColO + c0, o);
          if (nt > 1) tmem_load32<0>(tmem + lanes + kColO + 128 + c0, o1);
          tmem_wait_load();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            float v = __uint_as_float(o[e]) * w0;
            if (nt > 1) v = fmaf(__uint_as_float(o1[e]), w1, v);
            o[e] = __float_as_uint(v);
          }
          if (live) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              reinterpret_cast<uint4 *>(acc + c0)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
      }
      tiles += nt;
      units += mine;
    }
  } else if (warp < kFetchWarp) {
    // ================= decode ==========================================================
    // Tasks of 16 tokens of one side, eight per tile (four of K, four of V), dealt round-robin.
    const int g = lane & 7, t = lane >> 3;
    const uint32_t sel = mma::kLutAddr | (uint32_t)(lane << 2);
    const long long tasks = 8 * max(0LL, end - begin);
    auto task = [&](int T, int u, auto is_v_) -> bool {
      constexpr bool kV = decltype(is_v_)::value;
      constexpr int BW = kV ? BWV : BWK, kRowBytes = D * BW / 8;
      const int raw = T % M::kRawTiles, buf = T % kStages;
      if (!__all_sync(kFull, wait(kRawFull + 8u * raw, T / M::kRawTiles))) return false;
      const uint32_t at = M::kRaw + (uint32_t)raw * M::kRawBytes, valid = lds32(kValid + 4u * raw);
      const uint32_t codes = at + (kV ? M::kCodesK : 0u) + (uint32_t)(16 * u + g) * kRowBytes + (uint32_t)t * (kRowBytes / 4);
      const uint32_t norms = at + M::kCodesK + M::kCodesV + (kV ? 2u * kTile : 0u) + (uint32_t)(16 * u + g) * 2u;
      uint32_t w[2][kRowBytes / 16];
      float n[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_words<kRowBytes / 4>(codes + (uint32_t)(8 * h) * kRowBytes, w[h]);
        n[h] = (uint32_t)(16 * u + g + 8 * h) < valid ? lds_half(norms + 16u * h) : 0.f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(kRawFree + 8u * raw);
      if (T >= kStages)                                     // the tile's last reader is done
        if (!__all_sync(kFull, wait((kV ? kVFree : kKFree) + 8u * buf, T / kStages - 1))) return false;
      if constexpr (!kV) {
        if (t == 0) {
          const uint32_t to = kNorms + (uint32_t)(T % kNormRing) * (kTile * 4) + (uint32_t)(16 * u + g) * 4u;
          sts32(to, __float_as_uint(n[0]));
          sts32(to + 32, __float_as_uint(n[1]));
        }
      }
      const __half nh[2] = {__float2half_rn(n[0]), __float2half_rn(n[1])};
      decode_task<BW, D, kV>((kV ? kVTile : M::kKTile) + (uint32_t)buf * M::kTileBytes, u, g, t, kV ? sel | 0x80u : sel, w, nh);
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive((kV ? kVFull : kKFull) + 8u * buf);
        if (!kV) mbar_arrive(kNFull + 8u * (T % kNormRing));
      }
      return true;
    };
    for (long long q = warp - kSoftWarps; q < tasks; q += kDecodeWarps) {
      const int T = (int)(q >> 3), u = (int)q & 3;
      if (!((q & 4) ? task(T, u, std::true_type{}) : task(T, u, std::false_type{}))) break;
    }
  } else if (warp == kFetchWarp) {
    // ================= fetch ===========================================================
    // lane: 16-token group lane & 3 of K codes, V codes, K norms, V norms (lane >> 2)
    const int u = lane & 3, kind = lane >> 2;
    const int page_shift = 31 - __clz(p.S);
    const DecodeSideDev &sd = (kind & 1) ? p.v : p.k;
    const uint32_t bytes = kind == 0 ? M::kCodesK / 4 : kind == 1 ? M::kCodesV / 4 : 2u * 16u;
    const uint32_t to = (kind == 0 ? 0u : kind == 1 ? M::kCodesK : M::kCodesK + M::kCodesV + (kind == 3 ? 2u * kTile : 0u)) +
                        (uint32_t)u * bytes;
    int T = 0;
    bool ok = true;
    for (long long x = begin; x < end && ok;) {
      const Piece c = piece_at(p, prefix, x, begin, end);
      x += c.last - c.first;
      const int L = length_of(p, c.b);
      const int32_t *table = p.page_table + (int64_t)c.b * p.table_stride;
      const uint8_t *codes = sd.pages + (int64_t)c.h * sd.head_stride;
      const __half *norms = sd.norms + (int64_t)c.h * sd.norm_head_stride;
      auto page_of = [&](int tile) {                        // -2: past the end
        const int tok = tile * kTile + 16 * u;
        return tile < c.last && tok < L ? table[tok >> page_shift] : -2;
      };
      int page = page_of(c.first), next = page_of(c.first + 1);
      for (int tile = c.first; tile < c.last; ++tile, ++T) {
        const int after = page_of(tile + 2);
        const int raw = T % M::kRawTiles;
        if (T >= M::kRawTiles) {
          ok = __all_sync(kFull, wait(kRawFree + 8u * raw, T / M::kRawTiles - 1));
          if (!ok) break;
        }
        const uint32_t at = M::kRaw + (uint32_t)raw * M::kRawBytes, bar = kRawFull + 8u * raw;
        const bool good = (uint32_t)page < (uint32_t)p.P;
        if (kind < 4 && !good) {
          if (kind >= 2) {                                  // (codes of such tokens are whatever was there)
            sts128(at + to, 0u, 0u, 0u, 0u);
            sts128(at + to + 16, 0u, 0u, 0u, 0u);
          } else if (kind == 0 && page != -2 && p.status) {
            atomicOr(p.status, WTQ_STATUS_BAD_PAGE);
          }
        }
        const uint32_t fetched = __reduce_add_sync(kFull, kind < 4 && good ? bytes : 0u);
        if (lane == 0) {
          sts32(kValid + 4u * raw, (uint32_t)min(kTile, L - tile * kTile));
          arrive_expect(bar, fetched);
        }
        __syncwarp();
        if (kind < 4 && good) {
          const int64_t slot = (tile * kTile + 16 * u) & (p.S - 1);
          const void *from = kind < 2 ? (const void *)(codes + (int64_t)page * sd.page_stride + slot * (D / 8) * sd.bw)
                                      : (const void *)(norms + (int64_t)page * sd.norm_page_stride + slot);
          bulk_copy(at + to, from, bytes, bar);
        }
        page = next;
        next = after;
      }
    }
  } else {
    // ================= multiply: the whole warp waits, one lane issues ======================
    const uint32_t issuer = elect_one();
    int tiles = 0, pieces = 0, units[2] = {0, 0};
    bool ok = true;
    for (long long x = begin; x < end && ok; ++pieces) {
      const Piece c = piece_at(p, prefix, x, begin, end);
      const int nt = c.last - c.first;
      x += nt;
      ok = wait(kQFull, pieces);
      if (!__all_sync(kFull, ok)) break;
      fence_after();
      auto scores = [&](int j) -> bool {                    // S of the piece's tile j
        const int T = tiles + j, buf = T % kStages, st = j & 1, n = units[st] + (j >> 1);
        if (!wait(kKFull + 8u * buf, T / kStages)) return false;
        if (n > 0 && !wait(kSFree + 8u * st, n - 1)) return false;
        fence_after();
        if (issuer) {
          const uint64_t kb = descriptor(M::kKTile + (uint32_t)buf * M::kTileBytes, 128u, M::kGroup);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            umma_ts(tmem + kColS + 64u * st, tmem + kColQ + 8u * ks, kb + 16u * ks, M::kIdescQK, ks > 0);
          umma_commit(kSFull + 8u * st);
          umma_commit(kKFree + 8u * buf);
        }
        __syncwarp();
        return true;
      };
      auto values = [&](int j) -> bool {                    // O += P V of tile j
        const int T = tiles + j, buf = T % kStages, st = j & 1, n = units[st] + (j >> 1);
        if (!wait(kVFull + 8u * buf, T / kStages)) return false;
        if (!wait(kPFull + 8u * st, n)) return false;
        fence_after();
        if (issuer) {
          const uint64_t vb = descriptor(kVTile + (uint32_t)buf * M::kTileBytes, M::kGroup, 128u);
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks)
            umma_ts(tmem + kColO + 128u * st, tmem + kColP + 32u * st + 8u * ks, vb + (uint64_t)(2 * M::kGroup / 16) * ks,
                    M::kIdescPV, j > 1 || ks > 0);
          umma_commit(kODone + 8u * st);
          umma_commit(kVFree + 8u * buf);
        }
        __syncwarp();
        return true;
      };
      for (int j = -2; j < nt && ok; ++j) {
        if (j + 2 < nt) ok = scores(j + 2);
        ok = __all_sync(kFull, ok);
        if (ok && j >= 0) ok = values(j);
        ok = __all_sync(kFull, ok);
      }
      tiles += nt;
      units[0] += (nt + 1) / 2;
      units[1] += nt / 2;
    }
  }
  fence_before();
  __syncthreads();
  if (tid == 0 && lds32(kAbort) != 0u && p.status) atomicOr(p.status, WTQ_STATUS_SCAN_TIMEOUT);
  if (warp == kMmaWarp) {
    // A block that gave up may have products in flight: they end before their tensor memory
    // goes to somebody else (bounded, like every wait).
    fence_after();
    if (elect_one()) umma_commit(kLast);
    __syncwarp();
    for (int spin = 0; spin < kWaitTries && !mbar_try(kLast, 0u); ++spin) {
    }
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

template <int BWK, int BWV, int D> int launch(const Params &p, cudaStream_t stream) {
  using M = Map<BWK, BWV, D>;
  static std::atomic<bool> opted_in[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !opted_in[dev & 63].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(scan_kernel<BWK, BWV, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)M::kDynamic);
    if (e != cudaSuccess) return check_cuda(e, "wtq_tree: shared memory opt-in");
    opted_in[dev & 63].store(true, std::memory_order_release);
  }
  scan_kernel<BWK, BWV, D><<<p.blocks, kThreads, M::kDynamic, stream>>>(p);
  note_launches(1);
  return check_cuda(cudaGetLastError(), "wtq_tree scan launch");
}
template <int D> int launch_widths(const Params &p, cudaStream_t stream) {
  if (p.k.bw == 4 && p.v.bw == 4) return launch<4, 4, D>(p, stream);
  if (p.k.bw == 4 && p.v.bw == 6) return launch<4, 6, D>(p, stream);
  if (p.k.bw == 6 && p.v.bw == 6) return launch<6, 6, D>(p, stream);
  return launch<8, 8, D>(p, stream);
}

}  // namespace um

bool on_tensor_cores(const wtq_side_t &k, const wtq_side_t &v, int dtype, int D, int S) {
  const bool widths = (k.bw == 4 && (v.bw == 4 || v.bw == 6)) || (k.bw == v.bw && (k.bw == 6 || k.bw == 8));
  auto fits = [](const wtq_side_t &s) {
    return (((uintptr_t)s.pages | (uintptr_t)s.norms) & 15) == 0 && s.page_stride % 16 == 0 && s.head_stride % 16 == 0 &&
           s.norm_page_stride % 8 == 0 && s.norm_head_stride % 8 == 0;
  };
  return dtype != WTQ_F32 && (D == 64 || D == 128) && widths && S >= 16 && (S & (S - 1)) == 0 && fits(k) && fits(v);
}

int launch_scan_umma(const Params &p, cudaStream_t stream) {
  return p.D == 128 ? um::launch_widths<128>(p, stream) : um::launch_widths<64>(p, stream);
}

}  // namespace tree
}  // namespace wtq
