// Tensor-core scan of drafted trees' attention: 16-bit queries, head_dim 64 or 128, packed widths 4, 6
// and 8.  The schedule is in wtq_tree.cuh; a group has 128 query rows, a tile 64 tokens.
//
// The query rows of a group lie in tensor memory as the fp16 A operand of all score products.  The
// group's tiles alternate between two streams, each with scores, probabilities, accumulator, running
// maximum and sum of its own, so that one stream's softmax runs under the other's products; the two
// states are joined when the piece ends.  Twenty to twenty-eight warps in roles that meet at mbarriers only:
//
//   fetch     a warp per side: codes and norms of a tile into a ring of raw tiles, 16 bytes a copy;
//   decode    four or eight warps per side, one for every 16 or 8 tokens of a tile: codes through the
//             per-lane lookup tables (wtq_lut.cuh) to fp16 centroid times norm in the canonical operand
//             layout, three tiles deep;
//   multiply  a warp for S = Q K^T (N 64) and one for O += P V (A = P from tensor memory, V read with
//             tokens as the contraction), an elected lane of each issues;
//   softmax   a warpgroup per stream, a thread per query row: scores from tensor memory, handed back at
//             once; tree mask, running maximum, probabilities as fp16.  O is rescaled only when a row's
//             maximum grows by 2^8.
//
// The roles walk the static schedule by themselves: fetch and decode work into the next piece while
// the softmax warps write the last one's states.  Every wait is bounded; one that runs out raises a
// flag that ends all others, and the status word says so.
//
// A warp on its own gets through an instruction in about nine cycles here, so a role is only as fast
// as its instructions per tile are few and lie in the instruction cache: with code of its own for each side
// the roles' loops were more than that holds (hit rate 89 %, the level behind at 77 % of its rate), and a
// few dozen instructions more cost 5 to 25 %.  Now (98 %, 30 %) bound by the chain of a stream's tile, scores ready
// to probabilities stored; issue slots 46 % used, the tensor pipe active 29 % of the time.  16 x 8 kv heads x 8192 tokens, 128 rows a group, 4 bits (69 GFLOP): 146 us
// with both rotations; 8 x 131 072 tokens, 512 rows a group (275 GFLOP): 374 us, 735 TFLOP/s.
//
// Rounded to fp16, because the products' operands are: query rows, centroids, centroid times norm and
// probabilities; sums, maxima and states are fp32.  Measured on fp16 results against 64 bits: 8.2e-4 over
// 1000 tokens, 1.3e-3 over 65 536; applied alone in 64 bits the centroids of the keys give 4.5e-4 to 8.1e-4
// of it, the queries 3.4e-4, the values 3e-4, the probabilities 1e-4 (a bf16 result's own rounding: 1.7e-3).
// The scores' error grows with |q| |k|; rows whose maximum in a tile lies beyond kPreciseAbove (log2
// domain) take that tile's scores in fp32 from the packed codes.
#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

#include "wtq_lut.cuh"
#include "wtq_tree.cuh"
#include "wtq_umma.cuh"

namespace wtq {
namespace tree {
namespace um {

using namespace umma;

constexpr int kSoftWarps = 8;
// Decode warps of a side: a code of 6 or 8 bits takes a lookup of its own and twice the instructions of
// a 4-bit one, so those sides have a warp for every 8 tokens of a tile instead of 16.
__host__ __device__ constexpr int decode_warps(int bw) { return bw == 4 ? 4 : 8; }
constexpr int kRows = kUmmaRows, kTile = kUmmaTile;
constexpr int kStages = 3;                      // decoded tiles of a side
constexpr int kMostRaw = 5;                     // raw tiles of a side: as many of these as fit
constexpr uint32_t kFull = 0xffffffffu;
// shared memory; dynamic shared memory is assumed to start at or below kBase
constexpr uint32_t kBase = 1024;
constexpr uint32_t kTileFull = kBase, kTileFree = kTileFull + 16 * kStages;                 // [side][stage]
constexpr uint32_t kRawFull = kTileFree + 16 * kStages, kRawFree = kRawFull + 16 * kMostRaw;   // [side][raw tile]
constexpr uint32_t kSFull = kRawFree + 16 * kMostRaw, kSFree = kSFull + 16, kPFull = kSFree + 16,
                   kODone = kPFull + 16;                                   // [stream]
constexpr uint32_t kQFull = kODone + 16, kLast = kQFull + 8, kTmemSlot = kLast + 8, kAbort = kTmemSlot + 4,
                   kBadNorm = kAbort + 4;                                  // a value norm that is not finite was met
constexpr uint32_t kPrefix = kBase + 512;                                  // kMaxBatch + 1 words
constexpr uint32_t kStates = kPrefix + 4 * (kMaxBatch + 4);                // [piece's parity][stream][m, l][row]
constexpr uint32_t kVTile = 16384;
static_assert(kBadNorm + 4 <= kPrefix && kStates + 2 * 4 * kRows * 4 <= kVTile, "low region");
static_assert(kVTile + kStages * kTile * 256 <= mma::kLutAddr, "value tiles end where the tables begin");
// tensor memory columns
constexpr uint32_t kColQ = 0, kColS = 64, kColP = 192, kColO = 256, kCols = 512;   // S + 64, P + 32, O + 128 per stream
constexpr float kPreciseAbove = 24.f;
constexpr float kSlack = 8.f;
constexpr int kWaitTries = 1 << 20;

template <int BWK, int BWV, int D> struct Map {
  static constexpr int kEntries = mma::lut_entries(BWK) > mma::lut_entries(BWV) ? mma::lut_entries(BWK)
                                                                                : mma::lut_entries(BWV);
  static constexpr int kDecodeK = kSoftWarps, kDecodeV = kDecodeK + decode_warps(BWK), kFetch = kDecodeV + decode_warps(BWV);
  static constexpr int kScore = kFetch + 2, kValue = kScore + 1, kThreads = 32 * (kValue + 1);
  static constexpr uint32_t kGroup = (uint32_t)D * 16u;                    // eight rows of an operand tile
  static constexpr uint32_t kTileBytes = kTile / 8 * kGroup;
  static constexpr uint32_t kKTile = mma::kLutAddr + (uint32_t)kEntries * 256u;
  // a raw tile: codes as the pages have them, then norms
  static constexpr uint32_t kRawK = kTile * D * BWK / 8 + 2 * kTile, kRawV = kTile * D * BWV / 8 + 2 * kTile;
  static constexpr uint32_t kRaw = kKTile + kStages * kTileBytes;
  static constexpr int kFit = (int)((227u * 1024u - kRaw) / (kRawK + kRawV));
  static constexpr int kRawTiles = kFit < kMostRaw ? kFit : kMostRaw;
  static constexpr uint32_t kDynamic = kRaw + kRawTiles * (kRawK + kRawV);
  static_assert(kRawTiles >= 2 && kDynamic <= 227u * 1024u, "shared memory budget");
  static constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
  static constexpr uint32_t kIdescPV = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
};

// 16 bytes to shared memory, zeros behind the first `bytes` of them (which alone are read).
__device__ __forceinline__ void copy16(uint32_t to, const void *from, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(from), "r"(bytes) : "memory");
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
__device__ __forceinline__ bool warp_wait(uint32_t bar, int use) { return __all_sync(kFull, wait(bar, use)); }

// A place in a ring of N that is walked once: index and completion number without divisions.
template <int N> struct Ring {
  int at = 0, use = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) {
      at = 0;
      ++use;
    }
  }
};

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Codes 2 I, 2 I + 1 of a lane's quarter of a packed row as fp16 centroids.
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

// A bit for each of the 16 fp16 numbers at `from` that is not finite.  Out of line: rarely called.
__device__ __noinline__ uint32_t not_finite(const __half *from) {
  uint32_t bad = 0;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) bad |= (uint32_t)!(fabsf(__half2float(from[i])) < INFINITY) << i;
  return bad;
}
// Whether sixteen fp16 numbers all give zero when multiplied with zero.
__device__ __forceinline__ bool all_finite(const uint4 &a, const uint4 &b) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const __half2 zero = __float2half2_rn(0.f);
  __half2 t = zero;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = __hfma2(*reinterpret_cast<const __half2 *>(&w[i]), zero, t);
  return __hbeq2(t, zero);
}

// One side's fetch warp: page ids of eight tiles ahead, a lane per 16 tokens.  A value norm that is not finite
// is replaced by zero, since the product would carry it (0 x inf) to rows that do not see its token;
// those that do are found when the piece ends (spoiled()).  A look at a lane's norms every eight tiles does
// it here; in the decode warps' loop the same check took 7 % of a long scan.
template <int BW, int D, int RAW_TILES>
__device__ __forceinline__ void fetch_role(const Params &p, int side, const int *prefix, long long begin, long long end,
                                           uint32_t ring) {
  const DecodeSideDev sd = side ? p.v : p.k;
  constexpr int kBytes = 16 * D * BW / 8;                   // codes of 16 tokens
  constexpr uint32_t kRawBytes = 4 * kBytes + 2 * kTile;
  const int lane = threadIdx.x & 31, page_shift = 31 - __clz(p.S);
  Ring<RAW_TILES> raw;
  for (long long x = begin; x < end;) {
    const Piece c = piece_at(p, prefix, x, begin, end);
    x += c.last - c.first;
    const int L = length_of(p, c.b);
    const int32_t *table = p.page_table + (int64_t)c.b * p.table_stride;
    const uint8_t *codes = sd.pages + (int64_t)c.h * sd.head_stride;
    const __half *norms = sd.norms + (int64_t)c.h * sd.norm_head_stride;
    auto page_of = [&](int tile) {                          // of tokens 16 lane .. from that tile on; -2: past the end
      const int tok = tile * kTile + 16 * lane;
      return tok < L && tok < c.last * kTile ? table[tok >> page_shift] : -2;
    };
    int ahead = page_of(c.first);
    uint32_t from_lo = 0, from_hi = 0;                      // where this lane's 16 tokens' codes are
    const __half *norms_from = norms;
    uint32_t norm_bytes = 0, bad = 0;                       // of this lane's 16 tokens: those that exist; norms not finite
    bool good = false;
    uint32_t goods = 0;
    for (int tile = c.first; tile < c.last; ++tile, raw.next()) {
      const int step = (tile - c.first) & 7;
      if (step == 0) {
        const int page = ahead, slot = (tile * kTile + 16 * lane) & (p.S - 1);
        ahead = page_of(tile + 8);
        good = (uint32_t)page < (uint32_t)p.P;
        if (!good && page != -2 && p.status) atomicOr(p.status, WTQ_STATUS_BAD_PAGE);
        const uint64_t from = (uint64_t)(good ? codes + (int64_t)page * sd.page_stride + (int64_t)slot * (kBytes / 16) : codes);
        from_lo = (uint32_t)from;
        from_hi = (uint32_t)(from >> 32);
        norms_from = good ? norms + (int64_t)page * sd.norm_page_stride + slot : norms;
        norm_bytes = good ? 2u * (uint32_t)min(16, L - (tile * kTile + 16 * lane)) : 0u;
        goods = __ballot_sync(kFull, good);
        bad = 0u;
        if (good && side) {
          const uint4 *n = reinterpret_cast<const uint4 *>(norms_from);
          if (!all_finite(__ldg(n), __ldg(n + 1))) bad = not_finite(norms_from) & ((1u << (norm_bytes / 2)) - 1u);
        }
        if (bad != 0u) sts32(kBadNorm, 1u);
      }
      const uint32_t bar = (uint32_t)(side * kMostRaw + raw.at) * 8u, at = ring + (uint32_t)raw.at * kRawBytes;
      if (raw.use > 0 && !warp_wait(kRawFree + bar, raw.use - 1)) return;
      const int owner = 4 * step + (lane >> 3);             // whose 16 tokens this lane copies an eighth of
      const uint64_t lo = __shfl_sync(kFull, from_lo, owner), hi = __shfl_sync(kFull, from_hi, owner);
      const uint32_t there = (goods >> owner & 1u) << 4;    // bytes of a copy
      const uint8_t *from = (const uint8_t *)(lo | hi << 32) + (there ? 16 * (lane & 7) : 0);
      const uint32_t to = at + (uint32_t)(lane >> 3) * kBytes + 16u * (lane & 7);
#pragma unroll
      for (int e = 0; e < kBytes; e += 128) copy16(to + e, from + e, there);
      if (lane >> 2 == step) {                              // the lane that knows the page
        const uint32_t to = at + 4 * kBytes + 32u * (lane & 3);
        if (bad != 0u) {
#pragma unroll 1
          for (uint32_t i = 0; i < 16; i += 2) {
            auto kept = [&](uint32_t k) { return 2 * k < norm_bytes && !(bad >> k & 1u) ? norms_from[k] : __float2half(0.f); };
            const __half2 two = __halves2half2(kept(i), kept(i + 1));
            sts32(to + 2 * i, *reinterpret_cast<const uint32_t *>(&two));
          }
          __threadfence_block();
        } else {
          copy16(to, norms_from, min(norm_bytes, 16u));
          copy16(to + 16, norms_from + (good ? 8 : 0), norm_bytes > 16u ? norm_bytes - 16u : 0u);
        }
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(kRawFull + bar) : "memory");
    }
  }
}

// One decode warp: its eight or sixteen tokens of every tile of a side, lane (g, t) rows g (and g + 8) of
// them, coordinates t * D / 4 on.
template <int BW, int D, int RAW_TILES>
__device__ __forceinline__ void decode_role(int tiles, int side, int u, uint32_t ring, uint32_t tile_base) {
  constexpr int kRowBytes = D * BW / 8, kPairs = D / 8;     // code pairs of a quarter
  constexpr int kGroups = 8 / decode_warps(BW);             // groups of eight tokens
  constexpr uint32_t kRawBytes = kTile * kRowBytes + 2 * kTile, kTileBytes = kTile * D * 2;
  const int lane = threadIdx.x & 31, g = lane & 7, t = lane >> 3;
  const uint32_t sel = mma::kLutAddr | (uint32_t)(lane << 2) | (side ? 0x80u : 0u);
  const uint32_t row = (uint32_t)(8 * kGroups * u + g);
  const uint32_t codes = ring + row * kRowBytes + (uint32_t)t * (kRowBytes / 4), norms = ring + kTile * kRowBytes + 2u * row;
  const uint32_t to = tile_base + (uint32_t)(kGroups * u) * (uint32_t)(D * 16) + (uint32_t)t * (D / 32 * 128) + (uint32_t)g * 16u;
  const uint32_t raw_bar = kRawFull + (uint32_t)(side * kMostRaw) * 8u, tile_bar = kTileFull + (uint32_t)(side * kStages) * 8u;
  constexpr uint32_t kFreeRaw = kRawFree - kRawFull, kFreeTile = kTileFree - kTileFull;
  Ring<RAW_TILES> raw;
  Ring<kStages> buf;
  for (int T = 0; T < tiles; ++T, raw.next(), buf.next()) {
    if (!warp_wait(raw_bar + 8u * raw.at, raw.use)) return;
    // (looked at now, waited for only when the lookups are done)
    const bool is_free = buf.use == 0 || mbar_try(tile_bar + kFreeTile + 8u * buf.at, (uint32_t)(buf.use - 1) & 1u);
    const uint32_t off = (uint32_t)raw.at * kRawBytes;
    uint32_t w[kGroups][kRowBytes / 16];
    __half2 n[kGroups];
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      load_words<kRowBytes / 4>(codes + off + (uint32_t)(8 * h * kRowBytes), w[h]);
      n[h] = __float2half2_rn(lds_half(norms + off + 16u * h));
    }
#pragma unroll
    for (int h = 0; h < kGroups; ++h) {
      uint32_t f[kPairs];
      quarter_codes<BW>(w[h], sel, f, std::make_integer_sequence<int, kPairs>{});
#pragma unroll
      for (int i = 0; i < kPairs; ++i) f[i] = times(f[i], n[h]);
      if (h == 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(raw_bar + kFreeRaw + 8u * raw.at);
        if (!__all_sync(kFull, is_free) && !warp_wait(tile_bar + kFreeTile + 8u * buf.at, buf.use - 1)) return;
      }
      const uint32_t at = to + (uint32_t)buf.at * kTileBytes + (uint32_t)h * (uint32_t)(D * 16);
#pragma unroll
      for (int i = 0; i < kPairs / 4; ++i) sts128(at + 128u * i, f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(tile_bar + 8u * buf.at);
  }
}

// The row's mask words of query row `qr` of a piece's kv head.
__device__ __forceinline__ const int32_t *words_of(const Params &p, const Piece &c, int qr) {
  return p.mask + c.b * p.mask_b + (int64_t)(qr / p.n_rep) * p.mask_t;
}

// Bits of the 64 tokens from `tok0` on that query row `qr` sees.
__device__ __noinline__ uint2 seen_tokens(const Params &p, int b, int qr, int at) {
  const int32_t *words = p.mask + b * p.mask_b + (int64_t)(qr / p.n_rep) * p.mask_t;
  return make_uint2(visible(words, p.Q, at), visible(words, p.Q, at + 32));
}

// fp32 scores of query row `qr` (negative: zeros) with the 64 tokens from `tok0` on, from the packed codes,
// the same addresses for the whole warp, to `own` where they are wanted; those it does not see are -inf.
// Out of line: only for tiles whose scores came out large.
template <int BW, int D>
__device__ __noinline__ void precise_scores(const Params &p, Piece c, int qr, int tok0, bool masked, bool wanted, float *own) {
  constexpr int kRowBytes = D * BW / 8;
  const int end = length_of(p, c.b), i = qr / p.n_rep;
  uint2 seen = make_uint2(kFull, kFull);
  if (masked && qr >= 0) seen = seen_tokens(p, c.b, qr, tok0 - (end - p.Q));
  const float *q = qr < 0 ? nullptr : p.q_rot + (((int64_t)c.b * p.Q + i) * p.Hq + c.h * p.n_rep + qr - i * p.n_rep) * D;
#pragma unroll 1
  for (int blk = 0; blk < kTile / 16; ++blk) {                 // sixteen tokens of one page
    const int tok = tok0 + 16 * blk;
    const int page = tok < end ? p.page_table[(int64_t)c.b * p.table_stride + tok / p.S] : -1;
    float acc[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = 0.f;
    if ((uint32_t)page < (uint32_t)p.P) {
      const uint8_t *row = p.k.pages + (int64_t)c.h * p.k.head_stride + (int64_t)page * p.k.page_stride +
                           (int64_t)(tok % p.S) * kRowBytes;
#pragma unroll 1
      for (int d = 0; d < D / 4; ++d) {                        // four coordinates: BW / 2 bytes of each row
        const float4 x = q ? __ldcg(reinterpret_cast<const float4 *>(q) + d) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          uint32_t w = 0;
#pragma unroll
          for (int e = 0; e < BW / 2; ++e) w |= (uint32_t)__ldg(row + k * kRowBytes + d * (BW / 2) + e) << (8 * e);
          constexpr uint32_t kMask = (1u << BW) - 1u;
          acc[k] = fmaf(x.x, __ldg(p.k.centroids + (w & kMask)), acc[k]);
          acc[k] = fmaf(x.y, __ldg(p.k.centroids + ((w >> BW) & kMask)), acc[k]);
          acc[k] = fmaf(x.z, __ldg(p.k.centroids + ((w >> (2 * BW)) & kMask)), acc[k]);
          acc[k] = fmaf(x.w, __ldg(p.k.centroids + ((w >> (3 * BW)) & kMask)), acc[k]);
        }
      }
      const __half *nrm = p.k.norms + (int64_t)c.h * p.k.norm_head_stride + (int64_t)page * p.k.norm_page_stride + tok % p.S;
#pragma unroll
      for (int k = 0; k < 16; ++k) acc[k] *= tok + k < end ? __half2float(nrm[k]) : 0.f;
    }
    const uint32_t bits = (blk < 2 ? seen.x : seen.y) >> (16 * (blk & 1));
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (wanted) own[16 * blk + k] = (bits >> k & 1u) ? acc[k] : -INFINITY;
  }
}

// Whether query row `qr` (negative: none) sees a token of the piece whose value norm is not finite.
__device__ __noinline__ bool spoiled(const Params &p, Piece c, int qr) {
  const int L = length_of(p, c.b), hist = L - p.Q, lane = threadIdx.x & 31;
  const int32_t *words = p.mask + c.b * p.mask_b + (int64_t)(max(qr, 0) / p.n_rep) * p.mask_t;
  bool found = false;
  for (int tok0 = c.first * kTile; tok0 < min(L, c.last * kTile); tok0 += 32) {
    const int tok = tok0 + lane, page = tok < L ? p.page_table[(int64_t)c.b * p.table_stride + tok / p.S] : -1;
    bool bad = false;
    if ((uint32_t)page < (uint32_t)p.P) {
      const float n = __half2float(p.v.norms[(int64_t)c.h * p.v.norm_head_stride + (int64_t)page * p.v.norm_page_stride +
                                             tok % p.S]);
      bad = !(fabsf(n) < INFINITY);
    }
    const uint32_t all = __ballot_sync(kFull, bad);
    if (all != 0u && qr >= 0) found = found || (visible(words, p.Q, tok0 - hist) & all) != 0u;
  }
  return found;
}

// Scores of unseen tokens become -inf (`seen`: a bit per token).
__device__ __forceinline__ void hide(uint32_t (&s)[64], uint2 seen) {
#pragma unroll
  for (int i = 0; i < 64; ++i) s[i] = ((i < 32 ? seen.x >> i : seen.y >> (i - 32)) & 1u) ? s[i] : 0xff800000u;
}
__device__ __forceinline__ float maximum(const uint32_t (&s)[64]) {
  float a = -INFINITY, b = -INFINITY, c = -INFINITY, d = -INFINITY;
#pragma unroll
  for (int i = 0; i < 64; i += 8) {
    a = max3(a, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    b = max3(b, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
    c = max3(c, __uint_as_float(s[i + 4]), __uint_as_float(s[i + 5]));
    d = max3(d, __uint_as_float(s[i + 6]), __uint_as_float(s[i + 7]));
  }
  return fmaxf(max3(a, b, c), d);
}

template <int BWK, int BWV, int D>
__global__ void __launch_bounds__(Map<BWK, BWV, D>::kThreads, 1) scan_kernel(const __grid_constant__ Params p) {
  using M = Map<BWK, BWV, D>;
  extern __shared__ __align__(128) uint8_t dyn_smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((uint32_t)__cvta_generic_to_shared(dyn_smem) > kBase) {   // layout assumption broken
    if (p.status && tid == 0) atomicOr(p.status, WTQ_STATUS_LAYOUT);
    return;
  }
  int *prefix = reinterpret_cast<int *>(dyn_smem + (kPrefix - (uint32_t)__cvta_generic_to_shared(dyn_smem)));
  for (int e = tid; e < M::kEntries * 64; e += M::kThreads)
    sts32(mma::kLutAddr + 4u * e, mma::lut_word(e, BWK, BWV, p.k.centroids, p.v.centroids));
  if (warp == M::kScore) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(kTmemSlot),
                 "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < 2 * kStages; ++i) {
      mbar_init(kTileFull + 8u * i, decode_warps(i < kStages ? BWK : BWV));
      mbar_init(kTileFree + 8u * i, 1);
    }
#pragma unroll
    for (int i = 0; i < 2 * kMostRaw; ++i) {
      mbar_init(kRawFull + 8u * i, 32);                     // every lane's copies
      mbar_init(kRawFree + 8u * i, decode_warps(i < kMostRaw ? BWK : BWV));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(kSFull + 8u * i, 1);
      mbar_init(kSFree + 8u * i, 4);                        // the four warps of a stream
      mbar_init(kPFull + 8u * i, 4);
      mbar_init(kODone + 8u * i, 1);
    }
    mbar_init(kQFull, kSoftWarps);
    mbar_init(kLast, 2);
    sts32(kAbort, 0u);
    sts32(kBadNorm, 0u);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  fence_before();
  tile_prefix(p, prefix);                                   // (ends with a block barrier)
  fence_after();
  // Only now: the join's blocks take tensor memory too, and one that got it before this block's share was
  // taken would wait for this kernel's end while this block waited for it.
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const uint32_t tmem = lds32(kTmemSlot);
  const long long share = run_length(p, prefix), all = (long long)prefix[p.B] * p.row_blocks * p.Hkv;
  const long long begin = share * blockIdx.x, end = min(all, begin + share);

  // Registers go from the other warps to the softmax warps, which hold 64 scores a thread: of the 640 x 96,
  // 768 x 80 or 896 x 72 that the block was launched with, 256 x 144 and 384 x 64, 512 x 48 or 640 x 40.
  if (warp < kSoftWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;\n");
  else if constexpr (M::kThreads == 640) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n");
  else if constexpr (M::kThreads == 768) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;\n");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n");

  if (warp < kSoftWarps) {
    // ================= softmax: stream `st`, one query row per thread =======================
    const int st = warp >> 2, r = 32 * (warp & 3) + lane;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_addr = tmem + lanes + kColS + 64u * st, p_addr = tmem + lanes + kColP + 32u * st,
                   o_addr = tmem + lanes + kColO + 128u * st;
    int n = 0;                                              // units of this stream so far
    uint32_t states = kStates + 4u * r;                     // of this row, in the present piece's copy
    bool piece_odd = false;
    bool ok = true;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");   // the rotated queries (all else is there already)
    for (long long x = begin; x < end;) {
      const Piece c = piece_at(p, prefix, x, begin, end);
      const int nt = c.last - c.first;
      x += nt;
      const int L = length_of(p, c.b), hist = L - p.Q, qr = c.rb * kRows + r;
      const bool live = qr < p.R && !padding(words_of(p, c, qr), p.Q);
      const bool working = __any_sync(kFull, live);         // a warp without live rows only keeps step
      auto row_of = [&]() -> int64_t {                      // of the (B, Q, Hq) states
        const int i = qr / p.n_rep;
        return ((int64_t)c.b * p.Q + i) * p.Hq + c.h * p.n_rep + qr - i * p.n_rep;
      };
      {
        // this warpgroup's half of the query rows into tensor memory (the products of the last piece are done)
        const float *q = live ? p.q_rot + row_of() * D : nullptr;
        constexpr int kPart = D / 2;
        uint32_t v[kPart / 2];
#pragma unroll
        for (int k = 0; k < kPart / 4; ++k) {
          const float4 y = q ? __ldcg(reinterpret_cast<const float4 *>(q + kPart * st) + k) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[2 * k] = pack_half2(y.x, y.y);
          v[2 * k + 1] = pack_half2(y.z, y.w);
        }
        const uint32_t to = tmem + lanes + kColQ + (uint32_t)(kPart / 2 * st);
        if constexpr (D == 128) tmem_store32(to, v);
        else tmem_store16(to, v);
      }
      tmem_wait_store();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(kQFull);
      float ref = -INFINITY, sum = 0.f;
      const int mine = (nt + 1 - st) / 2;                   // units of this stream in the piece
      for (int k = 0; k < mine && ok; ++k, ++n) {
        const int tok0 = (c.first + 2 * k + st) * kTile;
        if (!(ok = warp_wait(kSFull + 8u * st, n))) break;
        if (!working) {
          if (lane == 0) mbar_arrive(kSFree + 8u * st);
          if (k > 0 && !(ok = warp_wait(kODone + 8u * st, n - 1))) break;
          if (lane == 0) mbar_arrive(kPFull + 8u * st);
          continue;
        }
        fence_after();
        uint32_t s[64];
        tmem_load32<0>(s_addr, s);
        tmem_load32<32>(s_addr + 32, s);
        tmem_wait_load();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(kSFree + 8u * st);       // the scores are in registers
        const bool masked = tok0 + kTile > hist;
        bool sees = live;
        if (masked) {
          uint2 seen = make_uint2(kFull, kFull);
          if (live) seen = seen_tokens(p, c.b, qr, tok0 - hist);
          hide(s, seen);
          sees = live && (seen.x | seen.y) != 0u;
        }
        float mx = maximum(s);
        // (no maximum although something is seen: scores that are not numbers, as of a query beyond fp16)
        const bool large = !(fabsf(mx) <= kPreciseAbove) && (mx != -INFINITY || sees);
        bool drained = k == 0;                              // the stream's last products have ended
        if (__any_sync(kFull, large || mx > ref + kSlack || (ref == -INFINITY && mx != -INFINITY))) {
          if (__any_sync(kFull, large)) {
            float own[64];
#pragma unroll
            for (int e = 0; e < 64; ++e) own[e] = __uint_as_float(s[e]);
            precise_scores<BWK, D>(p, c, live ? qr : -1, tok0, masked, large, own);
#pragma unroll
            for (int e = 0; e < 64; ++e) s[e] = __float_as_uint(own[e]);
            mx = maximum(s);
          }
          const float now = mx > ref + kSlack || ref == -INFINITY ? mx : ref;
          if (k > 0 && __any_sync(kFull, now != ref)) {     // rescale what is accumulated
            if (!(ok = warp_wait(kODone + 8u * st, n - 1))) break;
            fence_after();
            drained = true;
            const float scale = ref == now ? 1.f : ref == -INFINITY ? 0.f : ex2(ref - now);
            sum *= scale;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 16) {
              uint32_t o[16];
              tmem_load16(o_addr + c0, o);
              tmem_wait_load();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * scale);
              tmem_store16(o_addr + c0, o);
            }
            tmem_wait_store();
          }
          ref = now;
        }
        const uint64_t base = twice(ref == -INFINITY ? 0.f : -ref);
        uint32_t pr[32];
        uint64_t sums[2] = {0, 0};                          // (the bits of two zeros)
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float2 y = halves(add2(pair(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), base));
          const float a = ex2(y.x), b = ex2(y.y);
          sums[e & 1] = add2(sums[e & 1], pair(a, b));
          pr[e] = pack_half2(a, b);
        }
        const float2 both = halves(add2(sums[0], sums[1]));
        sum += both.x + both.y;
        if (!drained) {                                     // the last products have read their probabilities
          if (!(ok = warp_wait(kODone + 8u * st, n - 1))) break;
          fence_after();
        }
        tmem_store32(p_addr, pr);
        tmem_wait_store();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(kPFull + 8u * st);
      }
      // ---- the rows' states: the two streams joined, half of the coordinates to each warpgroup ----
      if (ok && mine > 0) ok = warp_wait(kODone + 8u * st, n - 1);
      // (two copies, by turns: a stream without a tile in the next piece waits for nothing in it, and may write its
      // state there while the other still reads this one; the barrier below keeps it from going a piece further)
      sts32(states + 4u * ((2 * st) * kRows), __float_as_uint(ref));
      sts32(states + 4u * ((2 * st + 1) * kRows), __float_as_uint(sum));
      fence_before();
      asm volatile("bar.sync 1, %0;\n" ::"r"(32 * kSoftWarps) : "memory");   // every softmax warp, whatever it gave up on
      fence_after();
      ok = __all_sync(kFull, ok && lds32(kAbort) == 0u);
      if (ok) {
        auto state = [&](int what) { return __uint_as_float(lds32(states + 4u * (what * kRows))); };
        const float m0 = state(0), m1 = state(2);
        float top = fmaxf(m0, m1);
        const float l0 = state(1), l1 = state(3);
        bool broken = l0 != l0 || l1 != l1;                 // a query that is not a number: so is its result
        if (lds32(kBadNorm) != 0u) broken = spoiled(p, c, live ? qr : -1) || broken;
        const float w0 = m0 == -INFINITY ? 0.f : ex2(m0 - top), w1 = m1 == -INFINITY ? 0.f : ex2(m1 - top);
        const float total = broken ? NAN : w0 * l0 + w1 * l1;
        if (broken) top = 0.f;
        float *acc;
        const int64_t row = row_of();
        if (c.slot < 0) {
          acc = p.acc + row * D;
          if (st == 0 && qr < p.R) p.m[row] = live ? top : -INFINITY, p.l[row] = live ? total : 0.f;
        } else {
          const int64_t at = ((int64_t)blockIdx.x * 2 + c.slot) * kRows + r;
          acc = p.part_acc + at * D;
          if (st == 0) p.part_m[at] = live ? top : -INFINITY, p.part_l[at] = live ? total : 0.f;
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
      states += piece_odd ? 0u - 16u * kRows : 16u * kRows;
      piece_odd = !piece_odd;
    }
  } else if (warp < M::kFetch) {
    const int tiles = (int)max(0LL, end - begin);
    // Sides of one width run the same instructions, for the instruction cache's sake: 16 x 8 k 152 -> 145 us
    // (with the fetch warps' shorter loop), 1 x 128 k 397 -> 373 us.
    if constexpr (BWK == BWV) {
      const bool v = warp >= M::kDecodeV;
      decode_role<BWK, D, M::kRawTiles>(tiles, v, warp - (v ? M::kDecodeV : M::kDecodeK),
                                        M::kRaw + (v ? M::kRawTiles * M::kRawK : 0u), v ? kVTile : M::kKTile);
    } else if (warp < M::kDecodeV) decode_role<BWK, D, M::kRawTiles>(tiles, 0, warp - M::kDecodeK, M::kRaw, M::kKTile);
    else decode_role<BWV, D, M::kRawTiles>(tiles, 1, warp - M::kDecodeV, M::kRaw + M::kRawTiles * M::kRawK, kVTile);
  } else if (warp < M::kScore) {
    if constexpr (BWK == BWV) {
      const bool v = warp != M::kFetch;
      fetch_role<BWK, D, M::kRawTiles>(p, v, prefix, begin, end, M::kRaw + (v ? M::kRawTiles * M::kRawK : 0u));
    } else if (warp == M::kFetch) fetch_role<BWK, D, M::kRawTiles>(p, 0, prefix, begin, end, M::kRaw);
    else fetch_role<BWV, D, M::kRawTiles>(p, 1, prefix, begin, end, M::kRaw + M::kRawTiles * M::kRawK);
    asm volatile("cp.async.wait_all;\n" ::: "memory");     // (a block that gave up leaves no copies behind)
  } else {
    // ================= multiply: one lane issues ===========================================
    const uint32_t issuer = elect_one();
    Ring<kStages> buf;
    int pieces = 0, n0 = 0, n1 = 0;                         // units of the streams so far
    bool ok = true;
    for (long long x = begin; x < end && ok; ++pieces) {
      const Piece c = piece_at(p, prefix, x, begin, end);
      const int nt = c.last - c.first;
      x += nt;
      if (warp == M::kScore) {
        ok = warp_wait(kQFull, pieces);
        fence_after();
        for (int j = 0; j < nt && ok; ++j, buf.next()) {    // S of the piece's tile j
          const uint32_t st = j & 1;
          const int n = st ? n1++ : n0++;
          ok = __all_sync(kFull, (n == 0 || wait(kSFree + 8u * st, n - 1)) && wait(kTileFull + 8u * buf.at, buf.use));
          fence_after();
          if (ok && issuer) {
            const uint64_t kb = descriptor(M::kKTile + (uint32_t)buf.at * M::kTileBytes, 128u, M::kGroup);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_ts(tmem + kColS + 64u * st, tmem + kColQ + 8u * ks, kb + 16u * ks, M::kIdescQK, ks > 0);
            umma_commit(kSFull + 8u * st);
            umma_commit(kTileFree + 8u * buf.at);
          }
          __syncwarp();
        }
      } else {
        for (int j = 0; j < nt && ok; ++j, buf.next()) {    // O += P V of tile j
          const uint32_t st = j & 1, at = kStages + buf.at;
          const int n = st ? n1++ : n0++;
          ok = __all_sync(kFull, wait(kTileFull + 8u * at, buf.use) && wait(kPFull + 8u * st, n));
          fence_after();
          if (ok && issuer) {
            const uint64_t vb = descriptor(kVTile + (uint32_t)buf.at * M::kTileBytes, M::kGroup, 128u);
#pragma unroll
            for (int ks = 0; ks < kTile / 16; ++ks)
              umma_ts(tmem + kColO + 128u * st, tmem + kColP + 32u * st + 8u * ks, vb + (uint64_t)(2 * M::kGroup / 16) * ks,
                      M::kIdescPV, j > 1 || ks > 0);
            umma_commit(kODone + 8u * st);
            umma_commit(kTileFree + 8u * at);
          }
          __syncwarp();
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (tid == 0 && lds32(kAbort) != 0u && p.status) atomicOr(p.status, WTQ_STATUS_SCAN_TIMEOUT);
  // A block that gave up may have products in flight: they end before their tensor memory
  // goes to somebody else (bounded, like every wait).  Each of the two warps answers for its own.
  if (warp >= M::kScore) {
    fence_after();
    if (elect_one()) umma_commit(kLast);
    __syncwarp();
  }
  if (warp == M::kScore) {
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
  return launch_behind(scan_kernel<BWK, BWV, D>, p.blocks, M::kThreads, M::kDynamic, stream, "wtq_tree scan launch", p);
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
