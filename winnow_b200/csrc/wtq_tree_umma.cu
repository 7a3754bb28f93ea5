// Tensor-core scan of drafted trees' attention: 16-bit queries, head_dim 64 or 128, packed widths 4, 6
// and 8.  The schedule is in wtq_tree.cuh; a group has 128 query rows, a tile 64 tokens.
//
// The query rows of a group lie in tensor memory as the A operand of all score products, in two fp16 parts.  The
// group's tiles alternate between two streams, each with scores, accumulator, running
// maximum and sum of its own, so that one stream's softmax runs under the other's products; the two
// states are joined when the piece ends.  Twenty-four or twenty-eight warps in roles that meet at mbarriers only:
//
//   fetch     a warp per side: codes and norms of a tile into a ring of raw tiles, 16 bytes a copy;
//   decode    eight warps per side, one for every 8 tokens of a tile (four for 4-bit values without low parts):
//             codes through the per-lane lookup tables to centroid times norm as fp16 high and low parts in the
//             canonical operand layout, as many tiles deep as shared memory has room for (two or three; one of the
//             values for fp16 results at head_dim 128, but for 6 bits);
//   multiply  a warp for S = Qlow Khigh + Qhigh Klow + Qhigh Khigh (N 64) and one for O += P V (A = P from tensor
//             memory, V read with tokens as the contraction), an elected lane of each issues;
//   softmax   a warpgroup per stream, a thread per query row: scores from tensor memory, tree mask, running maximum,
//             probabilities as fp16 over the scores they came from.  O is rescaled only when a row's
//             maximum grows by 2^8.
//
// The roles walk the static schedule by themselves: fetch and decode work into the next piece while
// the softmax warps write the last one's states.  Every wait is bounded; one that runs out raises a
// flag that ends all others, and the status word says so.
//
// Scores are sums of split products, off by 2^-21 of |q| |k|: the class of fp32, whatever their size.  One product of
// operands rounded to fp16 would be off by 3e-4 to 6e-4 nats at logits of one nat (queries) and as much again (centroids
// and their products with norms), which were four fifths of an fp16 result's error and grow with the logits; rescoring
// large scores in fp32 instead took 20 % of the tiles at logits of 3.3 nats and all at 5.5.  Rounded to fp16 are the
// probabilities and, for bf16 results only, the values (centroid, and its product with the norm: 3.4e-4, where the
// result's own rounding is 1.7e-3); fp16 results take the values' low parts too.  Sums, maxima and states are fp32.
// A tile with a score that is no number or infinite (queries beyond fp16) takes its scores in fp32 from the packed codes.
//
// A warp on its own gets through an instruction in about nine cycles here, so a role is only as fast
// as its instructions per tile are few and lie in the instruction cache, which is why sides of one width share theirs.
// Bound by shared memory: loads (lookups, 8 bytes a pair of codes with low parts) and operand stores take half of its
// cycles, and the products, whose pipe is active 46 % of the time, read their operands through the rest.  Queries' low parts
// in tensor memory, with the probabilities over the scores, and raw rows turned against bank conflicts took
// 16 x 8 kv heads x 8192 tokens, 128 rows a group, 4 bits, bf16 from 215 to 171 us with both rotations, and
// 8 x 131 072 tokens, 512 rows a group, fp16 from 820 to 560 us; now 173 (up to 194 where calls follow one another for
// long) and 575 (676), 478 TFLOP/s.  (Single products, without low parts on either side: 145 and 400 us.)
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
constexpr int kRows = kUmmaRows, kTile = kUmmaTile;
constexpr int kMostStages = 3;                  // decoded tiles of a side: as many of these as fit
constexpr int kMostRaw = 5;                     // raw tiles of a side: the same
constexpr uint32_t kFull = 0xffffffffu;
// shared memory; dynamic shared memory is assumed to start at or below kBase
constexpr uint32_t kBase = 1024;
constexpr uint32_t kTileFull = kBase, kTileFree = kTileFull + 16 * kMostStages;             // [side][stage]
constexpr uint32_t kRawFull = kTileFree + 16 * kMostStages, kRawFree = kRawFull + 16 * kMostRaw;   // [side][raw tile]
constexpr uint32_t kSFull = kRawFree + 16 * kMostRaw, kPFull = kSFull + 16, kODone = kPFull + 16;                                   // [stream]
constexpr uint32_t kQFull = kODone + 16, kLast = kQFull + 8, kTmemSlot = kLast + 8, kAbort = kTmemSlot + 4,
                   kBadNorm = kAbort + 4;                                  // a value norm that is not finite was met
constexpr uint32_t kPrefix = kBase + 512;                                  // kMaxBatch + 1 words
constexpr uint32_t kStates = kPrefix + 4 * (kMaxBatch + 4);                // [piece's parity][stream][m, l][row]
constexpr uint32_t kLow = 10240;                                           // tiles from here on
static_assert(kBadNorm + 4 <= kPrefix && kStates + 2 * 4 * kRows * 4 <= kLow, "low region");
// tensor memory columns
constexpr uint32_t kColQ = 0, kColQLow = 64, kColS = 128, kColO = 256, kCols = 512;   // S + 64, O + 128 per stream; P over S
constexpr float kSlack = 8.f;
constexpr int kWaitTries = 1 << 20;

// Where the tiles lie: decoded values, decoded keys, and the two rings of raw tiles, each below the lookup tables or
// behind them; the most stages and then the most raw tiles that fit.
struct Layout {
  int k_stages, v_stages, raws;
  uint32_t at[4], end;                    // values, keys, raw keys, raw values
};
constexpr Layout lay_out(uint32_t behind, uint32_t k_tile, uint32_t v_tile, uint32_t raw_k, uint32_t raw_v) {
  const int stages[4][2] = {{3, 3}, {2, 2}, {2, 1}, {1, 1}};
  for (int i = 0; i < 4; ++i)
    for (int raws = kMostRaw; raws >= 2; --raws)
      for (int where = 0; where < 16; ++where) {
        const uint32_t size[4] = {v_tile * stages[i][1], k_tile * stages[i][0], raw_k * raws, raw_v * raws};
        Layout l = {stages[i][0], stages[i][1], raws, {}, behind};
        uint32_t below = kLow;
        for (int e = 0; e < 4; ++e) {
          uint32_t &from = where >> e & 1 ? l.end : below;
          l.at[e] = from;
          from += size[e];
        }
        if (below <= mma::kLutAddr && l.end <= 227u * 1024u) return l;
      }
  return {};
}

// VLOW: the values' low parts are multiplied too.
template <int BWK, int BWV, int D, bool VLOW> struct Map {
  static constexpr int kEntries = mma::lut_entries(BWK) > mma::lut_entries(BWV) ? mma::lut_entries(BWK)
                                                                                : mma::lut_entries(BWV);
  // groups of eight tokens of a tile that a decode warp takes: one, or two where its work per token is least
  static constexpr int kGroupsV = BWV == 4 && !VLOW ? 2 : 1;
  static constexpr int kDecodeK = kSoftWarps, kDecodeV = kDecodeK + 8, kFetch = kDecodeV + 8 / kGroupsV;
  static constexpr int kScore = kFetch + 2, kValue = kScore + 1, kThreads = 32 * (kValue + 1);
  static constexpr uint32_t kGroup = (uint32_t)D * 16u;                    // eight rows of an operand tile
  static constexpr uint32_t kTileBytes = kTile / 8 * kGroup;               // fp16 parts of one kind
  static constexpr uint32_t kKBytes = 2 * kTileBytes, kVBytes = (VLOW ? 2 : 1) * kTileBytes;   // of a stage: high, then low
  // a raw tile: codes as the pages have them, then norms
  static constexpr uint32_t kRawK = kTile * D * BWK / 8 + 2 * kTile, kRawV = kTile * D * BWV / 8 + 2 * kTile;
  static constexpr Layout kLayout = lay_out(mma::kLutAddr + (uint32_t)kEntries * 256u, kKBytes, kVBytes, kRawK, kRawV);
  static constexpr int kRawTiles = kLayout.raws, kStagesK = kLayout.k_stages, kStagesV = kLayout.v_stages;
  static constexpr uint32_t kVTile = kLayout.at[0], kKTile = kLayout.at[1], kRingK = kLayout.at[2], kRingV = kLayout.at[3],
                            kDynamic = kLayout.end;
  static_assert(kRawTiles >= 2, "shared memory budget");
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

// A place in a ring of `count` that is walked once: index and completion number without divisions.
struct Ring {
  int count, at = 0, use = 0;
  __device__ __forceinline__ explicit Ring(int n) : count(n) {}
  __device__ __forceinline__ void next() {
    if (++at == count) {
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

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2 *>(&x); }
__device__ __forceinline__ uint32_t bits_of(__half2 x) { return *reinterpret_cast<const uint32_t *>(&x); }

// Lookup tables of centroids, in the address layout of wtq_lut.cuh.  4 bits: index = a packed byte; a side with low
// parts has eight bytes for each of sixteen lanes, the fp16 high parts of the two codes and what they leave (a 64-bit load
// serves half a warp at a time, without conflicts), one without has the high parts for each lane.  6 and 8 bits:
// index = a code, high and low part for each lane.
__device__ __forceinline__ uint32_t table_word(int e, int bw_k, int bw_v, const float *ck, const float *cv, bool v_low) {
  const int index = e >> 6, side = (e >> 5) & 1;
  const int bw = side ? bw_v : bw_k;
  const float *cent = side ? cv : ck;
  if (bw == 4) {
    const float a = __ldg(cent + (index & 15)), b = __ldg(cent + (index >> 4));
    const __half2 high = __floats2half2_rn(a, b);
    const float2 back = __half22float2(high);
    return (e & 1) && (!side || v_low) ? pack_half2(a - back.x, b - back.y) : bits_of(high);
  }
  if (index >= 1 << bw) return 0u;
  const float c = __ldg(cent + index);
  return pack_half2(c, c - __half2float(__float2half_rn(c)));
}
// Codes 2 I, 2 I + 1 of a lane's quarter of a packed row: high and, if wanted, low parts of their centroids.
template <int BW, bool LOW, int I, int NW>
__device__ __forceinline__ void two_codes(const uint32_t (&w)[NW], uint32_t sel, uint32_t &high, uint32_t &low) {
  if constexpr (BW == 4) {
    const uint32_t at = lut_addr<I % 4>(w[I / 4], sel);
    if constexpr (LOW) {
      const uint2 v = lds64(at);
      high = v.x;
      low = v.y;
    } else {
      high = lds32(at);
    }
  } else {
    const uint32_t x = lut_code<BW, 2 * I>(w, sel), y = lut_code<BW, 2 * I + 1>(w, sel);
    high = __byte_perm(x, y, 0x5410);
    if constexpr (LOW) low = __byte_perm(x, y, 0x7632);
  }
}
// Pairs FIRST .. of a quarter.
template <int BW, bool LOW, int FIRST, int NW, int... I>
__device__ __forceinline__ void some_codes(const uint32_t (&w)[NW], uint32_t sel, uint32_t *high, uint32_t *low,
                                           std::integer_sequence<int, I...>) {
  (two_codes<BW, LOW, FIRST + I>(w, sel, high[I], low[I]), ...);
}
// Pairs FIRST .. FIRST + 7 times the norm as operand pieces, rounded to fp16, at `at`; LOW: and what that leaves (of the
// centroids' own rounding, too) `low_at` behind them.
template <int BW, bool LOW, int FIRST, int NW>
__device__ __forceinline__ void store_pairs(const uint32_t (&w)[NW], uint32_t sel, __half2 n, uint32_t at, uint32_t low_at) {
  uint32_t h[8], l[8];
  some_codes<BW, LOW, FIRST>(w, sel, h, l, std::make_integer_sequence<int, 8>{});
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2 c = as_half2(h[i]), y = __hmul2(c, n);
    h[i] = bits_of(y);
    if constexpr (LOW) l[i] = bits_of(__hfma2(as_half2(l[i]), n, __hfma2(c, n, __hneg2(y))));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) sts128(at + 128u * (FIRST / 4 + i), h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
  if constexpr (LOW) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      sts128(at + low_at + 128u * (FIRST / 4 + i), l[4 * i], l[4 * i + 1], l[4 * i + 2], l[4 * i + 3]);
  }
}

// Raw rows of 64 or 128 bytes keep their 16-byte pieces in an order that depends on the row, so that eight rows' pieces
// of one number lie in different banks: piece c of row r is in place c ^ turn(r).
template <int ROW_BYTES> __host__ __device__ constexpr int turn(int row) {
  return ROW_BYTES == 64 ? row >> 1 & 3 : ROW_BYTES == 128 ? row & 7 : 0;
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
  constexpr int kRowBytes = D * BW / 8, kBytes = 16 * kRowBytes;   // codes of a token, of 16
  constexpr uint32_t kRawBytes = 4 * kBytes + 2 * kTile;
  const int lane = threadIdx.x & 31, page_shift = 31 - __clz(p.S);
  Ring raw(RAW_TILES);
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
      for (int e = 0; e < kBytes; e += 128) {
        // (row e / kRowBytes of the sixteen and, of shorter rows, those that follow it in 128 bytes: they turn alike)
        copy16((to ^ (uint32_t)(turn<kRowBytes>(e / kRowBytes) << 4)) + e, from + e, there);
      }
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

// One decode warp: its `groups` times eight tokens of every tile of a side, lane (g, t) row g of a group, coordinates
// t * D / 4 on.
template <int BW, int D, int RAW_TILES>
__device__ __forceinline__ void decode_role(int tiles, int side, int u, int groups, uint32_t ring, uint32_t tile_base, int stages,
                                            bool low) {
  constexpr int kRowBytes = D * BW / 8, kPairs = D / 8;     // code pairs of a quarter
  constexpr uint32_t kRawBytes = kTile * kRowBytes + 2 * kTile, kTileBytes = kTile * D * 2;
  const uint32_t stage_bytes = low ? 2 * kTileBytes : kTileBytes;
  const int lane = threadIdx.x & 31, g = lane & 7, t = lane >> 3;
  const uint32_t sel = mma::kLutAddr | (uint32_t)(BW == 4 && low ? (lane & 15) << 3 : lane << 2) | (side ? 0x80u : 0u);
  const uint32_t row = (uint32_t)(8 * groups * u + g);
  const uint32_t codes = ring + row * kRowBytes + (uint32_t)((t * (kRowBytes / 4)) ^ (turn<kRowBytes>(g) << 4)), norms = ring + kTile * kRowBytes + 2u * row;
  const uint32_t to = tile_base + (uint32_t)(groups * u) * (uint32_t)(D * 16) + (uint32_t)t * (D / 32 * 128) + (uint32_t)g * 16u;
  const uint32_t raw_bar = kRawFull + (uint32_t)(side * kMostRaw) * 8u, tile_bar = kTileFull + (uint32_t)(side * kMostStages) * 8u;
  constexpr uint32_t kFreeRaw = kRawFree - kRawFull, kFreeTile = kTileFree - kTileFull;
  Ring raw(RAW_TILES), buf(stages);
  for (int T = 0; T < tiles; ++T, raw.next(), buf.next()) {
    if (!warp_wait(raw_bar + 8u * raw.at, raw.use)) return;
    // (looked at now, waited for only when the first words are there)
    const bool is_free = buf.use == 0 || mbar_try(tile_bar + kFreeTile + 8u * buf.at, (uint32_t)(buf.use - 1) & 1u);
    uint32_t from = (uint32_t)raw.at * kRawBytes, at = to + (uint32_t)buf.at * stage_bytes;
#pragma unroll 1
    for (int h = 0; h < groups; ++h, from += 8 * kRowBytes, at += (uint32_t)(D * 16)) {
      uint32_t w[kRowBytes / 16];
      if constexpr (kRowBytes == 128) {                     // (pieces 2 t and 2 t + 1, which turn to a pair of places)
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          const uint4 v = lds128((codes + from) ^ (16u * i));
          w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
      } else {
        load_words<kRowBytes / 4>(codes + from, w);
      }
      const __half2 n = __float2half2_rn(lds_half(norms + (uint32_t)raw.at * kRawBytes + 16u * h));
      if (h == 0 && !__all_sync(kFull, is_free) && !warp_wait(tile_bar + kFreeTile + 8u * buf.at, buf.use - 1)) return;
      if (low) {
        store_pairs<BW, true, 0>(w, sel, n, at, kTileBytes);
        if constexpr (kPairs > 8) store_pairs<BW, true, 8>(w, sel, n, at, kTileBytes);
      } else {
        store_pairs<BW, false, 0>(w, sel, n, at, kTileBytes);
        if constexpr (kPairs > 8) store_pairs<BW, false, 8>(w, sel, n, at, kTileBytes);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(raw_bar + kFreeRaw + 8u * raw.at);
      mbar_arrive(tile_bar + 8u * buf.at);
    }
  }
}

// The row's mask words of query row `qr` of a piece's kv head.
__device__ __forceinline__ const int32_t *words_of(const Params &p, const Piece &c, int qr) {
  return p.mask + c.b * p.mask_b + (int64_t)(qr / p.n_rep) * p.mask_t;
}

// Bits of the 64 tokens from `tok0` on that query row `qr` sees.
__device__ __noinline__ uint2 seen_tokens(const Params &p, int b, int qr, int at) {
  const int32_t *words = p.mask + b * p.mask_b + (int64_t)(qr / p.n_rep) * p.mask_t;
  const int places = places_of(p, b);
  return make_uint2(visible(words, places, at), visible(words, places, at + 32));
}

// fp32 scores of query row `qr` (negative: zeros) with the 64 tokens from `tok0` on, from the packed codes,
// the same addresses for the whole warp, to `own` where they are wanted; those it does not see are -inf.
// Out of line: only for tiles whose scores came out large.
template <int BW, int D>
__device__ __noinline__ void precise_scores(const Params &p, Piece c, int qr, int tok0, bool masked, bool wanted, float *own) {
  constexpr int kRowBytes = D * BW / 8;
  const int end = length_of(p, c.b), i = qr / p.n_rep;
  uint2 seen = make_uint2(kFull, kFull);
  if (masked && qr >= 0) seen = seen_tokens(p, c.b, qr, tok0 - history_of(p, c.b));
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
  const int L = length_of(p, c.b), hist = history_of(p, c.b), places = places_of(p, c.b), lane = threadIdx.x & 31;
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
    if (all != 0u && qr >= 0) found = found || (visible(words, places, tok0 - hist) & all) != 0u;
  }
  return found;
}

// Scores of unseen tokens become -inf (`seen`: a bit per token).
__device__ __forceinline__ void hide(uint32_t (&s)[64], uint2 seen) {
#pragma unroll
  for (int i = 0; i < 64; ++i) s[i] = ((i < 32 ? seen.x >> i : seen.y >> (i - 32)) & 1u) ? s[i] : 0xff800000u;
}
template <bool NANS> __device__ __forceinline__ float most_of(float a, float b, float c) {
  float d;
  if constexpr (NANS) asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  else d = max3(a, b, c);
  return d;
}
// NANS: not a number if a score is none.
template <bool NANS> __device__ __forceinline__ float maximum(const uint32_t (&s)[64]) {
  float a = -INFINITY, b = -INFINITY, c = -INFINITY, d = -INFINITY;
#pragma unroll
  for (int i = 0; i < 64; i += 8) {
    a = most_of<NANS>(a, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    b = most_of<NANS>(b, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
    c = most_of<NANS>(c, __uint_as_float(s[i + 4]), __uint_as_float(s[i + 5]));
    d = most_of<NANS>(d, __uint_as_float(s[i + 6]), __uint_as_float(s[i + 7]));
  }
  return most_of<NANS>(most_of<NANS>(a, b, c), d, d);
}

template <int BWK, int BWV, int D, bool VLOW>
__global__ void __launch_bounds__(Map<BWK, BWV, D, VLOW>::kThreads, 1) scan_kernel(const __grid_constant__ Params p) {
  using M = Map<BWK, BWV, D, VLOW>;
  extern __shared__ __align__(128) uint8_t dyn_smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((uint32_t)__cvta_generic_to_shared(dyn_smem) > kBase) {   // layout assumption broken
    if (p.status && tid == 0) atomicOr(p.status, WTQ_STATUS_LAYOUT);
    return;
  }
  int *prefix = reinterpret_cast<int *>(dyn_smem + (kPrefix - (uint32_t)__cvta_generic_to_shared(dyn_smem)));
  for (int e = tid; e < M::kEntries * 64; e += M::kThreads)
    sts32(mma::kLutAddr + 4u * e, table_word(e, BWK, BWV, p.k.centroids, p.v.centroids, VLOW));
  if (warp == M::kScore) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(kTmemSlot),
                 "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < 2 * kMostStages; ++i) {
      mbar_init(kTileFull + 8u * i, i < kMostStages ? 8 : 8 / M::kGroupsV);
      mbar_init(kTileFree + 8u * i, 1);
    }
#pragma unroll
    for (int i = 0; i < 2 * kMostRaw; ++i) {
      mbar_init(kRawFull + 8u * i, 32);                     // every lane's copies
      mbar_init(kRawFree + 8u * i, i < kMostRaw ? 8 : 8 / M::kGroupsV);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(kSFull + 8u * i, 1);
      mbar_init(kPFull + 8u * i, 4);                        // the four warps of a stream
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

  // Registers go from the other warps to the softmax warps, which hold 64 scores a thread: of the 768 x 80 or
  // 896 x 72 that the block was launched with, 256 x 144 and 512 x 48 or 640 x 40.
  if (warp < kSoftWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 144;\n");
  else if constexpr (M::kThreads == 768) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;\n");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;\n");

  if (warp < kSoftWarps) {
    // ================= softmax: stream `st`, one query row per thread =======================
    const int st = warp >> 2, r = 32 * (warp & 3) + lane;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_addr = tmem + lanes + kColS + 64u * st, o_addr = tmem + lanes + kColO + 128u * st;
    int n = 0;                                              // units of this stream so far
    uint32_t states = kStates + 4u * r;                     // of this row, in the present piece's copy
    bool piece_odd = false;
    bool ok = true;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");   // the rotated queries (all else is there already)
    for (long long x = begin; x < end;) {
      const Piece c = piece_at(p, prefix, x, begin, end);
      const int nt = c.last - c.first;
      x += nt;
      const int hist = history_of(p, c.b), all_see = min(hist, p.max_tokens), qr = c.rb * kRows + r;
      const bool live = qr < p.R && !padding(words_of(p, c, qr), p.Q);
      const bool working = __any_sync(kFull, live);         // a warp without live rows only keeps step
      auto row_of = [&]() -> int64_t {                      // of the (B, Q, Hq) states
        const int i = qr / p.n_rep;
        return ((int64_t)c.b * p.Q + i) * p.Hq + c.h * p.n_rep + qr - i * p.n_rep;
      };
      {
        // this warpgroup's half of the query rows as high and low parts (the products of the last piece are done)
        const float *q = live ? p.q_rot + row_of() * D : nullptr;
        constexpr int kPart = D / 2;
        uint32_t v[kPart / 2], l[kPart / 2];
#pragma unroll
        for (int k = 0; k < kPart / 4; ++k) {
          const float4 y = q ? __ldcg(reinterpret_cast<const float4 *>(q + kPart * st) + k) : make_float4(0.f, 0.f, 0.f, 0.f);
          const __half2 a = __floats2half2_rn(y.x, y.y), b = __floats2half2_rn(y.z, y.w);
          const float2 af = __half22float2(a), bf = __half22float2(b);
          v[2 * k] = bits_of(a);
          v[2 * k + 1] = bits_of(b);
          l[2 * k] = pack_half2(y.x - af.x, y.y - af.y);
          l[2 * k + 1] = pack_half2(y.z - bf.x, y.w - bf.y);
        }
        const uint32_t to = tmem + lanes + (uint32_t)(kPart / 2 * st);
        __syncwarp();                                       // (rows with and without queries: all issue what follows together)
        if constexpr (D == 128) {
          tmem_store32(to + kColQ, v);
          tmem_store32(to + kColQLow, l);
        } else {
          tmem_store16(to + kColQ, v);
          tmem_store16(to + kColQLow, l);
        }
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
          if (lane == 0) mbar_arrive(kPFull + 8u * st);
          continue;
        }
        fence_after();
        uint32_t s[64];
        tmem_load32<0>(s_addr, s);
        tmem_load32<32>(s_addr + 32, s);
        tmem_wait_load();
        const bool masked = tok0 + kTile > all_see;
        bool sees = live;
        if (masked) {
          uint2 seen = make_uint2(kFull, kFull);
          if (live) seen = seen_tokens(p, c.b, qr, tok0 - hist);
          hide(s, seen);
          sees = live && (seen.x | seen.y) != 0u;
        }
        float mx = maximum<true>(s);
        // (not a number although something is seen: a query or a key beyond fp16, or one that is no number itself)
        const bool large = !(fabsf(mx) < INFINITY) && (mx != -INFINITY || sees);
        if (__any_sync(kFull, large || mx > ref + kSlack || (ref == -INFINITY && mx != -INFINITY))) {
          if (__any_sync(kFull, large)) {
            float own[64];
#pragma unroll
            for (int e = 0; e < 64; ++e) own[e] = __uint_as_float(s[e]);
            precise_scores<BWK, D>(p, c, live ? qr : -1, tok0, masked, large, own);
#pragma unroll
            for (int e = 0; e < 64; ++e) s[e] = __float_as_uint(own[e]);
            mx = maximum<false>(s);
          }
          const float now = mx > ref + kSlack || ref == -INFINITY ? mx : ref;
          if (k > 0 && __any_sync(kFull, now != ref)) {     // rescale what is accumulated (its products have ended)
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
          pr[e] = pack_half2(ex2(y.x), ex2(y.y));
          // The sum takes the probabilities as the product has them: where a few tokens carry the row, their
          // rounding then cancels in the quotient.
          const float2 rounded = __half22float2(as_half2(pr[e]));
          sums[e & 1] = add2(sums[e & 1], pair(rounded.x, rounded.y));
        }
        const float2 both = halves(add2(sums[0], sums[1]));
        sum += both.x + both.y;
        __syncwarp();
        tmem_store32(s_addr, pr);                           // over the scores just read
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
          __syncwarp();                                     // (rows that store nothing are back from the last columns)
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
    // Sides of one width run the same instructions, for the instruction cache's sake.
    const bool v = warp >= M::kDecodeV;
    if constexpr (BWK == BWV) {
      decode_role<BWK, D, M::kRawTiles>(tiles, v, warp - (v ? M::kDecodeV : M::kDecodeK), v ? M::kGroupsV : 1,
                                        v ? M::kRingV : M::kRingK, v ? M::kVTile : M::kKTile, v ? M::kStagesV : M::kStagesK,
                                        !v || VLOW);
    } else if (!v) decode_role<BWK, D, M::kRawTiles>(tiles, 0, warp - M::kDecodeK, 1, M::kRingK, M::kKTile, M::kStagesK, true);
    else decode_role<BWV, D, M::kRawTiles>(tiles, 1, warp - M::kDecodeV, M::kGroupsV, M::kRingV, M::kVTile, M::kStagesV, VLOW);
  } else if (warp < M::kScore) {
    if constexpr (BWK == BWV) {
      const bool v = warp != M::kFetch;
      fetch_role<BWK, D, M::kRawTiles>(p, v, prefix, begin, end, v ? M::kRingV : M::kRingK);
    } else if (warp == M::kFetch) fetch_role<BWK, D, M::kRawTiles>(p, 0, prefix, begin, end, M::kRingK);
    else fetch_role<BWV, D, M::kRawTiles>(p, 1, prefix, begin, end, M::kRingV);
    asm volatile("cp.async.wait_all;\n" ::: "memory");     // (a block that gave up leaves no copies behind)
  } else {
    // ================= multiply: one lane issues ===========================================
    const uint32_t issuer = elect_one();
    Ring buf(warp == M::kScore ? M::kStagesK : M::kStagesV);
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
          // (the stream's last products have read their probabilities, and its accumulator is at rest)
          ok = __all_sync(kFull, (n == 0 || wait(kODone + 8u * st, n - 1)) && wait(kTileFull + 8u * buf.at, buf.use));
          fence_after();
          if (ok && issuer) {
            // S = Qlow Khigh + Qhigh Klow + Qhigh Khigh, the small ones first
            const uint64_t kb = descriptor(M::kKTile + (uint32_t)buf.at * M::kKBytes, 128u, M::kGroup);
            const uint64_t kl = descriptor(M::kKTile + (uint32_t)buf.at * M::kKBytes + M::kTileBytes, 128u, M::kGroup);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_ts(tmem + kColS + 64u * st, tmem + kColQLow + 8u * ks, kb + 16u * ks, M::kIdescQK, ks > 0);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_ts(tmem + kColS + 64u * st, tmem + kColQ + 8u * ks, kl + 16u * ks, M::kIdescQK, 1u);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_ts(tmem + kColS + 64u * st, tmem + kColQ + 8u * ks, kb + 16u * ks, M::kIdescQK, 1u);
            umma_commit(kSFull + 8u * st);
            umma_commit(kTileFree + 8u * buf.at);
          }
          __syncwarp();
        }
      } else {
        for (int j = 0; j < nt && ok; ++j, buf.next()) {    // O += P V of tile j
          const uint32_t st = j & 1, at = kMostStages + buf.at;
          const int n = st ? n1++ : n0++;
          ok = __all_sync(kFull, wait(kTileFull + 8u * at, buf.use) && wait(kPFull + 8u * st, n));
          fence_after();
          if (ok && issuer) {
#pragma unroll
            for (int part = VLOW ? 1 : 0; part >= 0; --part) {        // low parts first
              const uint64_t vb = descriptor(M::kVTile + (uint32_t)buf.at * M::kVBytes + (uint32_t)part * M::kTileBytes, M::kGroup, 128u);
#pragma unroll
              for (int ks = 0; ks < kTile / 16; ++ks)
                umma_ts(tmem + kColO + 128u * st, tmem + kColS + 64u * st + 8u * ks, vb + (uint64_t)(2 * M::kGroup / 16) * ks,
                        M::kIdescPV, j > 1 || ks > 0 || (VLOW && part == 0));
            }
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

template <int BWK, int BWV, int D, bool VLOW> int launch(const Params &p, cudaStream_t stream) {
  using M = Map<BWK, BWV, D, VLOW>;
  static std::atomic<bool> opted_in[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !opted_in[dev & 63].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(scan_kernel<BWK, BWV, D, VLOW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)M::kDynamic);
    if (e != cudaSuccess) return check_cuda(e, "wtq_tree: shared memory opt-in");
    opted_in[dev & 63].store(true, std::memory_order_release);
  }
  return launch_behind(scan_kernel<BWK, BWV, D, VLOW>, p.blocks, M::kThreads, M::kDynamic, stream, "wtq_tree scan launch", p);
}
template <int D, bool VLOW> int launch_widths(const Params &p, cudaStream_t stream) {
  if (p.k.bw == 4 && p.v.bw == 4) return launch<4, 4, D, VLOW>(p, stream);
  if (p.k.bw == 4 && p.v.bw == 6) return launch<4, 6, D, VLOW>(p, stream);
  if (p.k.bw == 6 && p.v.bw == 6) return launch<6, 6, D, VLOW>(p, stream);
  return launch<8, 8, D, VLOW>(p, stream);
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
  // (a value's one rounding to fp16, 1.4e-4 of it in the mean, is a twelfth of what rounding to bf16 does to the result,
  // but would be the larger part of an fp16 result's error)
  if (p.dtype == WTQ_F16)
    return p.D == 128 ? um::launch_widths<128, true>(p, stream) : um::launch_widths<64, true>(p, stream);
  return p.D == 128 ? um::launch_widths<128, false>(p, stream) : um::launch_widths<64, false>(p, stream);
}

}  // namespace tree
}  // namespace wtq
