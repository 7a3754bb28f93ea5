// Block tables and slot maps of a step, built on the device from request lengths: how many pages
// every request needs more, which ones (off a stack of free pages, in batch order), and for every
// new token its sequence, position and slot.  With drafted trees also each token's depth and the
// words of its ancestors' mask.  The step is granted as a whole or not at all.
//
// Every block computes the two prefix sums over the batch (new tokens, new pages) for itself,
// which is cheaper than a second launch, and then takes its share of the tokens and of the new
// table entries.  The slot of a token on a new page is computed from the stack, not read back
// from the table, so no block waits for another's entries.  State that is advanced in place
// (lengths, held, free count) is written by the block that finishes last, when no other reads
// it any more; with separate outputs the first block writes it.  Bound by the launch and two
// dependent reads: a call takes 8 us, trees of 32 tokens for 32 sequences and 20 000 ragged tokens alike.
#include <algorithm>

#include "wtq_common.cuh"

namespace wtq {
namespace plan {

constexpr int kThreads = 256;
constexpr int kMaxBatch = 4096;                 // two prefixes of it in shared memory
constexpr int kMost = 1 << 30;                  // tokens and pages: a grid's stride past them is still an int

struct Params {
  const int32_t *lengths, *new_tokens, *parents;
  int64_t parent_stride;
  int32_t *table;
  int64_t table_stride;
  const int32_t *held;
  const int32_t *free_pages, *free_count;
  int B, W, S, tokens, drafted, stack;
  int32_t *seq_lens, *held_out, *free_out, *starts, *sequence, *positions, *slot_pages, *slot_ends, *mask;
  int32_t *ticket, *status;
};

// Sequence whose range of an exclusive prefix (B + 1 entries) holds x.
__device__ __forceinline__ int find(const int *prefix, int B, int x) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (prefix[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Bits of an exclusive prefix over the block's threads; returns the block's total.
__device__ __forceinline__ long long block_prefix(long long v, long long &before, long long *parts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) parts[warp] = incl;
  __syncthreads();
  long long base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) base += parts[w];
    total += parts[w];
  }
  __syncthreads();
  before = base + incl - v;
  return total;
}

__global__ void __launch_bounds__(kThreads) plan_kernel(Params p) {
  extern __shared__ int smem[];
  int *starts = smem, *pages = smem + p.B + 1;             // exclusive prefixes
  __shared__ long long parts[kThreads / 32];
  __shared__ int is_last;
  const int tid = threadIdx.x;
  const int per = (p.B + kThreads - 1) / kThreads;         // sequences of this thread: tid * per ..
  const int b_lo = min(p.B, tid * per), b_hi = min(p.B, b_lo + per);
  const bool tree = p.parents != nullptr;
  bool malformed = false, narrow = false;
  long long sum_new = 0, sum_pages = 0;
  auto demand = [&](int b, int &n, int &grow) {
    const int len = p.lengths[b], have = p.held[b];
    n = tree ? p.drafted : p.new_tokens[b];
    grow = 0;
    if (len < 0 || n < 0 || have < 0 || have > p.W) {
      malformed = true;
      n = 0;
      return;
    }
    if ((long long)len + n > INT32_MAX) {                    // a position beyond 32 bits
      malformed = true;
      n = 0;
      return;
    }
    const long long need = ((long long)len + n + p.S - 1) / p.S;
    if (need > p.W) narrow = true;
    else grow = max(0, (int)need - have);
  };
  for (int b = b_lo; b < b_hi; ++b) {
    int n, grow;
    demand(b, n, grow);
    sum_new += n;
    sum_pages += grow;
  }
  long long before_new, before_pages;
  const long long all_new = block_prefix(sum_new, before_new, parts);
  const long long all_pages = block_prefix(sum_pages, before_pages, parts);
  const int count = *p.free_count;
  const bool bad = __syncthreads_or(malformed) || all_new > p.tokens || count < 0 || count > p.stack;
  const bool short_of = __syncthreads_or(narrow) || all_pages > count;
  const bool granted = !bad && !short_of;
  for (int b = b_lo; b < b_hi; ++b) {
    int n, grow;
    demand(b, n, grow);
    starts[b] = granted ? (int)before_new : 0;
    pages[b] = granted ? (int)before_pages : 0;
    before_new += n;
    before_pages += grow;
  }
  if (tid == 0) {
    starts[p.B] = granted ? (int)all_new : 0;
    pages[p.B] = granted ? (int)all_pages : 0;
    if (!granted && p.status && blockIdx.x == 0)
      atomicOr(p.status, bad ? WTQ_STATUS_BAD_POSITION : WTQ_STATUS_NO_PAGES);
  }
  __syncthreads();
  const int total = starts[p.B], fresh = pages[p.B];
  const int stride = gridDim.x * kThreads, me = blockIdx.x * kThreads + tid;
  // new entries of the table
  for (int x = me; x < fresh; x += stride) {
    const int b = find(pages, p.B, x);
    p.table[(int64_t)b * p.table_stride + p.held[b] + x - pages[b]] = p.free_pages[count - 1 - x];
  }
  // tokens
  const int words = tree ? (p.drafted + 31) / 32 : 0;
  for (int t = me; t < p.tokens; t += stride) {
    int seq = -1, pos = -1, page = -1, end = 0;
    if (t < total) {
      seq = tree ? t / p.drafted : find(starts, p.B, t);
      const int i = t - starts[seq], at = p.lengths[seq] + i;
      const int column = at / p.S, have = p.held[seq];
      page = column < have ? p.table[(int64_t)seq * p.table_stride + column]
                           : p.free_pages[count - 1 - (pages[seq] + column - have)];
      end = at - column * p.S + 1;
      pos = at;
    }
    if (tree) {
      // Ancestors by walking up: a parent stands before its child, so the words fill from the
      // own one downwards.  -1: below the history's last token; -2, or below such a token: padding.
      const int b = t / p.drafted, i = t - b * p.drafted;
      const int32_t *parent = p.parents + (int64_t)b * p.parent_stride;
      int32_t *out = p.mask + (int64_t)t * words;
      int depth = -1, j = i, word = words - 1;
      uint32_t bits = 0;
      while (j >= 0) {
        for (; word > j >> 5; --word) {
          out[word] = (int32_t)bits;
          bits = 0;
        }
        bits |= 1u << (j & 31);
        ++depth;
        const int up = parent[j];
        if (up >= j || up < -2) {
          if (p.status) atomicOr(p.status, WTQ_STATUS_BAD_PARENT);
          j = -2;
        } else {
          j = up;
        }
      }
      const bool padding = j == -2 || t >= total;
      for (int w = words - 1; w >= 0; --w) {
        if (padding) out[w] = 0;
        else if (w <= word) out[w] = w == word ? (int32_t)bits : 0;
      }
      pos = padding ? -1 : p.lengths[b] + depth;
    }
    p.sequence[t] = seq;
    p.positions[t] = pos;
    p.slot_pages[t] = page;
    p.slot_ends[t] = end;
  }
  // the advanced state
  if (p.ticket != nullptr) {
    __threadfence();
    __syncthreads();
    if (tid == 0) is_last = atomicAdd(p.ticket, 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!is_last) return;
  } else if (blockIdx.x != 0) {
    return;
  }
  for (int b = b_lo; b < b_hi; ++b) {
    const int len = p.lengths[b], have = p.held[b];
    p.starts[b] = starts[b];
    p.seq_lens[b] = len + starts[b + 1] - starts[b];
    p.held_out[b] = have + pages[b + 1] - pages[b];
  }
  if (tid == 0) {
    p.starts[p.B] = total;
    *p.free_out = count - fresh;
    if (p.ticket != nullptr) *p.ticket = 0;
  }
}

// The pages of the marked sequences go back onto the stack, in batch order, the last page of a
// sequence first; their rows read -1 and their lengths 0.  One block.
__global__ void __launch_bounds__(kThreads) release_kernel(const int32_t *marks, int32_t *table, int64_t table_stride,
                                                           int32_t *lengths, int32_t *held, int32_t *free_pages,
                                                           int32_t *free_count, int B, int W, int stack,
                                                           int32_t *status) {
  extern __shared__ int smem[];
  int *pages = smem;
  __shared__ long long parts[kThreads / 32];
  const int tid = threadIdx.x, per = (B + kThreads - 1) / kThreads;
  const int b_lo = min(B, tid * per), b_hi = min(B, b_lo + per);
  long long sum = 0, before;
  bool malformed = false;
  for (int b = b_lo; b < b_hi; ++b) {
    const int have = marks[b] ? held[b] : 0;
    if (have < 0 || have > W) malformed = true;
    else sum += have;
  }
  const long long total = block_prefix(sum, before, parts);
  const int count = *free_count;
  if (__syncthreads_or(malformed) || count < 0 || count + total > stack) {   // more than the pool has: refused
    if (tid == 0 && status) atomicOr(status, WTQ_STATUS_BAD_POSITION);
    return;
  }
  for (int b = b_lo; b < b_hi; ++b) {
    pages[b] = (int)before;
    if (marks[b]) before += held[b];
  }
  if (tid == 0) pages[B] = (int)total;
  __syncthreads();
  for (int x = tid; x < total; x += kThreads) {
    // (an unmarked sequence has an empty range: the search passes over it)
    const int b = find(pages, B, x);
    const int64_t at = (int64_t)b * table_stride + held[b] - 1 - (x - pages[b]);
    free_pages[count + x] = table[at];
    table[at] = -1;
  }
  __syncthreads();
  for (int b = b_lo; b < b_hi; ++b)
    if (marks[b]) lengths[b] = held[b] = 0;
  if (tid == 0) *free_count = count + (int)total;
}

}  // namespace plan
}  // namespace wtq

using namespace wtq;

extern "C" int wtq_plan_tokens(const int32_t *lengths, const int32_t *new_tokens, const int32_t *parents,
                               int64_t parent_stride, int32_t *table, int64_t table_stride, const int32_t *held,
                               const int32_t *free_pages, const int32_t *free_count, int B, int max_pages, int S,
                               int tokens, int drafted, int stack, const wtq_plan_t *out, int32_t *ticket,
                               int32_t *status, void *stream_) {
  if (B < 0 || B > plan::kMaxBatch || max_pages < 1 || S < 1 || tokens < 0 || drafted < 0 || stack < 0)
    return fail(WTQ_ERR_ARG, "wtq_plan_tokens: need 0 <= B <= %d and sizes that are not negative", plan::kMaxBatch);
  if (tokens > plan::kMost || stack > plan::kMost)
    return fail(WTQ_ERR_ARG, "wtq_plan_tokens: tokens and free pages are limited to 2^30");
  if (!out) return fail(WTQ_ERR_ARG, "wtq_plan_tokens: null outputs");
  if (parents ? drafted < 1 || (int64_t)B * drafted != tokens : drafted != 0)
    return fail(WTQ_ERR_ARG, "wtq_plan_tokens: with parents there are B * drafted tokens, without none is drafted");
  if (!free_count || !out->free_count || !out->starts) return fail(WTQ_ERR_ARG, "wtq_plan_tokens: null counters");
  if (B > 0 && (!lengths || (!new_tokens && !parents) || !table || !held || !out->seq_lens || !out->held))
    return fail(WTQ_ERR_ARG, "wtq_plan_tokens: null input or output");
  if (stack > 0 && !free_pages) return fail(WTQ_ERR_ARG, "wtq_plan_tokens: null free pages");
  if (tokens > 0 && (!out->sequence || !out->positions || !out->slot_pages || !out->slot_ends || (parents && !out->mask)))
    return fail(WTQ_ERR_ARG, "wtq_plan_tokens: null token output");
  const bool in_place = out->seq_lens == lengths || out->held == held || out->free_count == free_count;
  if (in_place && !ticket) return fail(WTQ_ERR_ARG, "wtq_plan_tokens: state advanced in place needs a ticket word");
  // Every block reads the inputs for itself while others write their results already: these lie apart from them and from
  // one another, but for state that is advanced in place.
  const int64_t n = tokens, words = parents ? (drafted + 31) / 32 : 0;
  const Span read[6] = {{lengths, B * 4LL}, {held, B * 4LL}, {free_count, 4}, {parents ? nullptr : new_tokens, B * 4LL},
                        {parents, parents ? ((B - 1) * parent_stride + drafted) * 4 : 0}, {free_pages, stack * 4LL}};
  const Span written[11] = {{out->seq_lens, B * 4LL}, {out->held, B * 4LL}, {out->free_count, 4}, {out->starts, (B + 1) * 4LL},
                            {out->sequence, n * 4}, {out->positions, n * 4}, {out->slot_pages, n * 4}, {out->slot_ends, n * 4},
                            {parents ? out->mask : nullptr, n * words * 4}, {in_place ? ticket : nullptr, 4},
                            {table, ((B - 1) * table_stride + max_pages) * 4}};
  for (int i = 0; i < 11; ++i) {
    for (int j = 0; j < 6; ++j)
      if (!(i == j && i < 3 && written[i].at == read[j].at) && meet(written[i], read[j]))
        return fail(WTQ_ERR_ARG, "wtq_plan_tokens: results must not share memory with inputs, but for their own state");
    for (int j = 0; j < i; ++j)
      if (meet(written[i], written[j])) return fail(WTQ_ERR_ARG, "wtq_plan_tokens: results must not share memory");
  }
  plan::Params p = {lengths, new_tokens, parents, parent_stride, table, table_stride, held, free_pages, free_count,
                    B, max_pages, S, tokens, drafted, stack, out->seq_lens, out->held, out->free_count, out->starts,
                    out->sequence, out->positions, out->slot_pages, out->slot_ends, out->mask,
                    in_place ? ticket : nullptr, status};
  const int work = std::max({tokens, B, 1});
  const int grid = std::min((work + plan::kThreads - 1) / plan::kThreads, device_sms());
  plan::plan_kernel<<<grid, plan::kThreads, 2 * (B + 1) * sizeof(int), (cudaStream_t)stream_>>>(p);
  note_launches(1);
  return check_cuda(cudaGetLastError(), "wtq_plan_tokens launch");
}

extern "C" int wtq_release_tokens(const int32_t *marks, int32_t *table, int64_t table_stride, int32_t *lengths,
                                  int32_t *held, int32_t *free_pages, int32_t *free_count, int B, int max_pages,
                                  int stack, int32_t *status, void *stream_) {
  if (B < 0 || B > plan::kMaxBatch || max_pages < 1 || stack < 0)
    return fail(WTQ_ERR_ARG, "wtq_release_tokens: need 0 <= B <= %d", plan::kMaxBatch);
  if (stack > plan::kMost) return fail(WTQ_ERR_ARG, "wtq_release_tokens: free pages are limited to 2^30");
  if (B == 0) return WTQ_OK;
  if (!marks || !table || !lengths || !held || !free_pages || !free_count)
    return fail(WTQ_ERR_ARG, "wtq_release_tokens: null argument");
  plan::release_kernel<<<1, plan::kThreads, (B + 1) * sizeof(int), (cudaStream_t)stream_>>>(
      marks, table, table_stride, lengths, held, free_pages, free_count, B, max_pages, stack, status);
  note_launches(1);
  return check_cuda(cudaGetLastError(), "wtq_release_tokens launch");
}
