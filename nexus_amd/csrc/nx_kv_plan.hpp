// nx_kv_plan.hpp — the paged key/value cache's geometry, what its calls
// accept, and which tokens a batch names.
//
// Plain C++ (no HIP): the CPU tests compile this header on its own.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <new>
#include <string>
#include <vector>

#include "../../include/nexus_hip.h"

namespace nx {

int fail(int code, const std::string &msg);

// A C entry's body: no exception leaves it (what they do on the host allocates).  The messages
// are short enough for a string to hold without memory of its own.
template <typename F>
int guarded(F f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return fail(NX_ERR_OOM, "out of memory");
  } catch (...) {
    return fail(NX_ERR_DEVICE, "internal error");
  }
}

// A page holds, for each kv head, page_tokens / 32 groups of 32 tokens.  A
// group's keys and values lie in the order in which the matrix cores take them
// (es bytes an element; D = head_dim):
//
//   keys    [D / 8][32 rows][8 elements]    token t of the group in row kv_row(t)
//   values  [4][D][8 tokens]                tokens 8 c .. 8 c + 7 of chunk c
//
// so an operand fragment is a run of contiguous memory, and the value chunks
// are already transposed: eight tokens of one element, the contraction index of
// p . v.  INT8 caches keep one f32 scale per token and head beside the codes,
// in token order.
constexpr int kKvGroup = 32;

// The row of a group in which token t's keys are stored.  The scores of a tile
// come out of the matrix cores with the accumulator's rows spread over the lane
// groups; these orders make each lane's scores those of eight consecutive
// tokens, one value chunk, so the probabilities are the next product's operand
// as they stand.  F16: bits 2 and 3 swapped, the order of one 32-row tile.
// INT8: the two 16-row tiles' rows alternate, so one 16-byte load feeds both.
constexpr int kv_row(int fmt, int t) {
  return fmt == NX_KV_INT8 ? (t & 24) + 2 * (t & 3) + ((t >> 2) & 1)
                           : (t & 19) | ((t & 4) << 1) | ((t & 8) >> 1);
}
// the token stored in row r (the inverse)
constexpr int kv_token(int fmt, int r) {
  return fmt == NX_KV_INT8 ? (r & 24) + 4 * (r & 1) + ((r >> 1) & 3)
                           : (r & 19) | ((r & 4) << 1) | ((r & 8) >> 1);
}
constexpr int kv_elem_bytes(int fmt) { return fmt == NX_KV_INT8 ? 1 : 2; }
// element offsets within a group
constexpr int kv_key_at(int fmt, int t, int d) { return ((d >> 3) * kKvGroup + kv_row(fmt, t)) * 8 + (d & 7); }
constexpr int kv_value_at(int D, int t, int d) { return ((t >> 3) * D + d) * 8 + (t & 7); }

struct Refusal {
  int code = NX_OK;
  std::string why;
  explicit operator bool() const { return code != NX_OK; }
};

constexpr bool kv_head_dim(int D) { return D == 64 || D == 96 || D == 128 || D == 256; }

inline Refusal kv_check_geometry(int fmt, int pages, int page_tokens, int kv_heads, int D) {
  if (fmt != NX_KV_F16 && fmt != NX_KV_INT8)
    return {NX_ERR_INVALID_ARG, "unknown cache format " + std::to_string(fmt)};
  if (pages <= 0 || kv_heads <= 0 || D <= 0 || page_tokens <= 0)
    return {NX_ERR_INVALID_ARG, "cache dimensions must be positive"};
  if (page_tokens < kKvGroup || page_tokens > 1024 || (page_tokens & (page_tokens - 1)))
    return {NX_ERR_UNSUPPORTED, "a page holds 32, 64, 128, 256, 512 or 1024 tokens, not " +
                                    std::to_string(page_tokens)};
  if (!kv_head_dim(D))
    return {NX_ERR_UNSUPPORTED, "a cache's head_dim is 64, 96, 128 or 256, not " + std::to_string(D)};
  if (kv_heads > 4096)
    return {NX_ERR_UNSUPPORTED, "a cache has at most 4096 heads, not " + std::to_string(kv_heads)};
  return {};
}

// bytes of the planes: keys or values, and one of the two scale planes
inline size_t kv_plane_bytes(int fmt, int pages, int page_tokens, int kv_heads, int D) {
  return (size_t)pages * page_tokens * kv_heads * D * kv_elem_bytes(fmt);
}
inline size_t kv_scale_bytes(int fmt, int pages, int page_tokens, int kv_heads) {
  return fmt == NX_KV_INT8 ? (size_t)pages * page_tokens * kv_heads * 4 : 0;
}

// What every call checks of a batch: its sizes and that its arrays are there.
inline Refusal kv_check_batch(const nx_kv_batch *b, int page_tokens) {
  if (!b) return {NX_ERR_INVALID_ARG, "null batch"};
  if (b->num_seqs < 0 || b->num_tokens < 0 || b->max_pages < 0)
    return {NX_ERR_INVALID_ARG, "negative batch size"};
  if (b->num_seqs == 0 || b->num_tokens == 0) return {};
  if (!b->row_start || !b->kv_len || !b->pages) return {NX_ERR_INVALID_ARG, "null batch array"};
  if (b->max_pages == 0) return {NX_ERR_SHAPE, "a batch of sequences without pages"};
  if ((int64_t)b->max_pages * page_tokens > INT32_MAX - 65536)
    return {NX_ERR_UNSUPPORTED, "sequences of more than 2^31 tokens"};
  if (b->num_seqs > (1 << 20)) return {NX_ERR_UNSUPPORTED, "more than 2^20 sequences"};
  if (b->num_tokens > (1 << 24)) return {NX_ERR_UNSUPPORTED, "more than 2^24 rows"};
  return {};
}

inline Refusal kv_check_rows(const char *what, long stride, long width) {
  if (stride < width)
    return {NX_ERR_SHAPE, std::string(what) + " rows overlap: stride " + std::to_string(stride) +
                              ", width " + std::to_string(width)};
  return {};
}

inline Refusal attn_check(int heads, int kv_heads, float scale, int window, int sinks) {
  if (heads <= 0) return {NX_ERR_INVALID_ARG, "number of heads must be positive"};
  if (heads % kv_heads)
    return {NX_ERR_SHAPE, std::to_string(heads) + " heads do not share " + std::to_string(kv_heads) +
                              " key/value heads evenly"};
  if (heads > 65536) return {NX_ERR_UNSUPPORTED, "more than 65536 heads"};
  if (!std::isfinite(scale)) return {NX_ERR_INVALID_ARG, "the score scale is not finite"};
  if (window < 0 || sinks < 0) return {NX_ERR_INVALID_ARG, "negative window or sinks"};
  return {};
}

// What the calls on host memory check besides: that every row, length and page
// is one the cache has.  (Calls on device memory cannot look: their kernels
// leave out what is not there.)  `whole`: the call reads the sequences from
// their first token on (attention; with a window, but for the pages that no row sees); else
// only the batch's rows.  `writes`: no two sequences may write one token's place.
inline Refusal kv_check_tables(const nx_kv_batch &b, int num_pages, int page_tokens, bool whole, bool writes,
                               int window = 0, int sinks = 0) {
  struct Span {
    int page, lo, hi;
  };
  std::vector<Span> spans;
  for (int s = 0; s < b.num_seqs; ++s) {
    const int r0 = b.row_start[s], r1 = b.row_start[s + 1], len = b.kv_len[s];
    if (r0 < 0 || r1 < r0 || r1 > b.num_tokens)
      return {NX_ERR_SHAPE, "rows of sequence " + std::to_string(s) + " are not in the batch"};
    const int n = r1 - r0;
    if (len < n)
      return {NX_ERR_SHAPE, "sequence " + std::to_string(s) + " has " + std::to_string(n) + " rows and " +
                                std::to_string(len) + " tokens"};
    if (len > (int64_t)b.max_pages * page_tokens)
      return {NX_ERR_SHAPE, "sequence " + std::to_string(s) + " is longer than its pages"};
    if (n == 0) continue;
    for (int p = whole ? 0 : (len - n) / page_tokens; p <= (len - 1) / page_tokens; ++p) {
      const int64_t from = (int64_t)p * page_tokens;
      if (window > 0 && from >= sinks && from + page_tokens <= (int64_t)len - n - window + 1) continue;
      const int page = b.pages[(size_t)s * b.max_pages + p];
      if (page < 0 || page >= num_pages)
        return {NX_ERR_INVALID_ARG, "page " + std::to_string(page) + " of sequence " + std::to_string(s) +
                                        " is not in the cache"};
      if (writes) spans.push_back({page, std::max(len - n - p * page_tokens, 0), std::min(len - p * page_tokens, page_tokens)});
    }
  }
  std::sort(spans.begin(), spans.end(), [](const Span &x, const Span &y) {
    return x.page != y.page ? x.page < y.page : x.lo < y.lo;
  });
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].page == spans[i - 1].page && spans[i].lo < spans[i - 1].hi)
      return {NX_ERR_INVALID_ARG, "two sequences write the same tokens of page " + std::to_string(spans[i].page)};
  return {};
}

// The groups of 32 tokens that some of the tokens pmin .. pmax of a sequence of
// len tokens see: [0, sinks) and [from, to).
struct KeySpan {
  int sinks, from, to;
  constexpr int count() const { return sinks + to - from; }
  // group number i of them
  constexpr int group(int i) const { return i < sinks ? i : from + (i - sinks); }
};
constexpr KeySpan key_span(int pmin, int pmax, int len, int window, int sinks) {
  const int last = pmax < len - 1 ? pmax : len - 1;
  const int to = last < 0 ? 0 : last / kKvGroup + 1;
  int from = 0, first = 0;
  if (window > 0) {
    const int lo = (pmin > 0 ? pmin : 0) - window + 1;  // (a row before token 0 sees nothing)
    from = lo > 0 ? lo / kKvGroup : 0;
    if (from > to) from = to;
    first = sinks / kKvGroup + (sinks % kKvGroup != 0);
    if (first > from) first = from;
  }
  return {first, from, to};
}

// Which of a join's slots (D / 4 threads each) take what: a row has `share` of them, a power
// of two, which share its parts, and rows() rows are joined at once.  Slots behind the last
// whole row (there are 10 or 21 for heads of 96) have no row.
struct JoinSlots {
  int slots, share;
  constexpr int rows() const { return slots / share; }
  // whether the slot adds up its row's, slot .. slot + share - 1
  constexpr bool leads(int slot) const { return (slot & (share - 1)) == 0 && slot < rows() * share; }
};
constexpr JoinSlots join_slots(int slots, int rows, int parts) {
  int share = 1;
  while (2 * share * rows <= slots && share < parts) share *= 2;
  return {slots, share};
}

// Groups of 32 tokens that a batch's rows touch, at most: a sequence of n rows
// touches at most n, and at most n / 32 + 2.
inline long kv_touched_groups(long seqs, long rows) { return std::min(rows, rows / kKvGroup + 2 * seqs); }

// Threads of a workgroup that moves a head's group of tokens into or out of the cache, and the
// groups that one launch takes: it has fewer than 2^32 threads.  More go in several launches.
constexpr int kMoveThreads = 512;
constexpr long kv_groups_at_once(int heads) { return (long)(UINT32_MAX / kMoveThreads) / heads; }

}  // namespace nx
