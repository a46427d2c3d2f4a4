// nx_step_plan.hpp — what the calls around a step's cache and attention accept (heads normed
// and rotated, gathered weights, eviction, log probabilities), and how they share their work out.
//
// Plain C++ (no HIP): the CPU tests compile this header on its own.
#pragma once

#include "nx_kv_plan.hpp"

namespace nx {

constexpr int kMaxRopeHead = 512;  // the widest head
constexpr int kMaxTop = 64;        // alternatives of a row: one for each lane of a wave

// Whether rows of `wa` floats, `sa` apart, share memory with rows of `wb`, `sb` apart.  Rows of
// one stride may lie in each other's gaps; of two strides, anything between the first and the
// last counts.
inline bool rows_overlap(const float *a, size_t sa, size_t wa, const float *b, size_t sb, size_t wb, long rows) {
  using Wide = unsigned __int128;
  if (!a || !b || !wa || !wb || rows <= 0) return false;
  const Wide a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  const Wide a1 = a0 + 4 * ((Wide)(rows - 1) * sa + wa), b1 = b0 + 4 * ((Wide)(rows - 1) * sb + wb);
  if (a1 <= b0 || b1 <= a0) return false;
  if (rows == 1 || sa != sb) return true;
  const Wide pitch = 4 * (Wide)sa, off = b0 >= a0 ? (b0 - a0) % pitch : (pitch - (a0 - b0) % pitch) % pitch;
  return off < 4 * (Wide)wa || off + 4 * (Wide)wb > pitch;
}

// The buffers of a rotation's rows.
struct RopeRows {
  const float *q, *k;
  float *q_out, *k_out;
  size_t q_stride, k_stride, q_out_stride, k_out_stride;
};

inline Refusal rope_check(const nx_rope *r, const int32_t *positions, int rows, int heads, int kv_heads,
                          const RopeRows &x) {
  if (!r) return {NX_ERR_INVALID_ARG, "null rotation"};
  if (rows < 0 || heads < 0 || kv_heads < 0) return {NX_ERR_INVALID_ARG, "negative rows or heads"};
  if (r->head_dim <= 0 || r->rotary_dim < 0) return {NX_ERR_INVALID_ARG, "head_dim must be positive"};
  if (r->style != NX_ROPE_HALVES && r->style != NX_ROPE_PAIRS)
    return {NX_ERR_INVALID_ARG, "unknown order of pairs " + std::to_string(r->style)};
  if (r->rotary_dim > r->head_dim)
    return {NX_ERR_SHAPE, std::to_string(r->rotary_dim) + " rotated elements of heads of " + std::to_string(r->head_dim)};
  if (r->head_dim % 2 || r->rotary_dim % 2 || r->head_dim > kMaxRopeHead)
    return {NX_ERR_UNSUPPORTED, "head_dim and rotary_dim are even, up to " + std::to_string(kMaxRopeHead) + ", not " +
                                    std::to_string(r->head_dim) + " and " + std::to_string(r->rotary_dim)};
  if (!(r->eps >= 0.f) || !std::isfinite(r->eps)) return {NX_ERR_INVALID_ARG, "eps is negative or not finite"};
  if (heads > 65536 || kv_heads > 65536) return {NX_ERR_UNSUPPORTED, "more than 65536 heads"};
  if (rows > (1 << 24)) return {NX_ERR_UNSUPPORTED, "more than 2^24 rows"};
  if (rows == 0 || heads + kv_heads == 0) return {};
  if (r->rotary_dim > 0 && (!r->freq || !positions)) return {NX_ERR_INVALID_ARG, "null positions or frequencies"};
  if ((heads && (!x.q || !x.q_out)) || (kv_heads && (!x.k || !x.k_out))) return {NX_ERR_INVALID_ARG, "null buffer"};
  for (size_t s : {x.q_stride, x.k_stride, x.q_out_stride, x.k_out_stride})
    if (s > (size_t)1 << 40) return {NX_ERR_UNSUPPORTED, "row stride above 2^40"};
  const size_t wq = (size_t)heads * r->head_dim, wk = (size_t)kv_heads * r->head_dim;
  if (heads) {
    if (Refusal f = kv_check_rows("query", (long)x.q_stride, (long)wq)) return f;
    if (Refusal f = kv_check_rows("query output", (long)x.q_out_stride, (long)wq)) return f;
  }
  if (kv_heads) {
    if (Refusal f = kv_check_rows("key", (long)x.k_stride, (long)wk)) return f;
    if (Refusal f = kv_check_rows("key output", (long)x.k_out_stride, (long)wk)) return f;
  }
  const bool same_q = x.q_out == x.q && x.q_out_stride == x.q_stride;
  const bool same_k = x.k_out == x.k && x.k_out_stride == x.k_stride;
  if ((!same_q && rows_overlap(x.q, x.q_stride, wq, x.q_out, x.q_out_stride, wq, rows)) ||
      (!same_k && rows_overlap(x.k, x.k_stride, wk, x.k_out, x.k_out_stride, wk, rows)) ||
      rows_overlap(x.q, x.q_stride, wq, x.k_out, x.k_out_stride, wk, rows) ||
      rows_overlap(x.k, x.k_stride, wk, x.q_out, x.q_out_stride, wq, rows) ||
      rows_overlap(x.q_out, x.q_out_stride, wq, x.k_out, x.k_out_stride, wk, rows))
    return {NX_ERR_INVALID_ARG, "outputs overlap rows that are not their own"};
  return {};
}

inline Refusal logprobs_check(const float *logits, size_t stride, int rows, int vocab, const int32_t *tokens,
                              int given, const float *logprobs, int top, const int32_t *top_ids,
                              const float *top_logprobs) {
  if (rows < 0 || given < 0 || top < 0) return {NX_ERR_INVALID_ARG, "negative rows, tokens or alternatives"};
  if (vocab <= 0) return {NX_ERR_INVALID_ARG, "the number of logits must be positive"};
  if (rows > (1 << 24)) return {NX_ERR_UNSUPPORTED, "more than 2^24 rows"};
  if (vocab > (1 << 30)) return {NX_ERR_UNSUPPORTED, "more than 2^30 logits"};
  if (top > kMaxTop) return {NX_ERR_UNSUPPORTED, "more than " + std::to_string(kMaxTop) + " alternatives"};
  if (given > (1 << 20)) return {NX_ERR_UNSUPPORTED, "more than 2^20 tokens of a row"};
  if (stride > (size_t)1 << 40) return {NX_ERR_UNSUPPORTED, "row stride above 2^40"};
  if (Refusal f = kv_check_rows("logit", (long)stride, vocab)) return f;
  if (rows == 0) return {};
  if (!logits || (given > 0 && (!tokens || !logprobs)) || (top > 0 && (!top_ids || !top_logprobs)))
    return {NX_ERR_INVALID_ARG, "null buffer"};
  return {};
}

// How the rows of weights of a host call are read, need(sequence) of each row of a sequence: `rows` - 1 whole ones of
// `width`, and of the last sequence that has any its last row's `last` weights, for the caller's memory may
// end with them.
struct WeightRows {
  size_t rows, last;
};
template <typename Need>
WeightRows weight_rows(int seqs, int kv_heads, Need need) {
  for (int s = seqs - 1; s >= 0; --s)
    if (const size_t n = need(s)) return {(size_t)(s + 1) * kv_heads, n};
  return {0, 0};
}
// Whether they, `sa` apart, share memory with others, `sb` apart: between the first weights and the last ones of
// both, and there as rows of wa and wb.
inline bool weights_overlap(const float *a, size_t sa, size_t wa, const WeightRows &ra, const float *b, size_t sb, size_t wb,
                            const WeightRows &rb) {
  if (!ra.rows || !rb.rows) return false;
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  if (a0 + 4 * ((ra.rows - 1) * sa + ra.last) <= b0 || b0 + 4 * ((rb.rows - 1) * sb + rb.last) <= a0) return false;
  return rows_overlap(a, sa, wa, b, sb, wb, (long)std::max(ra.rows, rb.rows));
}

// What the calls that gather attention weights check besides attn_check.  Calls on device memory, whose lengths
// are not known, take rows of weights for whole ones; `host`: mass_check_tables looks at them.
inline Refusal mass_check(const nx_kv_batch *b, int kv_heads, int heads, size_t q_stride, size_t width, const float *q,
                          const float *before, const float *mass, size_t mass_stride, bool host = false) {
  if (!q || !mass) return {NX_ERR_INVALID_ARG, "null buffer"};
  if ((int64_t)b->num_tokens * heads > INT32_MAX) return {NX_ERR_UNSUPPORTED, "more than 2^31 query rows"};
  if (q_stride > (size_t)1 << 40 || mass_stride > (size_t)1 << 40) return {NX_ERR_UNSUPPORTED, "row stride above 2^40"};
  if (Refusal f = kv_check_rows("query", (long)q_stride, (long)width)) return f;
  if (mass_stride == 0) return {NX_ERR_SHAPE, "rows of no weights"};
  if (!host && before && before != mass &&
      rows_overlap(before, mass_stride, mass_stride, mass, mass_stride, mass_stride, (long)b->num_seqs * kv_heads))
    return {NX_ERR_INVALID_ARG, "the weights overlap those before in part"};
  return {};
}

// Of a host batch whose tables were checked: the tokens of a row of weights that are read (those before the
// step's own) and written.
inline size_t mass_read(const nx_kv_batch &b, int s, size_t mass_stride) {
  const int n = b.row_start[s + 1] - b.row_start[s];
  return n > 0 ? std::min((size_t)(b.kv_len[s] - n), mass_stride) : 0;
}
inline size_t mass_written(const nx_kv_batch &b, int s, size_t mass_stride) {
  return b.row_start[s + 1] > b.row_start[s] ? std::min((size_t)b.kv_len[s], mass_stride) : 0;
}
inline Refusal mass_check_tables(const nx_kv_batch &b, int kv_heads, const float *before, const float *mass,
                                 size_t mass_stride) {
  if (before && before != mass &&
      weights_overlap(before, mass_stride, mass_stride,
                      weight_rows(b.num_seqs, kv_heads, [&](int s) { return mass_read(b, s, mass_stride); }), mass,
                      mass_stride, mass_stride,
                      weight_rows(b.num_seqs, kv_heads, [&](int s) { return mass_written(b, s, mass_stride); })))
    return {NX_ERR_INVALID_ARG, "the weights overlap those before in part"};
  return {};
}

// How a batch's gathered weights are worked out (nx_mass.hip).  `groups`: of 32 tokens of the
// page table; `group`: query heads of a key/value head.
constexpr int kMassRows = 16, kMassTile = 128, kMassBlock = 32;
constexpr size_t kMassFloats = (size_t)1 << 26;  // of the workspace
constexpr long kMassAtOnce = 3 * 256;            // workgroups that run at once, three on a CU
// tiles of 16 rows whose scores are stored: `heads` key/value heads at once
struct MassNarrow {
  int heads;          // 0: not even one fits
  int share, chunks;  // groups of a chunk, chunks of the table
  int add_share, add_chunks;  // and of those that k_mass_add sums, which joins all chunks in each
  int tiles;          // at most, of `heads` heads
  bool one_each;      // a sequence has one tile of a head, or none: longer ones are not these kernels'
  size_t slots;       // rows of `heads` heads that there is room for
};
inline MassNarrow mass_narrow(int seqs, int rows, int group, int kv_heads, int groups, bool one_each) {
  MassNarrow m{};
  m.one_each = one_each;
  // 512 chunks of the whole batch, of 4 to 64 groups: a workgroup whose waves have one group each has nothing
  // on its way, and k_mass_add reads what each chunk leaves (4096 chunks: 100001 tokens of one INT8 sequence
  // of 4 heads 24 + 17 us for the two kernels, not 16 + 8; 61 sequences of 8191 alike)
  const long want = (long)seqs * kv_heads * groups / 512;
  m.share = 4;
  while (m.share < 64 && m.share < want) m.share *= 2;
  m.chunks = (groups + m.share - 1) / m.share;
  // (sequences of n rows have at most n group / 16 + 1 tiles of each head)
  const long all = (long)rows * group, tiles = one_each ? seqs : seqs + all / kMassRows;
  const size_t slots = one_each ? (size_t)seqs * kMassRows : (size_t)all;
  // a row's scores, and a maximum and a sum of each chunk; a launch has fewer than 2^32 threads
  const size_t row = (size_t)groups * kKvGroup + (size_t)m.chunks * 2;
  m.heads = (int)std::min({(long)kv_heads, (long)(kMassFloats / (slots * row)), (1L << 23) / (tiles * m.chunks)});
  m.tiles = (int)(tiles * m.heads);
  m.slots = slots * m.heads;
  m.add_share = m.share;
  while (m.add_share < 64 && (long)seqs * m.heads * groups / m.add_share > 512) m.add_share *= 2;
  m.add_chunks = (groups + m.add_share - 1) / m.add_share;
  return m;
}
// tiles of 128 rows against shares of the keys (k_mass_stats), and of keys against shares of the
// rows (k_mass_columns), whose parts are put together: as many rows at once as there is room for
struct MassWide {
  int rows;                  // of a launch
  size_t query;              // room for rows and heads (whole 16-byte runs)
  int key_share, key_parts;  // groups; parts of the table
  long key_units;            // tiles' parts, at most
  int row_share, row_parts;  // blocks of 32 rows; parts of a sequence of all rows
  long column_units;         // tiles of keys and their parts, at most
};
inline MassWide mass_wide(int seqs, int rows, int heads, int kv_heads, int groups, int key_tile, int D) {
  MassWide m{};
  // half of the workspace for the queries' halves, with two numbers of each row; the rest for parts
  m.rows = (int)std::max(1L, std::min((long)rows, (long)(kMassFloats / 2 / ((size_t)heads * (D + 2)))));
  const long group = heads / kv_heads, all = m.rows * group;
  m.query = ((size_t)m.rows * heads + 3) / 4 * 4;
  const long room = (long)(kMassFloats - m.query * (D + 2));
  // (sequences that these kernels take, and their tiles, at most)
  const long wide = std::min<long>(seqs, all / kMassRows + 1), tiles = kv_heads * (all / kMassTile + wide);
  const long blocks = (all + kMassBlock - 1) / kMassBlock;
  // Parts that differ in length, a prompt's, are many, so that workgroups end together: 161 to 164 us for one
  // of 4093 tokens in 2048 and 4096 units, 173 in 6144, 195 in 12288, where loads of queries add up.  Where the context is long against
  // the rows they are alike, and as many as workgroups run at once: 37 tokens behind 32003, two
  // sequences, 62 us in 744 units, 76 in 4000.
  const long units = (long)groups * kKvGroup >= 4L * rows ? kMassAtOnce : 4096;
  long parts = std::min({units / tiles, (long)groups / 4, room / ((long)m.rows * heads * 2)});
  parts = std::max(parts, 1L);
  m.key_share = (int)((groups + parts - 1) / parts);
  m.key_parts = (groups + m.key_share - 1) / m.key_share;
  // (where no scores are stored, sequences of one row are these kernels' too)
  m.key_units = kv_heads * (all / kMassTile + std::min(seqs, m.rows)) * m.key_parts;
  // The same for the rows: not shared out where there are tiles of keys for two rounds of workgroups
  // (those two sequences: 67 us, and no sum to follow, not 77 and 5), else in 2048 units (the
  // prompt: 190 us and 7 to sum up; 213 and 5 in 1024, 208 and 12 in 4096).
  const long columns = (long)kv_heads * ((groups + key_tile - 1) / key_tile);
  parts = columns * wide >= kMassAtOnce ? 1 : 2048 / columns;
  parts = std::min({parts, blocks / 4, room / ((long)seqs * kv_heads * groups * kKvGroup)});
  parts = std::max(parts, 1L);
  m.row_share = (int)((blocks + parts - 1) / parts);
  m.row_parts = (int)((blocks + m.row_share - 1) / m.row_share);
  // (of the sequences' parts each but the last is whole, and so is each of their blocks)
  m.column_units = columns * std::min((long)seqs * m.row_parts, m.row_parts + 2L * seqs);
  return m;
}

// The arguments of an eviction besides the cache and the batch.
struct EvictArgs {
  const int32_t *to_pages;
  int to_max_pages, keep, sinks, recent;
  const float *mass;
  size_t mass_stride;
  int32_t *kept, *new_len;
  float *new_mass;
  size_t new_mass_stride;
};

// `host`: evict_check_tables looks at the rows of weights
inline Refusal evict_check(const nx_kv_batch *b, int page_tokens, int kv_heads, const EvictArgs &a, bool host = false) {
  if (!b) return {NX_ERR_INVALID_ARG, "null batch"};
  if (b->num_seqs < 0 || b->max_pages < 0 || a.to_max_pages < 0) return {NX_ERR_INVALID_ARG, "negative batch size"};
  if (a.keep <= 0 || a.sinks < 0 || a.recent < 0)
    return {NX_ERR_INVALID_ARG, "a number of tokens to keep is negative, or none"};
  if ((int64_t)a.sinks + a.recent > a.keep)
    return {NX_ERR_SHAPE, std::to_string(a.sinks) + " first and " + std::to_string(a.recent) + " last tokens of " +
                              std::to_string(a.keep) + " to keep"};
  if (b->num_seqs == 0) return {};
  if (!b->kv_len || !b->pages || !a.to_pages) return {NX_ERR_INVALID_ARG, "null batch array"};
  if (!a.mass || !a.kept || !a.new_len) return {NX_ERR_INVALID_ARG, "null buffer"};
  if (b->max_pages == 0 || a.to_max_pages == 0) return {NX_ERR_SHAPE, "a batch of sequences without pages"};
  if ((int64_t)std::max(b->max_pages, a.to_max_pages) * page_tokens > INT32_MAX - 65536 || a.keep > INT32_MAX - 65536)
    return {NX_ERR_UNSUPPORTED, "sequences of more than 2^31 tokens"};
  if (b->num_seqs > (1 << 20)) return {NX_ERR_UNSUPPORTED, "more than 2^20 sequences"};
  // (every head's part of the call reads the lengths)
  const uintptr_t len = reinterpret_cast<uintptr_t>(b->kv_len), now = reinterpret_cast<uintptr_t>(a.new_len);
  const uintptr_t bytes = (uintptr_t)b->num_seqs * 4;
  if (now < len + bytes && len < now + bytes) return {NX_ERR_INVALID_ARG, "the new lengths overlap the old ones"};
  if (a.mass_stride == 0) return {NX_ERR_SHAPE, "rows of no weights"};
  if (a.mass_stride > (size_t)1 << 40 || a.new_mass_stride > (size_t)1 << 40)
    return {NX_ERR_UNSUPPORTED, "row stride above 2^40"};
  if (!a.new_mass) return {};
  if (Refusal f = kv_check_rows("weight", (long)a.new_mass_stride, a.keep)) return f;
  const size_t width = std::min(a.mass_stride, (size_t)b->max_pages * page_tokens);
  if (!host && rows_overlap(a.mass, a.mass_stride, width, a.new_mass, a.new_mass_stride, a.keep, (long)b->num_seqs * kv_heads))
    return {NX_ERR_INVALID_ARG, "the new weights overlap the old ones"};
  return {};
}

// What the call on host memory checks besides: lengths and weights (of kv_heads heads), and that the new pages
// are the cache's, nobody else's of the batch, and named once.
inline Refusal evict_check_tables(const nx_kv_batch &b, int num_pages, int page_tokens, const EvictArgs &a, int kv_heads = 1) {
  std::vector<int> from, to;
  for (int s = 0; s < b.num_seqs; ++s) {
    const int len = b.kv_len[s];
    const std::string who = "sequence " + std::to_string(s);
    if (len < 0 || len > (int64_t)b.max_pages * page_tokens) return {NX_ERR_SHAPE, who + " is not as long as its pages"};
    if ((size_t)len > a.mass_stride) return {NX_ERR_SHAPE, who + " has more tokens than weights"};
    const int n = std::min(len, a.keep);
    if (n > (int64_t)a.to_max_pages * page_tokens) return {NX_ERR_SHAPE, who + " keeps more tokens than its new pages hold"};
    for (int side = 0; side < 2; ++side) {
      const int32_t *pages = side ? a.to_pages + (size_t)s * a.to_max_pages : b.pages + (size_t)s * b.max_pages;
      for (int p = 0; p < ((side ? n : len) + page_tokens - 1) / page_tokens; ++p) {
        if (pages[p] < 0 || pages[p] >= num_pages)
          return {NX_ERR_INVALID_ARG, "page " + std::to_string(pages[p]) + " of " + who + " is not in the cache"};
        (side ? to : from).push_back(pages[p]);
      }
    }
  }
  size_t most = 0;
  for (int s = 0; s < b.num_seqs; ++s) most = std::max(most, (size_t)b.kv_len[s]);
  if (a.new_mass && weights_overlap(a.mass, a.mass_stride, most,
                                    weight_rows(b.num_seqs, kv_heads, [&](int s) { return (size_t)b.kv_len[s]; }),
                                    a.new_mass, a.new_mass_stride, a.keep, weight_rows(b.num_seqs, kv_heads, [&](int s) {
                                      return (size_t)std::min(b.kv_len[s], a.keep);
                                    })))
    return {NX_ERR_INVALID_ARG, "the new weights overlap the old ones"};
  std::sort(from.begin(), from.end());
  std::sort(to.begin(), to.end());
  for (size_t i = 0; i < to.size(); ++i)
    if ((i && to[i] == to[i - 1]) || std::binary_search(from.begin(), from.end(), to[i]))
      return {NX_ERR_INVALID_ARG, "new page " + std::to_string(to[i]) + " is in use"};
  return {};
}

// Workgroups that share a row's logits, and the logits of each (a multiple of 4).  (One of each row:
// 32000 logits 23 us, not 13, 61 rows of 131072 55 us, not 17.)
constexpr int kLogprobWgs = 1024;   // as many as fill the card, and no more where rows are split
constexpr int kLogprobLeast = 4096; // of one, in logits
constexpr int kLogprobParts = 64;
struct RowSplit {
  int parts, share;
};
inline RowSplit logprob_split(int rows, int vocab) {
  const int want = std::max(1, kLogprobWgs / rows), most = (vocab + kLogprobLeast - 1) / kLogprobLeast;
  const int parts = std::max(1, std::min({want, most, kLogprobParts}));
  const int share = ((vocab + parts - 1) / parts + 3) / 4 * 4;
  return {(vocab + share - 1) / share, share};
}

}  // namespace nx
