// nx_attn.hip — causal attention of new tokens over their sequences in the paged
// cache, whole or through a sliding window with first tokens that stay visible.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i)
//
// over the tokens j that token i sees, in one pass over the cache: m_i is the
// running maximum, and the sums taken so far are scaled by exp(m_old - m_new)
// when it grows.  Scores, weights, maxima and sums are f32.
//
// Three kernels.  k_attn_split reads the keys for 16 rows at a time and splits them over
// waves and workgroups: steps of few rows, bound by memory or, short ones, by latency.
// k_attn_tile reads them for 128 rows at a time: prompts, bound by the matrix cores and
// what feeds them.  k_attn_join puts the second one's split tiles together.  Which
// sequences go where: tile_from and kFewScores below.
#include <hip/hip_runtime.h>

#include "nx_attn_dev.hpp"

namespace nx {

struct AttnCall {
  const float *q;
  float *out;
  size_t q_stride, out_stride;
  int heads, group;  // query heads, and those that share a key/value head
  float scale;
  int window, sinks;
  bool wide_q, wide_out;  // rows of whole float4 runs
  uint32_t magic;         // by_group's
  int shift;
};

__device__ __forceinline__ int by_group(const AttnCall &a, int row) { return by_group(row, a.magic, a.shift); }

// whether token p sees token j <= p
__device__ __forceinline__ bool sees(const AttnCall &a, int p, int j) {
  return j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
}

// the largest (sum) over the wave's lanes, in all of them
template <typename Op>
__device__ __forceinline__ double across_wave(double v, Op op) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = op(v, __shfl_xor(v, d, 64));
  return v;
}

// One row by the formula alone, on the values that the cache reads back and summed in 64 bits
// (whose range holds any sum of f32 products): a wave, each lane a key's whole score, then each
// lane some elements of the sum over the keys.  For rows whose result on the matrix cores is
// not finite or sums to nothing: infinities and NaNs in the row's own keys, values or query, 0
// times a masked one, value scales that the halves do not reach (value_exp), or no token to
// see.  Rare, and not made fast: a wave walks a row's whole context, 45 ms, not 81 us, for one
// token after 100001 of 32 heads over 8 of 128 (F16).
template <int FMT, int D>
__device__ __forceinline__ void attn_row(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                         const KvSeq &s, int seq, int head, int p, const float *q,
                                         float *out) {
  using E = kv_elem<FMT>;
  constexpr bool I8 = FMT == NX_KV_INT8;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // what follows from it is not held in registers by the callers' loops
  const E *ck = reinterpret_cast<const E *>(kv.k), *cv = reinterpret_cast<const E *>(kv.v);
  double m = -INFINITY, l = 0., acc[(D + 63) / 64] = {};
  bool any = false;
  const int end = min(p + 1, s.len);
  for (int j0 = 0; j0 < end; j0 += 64) {
    if (a.window && j0 >= a.sinks && j0 + 64 <= p - a.window + 1) {
      j0 = (p - a.window + 1) / 64 * 64;  // the next tokens that the row sees
      if (j0 >= end) break;
    }
    const int j = j0 + lane;
    long group = -1;
    if (j < end && sees(a, p, j)) group = kv_group(kv, b, seq, head, j & ~(kKvGroup - 1));
    const int t = j & (kKvGroup - 1);
    double x = -INFINITY;
    if (group >= 0) {
      x = 0.;
      const E *k = ck + group * (kKvGroup * D);
      const float ks = I8 ? kv.ks[group * kKvGroup + t] : 1.f;
      for (int d = 0; d < D; ++d) x = fma((double)((float)k[kv_key_at(FMT, t, d)] * ks), (double)q[d], x);
      x *= a.scale;
    }
    const uint64_t seen = __ballot(group >= 0);
    if (!seen) continue;
    any = true;
    if (__any(x != x)) {  // a NaN score makes the row NaNs
      l = NAN;
      break;
    }
    const double m1 = fmax(m, across_wave(x, [](double u, double v) { return fmax(u, v); }));
    const double ref = m1 == -INFINITY ? 0. : m1;
    const float w = group >= 0 ? expf((float)(x - ref)) : 0.f;
    const double keep = m == -INFINITY ? 0. : (double)expf((float)(m - ref));
    m = m1;
    l = l * keep + across_wave((double)w, [](double u, double v) { return u + v; });
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i) acc[i] *= keep;
    const float vs = I8 && group >= 0 ? kv.vs[group * kKvGroup + t] : 1.f;
    for (int u = 0; u < 64; ++u) {
      if (!((seen >> u) & 1)) continue;
      const double wu = __shfl(w, u, 64);
      const float su = I8 ? __shfl(vs, u, 64) : 1.f;
      const E *v = cv + __shfl(group, u, 64) * (kKvGroup * D);
#pragma unroll
      for (int i = 0; i < (D + 63) / 64; ++i) {
        const int d = lane + 64 * i;
        if (d < D) acc[i] = fma(wu, (double)((float)v[kv_value_at(D, (j0 + u) & (kKvGroup - 1), d)] * su), acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < (D + 63) / 64; ++i) {
    const int d = lane + 64 * i;
    if (d < D) out[d] = any ? (float)(acc[i] / l) : 0.f;
  }
}

// ------------------------------------------------------------ decode: k_attn_split
//
// Rows of up to kTile (token, head) pairs that share a key/value head are one tile
// of the matrix cores; a unit of work is one tile against one group of 32 tokens.
// All units of the batch, in order of (sequence, head, tile, group), are dealt out
// in equal runs, one per workgroup, so a ragged batch loads every CU alike (or, in
// short steps, tile by tile: find_run_wave).  The waves of a workgroup take groups in
// turn and join in LDS; a tile that several workgroups have is joined by the last of them
// to end, in the order of its parts, so the result does not depend on who that is.
//
// Transposed products: S^T = K Q^T puts a query in each lane column, the scores of
// tokens 8 g .. 8 g + 7 in lane group g (kv_row), which is the operand layout of
// P^T in O^T = V^T P^T: no value moves between lanes but the maximum.  q and p
// are f32 split into two f16 halves (hi + lo: 22 bits), K and V enter as they are
// stored; int8 codes as exact f16 values, with the key's scale on the score and the
// value's on the weight.
//
// One token of one sequence uses a part of a matrix instruction, and still the loads are what
// it waits for: each lane's 16-byte loads of a group's keys are its operands as they lie in
// the cache, the next group's are on their way while one is worked on, its page number a
// group before that.  32 heads over 8 of 128: 61 sequences of up to 8191 tokens (F16, 1.29
// GB) 224-226 us, 5.7 TB/s; three of up to 131071 (INT8, 623 MB) 118, 5.3 TB/s; a large
// read reaches 6.5.  Eight waves, two on a SIMD, not four: 226 us against 233, and 29
// sequences through a window of 1024 tokens 18 against 22.  One token after 516: 10.0 us, of
// which an empty launch is 4.4 and the rest the round trips of the tables, a page number,
// the keys, the parts and their count.
// The largest weight of a row (p, or p times the value's scale) is 2^8 or more when the
// reference m is set; m is set anew, and the sums scaled, when one passes 2^15.  So
// halves stay in range, and weights down to 2^-18 of the largest keep all their bits.
constexpr float kHead = 9.f, kGrow = 15.f, kUnset = -1e30f;

// A row's running reference: m, and whether none is set yet (m is 0 then).
struct Ref {
  float m = 0.f;
  bool fresh = true;
  __device__ __forceinline__ float value() const { return fresh ? kUnset : m; }
};

// Takes sums of reference m to reference m1 >= m: by 2^(m - m1).  INT8: m follows the weights
// times their values' scales, and may move by more than 2^-126 reaches while the plain sum of
// the weights, of tokens whose scales are small, counts all the same.  So references are whole
// there, and that sum moves by its exponent (exactly, too).
template <bool I8>
struct Shift {
  float f;
  int e;
  __device__ __forceinline__ Shift(float m, float m1) {
    if constexpr (I8) {
      e = (int)fmaxf(m - m1, -1000.f);
      f = ldexp1(1.f, e);
    } else {
      f = exp2f(m - m1);
    }
  }
  __device__ __forceinline__ float weights(float l) const { return I8 ? ldexp1(l, e) : l * f; }
};

// A value scale's exponent: its log2 rounded up, + kExpBias.  Scales of 2^-90 to 2^95 count:
// then no weight without its scale passes 2^(90 + kGrow), the largest of them (which are summed
// too) lies above 2^-87, where 2^x still has 40 binades below it, and the weights with their
// scales stay in range.  A scale of 0 counts as one less than the least.  A larger or smaller one,
// or NaN (a token that is not finite), outgrows everything: rows that see it end without a sum,
// and attn_row gives what the formula does.
constexpr uint32_t kExpLeast = 37, kExps = 185;  // exponent fields
constexpr float kExpBias = 126.f - kExpLeast, kExpOut = 1e37f;
__device__ __forceinline__ uint32_t scale_field(float s) { return (__float_as_uint(s) >> 23) - kExpLeast; }
__device__ __forceinline__ float value_exp(float s) {
  const uint32_t e = scale_field(s);
  return e < kExps ? (float)e : s == 0.f ? -1.f : kExpOut;
}
__device__ __forceinline__ float finite_scale(float s) { return fmaxf(s, 0.f); }

// Scores to weights, in place: w = 2^(s c(j) - m) (INT8: times the values' scales dv(j),
// of exponents de(j)), added to l; where a weight has outgrown the reference of its
// row, m is set anew and l and acc are scaled.  vis: the scores that the row sees,
// unless `all` of the wave's rows see all of them; `top` makes a maximum that of the
// row's lanes.
template <bool I8, int N, typename Coef, typename Scale, typename Exp, typename Acc, int DT, typename Top>
__device__ __forceinline__ void weigh(float (&w)[N], Coef c, Scale dv, Exp de, bool all, int vis, Ref &ref,
                                      float &l, Acc (&acc)[DT], Top top) {
  float sum = 0.f, most = -INFINITY;
  if (all) {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = fmaf(w[j], c(j), -ref.m);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = (vis >> j) & 1 ? fmaf(w[j], c(j), -ref.m) : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) most = fmaxf(most, I8 ? w[j] + de(j) : w[j]);
  constexpr float bias = I8 ? kExpBias : 0.f;
  if (__any(most > (ref.fresh ? -INFINITY : kGrow + bias))) {
    most = top(most) - bias;
    const bool anew = most > (ref.fresh ? -INFINITY : kGrow);
    const float m1 = anew ? ref.m + (I8 ? floorf(most - kHead) : most - kHead) : ref.m;
    const Shift<I8> to(ref.m, m1);
    const float keep = ref.fresh ? 0.f : to.f;
    l = I8 ? (ref.fresh ? 0.f : to.weights(l)) : l * keep;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] *= keep;
    // (rounded in the last places of scores of this size, as they are themselves)
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] += ref.m - m1;
    ref.m = m1;
    ref.fresh = ref.fresh && !anew;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    w[j] = __builtin_amdgcn_exp2f(w[j]);
    sum += w[j];
  }
  l += sum;
  if constexpr (I8) {
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] *= dv(j);
  }
}

// A tile of a sequence: rows r0 .. r0 + nr - 1 of its n * group (token, head) rows
struct Tile {
  int seq, head, r0, nr;
};
__device__ __forceinline__ KeySpan tile_span(const KvSeq &s, const AttnCall &a, int r0, int nr) {
  return key_span(s.first + by_group(a, r0), s.first + by_group(a, r0 + nr - 1), s.len, a.window,
                  a.sinks);
}
// Partial results of tiles that were split: per workgroup, those of the tile that
// it ends (or passes through) and of the tile that it begins.
//   part [workgroups][2] {m[tile], l[tile], o[tile][D]}
// Of those tiles:
//   k_attn_split: done [workgroups] parts that are written of the tile it begins, 0 between calls
//   k_attn_tile: desc [workgroups][2], as part: {seq, head, r0, its parts 2^16 + which
//   one this is, or 0}
struct AttnWork {
  int4 *desc;
  int *done;
  float *part;
  int wgs_log2, min_share;
  int tile_cost, join_cost;   // what a tile, and one in parts, takes besides its groups, in units
  int rows_above, rows_upto;  // the kernel's sequences: those of so many rows
  long few;                   // or, above 0: all are k_attn_split's for up to so many scores
};

// whether the step has w.few scores or fewer (up to 64 sequences; in integers, so that
// both kernels find the same)
__device__ __forceinline__ bool few_scores(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                           const AttnWork &w) {
  const int lane = threadIdx.x & 63;
  const KvSeq q = lane < b.num_seqs ? kv_seq(b, lane, kv.page_log2) : KvSeq{0, 0, 0, 0};
  const long keys = a.window > 0 ? min((long)q.len, (long)a.window + a.sinks + q.n) : q.len;
  long scores = keys * q.n * a.heads;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) scores += __shfl_xor(scores, x, 64);
  return uniform(scores) <= w.few;
}

// Units of a tile: its cost, then one per group (at least one, so that rows which
// see nothing are written).
__device__ __forceinline__ int tile_units(const KvSeq &s, const AttnCall &a, int cost, int r0, int tile) {
  const int nr = min(tile, s.n * a.group - r0);
  return cost + max(tile_span(s, a, r0, nr).count(), 1);
}

// A workgroup's run of units: [begin, end) of all, which starts `off` units into
// the tile at (seq, head, r0).
struct Run {
  long begin, end, share;
  int seq, head, r0, off;
  int cost;  // what a tile takes besides its groups, in units
  KvSeq s;   // the sequence
};
struct RunLds {
  long sums[8];
  long at, in_head;
  int seq, bigs, big[512], r0, off;
};

__device__ __forceinline__ int quotient(long x, long y) {
  return x <= UINT32_MAX && y <= UINT32_MAX ? (int)((uint32_t)x / (uint32_t)y) : (int)(x / y);
}

// find_run for up to 64 sequences, the usual step: every wave by itself, a lane per
// sequence, without a barrier.  false: left to the workgroup (equal runs over many tiles).
//
// Two ways to deal the units out.  Equal runs of all of them load every CU alike.  Or the
// tiles apart: the same number of workgroups for each, and a workgroup has one tile.
// That is for steps whose time is latency: a run that crosses into another tile waits for
// its query and its keys again, and a tile in parts waits for them (join_cost), so
// tiles are also taken whole where that ends sooner.
template <int TILE>
__device__ __forceinline__ bool find_run_wave(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                              const AttnWork &w, int wg, Run &r, bool &some) {
  constexpr int kFew = 4;
  const int lane = threadIdx.x & 63;
  const KvSeq q = lane < b.num_seqs ? kv_seq(b, lane, kv.page_log2) : KvSeq{0, 0, 0, 0};
  int rows = q.n * a.group;
  if (rows <= w.rows_above || rows > w.rows_upto) rows = 0;
  const int tiles = (rows + TILE - 1) / TILE;
  if (__any(tiles > 1 << 12)) return false;
  // first, last and longest tile (through a window: a bound of the longest), and all by their mean
  const int begin_u = tiles > 0 ? tile_units(q, a, 0, 0, TILE) : 0;
  const int end_u = tiles > 1 ? tile_units(q, a, 0, (tiles - 1) * TILE, TILE) : begin_u;
  int longest = end_u;
  if (a.window > 0 && tiles > 1) {
    const long seen = min((long)a.sinks, (long)q.len) / kKvGroup + 1 +
                      ((long)a.window + by_group(a, TILE) + 2) / kKvGroup + 2;
    longest = (int)min(seen, (long)max(q.len, 1) / kKvGroup + 1);
  }
  const uint32_t guess = min((long)tiles * (begin_u + end_u) / 2 * kv.heads, 1L << 24);
  const uint32_t tiles_upto = scan64(tiles * kv.heads);
  const uint32_t all_tiles = __builtin_amdgcn_readlane(tiles_upto, 63);
  some = all_tiles > 0;
  if (!some) return true;
  const uint32_t wgs = 1u << w.wgs_log2;
  if (all_tiles <= wgs) {
    const uint32_t total = __builtin_amdgcn_readlane(scan64(guess), 63);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) longest = max(longest, __shfl_xor(longest, x, 64));
    const uint32_t most = uniform(longest), each = wgs / all_tiles;
    const uint32_t split = max((most + each - 1) / each, (uint32_t)w.min_share);
    const bool one = most <= split + w.join_cost;
    const uint32_t share = one ? most : split, cost = one ? most : split + w.join_cost;
    if (cost <= (total + all_tiles * w.tile_cost) / wgs + w.tile_cost + w.join_cost) {
      const uint32_t parts = (most + share - 1) / share, tile = wg / parts, part = wg - tile * parts;
      some = tile < all_tiles;
      if (!some) return true;
      const int s = __builtin_ctzll(__ballot(tiles_upto > tile));
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, s); };
      const uint32_t in_head = of(tiles), at = tile - (of(tiles_upto) - in_head * kv.heads);
      r.seq = s;
      r.s = {of(q.row), of(q.n), of(q.first), of(q.len)};
      r.head = at / in_head;
      r.r0 = (int)(at - r.head * in_head) * TILE;
      r.cost = 0;
      r.share = share;
      r.off = part * share;
      const int units = tile_units(r.s, a, 0, r.r0, TILE);
      some = r.off < units;
      r.begin = (long)wg * share;
      r.end = r.begin + min((int)share, units - r.off);
      return true;
    }
  }
  if (__any(rows > kFew * TILE)) return false;
  r.cost = w.tile_cost;
  int u[kFew];
  uint32_t c = 0;
#pragma unroll
  for (int i = 0; i < kFew; ++i) {
    u[i] = i * TILE < rows ? tile_units(q, a, r.cost, i * TILE, TILE) : 0;
    c += u[i];
  }
  if (__any((long)c * kv.heads > (1 << 24))) return false;
  const uint32_t mine = c * kv.heads, upto = scan64(mine), total = __builtin_amdgcn_readlane(upto, 63);
  const uint32_t share = max((total + wgs - 1) >> w.wgs_log2, (uint32_t)w.min_share), begin = wg * share;
  some = begin < total;
  if (!some) return true;
  const int s = __builtin_ctzll(__ballot(upto > begin));  // (its own units begin at or before)
  auto of = [&](int v) { return __builtin_amdgcn_readlane(v, s); };
  const uint32_t at = begin - (of(upto) - of(mine)), in_head = of(c);
  r.share = share;
  r.begin = begin;
  r.end = min(begin + share, total);
  r.seq = s;
  r.s = {of(q.row), of(q.n), of(q.first), of(q.len)};
  r.head = at / in_head;
  int rest = at - r.head * in_head, i = 0;
#pragma unroll
  for (int k = 0; k < kFew - 1; ++k) {
    const int uk = of(u[k]);
    const bool past = i == k && rest >= uk;
    rest -= past ? uk : 0;
    i += past;
  }
  r.r0 = i * TILE;
  r.off = rest;
  return true;
}

// Finds run `wg` in any batch.  A sequence's units are summed over its tiles by one
// thread, or by the workgroup where there are many; sequences are summed by a scan.
template <int TILE, int NW>
__device__ __forceinline__ bool find_run(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                         const AttnWork &w, int wg, RunLds &lds, Run &r) {
  if (b.num_seqs <= 64) {
    bool some;
    if (find_run_wave<TILE>(kv, b, a, w, wg, r, some)) return some;
  }
  constexpr int kFew = 8, kThreads = 64 * NW;
  const int tid = threadIdx.x;
  r.cost = w.tile_cost;
  auto rows_of = [&](const KvSeq &q) {
    const int rows = q.n * a.group;
    return rows > w.rows_above && rows <= w.rows_upto ? rows : 0;
  };
  // per-head units of sequence s0 + tid
  auto count = [&](int s0) {
    const KvSeq q = s0 + tid < b.num_seqs ? kv_seq(b, s0 + tid, kv.page_log2) : KvSeq{0, 0, 0, 0};
    const int rows = rows_of(q);
    long c = 0;
    if (tid == 0) lds.bigs = 0;
    __syncthreads();
    if (rows <= kFew * TILE)
      for (int r0 = 0; r0 < rows; r0 += TILE) c += tile_units(q, a, r.cost, r0, TILE);
    else
      lds.big[atomicAdd(&lds.bigs, 1)] = tid;
    __syncthreads();
    const int bigs = lds.bigs;
    for (int i = 0; i < bigs; ++i) {
      const int t = lds.big[i];
      const KvSeq o = kv_seq(b, s0 + t, kv.page_log2);
      long part = 0;
      for (long r0 = (long)tid * TILE; r0 < o.n * a.group; r0 += kThreads * TILE)
        part += tile_units(o, a, r.cost, (int)r0, TILE);
      long whole;
      scan_wg<NW>(part, lds.sums, whole);
      if (tid == t) c = whole;
    }
    return c;
  };
  long total = 0, c = 0, upto = 0, chunk;
  for (int s0 = 0; s0 < b.num_seqs; s0 += kThreads) {
    c = count(s0);
    upto = total + scan_wg<NW>(c * kv.heads, lds.sums, chunk);
    total += chunk;
  }
  total = uniform(total);
  r.share = max((total + (1 << w.wgs_log2) - 1) >> w.wgs_log2, (long)w.min_share);
  r.begin = wg * r.share;
  r.end = min(r.begin + r.share, total);
  if (r.begin >= r.end) return false;
  long before = 0;
  for (int s0 = 0; s0 < b.num_seqs; s0 += kThreads) {
    if (b.num_seqs > kThreads) {
      c = count(s0);
      upto = before + scan_wg<NW>(c * kv.heads, lds.sums, chunk);
      before += chunk;
    }
    if (r.begin >= upto - c * kv.heads && r.begin < upto) {
      lds.seq = s0 + tid;
      lds.at = r.begin - (upto - c * kv.heads);
      lds.in_head = c;
    }
    if (r.begin < before) break;  // uniform
  }
  __syncthreads();
  r.seq = uniform(lds.seq);
  const long at = uniform(lds.at), in_head = uniform(lds.in_head);
  r.head = quotient(at, in_head);
  long rest = at - r.head * in_head;
  const KvSeq s = r.s = kv_seq(b, r.seq, kv.page_log2);
  const int rows = s.n * a.group;
  if (rows <= kFew * TILE) {
    int units;
    r.r0 = 0;
    while (units = tile_units(s, a, r.cost, r.r0, TILE), rest >= units) rest -= units, r.r0 += TILE;
    r.off = (int)rest;
    return true;
  }
  long base = 0;
  for (long r0 = 0; r0 < rows && base <= rest; r0 += kThreads * TILE) {
    const long mine = r0 + (long)tid * TILE;
    const long u = mine < rows ? tile_units(s, a, r.cost, (int)mine, TILE) : 0;
    const long e = base + scan_wg<NW>(u, lds.sums, chunk);
    if (rest >= e - u && rest < e) {
      lds.r0 = (int)mine;
      lds.off = (int)(rest - (e - u));
    }
    base += chunk;
  }
  __syncthreads();
  r.r0 = uniform(lds.r0);
  r.off = uniform(lds.off);
  return true;
}

// the tile behind (seq, head, r0); the caller knows that there is one
template <int TILE>
__device__ __forceinline__ void next_tile(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                          const AttnWork &w, Run &r, KvSeq &s) {
  r.r0 += TILE;
  if (r.r0 < s.n * a.group) return;
  r.r0 = 0;
  if (++r.head < kv.heads) return;
  r.head = 0;
  int rows;
  do {
    s = kv_seq(b, ++r.seq, kv.page_log2);
    rows = s.n * a.group;
  } while (rows <= w.rows_above || rows > w.rows_upto);
}

// four values of a finished row; *bad is set where they are not finite: a weight 0
// times a value that is not finite, or a row whose result is not finite by the
// formula (or that sees nothing), which attn_row tells apart
template <int D>
__device__ __forceinline__ void store_out(const AttnCall &a, const KvSeq &s, int head, int row, int d,
                                          f32x4 o, float l, int *bad) {
  const float inv = 1.f / l;
  o *= inv;
  const int tok = by_group(a, row);
  float *out = a.out + (size_t)(s.row + tok) * a.out_stride +
               (size_t)(head * a.group + row - tok * a.group) * D + d;
  const bool fine = __builtin_isfinite(o.x) && __builtin_isfinite(o.y) && __builtin_isfinite(o.z) &&
                    __builtin_isfinite(o.w);
  if (!fine || !(l > 0.f && l < INFINITY)) *bad = 1;
  if (a.wide_out) {
    *reinterpret_cast<f32x4 *>(out) = o;
  } else {
    out[0] = o.x;
    out[1] = o.y;
    out[2] = o.z;
    out[3] = o.w;
  }
}

template <int FMT, int D, int NW>
__device__ __forceinline__ void finish_rows(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                            const KvSeq &s, const Tile &t, const int *bad) {
  for (int r = threadIdx.x >> 6; r < t.nr; r += NW) {
    if (!bad[r]) continue;
    const int row = t.r0 + r, i = by_group(a, row), h = t.head * a.group + row - i * a.group;
    attn_row<FMT, D>(kv, b, a, s, t.seq, t.head, s.first + i,
                     a.q + (size_t)(s.row + i) * a.q_stride + (size_t)h * D,
                     a.out + (size_t)(s.row + i) * a.out_stride + (size_t)h * D);
  }
}

__device__ __forceinline__ void store_through(float *p, f32x4 v) {
  const auto w = __builtin_bit_cast(ulong2, v);
  store_through(reinterpret_cast<unsigned long *>(p), w.x);
  store_through(reinterpret_cast<unsigned long *>(p) + 1, w.y);
}
template <bool THROUGH>
__device__ __forceinline__ float load1(const float *p) {
  return THROUGH ? __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *p;
}
template <bool THROUGH>
__device__ __forceinline__ f32x4 load4(const float *p) {
  if constexpr (!THROUGH) return *reinterpret_cast<const f32x4 *>(p);
  const unsigned long *q = reinterpret_cast<const unsigned long *>(p);
  const ulong2 w = {__hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
                    __hip_atomic_load(q + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)};
  return __builtin_bit_cast(f32x4, w);
}
constexpr int kTile = 16, kRows = 128;  // rows of a tile of k_attn_split, k_attn_tile

template <int D, int NW>
struct JoinLds {
  static constexpr int kSlots = 64 * NW / (D / 4);
  f32x4 o[kSlots][D / 4];
  float m[kSlots], l[kSlots];
  int bad[kRows];
};

// Joins rows y, y + dy, ... of a tile from its `parts` parts: the first one at `first`
// in slot 1 of its workgroup, the others in slot 0 of the workgroups behind.  A row
// takes D / 4 threads, or 2, 4, ... times as many that share its parts where rows are few.
// THROUGH: this kernel wrote them.
template <int FMT, int D, int NW, bool THROUGH>
__device__ __forceinline__ void join_tile(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                          const KvSeq &s, const Tile &t, const float *first, int tile,
                                          int parts, int y, int dy, JoinLds<D, NW> &lds) {
  using To = Shift<FMT == NX_KV_INT8>;
  constexpr int kSlots = JoinLds<D, NW>::kSlots;
  const int slot = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4), size = tile * (D + 2);
  const int mine = (t.nr - y + dy - 1) / dy;
  const JoinSlots by = join_slots(kSlots, mine, parts);
  const int share = by.share, sub = slot & (share - 1), at_once = by.rows();
  if (threadIdx.x < kRows) lds.bad[threadIdx.x] = 0;
  for (int k0 = 0; k0 < mine; k0 += at_once) {
    const int k = k0 + slot / share, r = y + min(k, mine - 1) * dy;
    float m = kUnset, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    auto take = [&](auto U, int i0) {  // U of the thread's parts, loaded ahead of their use
      float mp[U()], lp[U()];
      f32x4 op[U()];
#pragma unroll
      for (int x = 0; x < U(); ++x) {
        const int i = min(i0 + x * share, parts - 1);
        const float *p = first + (i == 0 ? 0 : (ptrdiff_t)(2 * i - 1) * size);
        mp[x] = load1<THROUGH>(p + r);
        lp[x] = load1<THROUGH>(p + tile + r);
        op[x] = load4<THROUGH>(p + 2 * tile + r * D + 4 * d);
      }
      float m1 = m;
#pragma unroll
      for (int x = 0; x < U(); ++x) m1 = fmaxf(m1, mp[x]);
      const To keep(m, m1);
      m = m1;
      l = keep.weights(l);
      o *= keep.f;
#pragma unroll
      for (int x = 0; x < U(); ++x) {
        const bool is = i0 + x * share < parts;
        To to(mp[x], m);
        to.f = is ? to.f : 0.f;
        l += is ? to.weights(lp[x]) : 0.f;
        o += (is ? op[x] : f32x4{0.f, 0.f, 0.f, 0.f}) * to.f;
      }
    };
    if (parts <= 2 * share)
      take(std::integral_constant<int, 2>(), sub);
    else
      for (int i = sub; i < parts; i += 4 * share) take(std::integral_constant<int, 4>(), i);
    __syncthreads();  // bad is clear, and the last rows' sums are read
    if (share > 1) {
      if (slot < kSlots) {
        lds.o[slot][d] = o;
        if (d == 0) {
          lds.m[slot] = m;
          lds.l[slot] = l;
        }
      }
      __syncthreads();
      if (by.leads(slot)) {
        float m1 = m;
        for (int x = 1; x < share; ++x) m1 = fmaxf(m1, lds.m[slot + x]);
        const To own(m, m1);
        l = own.weights(l);
        o *= own.f;
        for (int x = 1; x < share; ++x) {
          const To to(lds.m[slot + x], m1);
          l += to.weights(lds.l[slot + x]);
          o += lds.o[slot + x][d] * to.f;
        }
      }
    }
    if (by.leads(slot) && k < mine)
      store_out<D>(a, s, t.head, t.r0 + r, 4 * d, o, l, &lds.bad[r]);
  }
  __syncthreads();
  finish_rows<FMT, D, NW>(kv, b, a, s, t, lds.bad);
}

// waves of a decode workgroup: two per SIMD, or one where heads of 256 need the registers
template <int D>
constexpr int kDecodeWaves = D == 256 ? 4 : 8;

template <int D, int NW>
struct DecodeLds {
  float m[NW][kTile], l[NW][kTile];
  float o[NW][kTile][D + 4];
  int bad[kTile];
};

template <int FMT, int D>
__global__ __launch_bounds__(64 * kDecodeWaves<D>, D == 256 ? 1 : 2) void k_attn_split(KvView kv, nx_kv_batch b,
                                                                                    AttnCall a, AttnWork w) {
  using E = kv_elem<FMT>;
  constexpr int NW = kDecodeWaves<D>;
  constexpr bool I8 = FMT == NX_KV_INT8;
  constexpr int KS = D / 32, DT = D / 16;     // steps of a score, 16-element tiles of the output
  constexpr int KL = I8 ? KS : 2 * KS, VL = I8 ? DT / 2 : DT;  // 16-byte loads of a lane and group
  __shared__ union {
    RunLds run;
    DecodeLds<D, NW> rows;
    JoinLds<D, NW> join;
  } shared;
  __shared__ int lead, parts;  // the first workgroup of a split tile, and how many have it
  DecodeLds<D, NW> &lds = shared.rows;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  // neighbouring runs on one XCD: tiles of one head share its keys in that L2
  const int wg = (blockIdx.x & 7) << (w.wgs_log2 - 3) | blockIdx.x >> 3;
  if (w.few > 0 && few_scores(kv, b, a, w)) w.rows_upto = INT32_MAX;
  Run run;
  if (!find_run<kTile, NW>(kv, b, a, w, wg, shared.run, run)) return;
  __syncthreads();  // shared is free for the rows
  KvSeq s = run.s;
  const float one = opaque_one();

  for (long u = run.begin; u < run.end;) {
    const int seq = run.seq, head = run.head, r0 = run.r0;
    // groups [off, stop) of the tile's; units past its cost
    const int units = tile_units(s, a, run.cost, r0, kTile);
    const int till = (int)min((long)units, run.off + (run.end - u));
    const int off = max(run.off - run.cost, 0), stop = till - run.cost;
    const bool whole = off == 0 && till == units;
    const long next = u - run.off + units;  // the batch's units up to the next tile
    u += till - run.off;
    run.off = 0;
    if (stop <= off) {  // its cost alone: the next workgroup has it
      break;
    }
    const Tile t{seq, head, r0, min(kTile, s.n * a.group - r0)};
    const KeySpan span = tile_span(s, a, r0, t.nr);

    // ---- groups on their way: the page number a group ahead, then keys and values
    uint4 kf[KL], vf[VL];
    f32x4 dk[2], dv[2];  // INT8: scales of the lane's tokens
    auto page_of = [&](int i) {  // of group i (of the last one behind it)
      const int first = span.group(min(i, stop - 1)) * kKvGroup;
      return span.count() > 0 ? b.pages[(long)seq * b.max_pages + (first >> kv.page_log2)] : -1;
    };
    auto is_there = [&](int page) { return page >= 0 && page < kv.pages; };
    auto group_of = [&](int i, int page) {  // (pool group 0, masked, for one that is not there)
      const int in_page = (span.group(min(i, stop - 1)) * kKvGroup & ((1 << kv.page_log2) - 1)) / kKvGroup;
      return is_there(page) ? (((long)page * kv.heads + head) << (kv.page_log2 - 5)) + in_page : 0;
    };
    auto load_k = [&](long gr) {
      const E *base = reinterpret_cast<const E *>(kv.k) + gr * (kKvGroup * D);
      if constexpr (I8) {
        const f32x4 *s = reinterpret_cast<const f32x4 *>(kv.ks + gr * kKvGroup + 8 * g);
        dk[0] = s[0];
        dk[1] = s[1];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          kf[ks] = *reinterpret_cast<const uint4 *>(base + ((4 * ks + g) * kKvGroup + 2 * n) * 8);
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            kf[2 * ks + h] = *reinterpret_cast<const uint4 *>(
                base + ((4 * ks + g) * kKvGroup + 16 * (n >> 3) + 8 * h + (n & 7)) * 8);
      }
    };
    auto load_v = [&](long gr) {
      const E *base = reinterpret_cast<const E *>(kv.v) + gr * (kKvGroup * D);
      if constexpr (I8) {
        const f32x4 *s = reinterpret_cast<const f32x4 *>(kv.vs + gr * kKvGroup + 8 * g);
        dv[0] = s[0];
        dv[1] = s[1];
      }
#pragma unroll
      for (int i = 0; i < VL; ++i)
        vf[i] = *reinterpret_cast<const uint4 *>(base + (g * D + (I8 ? 32 * i + 2 * n : 16 * i + n)) * 8);
    };
    int page = page_of(off + wave), page1 = page_of(off + wave + NW);
    {
      const long gr = group_of(off + wave, page);
      load_k(gr);
      load_v(gr);
    }

    // ---- this lane's query
    const int row = r0 + min(n, t.nr - 1), tok = by_group(a, row);
    const int p = s.first + tok;  // its token
    f16x8 qh[KS], ql[KS];
    float c;
    {
      const float *q = a.q + (size_t)(s.row + tok) * a.q_stride +
                       (size_t)(head * a.group + row - tok * a.group) * D + 8 * g;
      float x[KS][8], mx = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        load8(q + 32 * ks, a.wide_q, x[ks]);
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[ks][i]));
      }
      mx = max_groups(mx);
      // scaled into [2^13, 2^14): both halves keep their bits
      const int E = mx < INFINITY ? max(__builtin_amdgcn_frexp_expf(mx), -112) : 0;
      const float up = ldexp1(1.f, 14 - E);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[ks][i] *= up;
        split2(x[ks], one, qh[ks], ql[ks]);
      }
      c = ldexp1(a.scale * kLog2e, E - 14 + (I8 ? 9 : 0));
    }

    Ref ref;
    float l = 0.f;
    f32x4 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    for (int i = off + wave; i < stop; i += NW) {
      const int first = span.group(i) * kKvGroup;
      const bool there = is_there(page);
      const long gr1 = group_of(i + NW, page1);
      page = page1;
      page1 = page_of(i + 2 * NW);
      // scores of tokens first + 8 g + 4 h + j
      f32x4 sc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f16x8 kx;
          if constexpr (I8)
            kx = h == 0 ? from_codes(kf[ks].x, kf[ks].y) : from_codes(kf[ks].z, kf[ks].w);
          else
            kx = __builtin_bit_cast(f16x8, kf[2 * ks + h]);
          sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kx, qh[ks], sc[h], 0, 0, 0);
          sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kx, ql[ks], sc[h], 0, 0, 0);
        }
      // (INT8: the keys' scales on the row's factor, not on sums that they could take past f32)
      f32x4 kc[2] = {};
      if constexpr (I8) {
        kc[0] = dk[0] * c;
        kc[1] = dk[1] * c;
      }
      load_k(gr1);  // the next group's keys, while this one's weights are made

      // which of them the lane's row sees: all, for groups inside every row's range
      const int pmin = s.first + by_group(a, r0), pmax = s.first + by_group(a, r0 + t.nr - 1);
      const bool all = there && first + kKvGroup - 1 <= pmin && first + kKvGroup <= s.len &&
                       (a.window == 0 || pmax - first < a.window || first + kKvGroup <= a.sinks);
      int vis = 0xff;
      if (!all) {
        vis = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = first + 8 * g + j;
          if (there && key < s.len && sees(a, p, key)) vis |= 1 << j;
        }
      }
      float de[8];
      if constexpr (I8) {
        uint32_t most_de = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t e = scale_field(dv[j >> 2][j & 3]);
          most_de = max(most_de, e);
          de[j] = (float)e;
        }
        if (__any(most_de >= kExps))
#pragma unroll
          for (int j = 0; j < 8; ++j) de[j] = value_exp(dv[j >> 2][j & 3]);
      }
      float pr[8] = {sc[0][0], sc[0][1], sc[0][2], sc[0][3], sc[1][0], sc[1][1], sc[1][2], sc[1][3]};
      weigh<I8>(pr, [&](int j) { return I8 ? kc[j >> 2][j & 3] : c; },
                [&](int j) { return finite_scale(dv[j >> 2][j & 3]); }, [&](int j) { return de[j]; }, all, vis, ref,
                l, acc, max_groups);
      f16x8 ph, pl;
      split2(pr, one, ph, pl);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        f16x8 vx;
        if constexpr (I8)
          vx = (d & 1) == 0 ? from_codes(vf[d / 2].x, vf[d / 2].y) : from_codes(vf[d / 2].z, vf[d / 2].w);
        else
          vx = __builtin_bit_cast(f16x8, vf[d]);
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vx, ph, acc[d], 0, 0, 0);
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vx, pl, acc[d], 0, 0, 0);
      }
      load_v(gr1);
    }

    // ---- join the waves
    l = sum_groups(l);
    const float un = I8 ? 512.f : 1.f;
    if (g == 0) {
      lds.m[wave][n] = ref.value();
      lds.l[wave][n] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        lds.o[wave][n][I8 ? 32 * (d / 2) + 2 * (4 * g + j) + (d & 1) : 16 * d + 4 * g + j] = acc[d][j] * un;
    if (threadIdx.x < kTile) lds.bad[threadIdx.x] = 0;
    __syncthreads();
    // a tile's first workgroup keeps its part in slot 1, the others in slot 0
    float *part = w.part + ((size_t)wg * 2 + (off == 0)) * (kTile * (D + 2));
    for (int e = threadIdx.x; e < t.nr * (D / 4); e += 64 * NW) {
      const int r = e / (D / 4), d = e % (D / 4) * 4;
      float m1 = lds.m[0][r];
#pragma unroll
      for (int v = 1; v < NW; ++v) m1 = fmaxf(m1, lds.m[v][r]);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float lt = 0.f;
#pragma unroll
      for (int v = 0; v < NW; ++v) {
        const Shift<I8> to(lds.m[v][r], m1);
        lt += to.weights(lds.l[v][r]);
        o += *reinterpret_cast<const f32x4 *>(&lds.o[v][r][d]) * to.f;
      }
      if (!whole) {
        if (d == 0) {
          store_through(part + r, m1);
          store_through(part + kTile + r, lt);
        }
        store_through(part + 2 * kTile + r * D + d, o);
      } else {
        const int rr = r0 + r;
        store_out<D>(a, s, head, rr, d, o, lt, &lds.bad[r]);
      }
    }
    if (whole) {
      __syncthreads();
      finish_rows<FMT, D, NW>(kv, b, a, s, t, lds.bad);
    } else {
      // The last workgroup to write its part joins them all, in their order.
      stores_done();  // this part, before the count says so
      __syncthreads();
      if (threadIdx.x == 0) {
        const long begin = next - units + run.cost;  // its first group
        const int by = off == 0 ? wg : quotient(begin, run.share);
        const int of = quotient(next - 1, run.share) - by + 1;
        const bool last = atomicAdd(&w.done[by], 1) == of - 1;
        if (last) w.done[by] = 0;  // for the next call
        lead = by;
        parts = last ? of : 0;
      }
      __syncthreads();
      if (parts > 0) {
        join_tile<FMT, D, NW, true>(kv, b, a, s, t, w.part + ((size_t)lead * 2 + 1) * (kTile * (D + 2)), kTile, parts,
                          0, 1, shared.join);
      }
    }
    __syncthreads();  // lds is free
    if (u < run.end) next_tile<kTile>(kv, b, a, w, run, s);
  }
}

// ------------------------------------------------------------ prompts: k_attn_tile
//
// Chunks of many rows: 128 rows of a key/value head against the groups of 32 tokens,
// which all four waves take from LDS, each for 32 rows of its own.  The same transposed
// products on 32 x 32 x 16 tiles: a group is one 32-row tile of scores, a lane holds
// tokens 16 s + 8 h .. + 7 of its query, the operand of value chunk 2 s + h.  The
// next group is on its way to registers while one is worked on and one lies in LDS;
// int8 codes become f16 on their way to LDS, once for the four waves.
//
// Each product is two matrix instructions (q's and p's halves; one alone would leave 11 bits
// of them).  Bound by the wave's own alternation: its scores, then maximum, exponentials and
// halves (F16 134, INT8 220 vector instructions for 32 matrix ones of a group), then its
// values; the CU's other workgroup fills the gaps, and the matrix cores are busy 43% of the
// time at about 2 GHz.  Over cards, 32 heads over 8 of 128, F16: a prompt of 4093 tokens 297-319
// us, 430-462 TFLOP/s with the halves counted once; 2039 tokens through a window of 4096
// 272-291 us, 471-504 (INT8 307, 447).  INT8, 32 heads over 4, two chunks of 509 tokens at up to
// 16127: 458-480 us, 446-467.  Scores
// of the next group ahead of this one's weights, with q's lower halves in LDS to make room:
// 346 us for the prompt, against 314.
template <int FMT, int D>
struct TileLds {
  // keys [D / 8][32 rows][8], then values [4][D][8], of two groups
  _Float16 kv[2][2 * kKvGroup * D];
  // INT8: scales of keys and values, and the latter's exponents, in token order
  float dk[2][kKvGroup], dv[2][kKvGroup], de[2][kKvGroup];
  // heads of 256: q's lower halves, each lane's its own, which registers do not hold
  f16x8 ql[D == 256 ? D / 16 : 1][D == 256 ? 256 : 1];
};

template <int FMT, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_tile(KvView kv, nx_kv_batch b,
                                                                    AttnCall a, AttnWork w) {
  using E = kv_elem<FMT>;
  constexpr bool I8 = FMT == NX_KV_INT8;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int C = kKvGroup * D * (int)sizeof(E) / 16;  // 16-byte chunks of a group's keys
  constexpr int L = (C + 255) / 256;                     // of which a thread moves
  __shared__ union {
    RunLds run;
    TileLds<FMT, D> tile;
  } shared;
  __shared__ int bad[kRows];
  TileLds<FMT, D> &lds = shared.tile;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const int wg = (blockIdx.x & 7) << (w.wgs_log2 - 3) | blockIdx.x >> 3;
  if (threadIdx.x < 2) w.desc[2 * wg + threadIdx.x] = int4{0, 0, 0, 0};
  if (w.few > 0 && few_scores(kv, b, a, w)) return;
  Run run;
  if (!find_run<kRows, 4>(kv, b, a, w, wg, shared.run, run)) return;
  KvSeq s = run.s;
  const float one = opaque_one();

  for (long u = run.begin; u < run.end;) {
    const int seq = run.seq, head = run.head, r0 = run.r0;
    // groups [off, stop) of the tile's; units past its cost
    const int units = tile_units(s, a, run.cost, r0, kRows);
    const int till = (int)min((long)units, run.off + (run.end - u));
    const int off = max(run.off - run.cost, 0), stop = till - run.cost;
    const bool whole = off == 0 && till == units;
    const long next = u - run.off + units;  // the batch's units up to the next tile
    u += till - run.off;
    run.off = 0;
    if (stop <= off) {  // its cost alone: the next workgroup has it
      break;
    }
    const int nr = min(kRows, s.n * a.group - r0);
    const KeySpan span = tile_span(s, a, r0, nr);

    // ---- this lane's query (rows behind the tile's last repeat it)
    const int row = r0 + min(32 * wave + n, nr - 1), tok = by_group(a, row);
    const int p = s.first + tok;
    // the wave's first and last token
    const int pmin = uniform(s.first + by_group(a, r0 + min(32 * wave, nr - 1)));
    const int pmax = uniform(s.first + by_group(a, r0 + min(32 * wave + 31, nr - 1)));
    f16x8 qh[KS], ql[D == 256 ? 1 : KS];
    float c;
    __syncthreads();  // the last tile's (or the run's) use of shared
    {
      const float *q = a.q + (size_t)(s.row + tok) * a.q_stride +
                       (size_t)(head * a.group + row - tok * a.group) * D + 8 * h;
      float x[KS][8], mx = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        load8(q + 16 * ks, a.wide_q, x[ks]);
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[ks][i]));
      }
      mx = max_halves(mx);
      const int X = mx < INFINITY ? max(__builtin_amdgcn_frexp_expf(mx), -112) : 0;
      const float up = ldexp1(1.f, 14 - X);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[ks][i] *= up;
        if constexpr (D == 256)
          split2(x[ks], one, qh[ks], lds.ql[ks][threadIdx.x]);
        else
          split2(x[ks], one, qh[ks], ql[ks]);
      }
      c = ldexp1(a.scale * kLog2e, X - 14 + (I8 ? 9 : 0));
    }
    Ref ref;
    float l = 0.f;
    f32x16 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;

    // ---- groups on their way: registers, then LDS
    uint4 rk[L], rv[L];
    float rs = 0.f;
    auto page_of = [&](int i) {  // of group i (of the last one behind it)
      const int first = span.group(min(i, stop - 1)) * kKvGroup;
      return span.count() > 0 ? b.pages[(long)seq * b.max_pages + (first >> kv.page_log2)] : -1;
    };
    int page = page_of(off);  // of the group to fetch next, looked up a group ahead
    auto fetch = [&](int i) {
      const bool found = page >= 0 && page < kv.pages;
      const int in_page = (span.group(i) * kKvGroup & ((1 << kv.page_log2) - 1)) / kKvGroup;
      // (pool group 0, masked, for one that is not there)
      const long gr = found ? (((long)page * kv.heads + head) << (kv.page_log2 - 5)) + in_page : 0;
      page = page_of(i + 1);
      const uint4 *gk = reinterpret_cast<const uint4 *>(kv.k) + gr * C;
      const uint4 *gv = reinterpret_cast<const uint4 *>(kv.v) + gr * C;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const int e = threadIdx.x + 256 * j;
        if (C % 256 == 0 || e < C) {
          rk[j] = gk[e];
          rv[j] = gv[e];
        }
      }
      if (I8 && threadIdx.x < 2 * kKvGroup)
        rs = (threadIdx.x < kKvGroup ? kv.ks : kv.vs)[gr * kKvGroup + (threadIdx.x & (kKvGroup - 1))];
      return found;
    };
    auto stage = [&](int buf) {
      f16x8 *k8 = reinterpret_cast<f16x8 *>(lds.kv[buf]), *v8 = k8 + kKvGroup * D / 8;
#pragma unroll
      for (int j = 0; j < L; ++j) {
        const int e = threadIdx.x + 256 * j;
        if (C % 256 != 0 && e >= C) break;
        if constexpr (I8) {
          // rows 2 x, 2 x + 1 of a key chunk: tokens t and t + 4
          const int d8 = e >> 4, t = kv_token(NX_KV_INT8, (e & 15) * 2);
          k8[d8 * kKvGroup + kv_row(NX_KV_F16, t)] = from_codes(rk[j].x, rk[j].y);
          k8[d8 * kKvGroup + kv_row(NX_KV_F16, t + 4)] = from_codes(rk[j].z, rk[j].w);
          v8[2 * e] = from_codes(rv[j].x, rv[j].y);
          v8[2 * e + 1] = from_codes(rv[j].z, rv[j].w);
        } else {
          k8[e] = __builtin_bit_cast(f16x8, rk[j]);
          v8[e] = __builtin_bit_cast(f16x8, rv[j]);
        }
      }
      if (I8 && threadIdx.x < 2 * kKvGroup) {
        (threadIdx.x < kKvGroup ? lds.dk : lds.dv)[buf][threadIdx.x & (kKvGroup - 1)] =
            threadIdx.x < kKvGroup ? rs : finite_scale(rs);
        if (threadIdx.x >= kKvGroup) lds.de[buf][threadIdx.x - kKvGroup] = value_exp(rs);
      }
    };

    bool there = fetch(off), there1 = false;
    stage(off & 1);
    if (off + 1 < stop) there1 = fetch(off + 1);
    for (int i = off; i < stop; ++i) {
      const int buf = i & 1;
      __syncthreads();  // group i is in LDS, and no wave reads group i - 1 any more
      const bool here = there;
      there = there1;
      if (i + 1 < stop) {
        stage(buf ^ 1);
        if (i + 2 < stop) there1 = fetch(i + 2);
      }
      const int first = span.group(i) * kKvGroup;
      // groups that none of the wave's rows see
      if (!here || first > pmax ||
          (a.window && first >= a.sinks && pmin - (first + kKvGroup - 1) >= a.window))
        continue;
      const f16x8 *k8 = reinterpret_cast<const f16x8 *>(lds.kv[buf]) + h * kKvGroup + n;
      const f16x8 *v8 = reinterpret_cast<const f16x8 *>(lds.kv[buf]) + kKvGroup * D / 8 + h * D + n;
      auto low = [&](int ks) {
        if constexpr (D == 256)
          return lds.ql[ks][threadIdx.x];
        else
          return ql[ks];
      };
      f32x16 sc;
#pragma unroll
      for (int j = 0; j < 16; ++j) sc[j] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const f16x8 kx = k8[2 * ks * kKvGroup];
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx, qh[ks], sc, 0, 0, 0);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx, low(ks), sc, 0, 0, 0);
      }
      // sc[8 s + j]: token first + 16 s + 8 h + j
      // (INT8: the keys' scales on the row's factor, as in k_attn_split)
      float kc[16];
      if constexpr (I8) {
#pragma unroll
        for (int j = 0; j < 16; ++j) kc[j] = lds.dk[buf][16 * (j >> 3) + 8 * h + (j & 7)] * c;
      }
      const bool all = first + kKvGroup - 1 <= pmin && first + kKvGroup <= s.len &&
                       (a.window == 0 || pmax - first < a.window || first + kKvGroup <= a.sinks);
      int vis = 0xffff;
      if (!all) {
        vis = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int key = first + 16 * (j >> 3) + 8 * h + (j & 7);
          if (key < s.len && sees(a, p, key)) vis |= 1 << j;
        }
      }
      float y[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = sc[j];
      const int at = 8 * h;  // score j's token is at + j + 8 (j >> 3)
      weigh<I8>(y, [&](int j) { return I8 ? kc[j] : c; },
                [&](int j) { return lds.dv[buf][at + j + (j & 8)]; },
                [&](int j) { return lds.de[buf][at + j + (j & 8)]; }, all, vis, ref, l, acc, max_halves);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float pr[8];
        f16x8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; ++j) pr[j] = y[8 * t + j];
        split2(pr, one, ph, pl);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const f16x8 vx = v8[2 * t * D + 32 * d];
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vx, ph, acc[d], 0, 0, 0);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vx, pl, acc[d], 0, 0, 0);
        }
      }
    }

    // ---- results: acc[d][4 x + j] is element 32 d + 8 x + 4 h + j of the lane's row
    l = across_halves(l, [](float x, float y) { return x + y; });
    const float un = I8 ? 512.f : 1.f;
    const int r = 32 * wave + n;
    if (threadIdx.x < kRows) bad[threadIdx.x] = 0;
    __syncthreads();
    float *part = w.part + ((size_t)wg * 2 + (off == 0)) * (kRows * (D + 2));
    if (r < nr) {
      if (!whole && h == 0) {
        part[r] = ref.value();
        part[kRows + r] = l;
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const f32x4 o = f32x4{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]} * un;
          const int d0 = 32 * d + 8 * x + 4 * h;
          if (whole)
            store_out<D>(a, s, head, row, d0, o, l, &bad[r]);
          else
            *reinterpret_cast<f32x4 *>(part + 2 * kRows + r * D + d0) = o;
        }
    }
    if (whole) {
      __syncthreads();
      finish_rows<FMT, D, 4>(kv, b, a, s, Tile{seq, head, r0, nr}, bad);
    } else if (threadIdx.x == 0) {
      const int by = off == 0 ? wg : quotient(next - units + run.cost, run.share);  // its first group's
      w.desc[2 * wg + (off == 0)] = int4{seq, head, r0, (quotient(next - 1, run.share) - by + 1) << 16 | (wg - by)};
    }
    if (u < run.end) next_tile<kRows>(kv, b, a, w, run, s);
  }
}

// Joins the tiles of k_attn_tile whose units several workgroups had: one workgroup here for
// each of theirs takes every (parts)th row, so all have as much to read, whatever the parts.
// Bound by the round trips of its few loads: 5 us for 2039 tokens through a window, 17-18 us
// for a prompt of 4093 (512 tiles of two parts).  Four rows of a thread at once changed nothing.
// (With the rows of any tile over 8 workgroups, 16 tiles of 32 parts took 88 us, not 36;
// with 4 or 2 times as many workgroups, 46 and 39.)
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_attn_join(KvView kv, nx_kv_batch b, AttnCall a, AttnWork w) {
  __shared__ JoinLds<D, 4> lds;
  const int4 t = w.desc[blockIdx.x];
  if (t.w == 0) return;
  const int seq = uniform(t.x), r0 = uniform(t.z), parts = uniform(t.w) >> 16, y = uniform(t.w) & 0xffff;
  const KvSeq s = kv_seq(b, seq, kv.page_log2);
  const int nr = min(kRows, s.n * a.group - r0);
  if (y >= nr) return;
  const int lead = (blockIdx.x >> 1) - y;
  join_tile<FMT, D, 4, false>(kv, b, a, s, Tile{seq, uniform(t.y), r0, nr},
                              w.part + ((size_t)lead * 2 + 1) * (kRows * (D + 2)), kRows, parts, y, parts, lds);
}

// Workgroups of a call (a power of two, so that whole XCDs get equal shares), and
// the workspace of their parts: of one size for every cache, so that it is
// allocated once.
constexpr int kAttnWgsPerCu = 2;
// What a tile costs besides its groups (its query, its results), in groups; without it runs
// of many short tiles end last.
//   k_attn_split: three sequences of up to 131071 tokens (INT8) 120.1 us at 4, 118.4 at 12,
//   117.2 at 24; 61 of up to 8191 (F16) 226 at 4 and 12, 228.5 at 24
//   k_attn_tile: a prompt of 4093 tokens 333 us at 2, 310 at 6, 314 at 12
constexpr int kTileCost = 12, kRowsCost = 6;
// The fewest groups of a workgroup where a tile is split.
//   k_attn_split (two for each wave): two sequences of up to 14304 tokens 25.0 us at 4, 23.7 at
//   8, 19.6 at 16, 22.2 at 32
//   k_attn_tile: three chunks of 37 tokens, 32 heads over 4 of 128, at up to 2592 tokens 41.5 us
//   at 2 and 4, 47.0 at 10, 63.6 at 20
constexpr int kMinShare = 16, kMinRows = 4;
// What the join of a split tile costs, in groups: a tile that ends no later is taken whole.
//   k_attn_split: one token after 516 11.6 us at 4, 10.0 at 16; 16 tokens and a chunk of 257
//   70.5 us at 16, 78.0 at 48
//   k_attn_tile: 709 tokens through a window of 13, 8 heads of 256, 49.1 us at 0, 38.7 at 8;
//   four prompts of 306 tokens 36.6 at 0, 33.3 at 8; three of 564 35.1 at 8, 40.4 at 16
constexpr int kJoinCost = 16, kJoinRows = 8;
// The kernel of a sequence.  A 16-row tile has a workgroup (or several) and a wave a group of
// its own: least latency, but every tile reads the keys again; a 128-row tile reads them once
// for all, at full cost whatever its rows.  So, in a step of many sequences, k_attn_tile
// takes those beyond two 16-row tiles (F16), or three (INT8, half the bytes); us for 64
// sequences of 1024 tokens, by k_attn_split and k_attn_tile:
//   rows of each                    24          40          56
//   F16,  32 heads over 4 of 128  47  47      66  49      84  52
//   INT8, 16 heads over 8 of 256 112 205     163 207     212 210
constexpr int tile_from(int fmt) { return kTile * (fmt == NX_KV_INT8 ? 3 : 2); }
// And all of a step goes to k_attn_split while it has a 16-row tile or less for each CU, and
// few scores: us for one chunk over 4 heads of 128,
//   rows                        1024          2048          4096              8192
//   tokens                    1024  16384   1024  16384   1024 4096 16384   1024 16384
//   F16,  k_attn_split          14     34     14     50     14   30    90     32   181
//         k_attn_tile           29     47     30     62     32   45    92     38   152
//   rows                        1024             2048             4096
//   tokens                    65536 131072     65536 131072     65536
//   INT8, k_attn_split          126    236       235    458       458
//         k_attn_tile            94    160       159    293       292
// Where the page table's width does not bound the scores so, both kernels are launched and
// sum up the lengths (1024 rows over 1024 tokens 19 us, not 14; 4096 18, not 32), but for the
// rows of an eighth of the CUs: 512 over 1024, 16384, 65536 and 131072 tokens take k_attn_split
// 14, 25, 60 and 113 us (INT8 16, 29, 75, 132) and k_attn_tile 25, 37, 64 and 100 (26, 39, 65, 99).
// (So those few rows lose 15 to 33% over INT8 contexts of 65536 tokens and more, and F16 ones of
// 131072 13%: the host knows the table's width, not the lengths, and a step behind a wide table
// that is short would pay some 5 us for the second kernel.)
constexpr long kFewScores = 40'000'000;  // rows times keys

static int attn_wgs_log2(const nx_ctx *c) { return std::max(4, 31 - __builtin_clz(c->num_cu * kAttnWgsPerCu)); }
static size_t part_floats(int tile, int D) { return (size_t)2 * tile * (D + 2); }
int attn_workspace(nx_ctx *c, void **out) {
  const size_t wgs = (size_t)1 << attn_wgs_log2(c);
  // (k_attn_tile runs half as many workgroups on heads of 256)
  const size_t wide = std::max(part_floats(kRows, 128), part_floats(kRows, 256) / 2);
  // (and a descriptor and a count of each)
  const size_t bytes = wgs * (2 * sizeof(int4) + sizeof(int) + 4 * (part_floats(kTile, 256) / 2 + wide));
  DevBuf &ws = c->ws[WS_ATTN];
  if (!ws.ptr) {  // of this size: it never grows
    NX_TRY(refuse_capture(c));
    void *p = nullptr;
    if (hipMalloc(&p, bytes) != hipSuccess) {
      (void)hipGetLastError();
      return fail(NX_ERR_OOM, "device allocation of " + std::to_string(bytes) + " bytes failed");
    }
    // counts begin at 0, and the workspace is there once they are: a call that finds others
    // would leave split tiles out
    if (hipMemsetAsync(static_cast<int4 *>(p) + 2 * wgs, 0, wgs * sizeof(int), c->stream) != hipSuccess ||
        hipStreamSynchronize(c->stream) != hipSuccess) {
      (void)hipGetLastError();
      (void)hipFree(p);
      return fail(NX_ERR_DEVICE, "clearing the attention's workspace failed");
    }
    ws = {p, bytes};
  }
  if (out) *out = ws.ptr;
  return NX_OK;
}

static int attention_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch &b, AttnCall a) {
  a.wide_q = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.q_stride % 4 == 0;
  a.wide_out = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && a.out_stride % 4 == 0;
  a.shift = group_shift(a.group);
  a.magic = group_magic(a.group);
  void *p;
  NX_TRY(attn_workspace(c, &p));
  // Which kernels the batch may need: only the device knows its sequences' rows.  With a row
  // or more in each, one has at most num_tokens - num_seqs + 1; a batch that leaves
  // sequences out for a long one is right on k_attn_split too, if slower.
  const int log2 = attn_wgs_log2(c), wgs = 1 << log2, from = tile_from(kv->fmt);
  const long rows = (long)b.num_tokens * a.heads, table = (long)b.max_pages * kv->page_tokens;
  const long keys = a.window > 0 ? std::min(table, (long)a.window + a.sinks + b.num_tokens) : table;
  const bool one_each = rows <= kTile * wgs / 2, few = one_each && (rows * keys <= kFewScores || rows <= kTile * wgs / 16);
  const bool wide = ((long)b.num_tokens - b.num_seqs + 1) * a.group > from && !few;
  const bool ask = wide && one_each && b.num_seqs <= 64;
  const bool narrow = !wide || ask || b.num_seqs > 1;
  int4 *desc = static_cast<int4 *>(p);
  int *done = reinterpret_cast<int *>(desc + 2 * wgs);
  float *part = reinterpret_cast<float *>(done + wgs);
  // (k_attn_split: one workgroup per CU)
  const AttnWork w0{nullptr, done, part, log2 - 1, kMinShare, kTileCost, kJoinCost, 0, wide ? from : INT32_MAX,
                    ask ? kFewScores : 0};
  const AttnWork w1{desc, nullptr, part + wgs / 2 * part_floats(kTile, 256), kv->D == 256 ? log2 - 1 : log2,
                    kMinRows, kRowsCost, kJoinRows, narrow ? from : 0, INT32_MAX, w0.few};
  const int wgs1 = 1 << w1.wgs_log2;
  const KvView view = view_of(kv);
  if (wide)
    NX_TRY(launch(c, "attn_tile", [&] {
      with_kernel(kv, [&](auto fmt, auto D) {
        go(c, k_attn_tile<fmt(), D()>, dim3(wgs1), dim3(256), 0, view, b, a, w1);
      });
    }));
  if (narrow)
    NX_TRY(launch(c, "attn_split", [&] {
      with_kernel(kv, [&](auto fmt, auto D) {
        go(c, k_attn_split<fmt(), D()>, dim3(wgs / 2), dim3(64 * kDecodeWaves<D()>), 0, view, b, a, w0);
      });
    }));
  if (!wide) return NX_OK;
  return launch(c, "attn_join", [&] {
    with_kernel(kv, [&](auto fmt, auto D) {
      go(c, k_attn_join<fmt(), D()>, dim3(2 * wgs1), dim3(256), 0, view, b, a, w1);
    });
  });
}

static int attention(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, const float *q,
                     size_t q_stride, int heads, float scale, int window, int sinks, float *out,
                     size_t out_stride, bool host) {
  NX_TRY(kv_check_call(c, kv, b));
  NX_TRY(refuse(attn_check(heads, kv->heads, scale, window, sinks)));
  if (b->num_seqs == 0 || b->num_tokens == 0) return NX_OK;
  if (!q || !out) return fail(NX_ERR_INVALID_ARG, "null buffer");
  if ((int64_t)b->num_tokens * heads > INT32_MAX)
    return fail(NX_ERR_UNSUPPORTED, "more than 2^31 query rows");
  const size_t width = (size_t)heads * kv->D;
  if (q_stride > (size_t)1 << 40 || out_stride > (size_t)1 << 40)
    return fail(NX_ERR_UNSUPPORTED, "row stride above 2^40");
  NX_TRY(refuse(kv_check_rows("query", (long)q_stride, (long)width)));
  NX_TRY(refuse(kv_check_rows("output", (long)out_stride, (long)width)));
  AttnCall a{q, out, q_stride, out_stride, heads, heads / kv->heads, scale, window, sinks, false, false, 0, 0};
  if (!host) return attention_dev(c, kv, *b, a);
  NX_TRY(refuse(kv_check_tables(*b, kv->pages, kv->page_tokens, true, false, window, sinks)));
  const size_t r0 = b->row_start[0], rows = b->row_start[b->num_seqs];
  if (rows == r0) return NX_OK;
  nx_kv_batch dev;
  NX_TRY(kv_upload_batch(c, *b, &dev));
  void *dq, *dout;
  NX_TRY(ws_get(c, WS_XIN, rows * width * 4, &dq));
  NX_TRY(ws_get(c, WS_OUT, rows * width * 4, &dout));
  const size_t line = width * 4;
  NX_HIP(hipMemcpy2DAsync(dq, line, q, q_stride * 4, line, rows, hipMemcpyHostToDevice, c->stream));
  a.q = static_cast<const float *>(dq);
  a.out = static_cast<float *>(dout);
  a.q_stride = a.out_stride = width;
  NX_TRY(attention_dev(c, kv, dev, a));
  NX_HIP(hipMemcpy2DAsync(out + r0 * out_stride, out_stride * 4, a.out + r0 * width, line, line,
                          rows - r0, hipMemcpyDeviceToHost, c->stream));
  NX_HIP(hipStreamSynchronize(c->stream));
  return NX_OK;
}

}  // namespace nx

using namespace nx;

extern "C" {

int nx_attention(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, const float *q, size_t q_stride,
                 int heads, float scale, int window, int sinks, float *out, size_t out_stride) {
  return guarded([&] {
    return attention(c, kv, b, q, q_stride, heads, scale, window, sinks, out, out_stride, true);
  });
}
int nx_attention_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, const float *q,
                     size_t q_stride, int heads, float scale, int window, int sinks, float *out,
                     size_t out_stride) {
  return guarded([&] {
    return attention(c, kv, b, q, q_stride, heads, scale, window, sinks, out, out_stride, false);
  });
}

}  // extern "C"
