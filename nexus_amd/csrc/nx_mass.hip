// nx_mass.hip — the weight that a step's queries give each cached token:
//
//   mass_j = before_j + sum_i p_ij,   p_ij = 2^(x_ij - e_i),   x_ij = log2(e) scale q_i . k_j,
//   e_i = m_i + log2 sum_j 2^(x_ij - m_i)
//
// over the rows i (of a token and a head that shares the key/value head) that see token j.  e_i
// takes all keys of a row, so the keys are gone through twice:
//
// Few rows (k_mass_scores, k_mass_add): the scores of 16 rows against a chunk of the keys are
// stored beside the chunk's maximum and sum, and read back once all chunks are there: less
// memory than the keys again.
// Many rows (k_mass_stats, k_mass_columns): the scores are worked out twice.  First 128 rows are
// held against the keys that stream by, for e_i; then keys are held against the rows that stream
// by, so a key's sum stays in its lanes.
//
// 32 heads over 8 of 128 in F16: one token of 61 sequences of up to 8191 155 us (667 MB), every token of a
// prompt of 4093 364 to 377 (69 GFLOP, four times that with two halves in two passes).  Cards differ by 5%:
// where two figures are compared below, both are of one card.
//
// The scores are nx_attn.hip's: transposed products K Q^T on the f16 matrix cores, q as two
// halves.  A score is one key's and one row's alone, so nothing that is masked reaches another.
#include <hip/hip_runtime.h>

#include "nx_attn_dev.hpp"
#include "nx_step_plan.hpp"

namespace nx {

struct MassCall {
  const float *q, *before;
  float *mass;
  size_t q_stride, mass_stride;
  int heads, group;  // query heads, and those that share a key/value head
  float scale;     // times log2(e)
  bool wide_q;     // rows of whole float4 runs
  uint32_t magic;  // by_group's
  int shift;
  int rows_above, rows_upto;  // the kernels' sequences: those of so many rows
};

// a row's maximum before its first score, which any may pass; less than this is only -infinity's stand-in
constexpr float kUnsetMax = -0x1.fffffcp127f;

__device__ __forceinline__ int rows_of(const MassCall &a, const KvSeq &q) {
  const int rows = q.n * a.group;
  return q.len > 0 && rows > a.rows_above && rows <= a.rows_upto ? rows : 0;
}

// -infinity stands for tokens that a row does not see: a score of -infinity is the lowest number
__device__ __forceinline__ float seen_score(float x) { return x == -INFINITY ? -3.4028234663852886e38f : x; }

// What a row's scores are multiplied by, with q scale log2(e) scaled into [2^13, 2^14) (both halves
// keep their bits) by `up`: powers of two.  mx: the largest of |q scale log2(e)|.
struct RowScale {
  float up, c;
  template <bool I8>
  static __device__ __forceinline__ RowScale of(float mx) {
    const int X = mx < INFINITY ? max(__builtin_amdgcn_frexp_expf(mx), -112) : 0;
    return {ldexp1(1.f, 14 - X), ldexp1(1.f, X - 14 + (I8 ? 9 : 0))};
  }
};

// x by - less, the product rounded first
__device__ __forceinline__ float score_less(float x, float by, float less) {
#pragma clang fp contract(off)
  const float y = x * by;
  return y - less;
}

// log2 of a row's sum: above everything where it is nothing
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l); }

// the sum of two parts of a row
__device__ __forceinline__ float2 joined(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x);
  return {top, a.y * __builtin_amdgcn_exp2f(a.x - top) + b.y * __builtin_amdgcn_exp2f(b.x - top)};
}

__device__ __forceinline__ void add_to(const MassCall &a, const KvSeq &s, size_t tile, int j, float sum) {
  if ((size_t)j >= a.mass_stride) return;
  const size_t at = tile * a.mass_stride + j;
  a.mass[at] = (a.before && j < s.first ? a.before[at] : 0.f) + sum;
}

// Groups of 32 tokens of a sequence and head, looked up in two steps: a page number is on its way
// while the keys of the groups before it are, and nothing waits for it in between.
struct Groups {
  const KvView &kv;
  const int32_t *pages;
  int head, end;  // (behind the last one: the last)
  __device__ __forceinline__ int page(int i) const {
    int at = min(i, end - 1) * kKvGroup >> kv.page_log2;
    asm volatile("" : "+v"(at));  // (a number that is known to be alike would be waited for at once)
    return pages[at];
  }
  __device__ __forceinline__ bool there(int page) const { return page >= 0 && page < kv.pages; }
  // in the pool (group 0, masked, for one that is not there); page: uniform
  __device__ __forceinline__ long at(int i, int page) const {
    const int in_page = (min(i, end - 1) * kKvGroup & ((1 << kv.page_log2) - 1)) / kKvGroup;
    return there(page) ? (((long)page * kv.heads + head) << (kv.page_log2 - 5)) + in_page : 0;
  }
};
__device__ __forceinline__ KvSeq uniform(const KvSeq &s) {
  return {uniform(s.row), uniform(s.n), uniform(s.first), uniform(s.len)};
}

// ------------------------------------------------------------ scores by the formula alone
// A query's halves may have signs of their own, or be 0 where the query is not: the products with an
// infinite key then add up to a NaN where the score is an infinity.  (An infinity that they do add up to is the
// score.)  So where a row's or a token's sum ends as a NaN, the scores that are NaNs are worked out again from q and
// the keys as they are, in 64 bits.  The loops of the products stay as they are.
template <int FMT, int D>
__device__ __forceinline__ float score_of(const KvView &kv, long group, int t, const float *q, float scale) {
  using E = kv_elem<FMT>;
  typedef E Chunk __attribute__((ext_vector_type(8)));
  const Chunk *k = reinterpret_cast<const Chunk *>(reinterpret_cast<const E *>(kv.k) + group * (kKvGroup * D)) + kv_row(FMT, t);
  double sum = 0.;
#pragma unroll 1
  for (int c = 0; c < D / 8; ++c) {
    const Chunk x = k[c * kKvGroup];
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fma((double)q[8 * c + i] * scale, (double)(float)x[i], sum);
  }
  if constexpr (FMT == NX_KV_INT8) sum *= kv.ks[group * kKvGroup + t];
  return (float)sum;
}

// ------------------------------------------------------------ few rows
struct NarrowWork {
  MassNarrow m;
  int head0;      // the launch's first key/value head
  int groups;     // of the page table
  // of each sequence's rows, head and 16-row tile: [groups][the tile's rows][32] scores, and a
  // maximum and sum [the tile's rows][chunks]
  float *scores;
  float2 *stats;
};
// the first row of a tile, in rows of the whole batch (or 16 of each sequence)
__device__ __forceinline__ size_t slot_of(const MassCall &a, const NarrowWork &w, const KvSeq &s, int seq, int head, int r0) {
  if (w.m.one_each) return ((size_t)seq * w.m.heads + (head - w.head0)) * kMassRows;
  return ((size_t)s.row * w.m.heads + (size_t)(head - w.head0) * s.n) * a.group + r0;
}

// 16-row tiles of a sequence
__device__ __forceinline__ int row_tiles(const MassCall &a, const KvSeq &q) {
  return (rows_of(a, q) + kMassRows - 1) / kMassRows;
}

constexpr int kMassWaves = 4, kMassThreads = 64 * kMassWaves;

template <int FMT, int D>
__global__ __launch_bounds__(kMassThreads, D == 256 ? 1 : 2) void k_mass_scores(KvView kv, nx_kv_batch b, MassCall a,
                                                                              NarrowWork w) {
  using E = kv_elem<FMT>;
  constexpr bool I8 = FMT == NX_KV_INT8;
  constexpr int KS = D / 32, KL = I8 ? KS : 2 * KS;
  __shared__ long sums[kMassWaves];
  __shared__ Place found;
  __shared__ float2 part[kMassWaves][kMassRows];
  // (a chunk of all tiles after the other: late chunks, which few sequences have, on all XCDs)
  const int tile = blockIdx.x % w.m.tiles, chunk = blockIdx.x / w.m.tiles;
  const Place at = find_item<kMassWaves>(
      kv, b, tile, [&](const KvSeq &q) { return row_tiles(a, q) * w.m.heads; }, sums, &found);
  if (at.s < 0) return;
  const KvSeq s = uniform(at.seq);
  const int seq = uniform(at.s), in_seq = uniform(at.at), tiles = row_tiles(a, s);
  const int head = w.head0 + in_seq / tiles, r0 = in_seq % tiles * kMassRows;
  if (head >= kv.heads) return;  // (the last heads may be fewer)
  const int nr = min(kMassRows, rows_of(a, s) - r0);
  const int begin = chunk * w.m.share, end = min(begin + w.m.share, (s.len + kKvGroup - 1) / kKvGroup);
  if (begin >= end) return;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), n = lane & 15, g = lane >> 4;

  uint4 kf[KL];
  f32x4 dk[2];  // INT8: scales of the lane's tokens
  const Groups groups{kv, b.pages + (long)seq * b.max_pages, head, end};
  // read once, past the scores in the L2 (142 us otherwise, not 138, and 21 for k_mass_add, not 18)
  auto once = [](const E *p) { return ld_stream16(reinterpret_cast<const uint8_t *>(p)); };
  auto load_k = [&](long gr) {
    const E *base = reinterpret_cast<const E *>(kv.k) + gr * (kKvGroup * D);
    if constexpr (I8) {
      const f32x4 *p = reinterpret_cast<const f32x4 *>(kv.ks + gr * kKvGroup + 8 * g);
      dk[0] = p[0];
      dk[1] = p[1];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        kf[ks] = once(base + ((4 * ks + g) * kKvGroup + 2 * n) * 8);
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          kf[2 * ks + h] = once(base + ((4 * ks + g) * kKvGroup + 16 * (n >> 3) + 8 * h + (n & 7)) * 8);
    }
  };
  int page = groups.page(begin + wave), page1 = groups.page(begin + wave + kMassWaves);
  page = uniform(page);
  load_k(groups.at(begin + wave, page));

  // this lane's query (rows behind the tile's last repeat it)
  const int row = r0 + min(n, nr - 1), tok = by_group(row, a.magic, a.shift);
  const float *q = a.q + (size_t)(s.row + tok) * a.q_stride + (size_t)(head * a.group + row - tok * a.group) * D + 8 * g;
  const int p = s.first + tok;
  const float one = opaque_one();
  f16x8 qh[KS], ql[KS];
  float c;
  {
    float x[KS][8], mx = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      load8(q + 32 * ks, a.wide_q, x[ks]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[ks][i] *= a.scale;
        mx = fmaxf(mx, fabsf(x[ks][i]));
      }
    }
    const RowScale by = RowScale::of<I8>(max_groups(mx));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[ks][i] *= by.up;
      split2(x[ks], one, qh[ks], ql[ks]);
    }
    c = by.c;
  }
  const size_t slot = slot_of(a, w, s, seq, head, r0);
  // Lanes without a row store out of range, where nothing is written: a branch around the stores would
  // make every wait for keys one for the stores before them as well.  (At most 2^28 bytes: kMassFloats.)
  const __amdgpu_buffer_rsrc_t scores =
      make_rsrc(w.scores + slot * ((size_t)w.groups * kKvGroup), (uint32_t)nr * w.groups * kKvGroup * 4);
  const uint32_t mine = n < nr ? (uint32_t)(n * kKvGroup + 8 * g) * 4 : 0x80000000u;
  float m = kUnsetMax, l = 0.f;
  for (int i = begin + wave; i < end; i += kMassWaves) {
    const int first = i * kKvGroup;
    const bool there = groups.there(page);
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
    float x[8], most = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float k = I8 ? dk[j >> 2][j & 3] * c : c;
      // token first + 8 g + j
      x[j] = there && first + 8 * g + j <= p ? seen_score(sc[j >> 2][j & 3] * k) : -INFINITY;
      most = fmaxf(most, x[j]);
    }
    page = uniform(page1);
    load_k(groups.at(i + kMassWaves, page));
    page1 = groups.page(i + 2 * kMassWaves);
    l *= __builtin_amdgcn_exp2f(m - most);
    m = most;
#pragma unroll
    for (int j = 0; j < 8; ++j) l += __builtin_amdgcn_exp2f(x[j] - m);
#pragma unroll
    for (int j = 0; j < 8; j += 4)
      __builtin_amdgcn_raw_buffer_store_b128(
          __builtin_bit_cast(u32x4_t, f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]}), scores,
          (int)(mine + (uint32_t)first * nr * 4 + 4 * j), 0, 0);
  }
  float all = max_groups(m);
  l = sum_groups(l * __builtin_amdgcn_exp2f(m - all));
  uint32_t odd = (uint32_t)__ballot(lane < nr && l != l);
  if (odd) stores_done();  // of the same scores, by other lanes
  for (; odd; odd &= odd - 1) {  // the wave's scores of a row, two groups at once
    const int r = __builtin_ctz(odd), now = by_group(r0 + r, a.magic, a.shift);
    const float *qr = a.q + (size_t)(s.row + now) * a.q_stride + (size_t)(head * a.group + r0 + r - now * a.group) * D;
    float *to = w.scores + slot * ((size_t)w.groups * kKvGroup);
    const int t = lane & (kKvGroup - 1);
    float2 o = {kUnsetMax, 0.f};
#pragma unroll 1
    for (int i0 = begin + wave; i0 < end; i0 += 2 * kMassWaves) {
      const int i = i0 + lane / kKvGroup * kMassWaves, at = i * kKvGroup + t;
      const long group = i < end && at <= s.first + now && at < s.len ? kv_group(kv, b, seq, head, i * kKvGroup) : -1;
      const float x = group >= 0 ? seen_score(score_of<FMT, D>(kv, group, t, qr, a.scale)) : -INFINITY;
      if (i < end) to[((size_t)i * nr + r) * kKvGroup + t] = x;
      const float most = fmaxf(o.x, x);
      o = {most, o.y * __builtin_amdgcn_exp2f(o.x - most) + __builtin_amdgcn_exp2f(x - most)};
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) o = joined(o, float2{__shfl_xor(o.x, d, 64), __shfl_xor(o.y, d, 64)});
    if (n == r) {
      all = o.x;
      l = o.y;
    }
  }
  if (g == 0) part[wave][n] = float2{all, l};
  __syncthreads();
  if ((int)threadIdx.x < nr) {
    float2 o = part[0][threadIdx.x];
#pragma unroll
    for (int v = 1; v < kMassWaves; ++v) o = joined(o, part[v][threadIdx.x]);
    w.stats[(slot + threadIdx.x) * w.m.chunks + chunk] = o;
  }
}

// Some of the tokens of a sequence and head: their weights, summed over its rows.  Every workgroup joins all
// chunks' maxima and sums by itself, with several loads of each thread on their way (a load at a time, 16
// threads a row, 128 tokens a workgroup: 52 us for 100001 tokens of one INT8 sequence, not 8).
__global__ __launch_bounds__(kMassThreads) void k_mass_add(KvView kv, nx_kv_batch b, MassCall a, NarrowWork w) {
  __shared__ float2 part[kMassWaves][kMassRows];
  __shared__ float e[kMassRows];
  const int units = b.num_seqs * w.m.heads, unit = blockIdx.x % units, chunk = blockIdx.x / units;
  const int seq = unit / w.m.heads, head = w.head0 + unit % w.m.heads;
  if (head >= kv.heads) return;
  const KvSeq s = kv_seq(b, seq, kv.page_log2);
  const int tiles = row_tiles(a, s), begin = chunk * w.m.add_share * kKvGroup;
  const int end = min(begin + w.m.add_share * kKvGroup, s.len), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (tiles == 0 || begin >= end) return;
  const int parts = (s.len + w.m.share * kKvGroup - 1) / (w.m.share * kKvGroup);
  constexpr int kTokens = 64 * kKvGroup / kMassThreads, kAtOnce = 4;
  float sum[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) sum[i] = 0.f;
  for (int t = 0; t < tiles; ++t) {
    // the tile's rows, a power of two of them, for as many threads each as there are
    const int nr = min(kMassRows, rows_of(a, s) - t * kMassRows), log2r = nr > 1 ? 32 - __builtin_clz(nr - 1) : 0;
    const int r = threadIdx.x & ((1 << log2r) - 1), subs = kMassThreads >> log2r;
    float2 o = {kUnsetMax, 0.f};
    const size_t slot = slot_of(a, w, s, seq, head, t * kMassRows);
    const float2 *stats = w.stats + (slot + min(r, nr - 1)) * w.m.chunks;
    for (int i = threadIdx.x >> log2r; i < parts; i += kAtOnce * subs) {
      float2 x[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) x[u] = stats[min(i + u * subs, parts - 1)];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (i + u * subs < parts) o = joined(o, x[u]);
    }
    for (int d = 1 << log2r; d < 64; d <<= 1) o = joined(o, float2{__shfl_xor(o.x, d, 64), __shfl_xor(o.y, d, 64)});
    if (lane == r) part[wave][r] = o;
    __syncthreads();
    if ((int)threadIdx.x < nr) {
      o = part[0][r];
#pragma unroll
      for (int i = 1; i < kMassWaves; ++i) o = joined(o, part[i][r]);
      e[r] = log_sum(o.x, o.y);
    }
    __syncthreads();
    const float *scores = w.scores + slot * ((size_t)w.groups * kKvGroup);
    for (int i = 0; i < nr; ++i) {
      const float ei = e[i];
#pragma unroll
      for (int u = 0; u < kTokens; ++u) {
        const int j = begin + (int)threadIdx.x + u * kMassThreads;
        const float x = j < end ? scores[((size_t)(j / kKvGroup) * nr + i) * kKvGroup + j % kKvGroup] : -INFINITY;
        sum[u] += x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(x - ei);
      }
    }
    __syncthreads();  // e and part are read
  }
#pragma unroll
  for (int u = 0; u < kTokens; ++u) {
    const int j = begin + (int)threadIdx.x + u * kMassThreads;
    if (j < end) add_to(a, s, (size_t)seq * kv.heads + head, j, sum[u]);
  }
}

// ------------------------------------------------------------ many rows
struct WideWork {
  MassWide m;
  int first;       // rows [first, first + m.rows) of the call: as many as the halves have room for
  int *next;       // units that k_mass_stats and k_mass_columns have given out besides a grid's; each clears the other's
  bool stats_once, columns_once;  // no more units than workgroups
  int groups;      // of the page table
  float *e, *coef;  // [rows x heads]: e_i, and what the products with the halves are multiplied by
  _Float16 *halves;  // [rows x heads][2][D] the queries as k_mass_stats splits them
  float *part;     // k_mass_stats: [rows x heads][key_parts] {maximum, sum}; k_mass_columns: [tiles][row_parts][tokens]
};

// The arguments of a kernel as it has them in memory, for what is hardly ever done: kept in registers for that they
// took others' (k_mass_columns 198 us for a prompt of 4093, not 191).
struct WideArgs {
  KvView kv;
  nx_kv_batch b;
  MassCall a;
  WideWork w;
};
__device__ __forceinline__ const WideArgs &arguments() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const WideArgs *)p;
}

// a sequence's part in the launch's rows, where it is these kernels' at all
__device__ __forceinline__ KvSeq part_of(const MassCall &a, const WideWork &w, const KvSeq &q) {
  const int r0 = max(q.row, w.first), r1 = rows_of(a, q) > 0 ? min(q.row + q.n, w.first + w.m.rows) : 0;
  return {r0, max(r1 - r0, 0), q.first + (r0 - q.row), q.len};
}
// where the launch has the rows of a sequence and head, one behind the other
__device__ __forceinline__ size_t stat_of(const MassCall &a, const WideWork &w, const KvSeq &s, int head) {
  return (size_t)(s.row - w.first) * a.heads + (size_t)head * s.n * a.group;
}
// adds a launch's sum to what the token has: in the sequence's first one, what it had before the call
__device__ __forceinline__ void add_more(const MassCall &a, const KvSeq &all, const KvSeq &s, size_t tile, int j, float sum) {
  if (s.row == all.row)
    add_to(a, all, tile, j, sum);
  else if ((size_t)j < a.mass_stride)
    a.mass[tile * a.mass_stride + j] += sum;
}

// the first block of rows that sees a tile of keys
__device__ __forceinline__ int first_block(const MassCall &a, const KvSeq &s, int token) {
  return (int)((long)max(token - s.first, 0) * a.group / kMassBlock);
}

// A sequence's units of k_mass_stats: for each share of the keys the tiles of rows that see any of
// it (of the first share all tiles), those that see most first, so that the last units are short: 170 us
// for a prompt of 4093, 178 with the others as units that end at once.  Where each workgroup has a
// unit or none, the others do no harm, and are not counted out (three prompts of 300
// behind 400 on 16 heads of 64: 41 us, not 50).
struct KeyUnits {
  int tiles, whole;  // of rows; shares that all of them see
  int first, len, group, tokens;
  __device__ __forceinline__ KeyUnits(const MassCall &a, const WideWork &w, const KvSeq &s)
      : tiles((s.n * a.group + kMassTile - 1) / kMassTile), first(s.first), len(s.len), group(a.group),
        tokens(w.m.key_share * kKvGroup) {
    whole = w.stats_once ? w.m.key_parts : min(max(min(first, len - 1), 0) / tokens + 1, w.m.key_parts);
  }
  // tiles that see a share from `whole` on
  __device__ __forceinline__ int of(int share) const {
    const long token = (long)share * tokens;
    return token < len ? (int)max(tiles - (token - first) * group / kMassTile, 0L) : 0;
  }
  __device__ __forceinline__ int all() const {
    int n = whole * tiles;
    for (int c = whole, k; tiles > 0 && (k = of(c)) > 0; ++c) n += k;
    return n;
  }
  __device__ __forceinline__ void find(int i, int &tile, int &share) const {
    int k = tiles;
    share = min(i / tiles, whole);
    i -= share * tiles;
    if (share == whole)
      for (k = of(share); k > 0 && i >= k; k = of(++share)) i -= k;
    tile = tiles - 1 - min(i, tiles - 1);
  }
};
// A sequence's units of k_mass_columns: for each part of the rows, the last one first, the tiles of keys that
// any of its rows see: 193 us for that prompt, 211 with all.  (Where there is one part, all tiles: keys
// that no row sees have what they had.)
template <int TOKENS>
struct RowUnits {
  const MassCall &a;
  int parts, tiles, whole;  // parts whose rows see into every tile
  int first, share, blocks;
  __device__ __forceinline__ RowUnits(const MassCall &a, const WideWork &w, const KvSeq &s)
      : a(a), first(s.first), share(w.m.row_share) {
    blocks = (s.n * a.group + kMassBlock - 1) / kMassBlock;
    tiles = (s.len + TOKENS - 1) / TOKENS;
    parts = whole = min(blocks, 1);
    if (w.m.row_parts == 1) return;
    parts = (blocks + share - 1) / share;
    if (parts < 2) return;
    const int seen = w.columns_once ? 0 : first_block(a, s, (tiles - 1) * TOKENS);
    whole = seen < blocks ? parts - seen / share : 0;
  }
  // tiles that a part sees
  __device__ __forceinline__ int of(int part) const {
    const int last = first + by_group((int)(min((part + 1) * share, blocks) * (uint32_t)kMassBlock - 1), a.magic, a.shift);
    return last < 0 ? 0 : min(last / TOKENS + 1, tiles);
  }
  __device__ __forceinline__ int all() const {
    int n = whole * tiles;
    for (int p = parts - whole - 1; p >= 0; --p) n += of(p);
    return n;
  }
  __device__ __forceinline__ void find(int i, int &tile, int &part) const {
    part = 0;
    tile = i;
    if (parts == 1) return;
    const int before = min(i / tiles, whole);
    i -= before * tiles;
    part = parts - 1 - before;
    if (before == whole)
      for (int k; part > 0 && i >= (k = of(part)); --part) i -= k;
    tile = min(i, tiles - 1);
  }
};

// The units of a batch in the order in which workgroups are free: those of rows that see little
// are short, and how many there are the host does not know.  Where they are not more than workgroups,
// each has one, and as many workgroups are started: 768 that ask one counter wait for each other
// (40 tokens of 32 heads over 4 of 128 behind 260: 47 us, not 33).
struct Units {
  int *next, *lds, now, ahead, turn;
  bool once;
  __device__ __forceinline__ Units(int *next, int *done, int *lds, bool once)
      : next(next), lds(lds), now(blockIdx.x), ahead(0), turn(0), once(once) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0;
  }
  // takes the next but one while the next is worked on
  __device__ __forceinline__ void ask() {
    if (!once && threadIdx.x == 0) ahead = atomicAdd(next, 1) + (int)gridDim.x;
  }
  __device__ __forceinline__ void go_on() {
    if (once) {
      now = -1;
      return;
    }
    turn ^= 1;  // (a wave may still read the last turn's)
    if (threadIdx.x == 0) lds[turn] = ahead;
    __syncthreads();  // the last unit's reads of LDS
    now = uniform(lds[turn]);
  }
};

// 128 rows against a share of the keys: each row's maximum and sum.  As in k_attn_tile, the
// four waves take a step's keys from LDS, each for 32 rows; a lane holds 16 keys' scores of a row.
// (Each wave loading its operands itself, without LDS and barriers: 214 us where this took 182, for a prompt of
// 4093: the loads' 64 bytes a clock are what a CU's four matrix cores take in.)
template <int FMT, int D>
__global__ __launch_bounds__(kMassThreads, D == 256 ? 1 : 3) void k_mass_stats(KvView kv, nx_kv_batch b, MassCall a,
                                                                             WideWork w) {
  using E = kv_elem<FMT>;
  constexpr bool I8 = FMT == NX_KV_INT8;
  constexpr int KS = D / 16, GS = D == 256 || I8 ? 1 : 2;  // groups of a step (as registers allow)
  constexpr int C = kKvGroup * D * (int)sizeof(E) / 16;  // 16-byte chunks of a group's keys
  constexpr int L = (C + kMassThreads - 1) / kMassThreads;
  __shared__ f16x8 keys[2][GS][kKvGroup * D / 8];
  __shared__ float scales[2][GS][kKvGroup];
  __shared__ long sums[kMassWaves];
  __shared__ Place found;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  const float one = opaque_one();
  __shared__ int unit[2];
  for (Units units(w.next, w.next + 1, unit, w.stats_once); units.now >= 0; units.go_on()) {
    units.ask();
    const Place at = find_item<kMassWaves>(
        kv, b, units.now, [&](const KvSeq &q) { return KeyUnits(a, w, part_of(a, w, q)).all() * kv.heads; }, sums, &found);
    if (at.s < 0) return;
    const KvSeq s = part_of(a, w, uniform(at.seq));
    const int seq = uniform(at.s), in_seq = uniform(at.at), head = in_seq % kv.heads;
    int tile, chunk;
    KeyUnits(a, w, s).find(in_seq / kv.heads, tile, chunk);
    const int rows = s.n * a.group, r0 = tile * kMassTile, nr = min(kMassTile, rows - r0);
    const int row = r0 + min(32 * wave + n, nr - 1), tok = by_group(row, a.magic, a.shift), p = s.first + tok;
    const int pmin = uniform(s.first + by_group(r0 + min(32 * wave, nr - 1), a.magic, a.shift));
    const int pmax = uniform(s.first + by_group(r0 + min(32 * wave + 31, nr - 1), a.magic, a.shift));
    const int last = min(s.first + by_group(r0 + nr - 1, a.magic, a.shift), s.len - 1);
    const int seen = last < 0 ? 0 : last / kKvGroup + 1;
    const int begin = chunk * w.m.key_share, end = min(begin + w.m.key_share, seen);
    if (chunk == 0) {  // the shares that are not the tile's
      const int from = max((seen + w.m.key_share - 1) / w.m.key_share, 1), none = w.m.key_parts - from;
      float2 *part = reinterpret_cast<float2 *>(w.part) + (stat_of(a, w, s, head) + r0) * w.m.key_parts + from;
      for (int i = threadIdx.x; i < none * nr; i += kMassThreads)
        part[(size_t)(i / none) * w.m.key_parts + i % none] = float2{kUnsetMax, 0.f};
    }
    float m = kUnsetMax, l = 0.f;
    const bool mine = 32 * wave + n < nr;  // (rows behind the tile's last repeat it)
    if (begin < end) {
      f16x8 qh[KS], ql[KS];
      float c;
      {
        const float *q = a.q + (size_t)(s.row + tok) * a.q_stride +
                         (size_t)(head * a.group + row - tok * a.group) * D + 8 * h;
        float x[KS][8], mx = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          load8(q + 16 * ks, a.wide_q, x[ks]);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[ks][i] *= a.scale;
            mx = fmaxf(mx, fabsf(x[ks][i]));
          }
        }
        const RowScale by = RowScale::of<I8>(max_halves(mx));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[ks][i] *= by.up;
          split2(x[ks], one, qh[ks], ql[ks]);
        }
        c = by.c;
      }
      if (chunk == 0 && mine) {
        const size_t o = stat_of(a, w, s, head) + row;
        f16x8 *to = reinterpret_cast<f16x8 *>(w.halves + o * (2 * D)) + h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          to[2 * ks] = qh[ks];
          to[2 * ks + D / 8] = ql[ks];
        }
        if (h == 0) w.coef[o] = c;
      }
      // steps of GS groups on their way: registers, then LDS
      uint4 rk[GS][L];
      float rs = 0.f;
      const Groups groups{kv, b.pages + (long)seq * b.max_pages, head, end};
      int page[GS];
      bool there[GS], there1[GS] = {};
#pragma unroll
      for (int g = 0; g < GS; ++g) page[g] = groups.page(begin + g);
      auto fetch = [&](int i, bool (&found)[GS]) {
#pragma unroll
        for (int g = 0; g < GS; ++g) {
          const int now = uniform(page[g]);
          found[g] = i + g < end && groups.there(now);
          const long from = groups.at(i + g, now);
          page[g] = groups.page(i + GS + g);
          const uint4 *gk = reinterpret_cast<const uint4 *>(kv.k) + from * C;
#pragma unroll
          for (int j = 0; j < L; ++j) {
            const int x = threadIdx.x + kMassThreads * j;
            if (C % kMassThreads == 0 || x < C) rk[g][j] = gk[x];
          }
          if (I8 && (int)threadIdx.x / kKvGroup == g) rs = kv.ks[from * kKvGroup + threadIdx.x % kKvGroup];
        }
      };
      auto stage = [&](int buf) {
#pragma unroll
        for (int g = 0; g < GS; ++g)
#pragma unroll
          for (int j = 0; j < L; ++j) {
            const int x = threadIdx.x + kMassThreads * j;
            if (C % kMassThreads != 0 && x >= C) continue;
            if constexpr (I8) {
              // rows 2 y, 2 y + 1 of a key chunk: tokens t and t + 4
              const int d8 = x >> 4, t = kv_token(NX_KV_INT8, (x & 15) * 2);
              keys[buf][g][d8 * kKvGroup + kv_row(NX_KV_F16, t)] = from_codes(rk[g][j].x, rk[g][j].y);
              keys[buf][g][d8 * kKvGroup + kv_row(NX_KV_F16, t + 4)] = from_codes(rk[g][j].z, rk[g][j].w);
            } else {
              keys[buf][g][x] = __builtin_bit_cast(f16x8, rk[g][j]);
            }
          }
        if (I8 && threadIdx.x < GS * kKvGroup) scales[buf][threadIdx.x / kKvGroup][threadIdx.x % kKvGroup] = rs;
      };
      fetch(begin, there);
      stage(0);
      if (begin + GS < end) fetch(begin + GS, there1);
      for (int i = begin, buf = 0; i < end; i += GS, buf ^= 1) {
        __syncthreads();  // the step is in LDS, and no wave reads the one before any more
        bool here[GS];
#pragma unroll
        for (int g = 0; g < GS; ++g) {
          here[g] = there[g];
          there[g] = there1[g];
        }
        if (i + GS < end) {
          stage(buf ^ 1);
          if (i + 2 * GS < end) fetch(i + 2 * GS, there1);
        }
        if (i * kKvGroup > pmax) continue;  // nothing that the wave's rows see
        f32x16 sc[GS];
#pragma unroll
        for (int g = 0; g < GS; ++g)
#pragma unroll
          for (int j = 0; j < 16; ++j) sc[g][j] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          f16x8 kx[GS];
#pragma unroll
          for (int g = 0; g < GS; ++g) {
            kx[g] = keys[buf][g][(2 * ks + h) * kKvGroup + n];
            sc[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx[g], qh[ks], sc[g], 0, 0, 0);
          }
#pragma unroll
          for (int g = 0; g < GS; ++g) sc[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx[g], ql[ks], sc[g], 0, 0, 0);
        }
#pragma unroll
        for (int g = 0; g < GS; ++g) {
          const int first = (i + g) * kKvGroup;
          // score j: token first + 16 (j / 8) + 8 h + j % 8
          float x[16], most = -INFINITY;
#pragma unroll
          for (int j = 0; j < 16; ++j)
            x[j] = I8 ? sc[g][j] * (scales[buf][g][16 * (j >> 3) + 8 * h + (j & 7)] * c) : sc[g][j];
          if (!here[g] || first + kKvGroup - 1 > pmin) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (!here[g] || 16 * (j >> 3) + (j & 7) > p - first - 8 * h) x[j] = -INFINITY;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) most = fmaxf(most, x[j]);
          most = fmaxf(m, I8 ? most : most * c);
          l *= __builtin_amdgcn_exp2f(m - most);
          m = most;
          float more[2] = {0.f, 0.f};
#pragma unroll
          for (int j = 0; j < 16; ++j) more[j & 1] += __builtin_amdgcn_exp2f(I8 ? score_less(x[j], 1.f, m) : fmaf(x[j], c, -m));
          l += more[0] + more[1];
        }
      }
      // Once more, with the scores that are NaNs by the formula.  The others are those of k_mass_columns to the last
      // bit, as the whole row's would not be: far from 0 that is a factor of any size.
      if (__any(mine && l != l)) {
        const WideArgs &in = arguments();
        const float *q = in.a.q + (size_t)(s.row + tok) * in.a.q_stride + (size_t)(head * in.a.group + row - tok * in.a.group) * D;
        m = kUnsetMax;
        l = 0.f;
#pragma unroll 1
        for (int i = chunk * in.w.m.key_share; i < end; ++i) {
          const int page = uniform(groups.page(i));
          if (!groups.there(page)) continue;
          const long group = groups.at(i, page);
          const E *base = reinterpret_cast<const E *>(in.kv.k) + group * (kKvGroup * D) + (h * kKvGroup + n) * 8;
          f32x16 sc;
#pragma unroll
          for (int j = 0; j < 16; ++j) sc[j] = 0.f;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            f16x8 kx;
            if constexpr (I8) {
              const uint2 x = *reinterpret_cast<const uint2 *>(base + 2 * ks * kKvGroup * 8);
              kx = from_codes(x.x, x.y);
            } else {
              kx = *reinterpret_cast<const f16x8 *>(base + 2 * ks * kKvGroup * 8);
            }
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx, qh[ks], sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx, ql[ks], sc, 0, 0, 0);
          }
#pragma unroll 1
          for (int j = 0; j < 16; ++j) {
            const int t = kv_token(FMT, 8 * (j >> 2) + 4 * h + (j & 3));
            float x = sc[0] * (I8 ? in.kv.ks[group * kKvGroup + t] * c : c);
#pragma unroll
            for (int next = 1; next < 16; ++next) sc[next - 1] = sc[next];
            if (i * kKvGroup + t > p) continue;
            if (x != x && l == l) x = score_of<FMT, D>(in.kv, group, t, q, in.a.scale);
            const float most = fmaxf(m, x);
            l = l * __builtin_amdgcn_exp2f(m - most) + __builtin_amdgcn_exp2f(score_less(x, 1.f, most));
            m = most;
          }
        }
      }
    }
    const float all = max_halves(m);
    l = across_halves(l * __builtin_amdgcn_exp2f(m - all), [](float x, float y) { return x + y; });
    if (h == 0 && mine) {
      const size_t o = stat_of(a, w, s, head) + row;
      if (w.m.key_parts == 1)
        w.e[o] = log_sum(all, l);
      else
        reinterpret_cast<float2 *>(w.part)[o * w.m.key_parts + chunk] = float2{all, l};
    }
  }
}

// e of each row, from its parts: 16 lanes take them
__global__ __launch_bounds__(kMassThreads) void k_mass_join(MassCall a, WideWork w, int rows) {
  const int r = blockIdx.x * (kMassThreads / 16) + threadIdx.x / 16, lane = threadIdx.x & 15;
  if (r >= rows) return;
  const float2 *p = reinterpret_cast<const float2 *>(w.part) + (size_t)r * w.m.key_parts;
  float2 o = {kUnsetMax, 0.f};
  for (int i = lane; i < w.m.key_parts; i += 16) o = joined(o, p[i]);
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) o = joined(o, float2{__shfl_xor(o.x, d, 16), __shfl_xor(o.y, d, 16)});
  if (lane == 0) w.e[r] = log_sum(o.x, o.y);
}

// groups of keys that a wave holds
template <int D>
constexpr int kHeldGroups = D == 256 ? 1 : 2;
template <int D>
constexpr int kKeyTile = kMassWaves * kHeldGroups<D>;  // of a workgroup

// In a 32-row tile's accumulator, register j of half h is row 8 (j / 4) + 4 h + j % 4: the token
// kv_token of h = 0, and so many behind it
template <int FMT>
constexpr int kTokenOfHalf = kv_token(FMT, 4);

// the weight that rows [from, to) give a token, in all lanes: NaN where any that sees it has no log sum
template <int FMT, int D>
__device__ __forceinline__ float column_by_formula(const WideArgs &all, const KvSeq &s, int seq, int head, int token,
                                                 int from, int to) {
  const KvView kv = all.kv;
  const nx_kv_batch b = all.b;
  const MassCall a = all.a;
  const WideWork w = all.w;
  const int lane = threadIdx.x & 63;
  const float *e = w.e + stat_of(a, w, s, head);
  from = max(from, max(token - s.first, 0) * a.group);
  for (int r = from + lane; r - lane < to; r += 64)
    if (__any(r < to && e[min(r, to - 1)] != e[min(r, to - 1)])) return NAN;
  const long group = kv_group(kv, b, seq, head, token & ~(kKvGroup - 1));
  float sum = 0.f;
#pragma unroll 1
  for (int r = from + lane; r < to; r += 64) {
    const int now = by_group(r, a.magic, a.shift);
    const float *q = a.q + (size_t)(s.row + now) * a.q_stride + (size_t)(head * a.group + r - now * a.group) * D;
    sum += __builtin_amdgcn_exp2f(score_of<FMT, D>(kv, group, token & (kKvGroup - 1), q, a.scale) - e[r]);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
  return sum;
}

// A tile of keys against a share of the rows: each wave holds its groups' keys in registers, and
// blocks of 32 rows go by in LDS, as two halves in operand order.  Score j of a lane is a key's,
// and the lane's column a row's: sums over rows stay in the lane until the end.
template <int FMT, int D>
__global__ __launch_bounds__(kMassThreads, D == 256 ? 1 : 2) void k_mass_columns(KvView kv, nx_kv_batch b, MassCall a,
                                                                               WideWork w) {
  using E = kv_elem<FMT>;
  constexpr bool I8 = FMT == NX_KV_INT8;
  constexpr int KS = D / 16, KG = kHeldGroups<D>, C8 = D / 8, Q = 2 * C8 * kMassBlock / kMassThreads;
  __shared__ f16x8 query[2][2][C8 * kMassBlock];  // [buffer][half]
  __shared__ float coef[2][kMassBlock], lse[2][kMassBlock];
  __shared__ int token[2][kMassBlock];
  __shared__ __align__(16) float scales[kMassWaves][KG][2][16];  // INT8: of the keys, as lanes hold their scores
  __shared__ long sums[kMassWaves];
  __shared__ Place found;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), n = lane & 31, h = lane >> 5;
  constexpr int kTokens = kKeyTile<D> * kKvGroup;
  __shared__ int unit[2];
  for (Units units(w.next + 1, w.next, unit, w.columns_once); units.now >= 0; units.go_on()) {
    units.ask();
    const Place at = find_item<kMassWaves>(
        kv, b, units.now, [&](const KvSeq &q) { return RowUnits<kTokens>(a, w, part_of(a, w, q)).all() * kv.heads; }, sums,
        &found);
    if (at.s < 0) return;
    const KvSeq all = uniform(at.seq), s = part_of(a, w, all);
    const int seq = uniform(at.s), in_seq = uniform(at.at), head = in_seq % kv.heads, rows = s.n * a.group;
    const RowUnits<kTokens> of(a, w, s);
    const int parts = of.parts;
    int kt, part;
    of.find(in_seq / kv.heads, kt, part);
    const int k0 = kt * kTokens;
    const int from = max(part * w.m.row_share, first_block(a, s, k0));
    const int to = min((part + 1) * w.m.row_share, (rows + kMassBlock - 1) / kMassBlock);
    const size_t tile = (size_t)seq * kv.heads + head;
    if (from >= to) {  // no row sees the keys: but in a sequence's first launch they have what they had
      const int j = k0 + (int)threadIdx.x;
      if (parts == 1 && s.row == all.row && j < min(k0 + kKeyTile<D> * kKvGroup, s.len)) add_to(a, all, tile, j, 0.f);
      continue;
    }

    // ---- the wave's keys: row n of a group in the cache's order
    f16x8 kx[KG][KS];
    bool there[KG];
    float scale[KG];
#pragma unroll
    for (int i = 0; i < KG; ++i) {
      const int first = k0 + (wave * KG + i) * kKvGroup;
      const long gr = first < s.len ? kv_group(kv, b, seq, head, first) : -1;
      there[i] = gr >= 0;
      const E *base = reinterpret_cast<const E *>(kv.k) + max(gr, 0L) * (kKvGroup * D) + (h * kKvGroup + n) * 8;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        if constexpr (I8) {
          const uint2 x = *reinterpret_cast<const uint2 *>(base + 2 * j * kKvGroup * 8);
          kx[i][j] = from_codes(x.x, x.y);
        } else {
          kx[i][j] = *reinterpret_cast<const f16x8 *>(base + 2 * j * kKvGroup * 8);
        }
      }
      if constexpr (I8) scale[i] = kv.ks[max(gr, 0L) * kKvGroup + kv_token(FMT, 8 * (n >> 2 & 3) + 4 * h + (n & 3))];
    }
    // INT8: a score is rounded times its key's scale, and the row's c and e follow in one step: c is a power of two,
    // so that is the score as k_mass_stats rounds it, times scale and c at once.  (Rounded with e taken off,
    // scores of 2^24 and more would be a factor of any size off.)  Scales that could pass f32's range so are held lower.
    float lift = 1.f;
    if constexpr (I8) {
      bool large = false;
#pragma unroll
      for (int i = 0; i < KG; ++i) large = large || scale[i] >= 0x1p100f;
      if (__any(large)) lift = 0x1p30f;
#pragma unroll
      for (int i = 0; i < KG; ++i)
        if (n < 16) scales[wave][i][h][n] = scale[i] * (1.f / lift);
    }
    float sum[KG][16];
#pragma unroll
    for (int i = 0; i < KG; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[i][j] = 0.f;

    // ---- blocks of rows on their way: 16-byte chunks of a row's halves by neighbouring threads.  A
    // row's place turns with the chunk, so that the 16 lanes that write at once hit all banks.
    auto slot = [](int c8, int row) { return c8 * kMassBlock + (row ^ 2 * (c8 & 7)); };
    f16x8 x[Q];
    float e = 0.f, c_next = 0.f;
    const size_t row0 = stat_of(a, w, s, head);
    const f16x8 *halves = reinterpret_cast<const f16x8 *>(w.halves + row0 * (2 * D));
    auto fetch = [&](int block) {
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        const int at = threadIdx.x + kMassThreads * i, r = at / (2 * C8), c8 = at - r * (2 * C8);
        x[i] = halves[(size_t)min(block * kMassBlock + r, rows - 1) * (2 * C8) + c8];
      }
      if (threadIdx.x < kMassBlock) {
        const int row = min(block * kMassBlock + (int)threadIdx.x, rows - 1);
        e = w.e[row0 + row];
        c_next = w.coef[row0 + row];
      }
    };
    auto stage = [&](int block, int buf) {
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        const int at = threadIdx.x + kMassThreads * i, r = at / (2 * C8), c8 = at - r * (2 * C8);
        query[buf][c8 / C8][slot(c8 % C8, r)] = x[i];
      }
      if (threadIdx.x < kMassBlock) {
        const int row = block * kMassBlock + (int)threadIdx.x;
        coef[buf][threadIdx.x] = c_next;
        lse[buf][threadIdx.x] = e;
        // (rows behind the last see nothing)
        token[buf][threadIdx.x] = row < rows ? s.first + by_group(row, a.magic, a.shift) : -1;
      }
    };
    fetch(from);
    stage(from, from & 1);
    if (from + 1 < to) fetch(from + 1);
    for (int block = from; block < to; ++block) {
      const int buf = block & 1;
      __syncthreads();  // the block is in LDS, and no wave reads the one before any more
      if (block + 1 < to) {
        stage(block + 1, buf ^ 1);
        if (block + 2 < to) fetch(block + 2);
      }
      const float c = coef[buf][n] * lift, ei = lse[buf][n];
      const int p = token[buf][n];
      const int pmin = uniform(block * kMassBlock + kMassBlock <= rows ? token[buf][0] : -1);
      const int pmax = s.first + by_group(min(block * kMassBlock + kMassBlock, rows) - 1, a.magic, a.shift);
      const int first = k0 + wave * KG * kKvGroup;
      if (first > pmax) continue;
      f32x16 sc[KG];
#pragma unroll
      for (int i = 0; i < KG; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) sc[i][j] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const f16x8 hi = query[buf][0][slot(2 * j + h, n)], lo = query[buf][1][slot(2 * j + h, n)];
#pragma unroll
        for (int i = 0; i < KG; ++i) {
          sc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx[i][j], hi, sc[i], 0, 0, 0);
          sc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx[i][j], lo, sc[i], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < KG; ++i) {
        const int g0 = first + i * kKvGroup;
        float y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float x = I8 ? sc[i][j] * scales[wave][i][h][j] : sc[i][j];
          y[j] = __builtin_amdgcn_exp2f(fmaf(x, c, -ei));
        }
        if (g0 + kKvGroup - 1 > pmin) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (kv_token(FMT, 8 * (j >> 2) + (j & 3)) > p - g0 - kTokenOfHalf<FMT> * h) y[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[i][j] += y[j];
        __builtin_amdgcn_sched_barrier(0);  // one group's weights at a time: registers
      }
    }

    // ---- over the lanes' rows; lane n takes sum n
#pragma unroll
    for (int i = 0; i < KG; ++i) {
      float mine = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float v = sum[i][j];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) v += __shfl_xor(v, d, 32);
        if (n == j) mine = v;
        __builtin_amdgcn_sched_barrier(0);
      }
      const int j = k0 + (wave * KG + i) * kKvGroup + kv_token(FMT, 8 * (n >> 2 & 3) + 4 * h + (n & 3));
      if (!there[i]) mine = 0.f;
      for (uint64_t odd = __ballot(n < 16 && j < s.len && mine != mine); odd; odd &= odd - 1) {
        const int l = __builtin_ctzll(odd), t = __builtin_amdgcn_readlane(j, l);
        const float x = column_by_formula<FMT, D>(arguments(), s, seq, head, t, from * kMassBlock, min(to * kMassBlock, rows));
        if (lane == l) mine = x;
      }
      if (n >= 16 || j >= s.len) continue;
      if (parts == 1)
        add_more(a, all, s, tile, j, mine);
      else
        w.part[(tile * w.m.row_parts + part) * ((size_t)w.groups * kKvGroup) + j] = mine;
    }
  }
}

// Sums the parts of sequences whose rows were shared out, in their order.
__global__ __launch_bounds__(kMassThreads) void k_mass_sum(KvView kv, nx_kv_batch b, MassCall a, WideWork w, int key_tile) {
  __shared__ long sums[kMassWaves];
  __shared__ Place found;
  for (int u = blockIdx.x;; u += gridDim.x) {
    __syncthreads();  // found is read
    auto parts = [&](const KvSeq &q) {
      const int blocks = (part_of(a, w, q).n * a.group + kMassBlock - 1) / kMassBlock;
      return (blocks + w.m.row_share - 1) / w.m.row_share;
    };
    const Place at = find_item<kMassWaves>(
        kv, b, u,
        [&](const KvSeq &q) { return parts(q) > 1 ? (q.len + kMassThreads - 1) / kMassThreads * kv.heads : 0; }, sums,
        &found);
    if (at.s < 0) return;
    const KvSeq s = part_of(a, w, at.seq);
    const int each = (s.len + kMassThreads - 1) / kMassThreads, head = at.at / each;
    const int j = (at.at - head * each) * kMassThreads + (int)threadIdx.x;
    if (j >= s.len) continue;
    const size_t unit = (size_t)at.s * kv.heads + head;
    // (where a slice ends in front of the keys, its last part would reach them by its size: none of it was written)
    const int seen = first_block(a, s, j / (key_tile * kKvGroup) * (key_tile * kKvGroup));
    const int to = seen < (s.n * a.group + kMassBlock - 1) / kMassBlock ? parts(at.seq) : 0;
    float sum = 0.f;
    for (int i = seen / w.m.row_share; i < to; ++i)
      sum += w.part[(unit * w.m.row_parts + i) * ((size_t)w.groups * kKvGroup) + j];
    add_more(a, at.seq, s, unit, j, sum);
  }
}

// The memory of scores and statistics: of one size for every call, allocated once, never moved.
static int mass_workspace(nx_ctx *c, float **out, int **next) {
  constexpr size_t kBytes = kMassFloats * 4, kCounts = 256;
  DevBuf &ws = c->ws[WS_MASS];
  if (!ws.ptr) {
    NX_TRY(refuse_capture(c));
    void *p = nullptr;
    if (hipMalloc(&p, kBytes + kCounts) != hipSuccess) {
      (void)hipGetLastError();
      return fail(NX_ERR_OOM, "device allocation of " + std::to_string(kBytes + kCounts) + " bytes failed");
    }
    // counts begin at 0, and the workspace is there once they are: a call that finds others
    // would leave units out
    if (hipMemsetAsync(static_cast<uint8_t *>(p) + kBytes, 0, kCounts, c->stream) != hipSuccess ||
        hipStreamSynchronize(c->stream) != hipSuccess) {
      (void)hipGetLastError();
      (void)hipFree(p);
      return fail(NX_ERR_DEVICE, "clearing the workspace of gathered weights failed");
    }
    ws = {p, kBytes + kCounts};
  }
  *out = static_cast<float *>(ws.ptr);
  *next = reinterpret_cast<int *>(*out + kMassFloats);
  return NX_OK;
}

// The most rows of a sequence whose scores are stored, where the batch has longer ones: one tile.
// us for 32 heads over 8 of 128, 16 rows of each, by stored scores and by scores worked out twice,
//   sequences, tokens, context   16 x 4, 4096   2 x 4, 32000   61 x 4, 1024   8 x 4, 512   1 x 4, 2000
//   F16                              52   87        57   90        49   80       21   24       13   20
//   INT8                             46   96        49   96        42   89       22   28       13   23
// (Two tiles would take more of the workspace, which sequences of one row beside a prompt need.)
constexpr int kMassFew = 16;

static int mass_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch &all, MassCall a) {
  a.wide_q = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.q_stride % 4 == 0;
  a.shift = group_shift(a.group);
  a.magic = group_magic(a.group);
  float *ws;
  int *next;
  NX_TRY(mass_workspace(c, &ws, &next));
  const KvView view = view_of(kv);
  const int groups = all.max_pages * (kv->page_tokens / kKvGroup);
  // Only the device knows the sequences' rows.  With one or more in each, one has at most
  // num_tokens - num_seqs + 1; a batch that leaves sequences out for a long one is right on 16-row tiles too.
  bool wide = ((long)all.num_tokens - all.num_seqs + 1) * a.group > kMassFew;
  MassNarrow n = mass_narrow(all.num_seqs, all.num_tokens, a.group, kv->heads, groups, wide);
  if (n.heads == 0) wide = true;
  if (wide && all.num_seqs == 1) n.heads = 0;  // (all rows are one sequence's)
  a.rows_above = 0;
  a.rows_upto = n.heads == 0 ? 0 : wide ? kMassFew : INT32_MAX;
  for (int head = 0; head < kv->heads && n.heads > 0; head += n.heads) {
    const NarrowWork w{n, head, groups, ws, reinterpret_cast<float2 *>(ws + n.slots * groups * kKvGroup)};
    NX_TRY(launch(c, "mass_scores", [&] {
      with_kernel(kv, [&](auto fmt, auto D) {
        go(c, k_mass_scores<fmt(), D()>, dim3((uint32_t)n.tiles * n.chunks), dim3(kMassThreads), 0, view, all, a, w);
      });
    }));
    NX_TRY(launch(c, "mass_add", [&] {
      go(c, k_mass_add, dim3((uint32_t)all.num_seqs * n.heads * n.add_chunks), dim3(kMassThreads), 0, view, all, a, w);
    }));
  }
  if (!wide) return NX_OK;
  a.rows_above = a.rows_upto;
  a.rows_upto = INT32_MAX;
  const int key_tile = kv->D == 256 ? kKeyTile<256> : kKeyTile<128>;
  const MassWide m = mass_wide(all.num_seqs, all.num_tokens, a.heads, kv->heads, groups, key_tile, kv->D);
  const long tiles = (long)all.num_seqs * kv->heads, columns = m.column_units;
  if (std::max(columns, tiles * (groups / 8 + 1)) > INT32_MAX)
    return fail(NX_ERR_UNSUPPORTED, "page tables of more than 2^31 tiles");
  const size_t query = m.query;
  WideWork w{m, 0, next, false, false, groups, ws, ws + query, reinterpret_cast<_Float16 *>(ws + 2 * query),
             ws + (2 + kv->D) * query};
  const dim3 block(kMassThreads);
  const long at_once = (kv->D == 256 ? 1 : 3) * c->num_cu, stats = std::min(at_once, m.key_units);
  const long columns_at_once = 2 * c->num_cu;
  w.stats_once = m.key_units <= at_once;
  w.columns_once = columns <= columns_at_once;
  for (; w.first < all.num_tokens; w.first += m.rows) {
    NX_TRY(launch(c, "mass_stats", [&] {
      const dim3 grid((uint32_t)stats);
      with_kernel(kv, [&](auto fmt, auto D) { go(c, k_mass_stats<fmt(), D()>, grid, block, 0, view, all, a, w); });
    }));
    if (m.key_parts > 1)
      NX_TRY(launch(c, "mass_join", [&] {
        const int rows = std::min(m.rows, all.num_tokens - w.first) * a.heads;
        go(c, k_mass_join, dim3((rows + kMassThreads / 16 - 1) / (kMassThreads / 16)), block, 0, a, w, rows);
      }));
    NX_TRY(launch(c, "mass_columns", [&] {
      const dim3 grid((uint32_t)std::min(columns_at_once, columns));
      with_kernel(kv, [&](auto fmt, auto D) { go(c, k_mass_columns<fmt(), D()>, grid, block, 0, view, all, a, w); });
    }));
    if (m.row_parts > 1)
      NX_TRY(launch(c, "mass_sum", [&] {
        go(c, k_mass_sum, dim3(2 * c->num_cu), block, 0, view, all, a, w, key_tile);
      }));
  }
  return NX_OK;
}

static int attention_mass(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, const float *q, size_t q_stride, int heads,
                          float scale, const float *before, float *mass, size_t mass_stride, bool host) {
  NX_TRY(kv_check_call(c, kv, b));
  NX_TRY(refuse(attn_check(heads, kv->heads, scale, 0, 0)));
  if (b->num_seqs == 0 || b->num_tokens == 0) return NX_OK;
  const size_t width = (size_t)heads * kv->D;
  NX_TRY(refuse(mass_check(b, kv->heads, heads, q_stride, width, q, before, mass, mass_stride, host)));
  MassCall a{q, before, mass, q_stride, mass_stride, heads, heads / kv->heads, scale * kLog2e};
  if (!host) return mass_dev(c, kv, *b, a);
  NX_TRY(refuse(kv_check_tables(*b, kv->pages, kv->page_tokens, true, false)));
  NX_TRY(refuse(mass_check_tables(*b, kv->heads, before, mass, mass_stride)));
  const size_t rows = b->row_start[b->num_seqs], tiles = (size_t)b->num_seqs * kv->heads;
  if (rows == (size_t)b->row_start[0]) return NX_OK;
  size_t most = 1;
  for (int s = 0; s < b->num_seqs; ++s) most = std::max(most, (size_t)b->kv_len[s]);
  most = std::min(most, mass_stride);
  nx_kv_batch dev;
  NX_TRY(kv_upload_batch(c, *b, &dev));
  void *dq, *dm;
  NX_TRY(ws_get(c, WS_XIN, rows * width * 4, &dq));
  NX_TRY(ws_get(c, WS_OUT, tiles * most * 4, &dm));
  NX_HIP(hipMemcpy2DAsync(dq, width * 4, q, q_stride * 4, width * 4, rows, hipMemcpyHostToDevice, c->stream));
  if (before)  // (of sequences that have rows, the tokens before them)
    NX_TRY(upload_weights(c, static_cast<float *>(dm), most, before, mass_stride,
                          weight_rows(b->num_seqs, kv->heads, [&](int s) { return mass_read(*b, s, most); })));
  a.q = static_cast<const float *>(dq);
  a.q_stride = width;
  a.mass = static_cast<float *>(dm);
  a.before = before ? a.mass : nullptr;
  a.mass_stride = most;
  dev.num_tokens = (int)rows;
  NX_TRY(mass_dev(c, kv, dev, a));
  for (int s = 0; s < b->num_seqs; ++s) {  // (sequences without rows, and what is behind the others, stay the caller's)
    const size_t len = std::min((size_t)b->kv_len[s], most), at = (size_t)s * kv->heads;
    if (len && b->row_start[s + 1] > b->row_start[s])
      NX_HIP(hipMemcpy2DAsync(mass + at * mass_stride, mass_stride * 4, a.mass + at * most, most * 4, len * 4, kv->heads,
                              hipMemcpyDeviceToHost, c->stream));
  }
  NX_HIP(hipStreamSynchronize(c->stream));
  return NX_OK;
}

}  // namespace nx

using namespace nx;

extern "C" {

int nx_attention_mass(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, const float *q, size_t q_stride, int heads,
                      float scale, const float *before, float *mass, size_t mass_stride) {
  return guarded([&] { return attention_mass(c, kv, b, q, q_stride, heads, scale, before, mass, mass_stride, true); });
}
int nx_attention_mass_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, const float *q, size_t q_stride, int heads,
                          float scale, const float *before, float *mass, size_t mass_stride) {
  return guarded([&] { return attention_mass(c, kv, b, q, q_stride, heads, scale, before, mass, mass_stride, false); });
}

}  // extern "C"
