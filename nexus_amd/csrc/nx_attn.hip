// nx_attn.hip — causal attention of new tokens over their sequences in the paged
// cache, whole or through a sliding window with first tokens that stay visible.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i)
//
// over the tokens j that token i sees, in one pass over the cache: m_i is the
// running maximum, and the sums taken so far are scaled by exp(m_old - m_new)
// when it grows.
#include <hip/hip_runtime.h>

#include "nx_kv_dev.hpp"
#include "nx_split_dev.hpp"

namespace nx {

struct AttnCall {
  const float *q;
  float *out;
  size_t q_stride, out_stride;
  int heads, group;  // query heads, and those that share a key/value head
  float scale;
  int window, sinks;
  bool wide_q, wide_out;  // rows of whole float4 runs
};

// whether token p sees token j <= p
__device__ __forceinline__ bool sees(const AttnCall &a, int p, int j) {
  return j <= p && (a.window == 0 || p - j < a.window || j < a.sinks);
}

// One row by the formula alone, in f32: a wave, each lane a key's whole score,
// then each lane some elements of the sum over the keys.
template <int FMT, int D>
__device__ __forceinline__ void attn_row(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                         const KvSeq &s, int seq, int head, int p, const float *q,
                                         float *out) {
  using E = kv_elem<FMT>;
  const int lane = threadIdx.x & 63;
  const E *ck = reinterpret_cast<const E *>(kv.k), *cv = reinterpret_cast<const E *>(kv.v);
  float m = -INFINITY, l = 0.f, acc[(D + 63) / 64] = {};
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
    float x = -INFINITY;
    if (group >= 0) {
      x = 0.f;
      const E *k = ck + group * (kKvGroup * D);
      for (int d = 0; d < D; ++d) x = fmaf((float)k[kv_key_at(FMT, t, d)], q[d], x);
      x *= a.scale;
      if (FMT == NX_KV_INT8) x *= kv.ks[group * kKvGroup + t];
    }
    const uint64_t seen = __ballot(group >= 0);
    if (!seen) continue;
    any = true;
    float top = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    const float m1 = fmaxf(m, top), ref = m1 == -INFINITY ? 0.f : m1;
    const float pr = group >= 0 ? expf(x - ref) : 0.f;
    const float keep = m == -INFINITY ? 0.f : expf(m - ref);
    m = m1;
    float sum = pr;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    l = l * keep + sum;
    // the 64 keys' sum apart: over long contexts a single chain of additions would
    // lose sqrt(keys) of its last places
    float part[(D + 63) / 64] = {};
    float w = pr;
    if (FMT == NX_KV_INT8 && group >= 0) w *= kv.vs[group * kKvGroup + t];
    for (int u = 0; u < 64; ++u) {
      if (!((seen >> u) & 1)) continue;
      const float wu = __shfl(w, u, 64);
      const long gu = __shfl(group, u, 64);
      const E *v = cv + gu * (kKvGroup * D);
#pragma unroll
      for (int i = 0; i < (D + 63) / 64; ++i) {
        const int d = lane + 64 * i;
        if (d < D) part[i] = fmaf(wu, (float)v[kv_value_at(D, (j0 + u) & (kKvGroup - 1), d)], part[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i) acc[i] = fmaf(acc[i], keep, part[i]);
  }
#pragma unroll
  for (int i = 0; i < (D + 63) / 64; ++i) {
    const int d = lane + 64 * i;
    if (d < D) out[d] = any ? acc[i] / l : 0.f;
  }
}

// ------------------------------------------------------------ decode: k_attn_split
//
// Rows of up to kTile (token, head) pairs that share a key/value head are one tile
// of the matrix cores; a unit of work is one tile against one group of 32 tokens.
// All units of the batch, in order of (sequence, head, tile, group), are dealt out
// in equal runs, one per workgroup, so a ragged batch loads every CU alike. A tile
// whose units end up in several workgroups is joined by k_attn_join.
//
// Transposed products: S^T = K Q^T puts a query in each lane column, the scores of
// tokens 8 g .. 8 g + 7 in lane group g (kv_row), which is the operand layout of
// P^T in O^T = V^T P^T: no value moves between lanes but the maximum.  q and p
// are f32 split into two f16 halves (hi + lo: 22 bits), K and V enter as they are
// stored; int8 codes as exact f16 values, with the key's scale on the score and the
// value's on the weight.
constexpr int kTile = 16;
constexpr float kLog2e = 1.4426950408889634f;
// weights reach 2^6 at the maximum that they are relative to, and 2^14 when the
// maximum has grown by 2^8 since: only then are the sums scaled anew
constexpr float kHead = 6.f, kGrow = 14.f, kUnset = -1e30f;

// int8 code -> f16 q 2^-9, exact: 0x80 ^ code as the low bits of a subnormal half
__device__ __forceinline__ f16x8 from_codes(uint32_t lo, uint32_t hi) { return operand8(lo, hi); }

__device__ __forceinline__ float ldexp1(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }

__device__ __forceinline__ void split2(const float (&x)[8], f16x8 &h, f16x8 &l) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    h[i] = (_Float16)x[i];
    l[i] = (_Float16)(x[i] - (float)h[i]);
  }
}

// the largest (sum) over the four lane groups, in all of them
template <typename Op>
__device__ __forceinline__ float across_groups(float v, Op op) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float max_groups(float v) {
  return across_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_groups(float v) {
  return across_groups(v, [](float a, float b) { return a + b; });
}

// A tile of a sequence: rows r0 .. r0 + nr - 1 of its n * group (token, head) rows
struct Tile {
  int seq, head, r0, nr;
};
__device__ __forceinline__ KeySpan tile_span(const KvSeq &s, const AttnCall &a, int r0, int nr) {
  return key_span(s.first + r0 / a.group, s.first + (r0 + nr - 1) / a.group, s.len, a.window, a.sinks);
}
// units of a tile: at least one, so that rows which see nothing are written
__device__ __forceinline__ int tile_units(const KvSeq &s, const AttnCall &a, int r0, int tile) {
  const int nr = min(tile, s.n * a.group - r0);
  return max(tile_span(s, a, r0, nr).count(), 1);
}
__device__ __forceinline__ long head_units(const KvSeq &s, const AttnCall &a, int tile) {
  long u = 0;
  for (int r0 = 0; r0 < s.n * a.group; r0 += tile) u += tile_units(s, a, r0, tile);
  return u;
}

// Partial results of tiles that were split: per workgroup, those of the tile that
// it ends (or passes through) and of the tile that it begins.
//   desc [workgroups] {seq, head, r0, workgroups of the tile that begins here or 0}
//   part [workgroups][2] {m[tile], l[tile], o[tile][D]}
struct AttnWork {
  int4 *desc;
  float *part;
  int wgs, min_share;
};

// four values of a finished row; *bad is set where they are not finite: a weight 0
// times a value that is not finite, or a row whose result is not finite by the
// formula (or that sees nothing), which attn_row tells apart
template <int D>
__device__ __forceinline__ void store_out(const AttnCall &a, const KvSeq &s, int head, int row, int d,
                                          f32x4 o, float l, int *bad) {
  const float inv = 1.f / l;
  o *= inv;
  float *out = a.out + (size_t)(s.row + row / a.group) * a.out_stride +
               (size_t)(head * a.group + row % a.group) * D + d;
  const bool fine = __builtin_isfinite(o.x) && __builtin_isfinite(o.y) && __builtin_isfinite(o.z) &&
                    __builtin_isfinite(o.w);
  if (!fine || !(l > 0.f)) *bad = 1;
  if (a.wide_out) {
    *reinterpret_cast<f32x4 *>(out) = o;
  } else {
    out[0] = o.x;
    out[1] = o.y;
    out[2] = o.z;
    out[3] = o.w;
  }
}

template <int FMT, int D>
struct DecodeLds {
  float m[4][kTile], l[4][kTile];
  float o[4][kTile][D + 4];
  int bad[kTile];
};

template <int FMT, int D>
__device__ __forceinline__ void finish_rows(const KvView &kv, const nx_kv_batch &b, const AttnCall &a,
                                            const KvSeq &s, const Tile &t, const int *bad) {
  for (int r = threadIdx.x >> 6; r < t.nr; r += 4) {
    if (!bad[r]) continue;
    const int row = t.r0 + r, h = t.head * a.group + row % a.group, i = row / a.group;
    attn_row<FMT, D>(kv, b, a, s, t.seq, t.head, s.first + i,
                     a.q + (size_t)(s.row + i) * a.q_stride + (size_t)h * D,
                     a.out + (size_t)(s.row + i) * a.out_stride + (size_t)h * D);
  }
}

template <int FMT, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_attn_split(KvView kv, nx_kv_batch b,
                                                                     AttnCall a, AttnWork w) {
  using E = kv_elem<FMT>;
  constexpr bool I8 = FMT == NX_KV_INT8;
  constexpr int KS = D / 32, DT = D / 16;     // steps of a score, 16-element tiles of the output
  constexpr int KL = I8 ? KS : 2 * KS, VL = I8 ? DT / 2 : DT;  // 16-byte loads of a lane and group
  __shared__ DecodeLds<FMT, D> lds;
  __shared__ long sums[4];
  __shared__ Place place;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
  // neighbouring runs on one XCD: tiles of one head share its keys in that L2
  const int wg = (blockIdx.x & 7) * (w.wgs >> 3) + (blockIdx.x >> 3);

  auto seq_units = [&](int s) {
    const KvSeq q = kv_seq(b, s, kv.page_log2);
    return q.n > 0 ? (long)kv.heads * head_units(q, a, kTile) : 0;
  };
  // all units, then the run of this workgroup
  long total = 0;
  for (int s0 = 0; s0 < b.num_seqs; s0 += 256) {
    const int s = s0 + (int)threadIdx.x;
    scan256(s < b.num_seqs ? seq_units(s) : 0, sums);
    total += sums[0] + sums[1] + sums[2] + sums[3];
  }
  const long share = max((total + w.wgs - 1) / w.wgs, (long)w.min_share);
  const long begin = wg * share, end = min(begin + share, total);
  if (threadIdx.x == 0) w.desc[wg] = int4{0, 0, 0, 0};
  if (begin >= end) return;
  const Place at = find_item(b.num_seqs, begin, seq_units, sums, &place);
  int seq = at.s;
  KvSeq s = kv_seq(b, seq, kv.page_log2);
  long in_head = head_units(s, a, kTile);
  int head = (int)(at.at / in_head), r0 = 0;
  int off = 0, units;
  {
    long rest = at.at - head * in_head;
    while (units = tile_units(s, a, r0, kTile), rest >= units) rest -= units, r0 += kTile;
    off = (int)rest;
  }

  for (long u = begin; u < end;) {
    const Tile t{seq, head, r0, min(kTile, s.n * a.group - r0)};
    const KeySpan span = tile_span(s, a, r0, t.nr);
    const int stop = (int)min((long)units, off + (end - u));  // units [off, stop) of the tile
    const bool whole = off == 0 && stop == units;

    // ---- this lane's query
    const int row = r0 + min(n, t.nr - 1), tok = row / a.group;
    const int p = s.first + tok;  // its token
    f16x8 qh[KS], ql[KS];
    float c;
    {
      const float *q = a.q + (size_t)(s.row + tok) * a.q_stride +
                       (size_t)(head * a.group + row % a.group) * D + 8 * g;
      float x[KS][8], mx = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (a.wide_q) {
          *reinterpret_cast<f32x4 *>(&x[ks][0]) = *reinterpret_cast<const f32x4 *>(q + 32 * ks);
          *reinterpret_cast<f32x4 *>(&x[ks][4]) = *reinterpret_cast<const f32x4 *>(q + 32 * ks + 4);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[ks][i] = q[32 * ks + i];
        }
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
        split2(x[ks], qh[ks], ql[ks]);
      }
      c = ldexp1(a.scale * kLog2e, E - 14 + (I8 ? 9 : 0));
    }

    float m = kUnset, l = 0.f;
    float wm = 0.f;  // INT8: the row's largest weight p scale when last looked at,
    int we = 0;      // and the power of two that keeps weights in half's range
    f32x4 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    uint4 kf[KL], vf[VL];
    auto locate = [&](int i, int &first, bool &there) {  // unit i's first token and pool group
      first = span.group(i) * kKvGroup;
      const long gr = span.count() > 0 ? kv_group(kv, b, seq, head, first) : -1;
      there = gr >= 0;
      return there ? gr : 0;
    };
    auto load_k = [&](long gr) {
      const E *base = reinterpret_cast<const E *>(kv.k) + gr * (kKvGroup * D);
      if constexpr (I8) {
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
#pragma unroll
      for (int i = 0; i < VL; ++i)
        vf[i] = *reinterpret_cast<const uint4 *>(base + (g * D + (I8 ? 32 * i + 2 * n : 16 * i + n)) * 8);
    };

    int first, first1;
    bool there, there1;
    long gr = 0, gr1;
    if (off + wave < stop) {
      gr = locate(off + wave, first, there);
      load_k(gr);
      load_v(gr);
    }
    for (int i = off + wave; i < stop; i += 4) {
      gr1 = locate(min(i + 4, stop - 1), first1, there1);
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
      float dv[8];
      if constexpr (I8) {
        const f32x4 *dk = reinterpret_cast<const f32x4 *>(kv.ks + gr * kKvGroup + 8 * g);
        const f32x4 *d2 = reinterpret_cast<const f32x4 *>(kv.vs + gr * kKvGroup + 8 * g);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sc[h] *= dk[h];
#pragma unroll
          for (int j = 0; j < 4; ++j) dv[4 * h + j] = d2[h][j];
        }
      }
      load_k(gr1);  // the next group's keys, while this one's weights are made

      // which of them the lane's row sees: all, for groups inside every row's range
      const int pmin = s.first + r0 / a.group, pmax = s.first + (r0 + t.nr - 1) / a.group;
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
      float y[8], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = (vis >> j) & 1 ? fmaf(sc[j >> 2][j & 3], c, -m) : -INFINITY;
        top = fmaxf(top, y[j]);
      }
      bool grew = false;
      if (__any(top > kGrow)) {
        float x = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if ((vis >> j) & 1) x = fmaxf(x, sc[j >> 2][j & 3] * c);
        x = max_groups(x);
        grew = x > m + kGrow;
        const float m1 = grew ? x - kHead : m, keep = exp2f(m - m1);
        m = m1;
        wm *= keep;
        l *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d] *= keep;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (vis >> j) & 1 ? fmaf(sc[j >> 2][j & 3], c, -m) : -INFINITY;
      }
      float pr[8], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pr[j] = __builtin_amdgcn_exp2f(y[j]);
        sum += pr[j];
      }
      l += sum;
      if constexpr (I8) {
        // weights p scale: the row's largest is kept near 2^12 (below 2^15), so that
        // the halves of those down to 2^-24 of it keep their bits
        float wt = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          pr[j] = (vis >> j) & 1 ? pr[j] * dv[j] : 0.f;
          wt = fmaxf(wt, pr[j]);
        }
        if (__any(grew || ldexp1(wt, we) > 32768.f)) {
          wt = max_groups(wt);
          if ((grew || ldexp1(wt, we) > 32768.f) && wt < INFINITY) {
            wm = fmaxf(wm, wt);
            const int e1 = wm > 0.f ? min(12 - __builtin_amdgcn_frexp_expf(wm), 126) : 0;
            const float f = ldexp1(1.f, min(e1 - we, 126));
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= f;
            we = e1;
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) pr[j] = ldexp1(pr[j], we);
      }
      f16x8 ph, pl;
      split2(pr, ph, pl);
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
      first = first1;
      there = there1;
      gr = gr1;
    }

    // ---- join the waves
    l = sum_groups(l);
    const float un = I8 ? ldexp1(1.f, 9 - we) : 1.f;
    if (g == 0) {
      lds.m[wave][n] = m;
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
    for (int e = threadIdx.x; e < t.nr * (D / 4); e += 256) {
      const int r = e / (D / 4), d = e % (D / 4) * 4;
      const float m1 = fmaxf(fmaxf(lds.m[0][r], lds.m[1][r]), fmaxf(lds.m[2][r], lds.m[3][r]));
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float lt = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float f = exp2f(lds.m[v][r] - m1);
        lt += lds.l[v][r] * f;
        o += *reinterpret_cast<const f32x4 *>(&lds.o[v][r][d]) * f;
      }
      if (!whole) {
        if (d == 0) {
          part[r] = m1;
          part[kTile + r] = lt;
        }
        *reinterpret_cast<f32x4 *>(part + 2 * kTile + r * D + d) = o;
      } else {
        const int rr = r0 + r;
        store_out<D>(a, s, head, rr, d, o, lt, &lds.bad[r]);
      }
    }
    __syncthreads();
    if (whole) {
      finish_rows<FMT, D>(kv, b, a, s, t, lds.bad);
    } else if (off == 0 && threadIdx.x == 0) {
      // how many workgroups hold the tile's units
      const long last = (u + units - 1) / share;
      w.desc[wg] = int4{seq, head, r0, (int)(last - wg) + 1};
    }
    __syncthreads();  // lds is free

    // ---- the next tile
    u += stop - off;
    off = 0;
    if (u >= end) break;
    r0 += kTile;
    if (r0 >= s.n * a.group) {
      r0 = 0;
      if (++head == kv.heads) {
        head = 0;
        do s = kv_seq(b, ++seq, kv.page_log2);
        while (s.n <= 0);  // (units are left, so a sequence is)
      }
    }
    units = tile_units(s, a, r0, kTile);
  }
}

// Joins the tiles whose units several workgroups had: rows y, y + 4, ... of the
// tile that workgroup x begins.
template <int FMT, int D>
__global__ __launch_bounds__(256) void k_attn_join(KvView kv, nx_kv_batch b, AttnCall a, AttnWork w) {
  constexpr int Q = 256 / (D / 4) >= 8 ? 8 : 256 / (D / 4);  // partial sums side by side
  __shared__ f32x4 lds[Q][D / 4];
  __shared__ float sum_l[Q];
  __shared__ int bad[1];
  const int4 t = w.desc[blockIdx.x];
  const int parts = t.w;
  if (parts == 0) return;
  const KvSeq s = kv_seq(b, t.x, kv.page_log2);
  auto at = [&](int i) {
    return w.part + ((size_t)(blockIdx.x + i) * 2 + (i == 0)) * (kTile * (D + 2));
  };
  const int lane = threadIdx.x & 63, q = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4);
  for (int r = blockIdx.y; r < kTile && t.z + r < s.n * a.group; r += 4) {
    float m = kUnset;
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, at(i)[r]);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    if (q < Q) {
      for (int i = q; i < parts; i += Q) {
        const float *p = at(i);
        const float f = exp2f(p[r] - m);
        l += p[kTile + r] * f;
        o += *reinterpret_cast<const f32x4 *>(p + 2 * kTile + r * D + 4 * d) * f;
      }
      lds[q][d] = o;
      if (d == 0) sum_l[q] = l;
    }
    if (threadIdx.x == 0) bad[0] = 0;
    __syncthreads();
    if (q == 0) {
#pragma unroll
      for (int i = 1; i < Q; ++i) {
        o += lds[i][d];
        l += sum_l[i];
      }
      store_out<D>(a, s, t.y, t.z + r, 4 * d, o, l, bad);
    }
    __syncthreads();
    if (threadIdx.x < 64) finish_rows<FMT, D>(kv, b, a, s, Tile{t.x, t.y, t.z + r, 1}, bad);
    __syncthreads();  // lds and bad are free
  }
}

// Workgroups of a call, and the workspace of their parts: of one size for every
// cache, so that it is allocated once.
constexpr int kAttnWgsPerCu = 2;
static int attn_wgs(const nx_ctx *c) { return c->num_cu * kAttnWgsPerCu / 8 * 8; }  // whole XCDs
static size_t attn_bytes(const nx_ctx *c) {
  return (size_t)attn_wgs(c) * (sizeof(int4) + 2 * kTile * (256 + 2) * 4);
}
int attn_workspace(nx_ctx *c, void **out) {
  void *p;
  NX_TRY(ws_get(c, WS_ATTN, attn_bytes(c), &p));
  if (out) *out = p;
  return NX_OK;
}

static int attention_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch &b, AttnCall a) {
  a.wide_q = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.q_stride % 4 == 0;
  a.wide_out = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && a.out_stride % 4 == 0;
  void *p;
  NX_TRY(attn_workspace(c, &p));
  const int wgs = attn_wgs(c);
  AttnWork w{static_cast<int4 *>(p), reinterpret_cast<float *>(static_cast<int4 *>(p) + wgs), wgs, 4};
  const KvView view = view_of(kv);
  NX_TRY(launch(c, "attn_split", [&] {
    with_kernel(kv, [&](auto fmt, auto D) {
      go(c, k_attn_split<fmt(), D()>, dim3(wgs), dim3(256), 0, view, b, a, w);
    });
  }));
  return launch(c, "attn_join", [&] {
    with_kernel(kv, [&](auto fmt, auto D) {
      go(c, k_attn_join<fmt(), D()>, dim3(wgs, 4), dim3(256), 0, view, b, a, w);
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
  AttnCall a{q, out, q_stride, out_stride, heads, heads / kv->heads, scale, window, sinks, false, false};
  if (!host) return attention_dev(c, kv, *b, a);
  NX_TRY(refuse(kv_check_tables(*b, kv->pages, kv->page_tokens, true, false)));
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
  return attention(c, kv, b, q, q_stride, heads, scale, window, sinks, out, out_stride, true);
}
int nx_attention_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, const float *q,
                     size_t q_stride, int heads, float scale, int window, int sinks, float *out,
                     size_t out_stride) {
  return attention(c, kv, b, q, q_stride, heads, scale, window, sinks, out, out_stride, false);
}

}  // extern "C"
