// nx_evict.hip — giving up cached tokens: which of them each key/value head keeps, by their
// weights, and moving those to new pages.
//
// k_evict_select, a workgroup of a sequence and head: the weight that the last kept token has,
// by counting the weights' leading 11, next 11 and last 10 bits (as keys that order as the values
// do); then every wave numbers the kept ones of its stretch of tokens, in their order.
// k_evict_move, a workgroup of 32 kept tokens of a head: out of their groups' operand order into
// that of the new group.
#include <hip/hip_runtime.h>

#include "nx_kv_dev.hpp"
#include "nx_step_plan.hpp"

namespace nx {

constexpr int kSelectWaves = 16, kSelectThreads = 64 * kSelectWaves, kBins = 2048;

// orders as the value, NaN below all of them; -0 is 0
__device__ __forceinline__ uint32_t weight_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int evict_len(const KvView &kv, const nx_kv_batch &b, int s) {
  return min(max(b.kv_len[s], 0), b.max_pages << kv.page_log2);
}

__global__ __launch_bounds__(kSelectThreads) void k_evict_select(KvView kv, nx_kv_batch b, EvictArgs a, long first) {
  __shared__ int bins[kBins], chosen, before;
  __shared__ long sums[kSelectWaves];
  __shared__ int above[kSelectWaves], even[kSelectWaves];
  const long tile = first + blockIdx.x;
  const int s = (int)(tile / kv.heads), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = evict_len(kv, b, s), n = min(len, a.keep);
  const float *w = a.mass + (size_t)tile * a.mass_stride;
  const int weights = (int)min((size_t)len, a.mass_stride);
  int32_t *kept = a.kept + (size_t)tile * a.keep;
  float *moved = a.new_mass ? a.new_mass + (size_t)tile * a.new_mass_stride : nullptr;
  if (tile % kv.heads == 0 && tid == 0) a.new_len[s] = n;
  for (int i = n + tid; i < a.keep; i += kSelectThreads) kept[i] = -1;
  auto key = [&](int j) { return j < weights ? weight_key(w[j]) : 0u; };
  // tokens [lo, hi) are chosen from: those above key t, and the first `need` of key t
  int lo = a.sinks, hi = len - a.recent, need = a.keep - a.sinks - a.recent;
  uint32_t t = 0xffffffffu;
  if (len <= a.keep) {
    lo = len;
    need = 0;
  }
  if (need > 0) {
    t = 0;
    int left = 32;
    while (left > 0) {
      const int bits = left == 10 ? 10 : 11, shift = left - bits, count = 1 << bits;
      for (int i = tid; i < count; i += kSelectThreads) bins[i] = 0;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += kSelectThreads) {
        const uint32_t k = key(j);
        if (left == 32 || k >> left == t) atomicAdd(&bins[k >> shift & (count - 1)], 1);
      }
      __syncthreads();
      // from the largest bin down: that in which the count passes `need`
      const int top = count - 1 - 2 * tid;
      const int c0 = top > 0 ? bins[top] : 0, c1 = top > 0 ? bins[top - 1] : 0;
      long total;
      const int upto = (int)scan_wg<kSelectWaves>((long)c0 + c1, sums, total), from = upto - c0 - c1;
      if (from < need && need <= upto) {
        chosen = need <= from + c0 ? top : top - 1;
        before = need <= from + c0 ? from : from + c0;
      }
      __syncthreads();
      t = t << bits | (uint32_t)chosen;
      need -= before;
      left = shift;
      __syncthreads();  // chosen and bins are read
    }
  }
  // the wave's stretch of tokens
  const int stretch = (len + kSelectThreads - 1) / kSelectThreads * 64;
  const int start = min(wave * stretch, len), stop = min(start + stretch, len);
  auto place = [&](int j, bool &over, bool &same) {
    const bool middle = j >= lo && j < hi && j < stop;
    const uint32_t k = middle ? key(j) : 0u;
    over = j < stop && (!middle || k > t);
    same = middle && need > 0 && k == t;
  };
  int sure = 0, maybe = 0;
  for (int j0 = start; j0 < stop; j0 += 64) {
    bool over, same;
    place(j0 + lane, over, same);
    sure += __popcll(__ballot(over));
    maybe += __popcll(__ballot(same));
  }
  if (lane == 0) {
    above[wave] = sure;
    even[wave] = maybe;
  }
  __syncthreads();
  sure = maybe = 0;
  for (int i = 0; i < wave; ++i) {
    sure += above[i];
    maybe += even[i];
  }
  const uint64_t lower = ((uint64_t)1 << lane) - 1;
  for (int j0 = start; j0 < stop; j0 += 64) {
    const int j = j0 + lane;
    bool over, same;
    place(j, over, same);
    const uint64_t o = __ballot(over), e = __ballot(same);
    const int rank = maybe + __popcll(e & lower);
    if (over || (same && rank < need)) {
      const int at = sure + __popcll(o & lower) + min(rank, need);
      kept[at] = j;
      if (moved) moved[at] = j < weights ? w[j] : 0.f;
    }
    sure += __popcll(o);
    maybe += __popcll(e);
  }
}

constexpr int kEvictThreads = 256;

template <int FMT, int D>
__global__ __launch_bounds__(kEvictThreads) void k_evict_move(KvView kv, nx_kv_batch b, EvictArgs a, int groups,
                                                              long first) {
  using E = kv_elem<FMT>;
  using Chunk = std::conditional_t<FMT == NX_KV_INT8, uint2, uint4>;  // 8 elements
  __shared__ long from[kKvGroup];  // the tokens' groups in the pool, -1: none
  __shared__ int in_group[kKvGroup];
  const long item = first + blockIdx.x, tile = item / groups;
  const int s = (int)(tile / kv.heads), head = (int)(tile % kv.heads), t0 = (int)(item % groups) * kKvGroup;
  const int n = min(evict_len(kv, b, s), a.keep), tid = threadIdx.x;
  if (t0 >= n) return;
  nx_kv_batch to = b;
  to.max_pages = a.to_max_pages;
  to.pages = a.to_pages;
  const long group = kv_group(kv, to, s, head, t0);
  if (group < 0) return;
  if (tid < kKvGroup) {
    const int j = t0 + tid < n ? a.kept[(size_t)tile * a.keep + t0 + tid] : -1;
    const long g = j >= 0 ? kv_group(kv, b, s, head, j & ~(kKvGroup - 1)) : -1;
    from[tid] = g;
    in_group[tid] = j & (kKvGroup - 1);
    if constexpr (FMT == NX_KV_INT8) {
      kv.ks[group * kKvGroup + tid] = g >= 0 ? kv.ks[g * kKvGroup + in_group[tid]] : 0.f;
      kv.vs[group * kKvGroup + tid] = g >= 0 ? kv.vs[g * kKvGroup + in_group[tid]] : 0.f;
    }
  }
  __syncthreads();
  Chunk *k = reinterpret_cast<Chunk *>(kv.k) + group * (kKvGroup * D / 8);
  Chunk *v = reinterpret_cast<Chunk *>(kv.v) + group * (kKvGroup * D / 8);
  for (int c = tid; c < kKvGroup * D / 8; c += kEvictThreads) {
    const int t = kv_token(FMT, c & (kKvGroup - 1));
    const long g = from[t];
    Chunk x = {};
    if (g >= 0)
      x = reinterpret_cast<const Chunk *>(kv.k)[g * (kKvGroup * D / 8) + (c & ~(kKvGroup - 1)) + kv_row(FMT, in_group[t])];
    k[c] = x;
  }
  for (int c = tid; c < kKvGroup * D / 8; c += kEvictThreads) {
    const int d = c % D, t1 = c / D * 8;
    union {
      E e[8];
      Chunk x;
    } o;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long g = from[t1 + i];
      o.e[i] = g >= 0 ? reinterpret_cast<const E *>(kv.v)[g * (kKvGroup * D) + kv_value_at(D, in_group[t1 + i], d)] : (E)0;
    }
    v[c] = o.x;
  }
}

static int evict_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch &b, const EvictArgs &a) {
  const KvView view = view_of(kv);
  const long tiles = (long)b.num_seqs * kv->heads;
  // (a launch has fewer than 2^32 threads)
  constexpr long kTiles = 1 << 20, kItems = 1 << 23;
  for (long first = 0; first < tiles; first += kTiles)
    NX_TRY(launch(c, "evict_select", [&] {
      go(c, k_evict_select, dim3((uint32_t)std::min(tiles - first, kTiles)), dim3(kSelectThreads), 0, view, b, a, first);
    }));
  const long tokens = std::min({(long)a.keep, (long)a.to_max_pages * kv->page_tokens, (long)b.max_pages * kv->page_tokens});
  const int groups = (int)((tokens + kKvGroup - 1) / kKvGroup);
  for (long first = 0; first < tiles * groups; first += kItems)
    NX_TRY(launch(c, "evict_move", [&] {
      with_kernel(kv, [&](auto fmt, auto D) {
        go(c, k_evict_move<fmt(), D()>, dim3((uint32_t)std::min(tiles * groups - first, kItems)), dim3(kEvictThreads), 0,
           view, b, a, groups, first);
      });
    }));
  return NX_OK;
}

static int evict(nx_ctx *c, nx_kv *kv, const nx_kv_batch *b, const EvictArgs &a, bool host) {
  NX_TRY(kv_check_cache(c, kv));
  NX_TRY(refuse(evict_check(b, kv->page_tokens, kv->heads, a)));
  if (b->num_seqs == 0) return NX_OK;
  if (!host) return evict_dev(c, kv, *b, a);
  NX_TRY(refuse(evict_check_tables(*b, kv->pages, kv->page_tokens, a)));
  const size_t S = b->num_seqs, tiles = S * kv->heads, table = S * b->max_pages, to = S * a.to_max_pages;
  const size_t kept = tiles * a.keep;
  size_t width = 1;  // weights that are looked at
  for (size_t s = 0; s < S; ++s) width = std::max(width, (size_t)b->kv_len[s]);
  void *pb, *pm, *po;
  NX_TRY(ws_get(c, WS_KV_BATCH, (2 * S + table + to) * 4, &pb));
  NX_TRY(ws_get(c, WS_XIN, tiles * width * 4, &pm));
  NX_TRY(ws_get(c, WS_OUT, 2 * kept * 4, &po));
  int32_t *len = static_cast<int32_t *>(pb), *new_len = len + S, *pages = new_len + S, *to_pages = pages + table;
  EvictArgs d = a;
  d.mass = static_cast<const float *>(pm);
  d.mass_stride = width;
  d.kept = static_cast<int32_t *>(po);
  d.new_len = new_len;
  d.new_mass = a.new_mass ? static_cast<float *>(po) + kept : nullptr;
  d.new_mass_stride = a.keep;
  d.to_pages = to_pages;
  nx_kv_batch on = *b;
  on.row_start = nullptr;
  on.kv_len = len;
  on.pages = pages;
  NX_HIP(hipMemcpyAsync(len, b->kv_len, S * 4, hipMemcpyHostToDevice, c->stream));
  NX_HIP(hipMemcpyAsync(pages, b->pages, table * 4, hipMemcpyHostToDevice, c->stream));
  NX_HIP(hipMemcpyAsync(to_pages, a.to_pages, to * 4, hipMemcpyHostToDevice, c->stream));
  NX_HIP(hipMemcpy2DAsync(pm, width * 4, a.mass, a.mass_stride * 4, width * 4, tiles, hipMemcpyHostToDevice, c->stream));
  NX_TRY(evict_dev(c, kv, on, d));
  NX_HIP(hipMemcpyAsync(a.kept, d.kept, kept * 4, hipMemcpyDeviceToHost, c->stream));
  NX_HIP(hipMemcpyAsync(a.new_len, new_len, S * 4, hipMemcpyDeviceToHost, c->stream));
  if (a.new_mass)
    for (size_t s = 0; s < S; ++s) {  // (what lies behind a sequence's kept tokens stays the caller's)
      const size_t n = std::min(b->kv_len[s], a.keep), at = s * kv->heads;
      if (n)
        NX_HIP(hipMemcpy2DAsync(a.new_mass + at * a.new_mass_stride, a.new_mass_stride * 4, d.new_mass + at * a.keep,
                                (size_t)a.keep * 4, n * 4, kv->heads, hipMemcpyDeviceToHost, c->stream));
    }
  NX_HIP(hipStreamSynchronize(c->stream));
  return NX_OK;
}

}  // namespace nx

using namespace nx;

extern "C" {

int nx_kv_evict(nx_ctx *c, nx_kv *kv, const nx_kv_batch *b, const int32_t *to_pages, int to_max_pages, int keep,
                int sinks, int recent, const float *mass, size_t mass_stride, int32_t *kept, int32_t *new_len,
                float *new_mass, size_t new_mass_stride) {
  return guarded([&] {
    return evict(c, kv, b, {to_pages, to_max_pages, keep, sinks, recent, mass, mass_stride, kept, new_len, new_mass,
                            new_mass_stride}, true);
  });
}
int nx_kv_evict_dev(nx_ctx *c, nx_kv *kv, const nx_kv_batch *b, const int32_t *to_pages, int to_max_pages, int keep,
                    int sinks, int recent, const float *mass, size_t mass_stride, int32_t *kept, int32_t *new_len,
                    float *new_mass, size_t new_mass_stride) {
  return guarded([&] {
    return evict(c, kv, b, {to_pages, to_max_pages, keep, sinks, recent, mass, mass_stride, kept, new_len, new_mass,
                            new_mass_stride}, false);
  });
}

}  // extern "C"
