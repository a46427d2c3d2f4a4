// nx_evict.hip — giving up cached tokens: which of them each key/value head keeps, by their
// weights, and moving those to new pages.
//
// k_evict_select, a workgroup of a sequence and head: the weight that the last kept token has,
// by counting the weights' leading 11, next 11 and last 10 bits (as keys that order as the values
// do); then every wave numbers the kept ones of its stretch of tokens, in their order.  What one
// CU can count bounds it: 16381 tokens of 8 heads 17 us, 5003 of 4 heads of 23 sequences 15, 100000 of
// one head, whose weights are read in every pass, 101.  Weights that are alike count into one bin: 53 and 300.
// k_evict_move, a workgroup of 32 kept tokens of a head: out of their groups' operand order into
// that of the new group.  4096 tokens of 8 heads in F16 15 us (34 MB), 3001 of 4 heads of 23
// sequences in INT8 44 us (128 MB, 2.9 TB/s): keys are read in pieces of 8 and 16 bytes, and a
// chunk of 8 tokens' values whole for those of it that stay.
#include <hip/hip_runtime.h>

#include "nx_kv_dev.hpp"
#include "nx_step_plan.hpp"

namespace nx {

constexpr int kSelectWaves = 16, kSelectThreads = 64 * kSelectWaves, kBins = 2 * kSelectThreads;
constexpr int kOwnKeys = 16, kAtOnce = 8;  // of a lane: in registers, loads at once
constexpr uint32_t kAlways = 0xffffffffu;  // above any weight: the first and the last tokens

// orders as the value, NaN below all of them; -0 is 0
__device__ __forceinline__ uint32_t weight_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int evict_len(const KvView &kv, const nx_kv_batch &b, int s) {
  return min(max(b.kv_len[s], 0), b.max_pages << kv.page_log2);
}

__global__ __launch_bounds__(kSelectThreads) void k_evict_select(KvView kv, nx_kv_batch b, EvictArgs a, long first) {
  __shared__ uint32_t bins[kBins], sums[kSelectWaves], chosen, before;
  __shared__ int above[kSelectWaves], even[kSelectWaves];
  const long tile = first + blockIdx.x;
  const int s = (int)(tile / kv.heads), tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int len = uniform(evict_len(kv, b, s)), n = min(len, a.keep);
  const float *w = a.mass + (size_t)tile * a.mass_stride;
  const int weights = (int)min((size_t)len, a.mass_stride);
  int32_t *kept = a.kept + (size_t)tile * a.keep;
  float *moved = a.new_mass ? a.new_mass + (size_t)tile * a.new_mass_stride : nullptr;
  if (tile % kv.heads == 0 && tid == 0) a.new_len[s] = n;
  for (int i = n + tid; i < a.keep; i += kSelectThreads) kept[i] = -1;
  if (len == 0) return;  // (mass_stride is not 0: there are weights)
  if (len <= a.keep) {
    for (int i = tid; i < len; i += kSelectThreads) {
      kept[i] = i;
      if (moved) moved[i] = i < weights ? w[i] : 0.f;
    }
    return;
  }
  // The wave's stretch of tokens, 64 at a step.  Their keys stay in registers where they fit (16381 tokens:
  // 17 us, not 23); those of longer sequences are worked out again in every pass, several steps' loads at once.
  const int stretch = (len + kSelectThreads - 1) / kSelectThreads * 64;
  const int start = min(wave * stretch, len), stop = min(start + stretch, len), steps = (stop - start + 63) / 64;
  auto weight = [&](int j) { return w[min(j, weights - 1)]; };  // (a load that nothing branches around)
  auto key = [&](int j, float x) {
    return j < a.sinks || j >= len - a.recent ? kAlways : j < weights ? weight_key(x) : 0u;
  };
  const bool holds = stretch <= 64 * kOwnKeys;
  uint32_t held[kOwnKeys];
  if (holds) {
    float x[kOwnKeys];
#pragma unroll
    for (int i = 0; i < kOwnKeys; ++i) x[i] = weight(min(start + 64 * i, len) + lane);
#pragma unroll
    for (int i = 0; i < kOwnKeys; ++i) held[i] = key(start + 64 * i + lane, x[i]);
  }
  auto each = [&](auto f) {  // f(token, key), all lanes of a step together; some are behind `stop`
    if (holds) {
#pragma unroll
      for (int i = 0; i < kOwnKeys; ++i)
        if (i < steps) f(start + 64 * i + lane, held[i]);
      return;
    }
    for (int i = 0; i < steps; i += kAtOnce) {
      float x[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) x[u] = weight(start + 64 * (i + u) + lane);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        if (i + u < steps) f(start + 64 * (i + u) + lane, key(start + 64 * (i + u) + lane, x[u]));
    }
  };
  // the key t of the last kept token: `need` of key t are kept, the first ones, and all above
  uint32_t need = a.keep, t = 0;
  for (int left = 32; left > 0;) {
    const int bits = left == 10 ? 10 : 11, shift = left - bits;
    bins[tid] = bins[tid + kSelectThreads] = 0;
    __syncthreads();
    each([&](int j, uint32_t k) {
      if (j < stop && (left == 32 || k >> left == t)) atomicAdd(&bins[k >> shift & ((1u << bits) - 1)], 1u);
    });
    __syncthreads();
    // from the largest bin down: that in which the count passes `need`
    const int top = kBins - 1 - 2 * tid;
    const uint32_t c0 = bins[top], c1 = bins[top - 1], in_wave = scan64(c0 + c1);
    if (lane == 63) sums[wave] = in_wave;
    __syncthreads();
    uint32_t upto = in_wave;
#pragma unroll
    for (int i = 0; i < kSelectWaves; ++i) upto += i < wave ? sums[i] : 0;
    const uint32_t from = upto - c0 - c1;
    if (from < need && need <= upto) {
      chosen = need <= from + c0 ? top : top - 1;
      before = need <= from + c0 ? from : from + c0;
    }
    __syncthreads();
    t = t << bits | chosen;
    need -= before;
    left = shift;
  }
  int sure = 0, maybe = 0;
  each([&](int j, uint32_t k) {
    sure += __popcll(__ballot(j < stop && k > t));
    maybe += __popcll(__ballot(j < stop && k == t));
  });
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
  each([&](int j, uint32_t k) {
    const bool over = j < stop && k > t, same = j < stop && k == t;
    const uint64_t o = __ballot(over), e = __ballot(same);
    const int rank = maybe + lanes_before(e);
    const int at = sure + lanes_before(o) + min(rank, (int)need);
    // (weights that something else writes meanwhile put nothing behind the row)
    if ((over || (same && rank < (int)need)) && at < n) kept[at] = j;
    sure += __popcll(o);
    maybe += __popcll(e);
  });
  if (!moved) return;
  __syncthreads();  // kept is there
  for (int i = tid; i < n; i += kSelectThreads) {
    const int j = kept[i];
    moved[i] = j < weights ? w[min(max(j, 0), weights - 1)] : 0.f;
  }
}

constexpr int kEvictThreads = 256;

template <int FMT, int D>
__global__ __launch_bounds__(kEvictThreads) void k_evict_move(KvView kv, nx_kv_batch b, EvictArgs a, int groups,
                                                              long first) {
  using Bits = std::conditional_t<FMT == NX_KV_INT8, uint8_t, uint16_t>;
  typedef uint32_t Chunk __attribute__((ext_vector_type(FMT == NX_KV_INT8 ? 2 : 4)));  // 8 elements
  __shared__ long from[kKvGroup];  // the tokens' groups in the pool, -1: none
  __shared__ int in_group[kKvGroup];
  __shared__ int run[kKvGroup + 1], runs;  // the first token of each run that came out of one value chunk
  __shared__ __align__(16) Bits values[kKvGroup * D];
  const long item = first + blockIdx.x, tile = item / groups;
  const int s = (int)(tile / kv.heads), head = (int)(tile % kv.heads), t0 = (int)(item % groups) * kKvGroup;
  const int len = evict_len(kv, b, s), n = min(len, a.keep), tid = threadIdx.x;
  if (t0 >= n) return;
  nx_kv_batch to = b;
  to.max_pages = a.to_max_pages;
  to.pages = a.to_pages;
  const long group = kv_group(kv, to, s, head, t0);
  if (group < 0) return;
  if (tid < kKvGroup) {
    const int j = t0 + tid < n ? a.kept[(size_t)tile * a.keep + t0 + tid] : -1;
    // (a number that something else wrote there names no token)
    const long g = j >= 0 && j < len ? kv_group(kv, b, s, head, j & ~(kKvGroup - 1)) : -1;
    from[tid] = g;
    in_group[tid] = j & (kKvGroup - 1);
    const int chunk = g >= 0 ? j >> 3 : -1;
    const int before = __shfl_up(chunk, 1, 64);  // (all 32 lanes: one that is not there hands nothing over)
    const uint32_t starts = (uint32_t)__ballot(tid == 0 || chunk != before);
    if (starts >> tid & 1) run[__popc(starts & ((1u << tid) - 1))] = tid;
    if (tid == 0) {
      runs = __popc(starts);
      run[runs] = kKvGroup;
    }
    if constexpr (FMT == NX_KV_INT8) {
      kv.ks[group * kKvGroup + tid] = g >= 0 ? kv.ks[g * kKvGroup + in_group[tid]] : 0.f;
      kv.vs[group * kKvGroup + tid] = g >= 0 ? kv.vs[g * kKvGroup + in_group[tid]] : 0.f;
    }
  }
  __syncthreads();
  // keys: chunks of eight elements of a token, in registers until the values are on their way too
  constexpr int kKeys = (kKvGroup * D / 8 + kEvictThreads - 1) / kEvictThreads, kAhead = 4;
  Chunk x[kKeys];
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    const int c = min(tid + i * kEvictThreads, kKvGroup * D / 8 - 1), t = kv_token(FMT, c & (kKvGroup - 1));
    x[i] = reinterpret_cast<const Chunk *>(kv.k)[max(from[t], 0L) * (kKvGroup * D / 8) + (c & ~(kKvGroup - 1)) +
                                                 kv_row(FMT, in_group[t])];
  }
  // values: each chunk of eight tokens that any of these lay in, once, and its kept elements to
  // their places (element by element out of the cache: 62 us, not 44, for 23 INT8 sequences)
  for (int c0 = tid; c0 < runs * D; c0 += kAhead * kEvictThreads) {
    Chunk y[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = min(c0 + u * kEvictThreads, runs * D - 1), r = c / D, t = run[r];
      y[u] = reinterpret_cast<const Chunk *>(kv.v)[max(from[t], 0L) * (kKvGroup * D / 8) + (in_group[t] >> 3) * D + (c - r * D)];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + u * kEvictThreads, r = min(c, runs * D - 1) / D, d = c - r * D;
      const int last = c < runs * D ? run[r + 1] : 0;
      const bool there = from[run[r]] >= 0;
      for (int t = run[r]; t < last; ++t) {
        const int i = in_group[t] & 7;
        uint32_t word;
        if constexpr (FMT == NX_KV_INT8)
          word = (i & 4 ? y[u].y : y[u].x) >> 8 * (i & 3);
        else
          word = (i & 4 ? (i & 2 ? y[u].w : y[u].z) : (i & 2 ? y[u].y : y[u].x)) >> 16 * (i & 1);
        values[kv_value_at(D, t, d)] = there ? (Bits)word : (Bits)0;
      }
    }
  }
  Chunk *k = reinterpret_cast<Chunk *>(kv.k) + group * (kKvGroup * D / 8);
  Chunk *v = reinterpret_cast<Chunk *>(kv.v) + group * (kKvGroup * D / 8);
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    const int c = tid + i * kEvictThreads;
    if (c < kKvGroup * D / 8) k[c] = from[kv_token(FMT, c & (kKvGroup - 1))] >= 0 ? x[i] : Chunk(0);
  }
  __syncthreads();
  for (int c = tid; c < kKvGroup * D / 8; c += kEvictThreads) v[c] = reinterpret_cast<const Chunk *>(values)[c];
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
  NX_TRY(refuse(evict_check(b, kv->page_tokens, kv->heads, a, host)));
  if (b->num_seqs == 0) return NX_OK;
  if (!host) return evict_dev(c, kv, *b, a);
  NX_TRY(refuse(evict_check_tables(*b, kv->pages, kv->page_tokens, a, kv->heads)));
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
  NX_TRY(upload_weights(c, static_cast<float *>(pm), width, a.mass, a.mass_stride,
                        weight_rows(b->num_seqs, kv->heads, [&](int s) { return (size_t)b->kv_len[s]; })));
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
