// nx_kv_dev.hpp — what the kernels of the paged cache (nx_kv.hip) and of the
// attention that reads it (nx_attn.hip) share: the device view of a cache and
// of a batch, and finding a workgroup's work in a batch whose lengths only the
// device knows.
#pragma once

#include <type_traits>

#include "nx_device.hpp"
#include "nx_internal.hpp"
#include "nx_kv_plan.hpp"

struct nx_kv {
  nx_ctx *ctx = nullptr;  // compared, never followed, once the cache exists
  int device = 0;
  int fmt = 0, pages = 0, page_tokens = 0, heads = 0, D = 0;
  uint8_t *k = nullptr, *v = nullptr;
  float *ks = nullptr, *vs = nullptr;  // INT8: scales [pages][heads][page_tokens]
  size_t device_bytes = 0;
};

namespace nx {

// the attention's workspace on a context: allocated once, never moved
int attn_workspace(nx_ctx *c, void **out);
// refuses what allocates and clears memory while the context's stream is captured: the graph
// would clear it again with every replay, and not before the first
int refuse_capture(nx_ctx *c);
// a context, a cache, and both on one device; then the batch's sizes
int kv_check_cache(nx_ctx *c, const nx_kv *kv);
int kv_check_call(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b);
// copies a host batch's arrays to the device; *dev describes them there
int kv_upload_batch(nx_ctx *c, const nx_kv_batch &b, nx_kv_batch *dev);

struct KvView {
  uint8_t *k, *v;
  float *ks, *vs;
  int pages, page_log2, heads;
};
inline KvView view_of(const nx_kv *kv) {
  return {kv->k, kv->v, kv->ks, kv->vs, kv->pages, __builtin_ctz(kv->page_tokens), kv->heads};
}

// One sequence of a batch, cut to what is there.
struct KvSeq {
  int row, n;  // first row, rows
  int first;   // token of row `row` (below 0 where the batch says so)
  int len;     // tokens that can be read: kv_len, at most the table's
};

__device__ __forceinline__ KvSeq kv_seq(const nx_kv_batch &b, int s, int page_log2) {
  const int r0 = min(max(b.row_start[s], 0), b.num_tokens);
  const int r1 = min(max(b.row_start[s + 1], r0), b.num_tokens);
  const int len = max(b.kv_len[s], 0);
  return {r0, r1 - r0, len - (r1 - r0), min(len, b.max_pages << page_log2)};
}

// The group of 32 tokens that holds token `first` of sequence s, as an index of
// groups over the whole pool ([pages][heads][groups of a page]); -1 if the cache has no such page.
__device__ __forceinline__ long kv_group(const KvView &kv, const nx_kv_batch &b, int s, int head,
                                         int first) {
  const int page = b.pages[(long)s * b.max_pages + (first >> kv.page_log2)];
  if (page < 0 || page >= kv.pages) return -1;
  const int in_page = (first & ((1 << kv.page_log2) - 1)) / kKvGroup;
  return (((long)page * kv.heads + head) << (kv.page_log2 - 5)) + in_page;
}

// what every lane has alike, as a scalar: addresses, bounds and branches on it
// then cost no vector registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ long uniform(long v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  return (long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 | lo);
}

// inclusive sum over the workgroup's NW waves, and the whole sum
template <int NW>
__device__ __forceinline__ long scan_wg(long v, long *sums, long &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  __syncthreads();  // the last call's reads of sums
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    v += w < wave ? sums[w] : 0;
    total += sums[w];
  }
  return v;
}

// inclusive sum over the wave's lanes
__device__ __forceinline__ uint32_t scan64(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// how many lanes of the mask come before this one
__device__ __forceinline__ int lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Which sequence holds item `item` when sequence s has count(its KvSeq) of them, at
// most 2^31 in all, and which of its items that is; s = -1 past the last one.  All threads
// of a workgroup of NW waves; up to 64 sequences each wave finds it by itself.
struct Place {
  int s, at;
  KvSeq seq;
};
template <int NW, typename Count>
__device__ __forceinline__ Place find_item(const KvView &kv, const nx_kv_batch &b, int item, Count count,
                                           long *sums, Place *lds) {
  if (b.num_seqs <= 64) {
    const int lane = threadIdx.x & 63;
    const KvSeq q = lane < b.num_seqs ? kv_seq(b, lane, kv.page_log2) : KvSeq{0, 0, 0, 0};
    const uint32_t c = count(q), upto = scan64(c);
    const uint64_t past = __ballot(upto > (uint32_t)item);
    if (!past) return {-1, 0, q};
    const int s = __builtin_ctzll(past);
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, s); };
    return {s, item - (of(upto) - of(c)), {of(q.row), of(q.n), of(q.first), of(q.len)}};
  }
  if (threadIdx.x == 0) lds->s = -1;
  long before = 0, chunk;
  for (int s0 = 0; s0 < b.num_seqs; s0 += 64 * NW) {
    const int s = s0 + (int)threadIdx.x;
    const KvSeq q = s < b.num_seqs ? kv_seq(b, s, kv.page_log2) : KvSeq{0, 0, 0, 0};
    const long c = count(q), end = before + scan_wg<NW>(c, sums, chunk);
    if (item >= end - c && item < end) *lds = {s, (int)(item - (end - c)), q};
    before += chunk;
    if (item < before) break;  // uniform: every thread has the same sums
  }
  __syncthreads();
  return *lds;
}

// Memory that workgroups of one kernel pass on, on any XCD: each has an L2 of its own,
// so these stores write through it and these loads go past it (device-scope atomics,
// relaxed).  A device-wide fence instead writes back everything that the L2 holds:
// with one per workgroup a decode batch took 442 us of attention, not 233.
template <typename T>
__device__ __forceinline__ void store_through(T *p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T load_past(const T *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// waits until this wave's stores are where they go
__device__ __forceinline__ void stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// f(format, head_dim) as constants
template <typename F>
void with_kernel(const nx_kv *kv, F f) {
  auto dims = [&](auto fmt) {
    switch (kv->D) {
    case 64: f(fmt, std::integral_constant<int, 64>()); break;
    case 96: f(fmt, std::integral_constant<int, 96>()); break;
    case 128: f(fmt, std::integral_constant<int, 128>()); break;
    default: f(fmt, std::integral_constant<int, 256>()); break;
    }
  };
  if (kv->fmt == NX_KV_INT8)
    dims(std::integral_constant<int, NX_KV_INT8>());
  else
    dims(std::integral_constant<int, NX_KV_F16>());
}

template <int FMT>
using kv_elem = std::conditional_t<FMT == NX_KV_INT8, int8_t, _Float16>;

// rows of weights (nx_step_plan.hpp's WeightRows) from the host, `from_stride` apart, to rows of `width`
template <typename Rows>
int upload_weights(nx_ctx *c, float *to, size_t width, const float *from, size_t from_stride, const Rows &r) {
  if (r.rows > 1)
    NX_HIP(hipMemcpy2DAsync(to, width * 4, from, from_stride * 4, width * 4, r.rows - 1, hipMemcpyHostToDevice, c->stream));
  if (r.rows > 0)
    NX_HIP(hipMemcpyAsync(to + (r.rows - 1) * width, from + (r.rows - 1) * from_stride, r.last * 4, hipMemcpyHostToDevice,
                          c->stream));
  return NX_OK;
}

inline int refuse(const Refusal &r) { return r ? fail(r.code, r.why) : NX_OK; }

}  // namespace nx
