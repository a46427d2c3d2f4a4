// nx_kv.hip — the paged key/value cache: its pages, writing tokens into them
// (quantised to the cache's format) and reading them back.
//
// Both kernels move each value once: they are bound by memory, and a workgroup
// takes one head's group of 32 tokens (nx_kv_plan.hpp), turning rows of f32 into
// the group's operand order, or back, through LDS, so that both sides are whole
// 16-byte runs.
//
// Four waves have the keys and four the values, and each side waits for its own rows only
// (all for one, then all for the other: 46 us against 42 below).  4 heads of 128, two
// sequences with 8191 new tokens each: INT8 84 MB written in 19 us and read in 15.5, 4.4
// and 5.5 TB/s; F16 101 MB in 17.8 and 17.1, 5.6 and 5.9 (one after the other, out of the
// caches in part); a large copy reaches 4.7.  Single tokens on 8 heads are launches and two
// round trips: F16, one 3.3 us written and 3.6 read, 61 of them 3.9 and 4.4; INT8, one 5.4 and
// 3.6, 61 of them 6.6 and 4.4.  INT8 writes take 2 to 3 us more: a row's maximum over its
// lanes, the division, and values that leave as single bytes.
#include <hip/hip_runtime.h>

#include "nx_kv_dev.hpp"

namespace nx {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// x / s rounded to nearest, ties to even, from the exact quotient: n = rint of
// the rounded quotient is off by one at most, and x - n s is exact (both are
// multiples of a last place of x or s and |x - n s| < s), so comparing it with
// s / 2 decides as the quotient would.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  float n = rintf(x * inv);
  const float r = fmaf(-n, s, x), h = 0.5f * s;
  const bool odd = ((int)n & 1) != 0;
  if (r > h || (r == h && odd)) n += 1.f;
  if (r < -h || (r == -h && odd)) n -= 1.f;
  return (int)n;
}

// 8 threads of a token: float4 `4 (sub + 8 j)` of its row in v[j]
template <int D>
__device__ __forceinline__ void load_row(const float *row, int sub, bool wide, float4 (&v)[D / 32]) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const float *p = row + 4 * (sub + 8 * j);
    v[j] = wide ? *reinterpret_cast<const float4 *>(p) : float4{p[0], p[1], p[2], p[3]};
  }
}

// The row's values in the cache's format into `tile` (a group in its layout).
// Returns the row's scale (INT8).
template <int FMT, int D, bool KEYS>
__device__ __forceinline__ float stage_row(const float4 (&v)[D / 32], int t, int sub,
                                           kv_elem<FMT> *tile) {
  float scale = 0.f, inv = 0.f;
  bool fine = true;
  if constexpr (FMT == NX_KV_INT8) {
    float mx = 0.f;  // (a maximum loses NaNs)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      mx = fmaxf(fmaxf(mx, fmaxf(fabsf(v[j].x), fabsf(v[j].y))), fmaxf(fabsf(v[j].z), fabsf(v[j].w)));
      fine = fine && __builtin_isfinite(v[j].x) && __builtin_isfinite(v[j].y) &&
             __builtin_isfinite(v[j].z) && __builtin_isfinite(v[j].w);
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
      mx = fmaxf(mx, __shfl_xor(mx, d, 8));
      fine &= __shfl_xor((int)fine, d, 8) != 0;
    }
    scale = fine ? mx / 127.0f : NAN;
    inv = 1.0f / scale;
    // a scale so small that its inverse may not be finite, or that is itself
    // rounded far down, divides in 64 bits below
  }
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const float e[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
    const int d0 = 4 * (sub + 8 * j);
    kv_elem<FMT> q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (FMT == NX_KV_INT8) {
        if (!fine || scale == 0.f)
          q[i] = 0;
        else if (scale < 0x1p-120f)
          q[i] = (int8_t)fmin(fmax(rint((double)e[i] / (double)scale), -127.0), 127.0);
        else
          q[i] = (int8_t)code_of(e[i], scale, inv);
      } else {
        q[i] = (_Float16)e[i];
      }
    }
    if constexpr (KEYS) {  // four neighbouring elements of one chunk
      kv_elem<FMT> *o = tile + kv_key_at(FMT, t, d0);
      if constexpr (FMT == NX_KV_INT8)
        *reinterpret_cast<char4 *>(o) = make_char4(q[0], q[1], q[2], q[3]);
      else
        *reinterpret_cast<f16x4 *>(o) = f16x4{q[0], q[1], q[2], q[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) tile[kv_value_at(D, t, d0 + i)] = q[i];
    }
  }
  return scale;
}

// item of a batch: group `at` of sequence s's touched groups
__device__ __forceinline__ int touched(const KvSeq &q) {
  const int lo = max(q.first, 0);
  return q.n > 0 && q.len > lo ? (q.len - 1) / kKvGroup - lo / kKvGroup + 1 : 0;
}

// Eight waves: four for the keys, four for the values.
constexpr int kMoveWaves = kMoveThreads / 64;
static_assert(kMoveWaves == 8);

template <int FMT, int D>
__global__ __launch_bounds__(kMoveThreads) void k_kv_write(KvView kv, nx_kv_batch b, int first, const float *k,
                                                          const float *v, size_t stride, bool wide) {
  using E = kv_elem<FMT>;
  using Chunk = std::conditional_t<FMT == NX_KV_INT8, uint2, uint4>;  // 8 elements
  __shared__ __align__(16) E tile[2][kKvGroup * D];
  __shared__ long sums[kMoveWaves];
  __shared__ Place place;
  const int head = blockIdx.x % kv.heads;
  const Place at = find_item<kMoveWaves>(kv, b, first + blockIdx.x / kv.heads, touched, sums, &place);
  if (at.s < 0) return;
  const KvSeq q = at.seq;
  const int g0 = (max(q.first, 0) / kKvGroup + at.at) * kKvGroup;  // the group's first token
  const long group = kv_group(kv, b, at.s, head, g0);
  if (group < 0) return;
  // its tokens that the batch has: [lo, hi)
  const int lo = max(q.first - g0, 0), hi = min(q.len - g0, kKvGroup);

  const bool keys = threadIdx.x < 256;
  const int tid = threadIdx.x & 255, t = tid >> 3, sub = tid & 7;
  if (t >= lo && t < hi) {
    const size_t row = (size_t)(q.row + (g0 + t - q.first)) * stride + (size_t)head * D;
    float4 r[D / 32];
    load_row<D>((keys ? k : v) + row, sub, wide, r);
    const float s = keys ? stage_row<FMT, D, true>(r, t, sub, tile[0]) : stage_row<FMT, D, false>(r, t, sub, tile[1]);
    if (FMT == NX_KV_INT8 && sub == 0) (keys ? kv.ks : kv.vs)[group * kKvGroup + t] = s;
  }
  __syncthreads();
  if (keys) {
    Chunk *gk = reinterpret_cast<Chunk *>(kv.k) + group * (kKvGroup * D / 8);
    for (int c = tid; c < kKvGroup * D / 8; c += 256) {
      const int token = kv_token(FMT, c & (kKvGroup - 1));
      if (token >= lo && token < hi) gk[c] = reinterpret_cast<const Chunk *>(tile[0])[c];
    }
    return;
  }
  E *gv = reinterpret_cast<E *>(kv.v) + group * (kKvGroup * D);
  for (int c = tid; c < kKvGroup * D / 8; c += 256) {
    // a value chunk: tokens t0 .. t0 + 7 of one element; other tokens of it may
    // be in the cache already
    const int t0 = c / D * 8;
    if (t0 >= lo && t0 + 8 <= hi) {
      reinterpret_cast<Chunk *>(gv)[c] = reinterpret_cast<const Chunk *>(tile[1])[c];
    } else {
      for (int i = max(lo - t0, 0); i < min(hi - t0, 8); ++i) gv[8 * c + i] = tile[1][8 * c + i];
    }
  }
}

template <int FMT, int D>
__global__ __launch_bounds__(kMoveThreads) void k_kv_read(KvView kv, nx_kv_batch b, int first, float *k, float *v,
                                                         size_t stride, bool wide) {
  using E = kv_elem<FMT>;
  using Chunk = std::conditional_t<FMT == NX_KV_INT8, uint2, uint4>;
  __shared__ __align__(16) E tile[2][kKvGroup * D];
  __shared__ long sums[kMoveWaves];
  __shared__ Place place;
  const int head = blockIdx.x % kv.heads;
  // rows without a token (before the first, behind the table) are read as zeros:
  // items cover the rows, in the groups that their tokens would have
  const Place at = find_item<kMoveWaves>(
      kv, b, first + blockIdx.x / kv.heads,
      [](const KvSeq &q) { return q.n > 0 ? ((q.first + q.n - 1) >> 5) - (q.first >> 5) + 1 : 0; }, sums, &place);
  if (at.s < 0) return;
  const KvSeq q = at.seq;
  const int g0 = ((q.first >> 5) + at.at) * kKvGroup;
  const bool there = g0 >= 0 && g0 < (b.max_pages << kv.page_log2);
  const long group = there ? kv_group(kv, b, at.s, head, g0) : -1;
  const int lo = max(q.first - g0, 0), hi = min(q.first + q.n - g0, kKvGroup);
  const bool keys = threadIdx.x < 256;
  const int tid = threadIdx.x & 255, t = tid >> 3, sub = tid & 7;
  float scale = 1.f;
  if (group >= 0) {
    if (FMT == NX_KV_INT8 && t >= lo && t < hi) scale = (keys ? kv.ks : kv.vs)[group * kKvGroup + t];
    const Chunk *from = reinterpret_cast<const Chunk *>(keys ? kv.k : kv.v) + group * (kKvGroup * D / 8);
    Chunk *to = reinterpret_cast<Chunk *>(tile[keys ? 0 : 1]);
#pragma unroll
    for (int j = 0; j < kKvGroup * D / 8 / 256; ++j) {
      const int c = tid + 256 * j, token = kv_token(FMT, c & (kKvGroup - 1)), t0 = c / D * 8;
      if (keys ? token >= lo && token < hi : t0 + 8 > lo && t0 < hi) to[c] = from[c];
    }
    if constexpr (kKvGroup * D / 8 % 256 != 0) {
      const int c = tid + kKvGroup * D / 8 / 256 * 256, token = kv_token(FMT, c & (kKvGroup - 1)), t0 = c / D * 8;
      if (c < kKvGroup * D / 8 && (keys ? token >= lo && token < hi : t0 + 8 > lo && t0 < hi)) to[c] = from[c];
    }
  }
  __syncthreads();
  if (t < lo || t >= hi) return;
  float *out = (keys ? k : v) + (size_t)(q.row + (g0 + t - q.first)) * stride + (size_t)head * D;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const int d0 = 4 * (sub + 8 * j);
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const E x = keys ? tile[0][kv_key_at(FMT, t, d0 + i)] : tile[1][kv_value_at(D, t, d0 + i)];
      e[i] = group >= 0 ? (float)x * scale : 0.f;
    }
    if (wide) {
      *reinterpret_cast<float4 *>(out + d0) = float4{e[0], e[1], e[2], e[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) out[d0 + i] = e[i];
    }
  }
}

static bool wide_rows(const void *a, const void *b, size_t stride) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0 && stride % 4 == 0;
}

static int kv_move_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch &b, const float *rk,
                       const float *rv, float *wk, float *wv, size_t stride, bool write) {
  const long groups = kv_touched_groups(b.num_seqs, b.num_tokens), at_once = kv_groups_at_once(kv->heads);
  const KvView view = view_of(kv);
  for (long first = 0; first < groups; first += at_once) {
    const dim3 grid((uint32_t)(std::min(groups - first, at_once) * kv->heads)), block(kMoveThreads);
    NX_TRY(launch(c, write ? "kv_write" : "kv_read", [&] {
      with_kernel(kv, [&](auto fmt, auto D) {
        if (write)
          go(c, k_kv_write<fmt(), D()>, grid, block, 0, view, b, (int)first, rk, rv, stride,
             wide_rows(rk, rv, stride));
        else
          go(c, k_kv_read<fmt(), D()>, grid, block, 0, view, b, (int)first, wk, wv, stride,
             wide_rows(wk, wv, stride));
      });
    }));
  }
  return NX_OK;
}

int refuse_capture(nx_ctx *c) {
  hipStreamCaptureStatus status;
  if (hipStreamIsCapturing(c->stream, &status) == hipSuccess && status == hipStreamCaptureStatusNone)
    return NX_OK;
  (void)hipGetLastError();
  return fail(NX_ERR_UNSUPPORTED, "a context's first cache or attention call, and every cache, is made "
                                  "outside of stream capture");
}

int kv_check_call(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b) {
  if (!c) return fail(NX_ERR_INVALID_ARG, "null context");
  NX_HIP(hipSetDevice(c->device));
  if (!kv) return fail(NX_ERR_INVALID_ARG, "null cache");
  if (kv->device != c->device)
    return fail(NX_ERR_INVALID_ARG, "the cache lives on device " + std::to_string(kv->device) +
                                        ", the context on " + std::to_string(c->device));
  return refuse(kv_check_batch(b, kv->page_tokens));
}

int kv_upload_batch(nx_ctx *c, const nx_kv_batch &b, nx_kv_batch *dev) {
  const size_t S = b.num_seqs, table = S * b.max_pages;
  void *p = nullptr;
  NX_TRY(ws_get(c, WS_KV_BATCH, (2 * S + 1 + table) * 4, &p));
  int32_t *d = static_cast<int32_t *>(p);
  NX_HIP(hipMemcpyAsync(d, b.row_start, (S + 1) * 4, hipMemcpyHostToDevice, c->stream));
  NX_HIP(hipMemcpyAsync(d + S + 1, b.kv_len, S * 4, hipMemcpyHostToDevice, c->stream));
  NX_HIP(hipMemcpyAsync(d + 2 * S + 1, b.pages, table * 4, hipMemcpyHostToDevice, c->stream));
  *dev = b;
  dev->row_start = d;
  dev->kv_len = d + S + 1;
  dev->pages = d + 2 * S + 1;
  return NX_OK;
}

static int kv_move(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, const float *rk,
                   const float *rv, float *wk, float *wv, size_t stride, bool write, bool host) {
  NX_TRY(kv_check_call(c, kv, b));
  const long width = (long)kv->heads * kv->D;
  if (b->num_seqs == 0 || b->num_tokens == 0) return NX_OK;
  if (write ? !rk || !rv : !wk || !wv) return fail(NX_ERR_INVALID_ARG, "null buffer");
  if (stride > (size_t)1 << 40) return fail(NX_ERR_UNSUPPORTED, "row stride above 2^40");
  NX_TRY(refuse(kv_check_rows("key and value", (long)stride, width)));
  if (!host) return kv_move_dev(c, kv, *b, rk, rv, wk, wv, stride, write);
  NX_TRY(refuse(kv_check_tables(*b, kv->pages, kv->page_tokens, false, write)));
  // rows are packed on the device; padding rows do not travel
  const size_t rows = b->row_start[b->num_seqs];
  if (rows == 0) return NX_OK;
  nx_kv_batch dev;
  NX_TRY(kv_upload_batch(c, *b, &dev));
  void *dk, *dv;
  NX_TRY(ws_get(c, WS_XIN, rows * width * 4, &dk));
  NX_TRY(ws_get(c, WS_OUT, rows * width * 4, &dv));
  float *fk = static_cast<float *>(dk), *fv = static_cast<float *>(dv);
  const size_t line = (size_t)width * 4, pitch = stride * 4;
  if (write) {
    NX_HIP(hipMemcpy2DAsync(fk, line, rk, pitch, line, rows, hipMemcpyHostToDevice, c->stream));
    NX_HIP(hipMemcpy2DAsync(fv, line, rv, pitch, line, rows, hipMemcpyHostToDevice, c->stream));
  }
  NX_TRY(kv_move_dev(c, kv, dev, fk, fv, fk, fv, width, write));
  if (!write) {
    // rows that no sequence owns (below row_start[0]) keep what the caller had
    const size_t r0 = b->row_start[0];
    NX_HIP(hipMemcpy2DAsync(wk + r0 * stride, pitch, fk + r0 * width, line, line, rows - r0,
                            hipMemcpyDeviceToHost, c->stream));
    NX_HIP(hipMemcpy2DAsync(wv + r0 * stride, pitch, fv + r0 * width, line, line, rows - r0,
                            hipMemcpyDeviceToHost, c->stream));
  }
  NX_HIP(hipStreamSynchronize(c->stream));
  return NX_OK;
}

static int kv_create(nx_ctx *c, int fmt, int pages, int page_tokens, int heads, int D, nx_kv **out) {
  if (out) *out = nullptr;
  if (!c) return fail(NX_ERR_INVALID_ARG, "null context");
  if (!out) return fail(NX_ERR_INVALID_ARG, "null output pointer");
  NX_TRY(refuse(kv_check_geometry(fmt, pages, page_tokens, heads, D)));
  NX_HIP(hipSetDevice(c->device));
  NX_TRY(refuse_capture(c));
  NX_TRY(attn_workspace(c, nullptr));
  const size_t plane = kv_plane_bytes(fmt, pages, page_tokens, heads, D);
  const size_t scales = kv_scale_bytes(fmt, pages, page_tokens, heads);
  nx_kv *kv = new nx_kv();
  kv->ctx = c;
  kv->device = c->device;
  kv->fmt = fmt;
  kv->pages = pages;
  kv->page_tokens = page_tokens;
  kv->heads = heads;
  kv->D = D;
  // cleared once: what lies behind a sequence's last token enters products with
  // probability 0 and has to be finite for that to be 0
  auto alloc = [&](size_t bytes, void **p) {
    if (!bytes) return (int)NX_OK;
    if (hipMalloc(p, bytes) != hipSuccess) {
      (void)hipGetLastError();
      *p = nullptr;
      return fail(NX_ERR_OOM, "device allocation of " + std::to_string(bytes) + " bytes failed");
    }
    kv->device_bytes += bytes;
    NX_HIP(hipMemsetAsync(*p, 0, bytes, c->stream));
    return (int)NX_OK;
  };
  int rc = alloc(plane, reinterpret_cast<void **>(&kv->k));
  if (!rc) rc = alloc(plane, reinterpret_cast<void **>(&kv->v));
  if (!rc) rc = alloc(scales, reinterpret_cast<void **>(&kv->ks));
  if (!rc) rc = alloc(scales, reinterpret_cast<void **>(&kv->vs));
  if (!rc && hipStreamSynchronize(c->stream) != hipSuccess) rc = fail(NX_ERR_DEVICE, "clearing the cache failed");
  if (rc) {
    const std::string why = nx_last_error();
    nx_kv_destroy(kv);
    return fail(rc, why);
  }
  *out = kv;
  return NX_OK;
}

}  // namespace nx

using namespace nx;

extern "C" {

int nx_kv_create(nx_ctx *c, int fmt, int pages, int page_tokens, int heads, int D, nx_kv **out) {
  return guarded([&] { return kv_create(c, fmt, pages, page_tokens, heads, D, out); });
}

int nx_kv_info(const nx_kv *kv, int *fmt, int *pages, int *page_tokens, int *heads, int *D, size_t *bytes) {
  if (!kv) return fail(NX_ERR_INVALID_ARG, "null cache");
  if (fmt) *fmt = kv->fmt;
  if (pages) *pages = kv->pages;
  if (page_tokens) *page_tokens = kv->page_tokens;
  if (heads) *heads = kv->heads;
  if (D) *D = kv->D;
  if (bytes) *bytes = kv->device_bytes;
  return NX_OK;
}

int nx_kv_destroy(nx_kv *kv) {
  if (!kv) return NX_OK;
  (void)hipSetDevice(kv->device);
  for (void *p : {(void *)kv->k, (void *)kv->v, (void *)kv->ks, (void *)kv->vs})
    if (p) (void)hipFree(p);
  delete kv;
  return NX_OK;
}

int nx_kv_write(nx_ctx *c, nx_kv *kv, const nx_kv_batch *b, const float *k, const float *v, size_t stride) {
  return guarded([&] { return kv_move(c, kv, b, k, v, nullptr, nullptr, stride, true, true); });
}
int nx_kv_write_dev(nx_ctx *c, nx_kv *kv, const nx_kv_batch *b, const float *k, const float *v,
                    size_t stride) {
  return guarded([&] { return kv_move(c, kv, b, k, v, nullptr, nullptr, stride, true, false); });
}
int nx_kv_read(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, float *k, float *v, size_t stride) {
  return guarded([&] { return kv_move(c, kv, b, nullptr, nullptr, k, v, stride, false, true); });
}
int nx_kv_read_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch *b, float *k, float *v, size_t stride) {
  return guarded([&] { return kv_move(c, kv, b, nullptr, nullptr, k, v, stride, false, false); });
}

}  // extern "C"
