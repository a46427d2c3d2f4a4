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

namespace nx {

struct AttnCall {
  const float *q;
  float *out;
  size_t q_stride, out_stride;
  int heads, group;  // query heads, and those that share a key/value head
  float scale;
  int window, sinks;
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

template <int FMT, int D>
__global__ __launch_bounds__(256) void k_attn_rows(KvView kv, nx_kv_batch b, AttnCall a) {
  __shared__ int owner;
  const int row = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int seq = find_row(b, row, kv.page_log2, &owner);
  if (seq < 0 || h >= a.heads) return;
  const KvSeq s = kv_seq(b, seq, kv.page_log2);
  attn_row<FMT, D>(kv, b, a, s, seq, h / a.group, s.first + (row - s.row),
                   a.q + row * a.q_stride + (size_t)h * D, a.out + row * a.out_stride + (size_t)h * D);
}

int attn_workspace(nx_ctx *c, void **out) {
  void *p;
  NX_TRY(ws_get(c, WS_ATTN, 256, &p));
  if (out) *out = p;
  return NX_OK;
}

static int attention_dev(nx_ctx *c, const nx_kv *kv, const nx_kv_batch &b, const AttnCall &a) {
  const dim3 grid(b.num_tokens, (a.heads + 3) / 4);
  return launch(c, "attention", [&] {
    with_kernel(kv, [&](auto fmt, auto D) {
      go(c, k_attn_rows<fmt(), D()>, grid, dim3(256), 0, view_of(kv), b, a);
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
  const size_t width = (size_t)heads * kv->D;
  if (q_stride > (size_t)1 << 40 || out_stride > (size_t)1 << 40)
    return fail(NX_ERR_UNSUPPORTED, "row stride above 2^40");
  NX_TRY(refuse(kv_check_rows("query", (long)q_stride, (long)width)));
  NX_TRY(refuse(kv_check_rows("output", (long)out_stride, (long)width)));
  AttnCall a{q, out, q_stride, out_stride, heads, heads / kv->heads, scale, window, sinks};
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
