// nx_rope.hip — a step's query and key heads, normed and rotated by their tokens' positions,
// in one pass between the fused projection and the cache.
//
// A head x of D elements:   y = x w / sqrt(sum x^2 / D + eps)        (no norm: y = x)
// pair i of the first R:    (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position freq_i
//
// Every element is read once and written once: memory is the bound.  A workgroup takes one
// token, whose angles its threads work out once for all heads, while the heads' rows are on
// their way; 16 lanes have a head of 128, a lane eight elements whose pairs are its own.
// 8191 tokens of 36 heads of 128, normed: 52 us for 302 MB (5.8 TB/s; a copy of 4 GiB reaches
// 4.9).  2039 of 24 heads of 96: 10 us for 38 MB.  One token: 2.6 us, a launch.
#include <hip/hip_runtime.h>

#include "nx_device.hpp"
#include "nx_internal.hpp"
#include "nx_kv_dev.hpp"
#include "nx_step_plan.hpp"

namespace nx {

struct RopeCall {
  RopeRows x;
  const int32_t *positions;
  const float *freq, *q_norm, *k_norm;
  int first;             // the launch's first row
  int heads, all;        // query heads, and key heads behind them
  int D, R;
  bool halves;
  float eps;
};

// cos and sin of position freq.  The product has up to 55 bits; what 53 of them leave is added
// back after whole turns are taken off, so the farthest positions keep their angle to 2^-50.
__device__ __forceinline__ float2 turn_of(int position, float freq) {
  const double p = position, f = freq, t = p * f, rest = fma(p, f, -t);
  constexpr double kTurn = 6.283185307179586, kTurnRest = 2.4492935982947064e-16;
  const double k = rint(t * (1.0 / kTurn));
  const double r = (fma(-k, kTurn, t) - k * kTurnRest + rest) * 0.3183098861837907;  // in half turns, -1 .. 1
  const float hi = (float)r, lo = (float)(r - (double)hi) * 3.14159274f;
  float s, c;
  sincospif(hi, &s, &c);
  return {fmaf(-lo, s, c), fmaf(lo, c, s)};
}

// What a head's elements are multiplied by, from its lanes' sums (L of them, a power of two): first by `up`, a
// power of two that is 1 but where eps is 0 and the head all but is, whose factor f32 does not hold.
struct NormScale {
  float up, s;
};
template <int L>
__device__ __forceinline__ NormScale scale_of(double sum, int D, float eps) {
#pragma unroll
  for (int d = 1; d < L; d <<= 1) sum += __shfl_xor(sum, d, L);
  const double s = 1.0 / sqrt(sum / D + (double)eps);
  const bool large = s > 0x1p100;
  return {large ? 0x1p100f : 1.f, (float)(large ? s * 0x1p-100 : s)};
}

struct Head {
  const float *in, *w;
  float *out;
};
__device__ __forceinline__ Head head_of(const RopeCall &a, int t, int h) {
  if (h < a.heads)
    return {a.x.q + (size_t)t * a.x.q_stride + (size_t)h * a.D, a.q_norm,
            a.x.q_out + (size_t)t * a.x.q_out_stride + (size_t)h * a.D};
  h -= a.heads;
  return {a.x.k + (size_t)t * a.x.k_stride + (size_t)h * a.D, a.k_norm,
          a.x.k_out + (size_t)t * a.x.k_out_stride + (size_t)h * a.D};
}

constexpr int kRopeThreads = 256, kRopeRounds = 4;

// Rows of whole float4, D and R multiples of 8: L lanes of a head, eight elements each.  Up to
// kRopeRounds heads of a lane are on their way together (one or two at once, in as many more
// workgroups: no different, 51 and 52 us).
template <int L>
__global__ __launch_bounds__(kRopeThreads) void k_rope_wide(RopeCall a, int rounds) {
  constexpr int kHeads = kRopeThreads / L;
  __shared__ __align__(16) float2 turns[kMaxRopeHead / 2];
  const int t = a.first + blockIdx.x, u = threadIdx.x % L;
  const int h0 = blockIdx.y * rounds * kHeads + threadIdx.x / L;
  const bool rotated = 8 * u < a.R, whole = 8 * u < a.D;
  const int at0 = rotated && a.halves ? 4 * u : 8 * u, at1 = rotated && a.halves ? a.R / 2 + 4 * u : 8 * u + 4;
  float4 x[kRopeRounds][2];
#pragma unroll
  for (int r = 0; r < kRopeRounds; ++r) {
    x[r][0] = x[r][1] = float4{0.f, 0.f, 0.f, 0.f};
    const int h = h0 + r * kHeads;
    if (r < rounds && h < a.all && whole) {
      const float *in = head_of(a, t, h).in;
      x[r][0] = *reinterpret_cast<const float4 *>(in + at0);
      x[r][1] = *reinterpret_cast<const float4 *>(in + at1);
    }
  }
  if ((int)threadIdx.x < a.R / 2) turns[threadIdx.x] = turn_of(a.positions[t], a.freq[threadIdx.x]);
  __syncthreads();
  float2 turn[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) turn[i] = rotated ? turns[4 * u + i] : float2{1.f, 0.f};
#pragma unroll
  for (int r = 0; r < kRopeRounds; ++r) {
    const int h = h0 + r * kHeads;
    if (r >= rounds || h >= a.all) break;
    const Head head = head_of(a, t, h);
    float e[8] = {x[r][0].x, x[r][0].y, x[r][0].z, x[r][0].w, x[r][1].x, x[r][1].y, x[r][1].z, x[r][1].w};
    if (head.w) {
      // in 64 bits: squares of any f32 stay in range
      double sum = 0.;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fma((double)e[i], (double)e[i], sum);
      const NormScale s = scale_of<L>(sum, a.D, a.eps);
      float w[8] = {};
      if (whole) {
        const float4 w0 = *reinterpret_cast<const float4 *>(head.w + at0);
        const float4 w1 = *reinterpret_cast<const float4 *>(head.w + at1);
        w[0] = w0.x, w[1] = w0.y, w[2] = w0.z, w[3] = w0.w, w[4] = w1.x, w[5] = w1.y, w[6] = w1.z, w[7] = w1.w;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = e[i] * s.up * s.s * w[i];
    }
    if (rotated) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float &p = a.halves ? e[i] : e[2 * i], &q = a.halves ? e[4 + i] : e[2 * i + 1];
        const float y = fmaf(p, turn[i].x, -(q * turn[i].y)), z = fmaf(p, turn[i].y, q * turn[i].x);
        p = y;
        q = z;
      }
    }
    if (whole) {
      *reinterpret_cast<float4 *>(head.out + at0) = float4{e[0], e[1], e[2], e[3]};
      *reinterpret_cast<float4 *>(head.out + at1) = float4{e[4], e[5], e[6], e[7]};
    }
  }
}

// Any even D and R, at any float address: a wave has a head, a lane every 64th pair.  (Those
// 8191 tokens: 126 us, not 52; 2039 tokens of 96: 22, not 10; one token: alike.)
__global__ __launch_bounds__(kRopeThreads) void k_rope_any(RopeCall a, int per_wave) {
  constexpr int kPairs = kMaxRopeHead / 2 / 64, kWaves = kRopeThreads / 64;
  const int t = a.first + blockIdx.x, lane = threadIdx.x & 63;
  float2 turn[kPairs];
  int at0[kPairs], at1[kPairs];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const int p = lane + 64 * j;
    const bool rotated = 2 * p < a.R;
    turn[j] = rotated ? turn_of(a.positions[t], a.freq[p]) : float2{1.f, 0.f};
    at0[j] = rotated && a.halves ? p : 2 * p;
    at1[j] = rotated && a.halves ? p + a.R / 2 : 2 * p + 1;
  }
  for (int i = 0; i < per_wave; ++i) {
    const int h = (blockIdx.y * per_wave + i) * kWaves + (threadIdx.x >> 6);
    if (h >= a.all) return;
    const Head head = head_of(a, t, h);
    float2 e[kPairs];
    double sum = 0.;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      e[j] = 2 * (lane + 64 * j) < a.D ? float2{head.in[at0[j]], head.in[at1[j]]} : float2{0.f, 0.f};
      sum = fma((double)e[j].x, (double)e[j].x, fma((double)e[j].y, (double)e[j].y, sum));
    }
    const NormScale s = head.w ? scale_of<64>(sum, a.D, a.eps) : NormScale{1.f, 1.f};
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int p = lane + 64 * j;
      if (2 * p >= a.D) continue;
      const float x = head.w ? e[j].x * s.up * s.s * head.w[at0[j]] : e[j].x;
      const float y = head.w ? e[j].y * s.up * s.s * head.w[at1[j]] : e[j].y;
      const bool rotated = 2 * p < a.R;
      head.out[at0[j]] = rotated ? fmaf(x, turn[j].x, -(y * turn[j].y)) : x;
      head.out[at1[j]] = rotated ? fmaf(x, turn[j].y, y * turn[j].x) : y;
    }
  }
}

constexpr int kRopeRows = 1 << 22;  // of a launch, which has fewer than 2^32 threads

static int rope_dev(nx_ctx *c, RopeCall a, int rows) {
  uintptr_t low = 0;  // of all addresses and strides, in bytes
  if (a.heads) low |= (uintptr_t)a.x.q | (uintptr_t)a.x.q_out | a.x.q_stride * 4 | a.x.q_out_stride * 4 | (uintptr_t)a.q_norm;
  if (a.all > a.heads)
    low |= (uintptr_t)a.x.k | (uintptr_t)a.x.k_out | a.x.k_stride * 4 | a.x.k_out_stride * 4 | (uintptr_t)a.k_norm;
  const bool wide = (low & 15) == 0 && a.D % 8 == 0 && a.R % 8 == 0;
  for (a.first = 0; a.first < rows; a.first += kRopeRows) {
    const int now = std::min(rows - a.first, kRopeRows);
    auto start = [&](auto L) {
      constexpr int kHeads = kRopeThreads / L();
      const int rounds = (a.all + kHeads - 1) / kHeads, groups = (rounds + kRopeRounds - 1) / kRopeRounds;
      const int each = (rounds + groups - 1) / groups;
      go(c, k_rope_wide<L()>, dim3(now, (rounds + each - 1) / each), dim3(kRopeThreads), 0, a, each);
    };
    NX_TRY(launch(c, "qk_rope", [&] {
      constexpr int per_wave = 4, heads = per_wave * kRopeThreads / 64;
      if (!wide)
        go(c, k_rope_any, dim3(now, (a.all + heads - 1) / heads), dim3(kRopeThreads), 0, a, per_wave);
      else if (a.D <= 64)
        start(std::integral_constant<int, 8>());
      else if (a.D <= 128)
        start(std::integral_constant<int, 16>());
      else if (a.D <= 256)
        start(std::integral_constant<int, 32>());
      else
        start(std::integral_constant<int, 64>());
    }));
  }
  return NX_OK;
}

static int qk_rope(nx_ctx *c, const nx_rope *r, const int32_t *positions, int rows, int heads, int kv_heads,
                   const RopeRows &x, bool host) {
  if (!c) return fail(NX_ERR_INVALID_ARG, "null context");
  NX_HIP(hipSetDevice(c->device));
  NX_TRY(refuse(rope_check(r, positions, rows, heads, kv_heads, x)));
  if (rows == 0 || heads + kv_heads == 0) return NX_OK;
  RopeCall a{x, positions, r->freq, r->q_norm, r->k_norm, 0, heads, heads + kv_heads, r->head_dim, r->rotary_dim,
             r->style == NX_ROPE_HALVES, r->eps};
  if (!host) return rope_dev(c, a, rows);
  const size_t D = r->head_dim, wq = heads * D, wk = kv_heads * D, half = (r->rotary_dim / 2 + 3) / 4 * 4;
  void *px, *pw;
  NX_TRY(ws_get(c, WS_XIN, rows * (wq + wk) * 4, &px));
  NX_TRY(ws_get(c, WS_NORM_W, (half + 2 * ((D + 3) / 4 * 4) + rows) * 4, &pw));
  float *dx = static_cast<float *>(px), *w = static_cast<float *>(pw);
  auto up = [&](const void *from, size_t n, const void **to) {
    *to = nullptr;
    if (!from || !n) return hipSuccess;
    *to = w;
    w += (n + 3) / 4 * 4;
    return hipMemcpyAsync(const_cast<void *>(*to), from, n * 4, hipMemcpyHostToDevice, c->stream);
  };
  NX_HIP(up(r->freq, r->rotary_dim / 2, reinterpret_cast<const void **>(&a.freq)));
  NX_HIP(up(r->q_norm, D, reinterpret_cast<const void **>(&a.q_norm)));
  NX_HIP(up(r->k_norm, D, reinterpret_cast<const void **>(&a.k_norm)));
  // (the last: it may end off a multiple of 4)
  if (r->rotary_dim) {
    a.positions = reinterpret_cast<const int32_t *>(w);
    NX_HIP(hipMemcpyAsync(w, positions, (size_t)rows * 4, hipMemcpyHostToDevice, c->stream));
  }
  float *dk = dx + (size_t)rows * wq;
  a.x = {dx, dk, dx, dk, wq, wk, wq, wk};
  if (heads) NX_HIP(hipMemcpy2DAsync(dx, wq * 4, x.q, x.q_stride * 4, wq * 4, rows, hipMemcpyHostToDevice, c->stream));
  if (kv_heads)
    NX_HIP(hipMemcpy2DAsync(dk, wk * 4, x.k, x.k_stride * 4, wk * 4, rows, hipMemcpyHostToDevice, c->stream));
  NX_TRY(rope_dev(c, a, rows));
  if (heads)
    NX_HIP(hipMemcpy2DAsync(x.q_out, x.q_out_stride * 4, dx, wq * 4, wq * 4, rows, hipMemcpyDeviceToHost, c->stream));
  if (kv_heads)
    NX_HIP(hipMemcpy2DAsync(x.k_out, x.k_out_stride * 4, dk, wk * 4, wk * 4, rows, hipMemcpyDeviceToHost, c->stream));
  NX_HIP(hipStreamSynchronize(c->stream));
  return NX_OK;
}

}  // namespace nx

using namespace nx;

extern "C" {

int nx_qk_rope(nx_ctx *c, const nx_rope *rope, const int32_t *positions, int rows, int heads, int kv_heads,
               const float *q, size_t q_stride, const float *k, size_t k_stride, float *q_out, size_t q_out_stride,
               float *k_out, size_t k_out_stride) {
  return guarded([&] {
    return qk_rope(c, rope, positions, rows, heads, kv_heads,
                   {q, k, q_out, k_out, q_stride, k_stride, q_out_stride, k_out_stride}, true);
  });
}
int nx_qk_rope_dev(nx_ctx *c, const nx_rope *rope, const int32_t *positions, int rows, int heads, int kv_heads,
                   const float *q, size_t q_stride, const float *k, size_t k_stride, float *q_out, size_t q_out_stride,
                   float *k_out, size_t k_out_stride) {
  return guarded([&] {
    return qk_rope(c, rope, positions, rows, heads, kv_heads,
                   {q, k, q_out, k_out, q_stride, k_stride, q_out_stride, k_out_stride}, false);
  });
}

}  // extern "C"
