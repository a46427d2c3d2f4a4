// nx_logprobs.hip — log probabilities, entropy and the likeliest tokens of rows of logits.
//
//   l = m + log sum_j e^(x_j - m),   entropy = log S - W / S,  S = sum_j e^(x_j - m),
//   W = sum_j e^(x_j - m) (x_j - m),
// with a running m, the maximum of what was read or up to 1 below: one pass over the logits, which memory bounds.
// Where few rows do not fill the card, several workgroups share a row, and the last of them to
// end puts their sums together in the order of the parts.
//
// The likeliest tokens in the same pass: a wave keeps those that passed a threshold in LDS, as
// keys (value, then lower id first) that are all distinct.  The first threshold is what `top` of the
// lanes' own maxima reach; when the list is full, the `top` largest stay and the least of them is
// the next, so most steps pass nothing and cost one comparison with their maximum.
//
// 2039 rows of 100003 with the likeliest: 147 us for 815 MB (5.5 TB/s).  61 rows of 131072 with
// five: 17 us for 32 MB, and one row of 32000 with 20: 13 us, in its parts' dependent steps (a
// first threshold, a list, the join).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "nx_device.hpp"
#include "nx_internal.hpp"
#include "nx_kv_dev.hpp"
#include "nx_step_plan.hpp"

namespace nx {

struct LogprobCall {
  const float *x;
  size_t stride;
  const int32_t *tokens;
  float *logprobs, *entropy, *top_logprobs;
  int32_t *top_ids;
  int first;  // the launch's first row
  int vocab, given, top;
  RowSplit split;
  int *done;       // [rows] parts that are written, 0 between calls
  uint64_t *part;  // [rows][parts] records
};

constexpr int kLogprobWaves = 4, kLogprobThreads = 64 * kLogprobWaves;
constexpr int kHeld = 512;               // keys of a wave's list
constexpr int kStep = 64 * 4;            // of a step of its lanes, at most; a few more may come behind the last
constexpr int kAhead = 4;                // steps on their way
constexpr int kRecord = 3 + kMaxTop;     // of a part: S, W, m, its keys
constexpr float kLowest = -3.4028234663852886e38f, kLog2e1 = 1.4426950408889634f;

// orders as the value (-0 is 0); above 0 for anything but NaNs
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __uint_as_float(order ^ ((int)order < 0 ? 0x80000000u : 0xffffffffu));
}
// then by the lower id
__device__ __forceinline__ uint64_t key_of(float x, int id) { return (uint64_t)order_of(x) << 32 | (uint32_t)~id; }
__device__ __forceinline__ float value_of(uint64_t key) { return value_of((uint32_t)(key >> 32)); }
__device__ __forceinline__ int id_of(uint64_t key) { return (int)~(uint32_t)key; }

// A t that k of the lanes' N keys reach and no more than have to: the largest such t, found bit by
// bit, or its leading bits, where they tell those k apart (0: there are no others).  Of all, `reach`
// are not 0, k or more.
template <int N, typename K>
__device__ __forceinline__ K kth_of(const K (&key)[N], int k, int reach) {
  K t = 0;
  for (int bit = 8 * sizeof(K) - 1; bit >= 0 && reach != k; --bit) {
    const K with = t | (K)1 << bit;
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __popcll(__ballot(key[i] >= with));
    if (count < k) continue;
    t = with;
    reach = count;
  }
  return t;
}

// Leaves the k largest of n <= 64 R keys (0: none) in a list, in no order; all lanes of a wave.
template <int R>
__device__ __forceinline__ void keep_some(uint64_t *list, int &n, int k) {
  const int lane = threadIdx.x & 63;
  wave_handoff();
  uint64_t key[R];
#pragma unroll
  for (int i = 0; i < R; ++i) key[i] = lane + 64 * i < n ? list[lane + 64 * i] : 0;
  const uint64_t t = kth_of(key, k, n);
  wave_handoff();
  int at = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const bool stays = key[i] >= t && key[i] != 0;
    const uint64_t mask = __ballot(stays);
    if (stays) list[at + lanes_before(mask)] = key[i];
    at += __popcll(mask);
  }
  wave_handoff();
  n = at;
}
// (as many registers as the keys take: one row of 32000 14 us otherwise, not 13, 61 of 131072 20, not 17)
__device__ __forceinline__ void keep_top(uint64_t *list, int &n, int k) {
  if (n <= k) return;
  if (n <= 64)
    keep_some<1>(list, n, k);
  else if (n <= 128)
    keep_some<2>(list, n, k);
  else
    keep_some<kHeld / 64>(list, n, k);
}

// Sums of many terms in 64 bits, a step's own in 32: equal terms all round the same way, so in 32 bits 2^20 equal
// logits behind a largest one left an entropy four times the documented bound away.
struct Sums {
  float m;
  double s, w;
};
// w's terms e (x - m), where e is 0 and x - m may be infinite
__device__ __forceinline__ float far(float d) { return fmaxf(d, -1e4f); }
// takes the sums to a larger m
__device__ __forceinline__ void raise(Sums &a, float m) {
  const float d = a.m - m;
  const double f = __builtin_amdgcn_exp2f(d * kLog2e1);
  a.w = (a.w + far(d) * a.s) * f;
  a.s *= f;
  a.m = m;
}
// op over the wave's lanes, a commutative one, in all of them: neighbours, pairs, runs of 4, 8, 16 and 32
template <typename T, typename Op>
__device__ __forceinline__ T over_wave(T v, Op op) {
  constexpr int W = sizeof(T) / 4;
  struct Words {
    uint32_t w[W];
  };
  auto with_lane = [&](auto ctrl) {
    Words x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < W; ++i) x.w[i] = __builtin_amdgcn_update_dpp(0, x.w[i], ctrl(), 0xf, 0xf, true);
    v = op(v, __builtin_bit_cast(T, x));
  };
  with_lane(std::integral_constant<int, 0xb1>());   // quad_perm 1, 0, 3, 2
  with_lane(std::integral_constant<int, 0x4e>());   // quad_perm 2, 3, 0, 1
  with_lane(std::integral_constant<int, 0x141>());  // row_half_mirror
  with_lane(std::integral_constant<int, 0x140>());  // row_mirror
  auto with_run = [&](auto swap) {
    const Words x = __builtin_bit_cast(Words, v);
    Words a, b;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const auto both = swap(x.w[i]);
      a.w[i] = both[0];
      b.w[i] = both[1];
    }
    v = op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
  };
  with_run([](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false); });
  with_run([](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false); });
  return v;
}
// (the maximum first, then plain sums: an exponential of each lane, not one of each step)
__device__ __forceinline__ Sums across(Sums a) {
  raise(a, over_wave(a.m, [](float x, float y) { return fmaxf(x, y); }));
  auto sum = [](double x, double y) { return x + y; };
  return {a.m, over_wave(a.s, sum), over_wave(a.w, sum)};
}
// m stays where the largest logit is at most 1 above it: rows that rise by little are not rounded with every step.
// (A branch around raise: 154 us for 2039 rows of 100003, not 151.)
template <int N>
__device__ __forceinline__ void add(Sums &a, const float (&x)[N], float most) {
  raise(a, most > a.m + 1.f ? most : a.m);
  float s = 0.f, w = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = x[i] - a.m, e = __builtin_amdgcn_exp2f(y * kLog2e1);
    s += e;
    w = fmaf(e, far(y), w);
  }
  a.s += s;
  a.w += w;
}

// A wave's list of the likeliest so far.
struct List {
  uint64_t *keys;
  int n, top;
  float least;  // what a logit has to pass
  // Before the list is used: of `most`, the largest of each lane's first logits, `top` reach t, so
  // the row's own `top` do.
  __device__ __forceinline__ void begin(float most) {
    const uint32_t o[1] = {most > -INFINITY ? order_of(most) : 0u};
    // (a NaN has no order; equal ones may reach t in greater number)
    const int some = __popcll(__ballot(o[0] != 0));
    if (some < top) return;
    const uint32_t t = kth_of(o, top, some);
    // the next lower value: t itself passes (-0 is none)
    if (t != 0) least = value_of(t - (t == 0x80000000u ? 2 : 1));
  }
  // N of each lane, of ids that all come behind those taken so far, for which there is room
  template <int N, typename Id>
  __device__ __forceinline__ void push(const float (&x)[N], Id id) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint64_t mask = __ballot(x[i] > least);
      if (!mask) continue;
      if (x[i] > least) keys[n + lanes_before(mask)] = key_of(x[i], id(i));
      n += __popcll(mask);
    }
  }
  // makes room for a step's
  __device__ __forceinline__ void shrink() {
    keep_top(keys, n, top);
    // the least of those kept: what equals it has a higher id
    const int lane = threadIdx.x & 63;
    uint32_t o = lane < n ? (uint32_t)(keys[lane] >> 32) : 0xffffffffu;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) o = min(o, (uint32_t)__shfl_xor((int)o, d, 64));
    least = value_of(o);
  }
};

struct RowLds {
  uint64_t keys[kLogprobWaves][kHeld];
  uint64_t best[kHeld];
  int count[kLogprobWaves];
  Sums sums[kLogprobWaves];
  bool last;
};

// the workgroup's sums, in all of its threads, and its top keys (or none) in best[0 .. top)
__device__ __forceinline__ Sums gather(RowLds &lds, Sums mine, List &list, int top) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  mine = across(mine);
  if (top > 0 && list.n > kHeld / kLogprobWaves) keep_top(list.keys, list.n, top);
  if (lane == 0) {
    lds.sums[wave] = mine;
    lds.count[wave] = list.n;
  }
  __syncthreads();
  Sums all{kLowest, 0., 0.};
  int before = 0, n = 0;
#pragma unroll
  for (int i = 0; i < kLogprobWaves; ++i) all.m = fmaxf(all.m, lds.sums[i].m);
#pragma unroll
  for (int i = 0; i < kLogprobWaves; ++i) {
    Sums of = lds.sums[i];
    raise(of, all.m);
    all.s += of.s;
    all.w += of.w;
    before += i < wave ? lds.count[i] : 0;
    n += lds.count[i];
  }
  if (top > 0) {
    wave_handoff();
    for (int i = lane; i < list.n; i += 64) lds.best[before + i] = list.keys[i];
    __syncthreads();
    if (wave == 0) {
      keep_top(lds.best, n, top);
      if (lane >= n && lane < top) lds.best[lane] = 0;
    }
  }
  __syncthreads();
  return all;
}

__device__ __forceinline__ void write_row(const LogprobCall &a, size_t row, const Sums &all, RowLds &lds) {
  const float *x = a.x + row * a.stride, total = logf((float)all.s);
  auto logprob = [&](float v) {  // (nothing is likely in a row of masked tokens)
    return all.s == 0. || v == -INFINITY ? (all.s == all.s ? -INFINITY : NAN) : v - all.m - total;
  };
  if (threadIdx.x == 0 && a.entropy) {
    const float e = total - (float)(all.w / all.s);
    a.entropy[row] = all.s == 0. || e < 0.f ? 0.f : e;
  }
  for (int i = threadIdx.x; i < a.given; i += kLogprobThreads) {
    const int id = a.tokens[row * a.given + i];
    a.logprobs[row * a.given + i] = id >= 0 && id < a.vocab ? logprob(x[id]) : 0.f;
  }
  if (a.top == 0 || threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  uint64_t key = lane < a.top ? lds.best[lane] : 0;
  // the largest first (a bitonic sort of the lanes that have any)
  for (int size = 2; size < 2 * a.top; size <<= 1)
    for (int d = size >> 1; d > 0; d >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)key, d, 64);
      const bool larger = ((lane & d) == 0) == ((lane & size) == 0);
      key = larger == (key > other) ? key : other;
    }
  if (lane < a.top) {
    a.top_ids[row * a.top + lane] = key ? id_of(key) : -1;
    a.top_logprobs[row * a.top + lane] = key ? logprob(value_of(key)) : -INFINITY;
  }
}

__global__ __launch_bounds__(kLogprobThreads) void k_logprobs(LogprobCall a) {
  __shared__ RowLds lds;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int parts = a.split.parts, part = blockIdx.x % parts;
  const size_t row = a.first + blockIdx.x / parts;
  const float *x = a.x + row * a.stride;
  // the part's logits [lo, hi): any in front of a 16-byte boundary, whole float4, and a rest
  const int front = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) / 4 & 3), a.vocab);
  const int whole = (a.vocab - front) / 4, rest = front + 4 * whole;
  const int lo = min(part * (a.split.share / 4), whole);
  const int hi = part + 1 == parts ? whole : min(lo + a.split.share / 4, whole);
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  const f32x4 *x4 = reinterpret_cast<const f32x4 *>(x + front);

  Sums sums{kLowest, 0., 0.};
  List list{lds.keys[wave], 0, a.top, -INFINITY};
  auto single = [&](int from, int to) {  // a few logits, one of each lane
    const int i = from + lane;
    const float v[1] = {i < to ? x[i] : -INFINITY};
    add(sums, v, v[0]);
    if (a.top > 0) list.push(v, [&](int) { return i; });
  };
  if (part == 0 && wave == 0 && front > 0) single(0, front);
  constexpr f32x4 kNone = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  f32x4 next[kAhead];
  auto fetch = [&](int at) {  // (behind the part: its last ones, which are not looked at)
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      next[j] = __builtin_nontemporal_load(x4 + min(at + j * kLogprobThreads + (int)threadIdx.x, hi - 1));
  };
  if (lo < hi) fetch(lo);
  for (int at = lo; at < hi; at += kAhead * kLogprobThreads) {
    float v[4 * kAhead], all = -INFINITY;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (at + kAhead * kLogprobThreads > hi && at + j * kLogprobThreads + (int)threadIdx.x >= hi) next[j] = kNone;
      v[4 * j] = next[j].x, v[4 * j + 1] = next[j].y, v[4 * j + 2] = next[j].z, v[4 * j + 3] = next[j].w;
      all = fmaxf(all, fmaxf(fmaxf(next[j].x, next[j].y), fmaxf(next[j].z, next[j].w)));
    }
    if (at + kAhead * kLogprobThreads < hi) fetch(at + kAhead * kLogprobThreads);
    add(sums, v, all);
    if (a.top > 0 && at == lo) list.begin(all);
    if (a.top > 0 && __any(all > list.least)) {
      int count = 0;
#pragma unroll
      for (int j = 0; j < 4 * kAhead; ++j) count += __popcll(__ballot(v[j] > list.least));
      const bool fits = list.n + count <= kHeld - 4;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (!fits && list.n > kHeld - 4 - kStep) list.shrink();
        const float u[4] = {v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
        const int id = front + 4 * (at + j * kLogprobThreads + (int)threadIdx.x);
        list.push(u, [&](int i) { return id + i; });
      }
    }
  }
  if (part + 1 == parts && wave == 0 && rest < a.vocab) single(rest, a.vocab);
  // the workgroup's own; then, in the row's last workgroup, those of all
  for (bool own = true;; own = false) {
    const Sums all = gather(lds, sums, list, a.top);
    if (parts == 1 || !own) {
      write_row(a, row, all, lds);
      return;
    }
    const size_t local = blockIdx.x / parts;
    uint64_t *record = a.part + (local * parts + part) * kRecord;
    if (threadIdx.x == 0) {
      store_through(record, __builtin_bit_cast(uint64_t, all.s));
      store_through(record + 1, __builtin_bit_cast(uint64_t, all.w));
      store_through(record + 2, (uint64_t)__float_as_uint(all.m));
    }
    if ((int)threadIdx.x < a.top) store_through(record + 3 + threadIdx.x, lds.best[threadIdx.x]);
    stores_done();  // this part, before the count says so
    __syncthreads();
    if (threadIdx.x == 0) {
      lds.last = atomicAdd(&a.done[local], 1) == parts - 1;
      if (lds.last) a.done[local] = 0;  // for the next call
    }
    __syncthreads();
    if (!lds.last) return;
    // a part to each lane for the sums; to each wave in turn for its keys
    sums = {kLowest, 0., 0.};
    const uint64_t *first = a.part + local * parts * kRecord;
    if ((int)threadIdx.x < parts) {
      const uint64_t *of = first + threadIdx.x * kRecord, s = load_past(of), w = load_past(of + 1);
      sums = {__uint_as_float((uint32_t)load_past(of + 2)), __builtin_bit_cast(double, s), __builtin_bit_cast(double, w)};
    }
    list.n = 0;
    for (int i0 = wave * 64; i0 < parts * a.top; i0 += kLogprobThreads) {
      const int i = i0 + lane, p = i / a.top;
      const uint64_t key = p < parts ? load_past(first + p * kRecord + 3 + (i - p * a.top)) : 0;
      const uint64_t mask = __ballot(key != 0);
      if (list.n + 64 > kHeld) keep_top(list.keys, list.n, a.top);
      if (key) list.keys[list.n + lanes_before(mask)] = key;
      list.n += __popcll(mask);
    }
  }
}

// Memory of the split rows: of one size for every call, allocated once, never moved.
static int logprob_workspace(nx_ctx *c, void **out) {
  constexpr size_t kCounts = kLogprobWgs * sizeof(int);
  constexpr size_t kBytes = kCounts + (size_t)kLogprobWgs * kRecord * 8;
  DevBuf &ws = c->ws[WS_LOGPROBS];
  if (!ws.ptr) {
    NX_TRY(refuse_capture(c));
    void *p = nullptr;
    if (hipMalloc(&p, kBytes) != hipSuccess) {
      (void)hipGetLastError();
      return fail(NX_ERR_OOM, "device allocation of " + std::to_string(kBytes) + " bytes failed");
    }
    // counts begin at 0, and the workspace is there once they are
    if (hipMemsetAsync(p, 0, kCounts, c->stream) != hipSuccess || hipStreamSynchronize(c->stream) != hipSuccess) {
      (void)hipGetLastError();
      (void)hipFree(p);
      return fail(NX_ERR_DEVICE, "clearing the workspace of log probabilities failed");
    }
    ws = {p, kBytes};
  }
  *out = ws.ptr;
  return NX_OK;
}

static int logprobs_dev(nx_ctx *c, LogprobCall a, int rows) {
  a.split = logprob_split(rows, a.vocab);
  if (a.split.parts > 1) {
    void *p;
    NX_TRY(logprob_workspace(c, &p));
    a.done = static_cast<int *>(p);
    a.part = reinterpret_cast<uint64_t *>(a.done + kLogprobWgs);
  }
  constexpr int kRows = 1 << 22;  // of a launch, which has fewer than 2^32 threads
  for (a.first = 0; a.first < rows; a.first += kRows) {
    const int now = std::min(rows - a.first, kRows);
    NX_TRY(launch(c, "logprobs", [&] {
      go(c, k_logprobs, dim3(now * a.split.parts), dim3(kLogprobThreads), 0, a);
    }));
  }
  return NX_OK;
}

static int logprobs(nx_ctx *c, LogprobCall a, int rows, bool host) {
  if (!c) return fail(NX_ERR_INVALID_ARG, "null context");
  NX_HIP(hipSetDevice(c->device));
  NX_TRY(refuse(logprobs_check(a.x, a.stride, rows, a.vocab, a.tokens, a.given, a.logprobs, a.top, a.top_ids,
                               a.top_logprobs)));
  if (rows == 0) return NX_OK;
  if (!host) return logprobs_dev(c, a, rows);
  const size_t V = a.vocab, T = rows, n = T * a.given, m = T * a.top;
  void *px, *pt, *po;
  NX_TRY(ws_get(c, WS_LOGITS, T * V * 4, &px));
  NX_TRY(ws_get(c, WS_XIN, n * 4, &pt));
  NX_TRY(ws_get(c, WS_OUT, (n + T + 2 * m) * 4, &po));
  LogprobCall d = a;
  d.x = static_cast<const float *>(px);
  d.stride = V;
  d.tokens = static_cast<const int32_t *>(pt);
  d.logprobs = static_cast<float *>(po);
  d.entropy = d.logprobs + n;
  d.top_logprobs = d.entropy + T;
  d.top_ids = reinterpret_cast<int32_t *>(d.top_logprobs + m);
  NX_HIP(hipMemcpy2DAsync(px, V * 4, a.x, a.stride * 4, V * 4, T, hipMemcpyHostToDevice, c->stream));
  if (n) NX_HIP(hipMemcpyAsync(pt, a.tokens, n * 4, hipMemcpyHostToDevice, c->stream));
  NX_TRY(logprobs_dev(c, d, rows));
  if (n) NX_HIP(hipMemcpyAsync(a.logprobs, d.logprobs, n * 4, hipMemcpyDeviceToHost, c->stream));
  if (a.entropy) NX_HIP(hipMemcpyAsync(a.entropy, d.entropy, T * 4, hipMemcpyDeviceToHost, c->stream));
  if (m) {
    NX_HIP(hipMemcpyAsync(a.top_logprobs, d.top_logprobs, m * 4, hipMemcpyDeviceToHost, c->stream));
    NX_HIP(hipMemcpyAsync(a.top_ids, d.top_ids, m * 4, hipMemcpyDeviceToHost, c->stream));
  }
  NX_HIP(hipStreamSynchronize(c->stream));
  return NX_OK;
}

}  // namespace nx

using namespace nx;

extern "C" {

int nx_logprobs(nx_ctx *c, const float *logits, size_t stride, int rows, int vocab, const int32_t *tokens, int given,
                float *logprobs, float *entropy, int top, int32_t *top_ids, float *top_logprobs) {
  return guarded([&] {
    return nx::logprobs(c, {logits, stride, tokens, logprobs, entropy, top_logprobs, top_ids, 0, vocab, given, top}, rows,
                        true);
  });
}
int nx_logprobs_dev(nx_ctx *c, const float *logits, size_t stride, int rows, int vocab, const int32_t *tokens,
                    int given, float *logprobs, float *entropy, int top, int32_t *top_ids, float *top_logprobs) {
  return guarded([&] {
    return nx::logprobs(c, {logits, stride, tokens, logprobs, entropy, top_logprobs, top_ids, 0, vocab, given, top}, rows,
                        false);
  });
}

}  // extern "C"
