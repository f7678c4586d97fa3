// Norms of queries and keys per head together with the rotation of their positions, forward and backward, and with the write to a key/value cache.
//
//   norm first:  y = R(x r w),  r = 1 / sqrt(mean(x^2) + eps)          after:  u = R x,  y = u r w,  r = 1 / sqrt(mean(u^2) + eps)
//
// R turns pairs of channels, (2i, 2i + 1) or (i, i + d/2), by the table's angle at the token's position; the table's (cos, sin) need not have length 1, so R^T below is the transpose and r
// in the second order is taken from u.  With dz = R^T dy (norm first) or dy, n = x r (or u r) and dn = dz w:
//   dw = sum dz n over tokens and heads,   dx (or du) = r (dn - n mean(dn n)),   dx = R^T du in the second order.
// All of it is fp32 with one rounding at the end; as a norm and a rotation of their own it is two roundings and, of two tensors, four launches and twice the traffic.
//
// A head row is shared by G lanes (a power of two), each with N channels of the first half and the same N of the second: in the half-split layout these are pairs, in the interleaved one
// pairs lie within the N, so that no value crosses lanes but the sums.  A group of lanes takes up to HEADS heads of one token, whose angles it keeps.
// The gains' gradients are sums in registers over all that a CTA does, then rows of a workspace that a second launch adds up, both in an order that depends on sizes alone.
//
// Bound by no one unit: with a third of the warps' places taken (registers) 64 % of the cycles issue and 4.3 TB/s flow; a value costs 18 instructions forward and 29 backward, conversions, two products of
// the turn, the square, the gain and its part of the sums.  Few tokens: by latency.
// Measured (bf16, 32 query and 8 key heads of 128 channels, cold L2, out of a graph): one token of 16 rows with the write to the cache 3.1 us; 4 x 1999 tokens with it 47 us (196 MB: 4.2 TB/s); 4 x 2048
// tokens forward 39 us (168 MB: 4.3 TB/s), backward 58 us (252 MB: 4.3 TB/s) and 3 us for the gains.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common/tmap.h"

TTB_DEFINE_VIOLATION_COUNTER(qk_norm)

namespace ttb {
namespace qkn {

static constexpr int kThreads = 256;

struct Part {  // of queries, keys or (copied) values; strides in elements
  const void* x;
  const void* dy;     // backward
  void* y;            // forward: output; backward: dx
  const void* gain;   // [d] or nullptr
  long long x_b, x_s, x_h, dy_b, dy_s, dy_h, y_b, y_s, y_h;
  int heads, chunks;
};
struct Params {
  Part part[3];
  const float* table;      // [table_len, d / 2, 2] cosine and sine
  const int* pos;          // [tokens] or nullptr: token % s
  const long long* slots;  // [s]: where keys and values go along the second dimension of y, or nullptr: to their token's place
  float* work;             // backward: rows of d sums, those of queries first
  int b, s, d, table_len, slot_count, wide_gain;
  int chunks;              // of a token, all parts
  float eps, per_d;        // per_d: 1 / d
  int ctas_q;              // backward: CTAs of queries; the others are of keys
};

__device__ __forceinline__ float widened(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widened(__half x) { return __half2float(x); }
__device__ __forceinline__ float widened(float x) { return x; }
template <typename T>
__device__ __forceinline__ T narrowed(float x) {
  if constexpr (std::is_same_v<T, float>) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Run {  // channels as they lie in memory
  T v[N];
  static constexpr int kBytes = N * sizeof(T);
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(p)[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(v)[i];
    }
  }
};

// The channels of a lane: [0, N) of the first half, [N, 2N) of the second.
template <typename T, int N>
__device__ __forceinline__ void widen(const Run<T, N> (&from)[2], float (&f)[2 * N]) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(from[i / (N / 2)].v)[i % (N / 2)];
      f[2 * i] = __uint_as_float(w << 16), f[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) f[i] = widened(from[i / N].v[i % N]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void narrow(const float (&f)[2 * N], Run<T, N> (&to)[2]) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<__nv_bfloat162*>(to[i / (N / 2)].v)[i % (N / 2)] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) to[i / N].v[i % N] = narrowed<T>(f[i]);
  }
}
template <bool INTERLEAVED, int N>
__device__ __forceinline__ void load_angles(const float* at, int d, int v, float (&cs)[2 * N]) {  // pair i: cs[2i], cs[2i + 1]
  const float* a = INTERLEAVED ? at + N * v : at + 2 * N * v;
  const float* b = INTERLEAVED ? at + d / 2 + N * v : at + 2 * N * v + N;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    *reinterpret_cast<float4*>(cs + 4 * i) = reinterpret_cast<const float4*>(a)[i];
    *reinterpret_cast<float4*>(cs + N + 4 * i) = reinterpret_cast<const float4*>(b)[i];
  }
}
template <bool INTERLEAVED, bool BACK, int N>
__device__ __forceinline__ void turn(float (&f)[2 * N], const float (&cs)[2 * N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float& x = f[INTERLEAVED ? 2 * i : i];
    float& y = f[INTERLEAVED ? 2 * i + 1 : i + N];
    const float c = cs[2 * i], s = BACK ? -cs[2 * i + 1] : cs[2 * i + 1], x0 = x;
    x = x0 * c - y * s;
    y = y * c + x0 * s;
  }
}
template <typename T, int N>
__device__ __forceinline__ void load_gain(const void* gain, int wide, int d, int v, float (&w)[2 * N]) {
  if (gain == nullptr) {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) w[i] = 1.f;
  } else if (wide) {
    Run<float, N> t[2];
    t[0].load(static_cast<const float*>(gain) + N * v), t[1].load(static_cast<const float*>(gain) + d / 2 + N * v);
    widen<float, N>(t, w);
  } else {
    Run<T, N> t[2];
    t[0].load(static_cast<const T*>(gain) + N * v), t[1].load(static_cast<const T*>(gain) + d / 2 + N * v);
    widen<T, N>(t, w);
  }
}
__device__ __forceinline__ int position(const Params& p, long long token, int i, bool first) {
  const int at = p.pos != nullptr ? p.pos[token] : i;
  if (at >= 0 && at < p.table_len) return at;
  if (first) TTB_NOTE_VIOLATION(qk_norm);  // position 0 stands in, and the event is counted
  return 0;
}

// A unit is a chunk of HEADS heads of one token, whose sums go around side by side: a head that a unit lacks counts as zeros, so that no branch keeps the chains of shuffles apart.
struct Place {  // of a unit
  long long x, dy, y;  // elements from the start of the part's tensors
  int which, token_in_row, count;
  uint32_t token;
  bool first;  // of its part
};
template <int N, int HEADS>
__device__ __forceinline__ Place place_of(const Params& p, uint32_t unit, uint32_t units, int chunks, int which, int v) {
  Place u;
  const bool live = unit < units;
  u.token = live ? unit / chunks : 0;
  int chunk = live ? static_cast<int>(unit - u.token * chunks) : 0;
  if (which < 0) {
    which = 0;
    while (chunk >= p.part[which].chunks) chunk -= p.part[which].chunks, ++which;
  }
  u.which = which, u.first = live && chunk == 0;
  const Part& part = p.part[which];
  const int bi = static_cast<int>(u.token / p.s), h0 = chunk * HEADS;
  u.token_in_row = static_cast<int>(u.token - static_cast<uint32_t>(bi) * p.s);
  u.count = live && v < p.d / (2 * N) ? min(HEADS, part.heads - h0) : 0;  // a group's lanes stay together: its sums take all of them
  u.x = bi * part.x_b + u.token_in_row * part.x_s + h0 * part.x_h + N * v;
  u.dy = bi * part.dy_b + u.token_in_row * part.dy_s + h0 * part.dy_h + N * v;
  long long to = u.token_in_row;
  if (which > 0 && p.slots != nullptr) {
    to = p.slots[u.token_in_row];
    if (to < 0 || to >= p.slot_count) to = -1;
  }
  u.y = to < 0 ? -1 : bi * part.y_b + to * part.y_s + h0 * part.y_h + N * v;
  return u;
}

template <int HEADS, int G>
__device__ __forceinline__ void group_sums(float (&x)[HEADS]) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
    for (int h = 0; h < HEADS; ++h) x[h] += __shfl_xor_sync(0xffffffffu, x[h], o);
}

template <typename T, bool INTERLEAVED, bool AFTER, int N, int G, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS == 1 ? 4 : N * sizeof(T) <= 8 ? 3 : 1) forward_kernel(const __grid_constant__ Params p) {
  const int v = threadIdx.x & (G - 1), lane = v < p.d / (2 * N) ? v : 0;
  const uint32_t units = static_cast<uint32_t>(p.b) * p.s * p.chunks;
  const Place u = place_of<N, HEADS>(p, blockIdx.x * (kThreads / G) + threadIdx.x / G, units, p.chunks, -1, v);
  const Part& part = p.part[u.which];
  const T* x = static_cast<const T*>(part.x) + u.x;
  Run<T, N> raw[HEADS][2];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    raw[h][0] = raw[h][1] = Run<T, N>{};
    if (h < u.count) raw[h][0].load(x + h * part.x_h), raw[h][1].load(x + h * part.x_h + p.d / 2);
  }
  float cs[2 * N], w[2 * N];
  const int at = u.count > 0 ? position(p, u.token, u.token_in_row, u.first && u.which == 0 && v == 0) : 0;
  load_angles<INTERLEAVED, N>(p.table + static_cast<long long>(at) * p.d, p.d, lane, cs);
  load_gain<T, N>(part.gain, p.wide_gain, p.d, lane, w);
  T* y = static_cast<T*>(part.y) + u.y;
  const int kept = u.y >= 0 ? u.count : 0;  // nothing is written outside a cache
  if (u.y < 0 && u.first && u.which == 1 && v == 0) TTB_NOTE_VIOLATION(qk_norm);
  if (u.which == 2) {
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
      if (h < kept) raw[h][0].store(y + h * part.y_h), raw[h][1].store(y + h * part.y_h + p.d / 2);
  }
  float f[HEADS][2 * N], sum[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    widen<T, N>(raw[h], f[h]);
    if (AFTER) turn<INTERLEAVED, false, N>(f[h], cs);
    sum[h] = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * N; ++j) sum[h] += f[h][j] * f[h][j];
  }
  group_sums<HEADS, G>(sum);
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    const float r = rsqrtf(sum[h] * p.per_d + p.eps);
#pragma unroll
    for (int j = 0; j < 2 * N; ++j) f[h][j] = f[h][j] * r * w[j];
    if (!AFTER) turn<INTERLEAVED, false, N>(f[h], cs);
    Run<T, N> out[2];
    narrow<T, N>(f[h], out);
    if (u.which < 2 && h < kept) out[0].store(y + h * part.y_h), out[1].store(y + h * part.y_h + p.d / 2);
  }
}

template <typename T, bool INTERLEAVED, bool AFTER, int N, int G, int HEADS>
__global__ void __launch_bounds__(kThreads, N * sizeof(T) <= 8 ? 3 : 1) backward_kernel(const __grid_constant__ Params p) {
  __shared__ float sums[kThreads / 32][2 * N * G];
  const int v = threadIdx.x & (G - 1);
  const int which = static_cast<int>(blockIdx.x) >= p.ctas_q;
  const Part& part = p.part[which];
  const int cta = blockIdx.x - (which ? p.ctas_q : 0), ctas = which ? gridDim.x - p.ctas_q : p.ctas_q;
  const uint32_t units = static_cast<uint32_t>(p.b) * p.s * part.chunks;
  constexpr int kGroups = kThreads / G;
  const bool lane_live = v < p.d / (2 * N);
  const int lane = lane_live ? v : 0;
  float w[2 * N], dw[2 * N];
  load_gain<T, N>(part.gain, p.wide_gain, p.d, lane, w);
#pragma unroll
  for (int j = 0; j < 2 * N; ++j) dw[j] = 0.f;
  for (uint32_t first = cta * kGroups; first < units; first += ctas * kGroups) {  // the same for all lanes of a warp; units are below 2^31
    const Place u = place_of<N, HEADS>(p, first + threadIdx.x / G, units, part.chunks, which, v);
    const T* x = static_cast<const T*>(part.x) + u.x;
    const T* dy = static_cast<const T*>(part.dy) + u.dy;
    T* dx = static_cast<T*>(part.y) + u.y;
    Run<T, N> raw_x[HEADS][2], raw_dy[HEADS][2];
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      raw_x[h][0] = raw_x[h][1] = raw_dy[h][0] = raw_dy[h][1] = Run<T, N>{};
      if (h < u.count) {
        raw_x[h][0].load(x + h * part.x_h), raw_x[h][1].load(x + h * part.x_h + p.d / 2);
        raw_dy[h][0].load(dy + h * part.dy_h), raw_dy[h][1].load(dy + h * part.dy_h + p.d / 2);
      }
    }
    float cs[2 * N], f[HEADS][2 * N], g[HEADS][2 * N], sums_of[2 * HEADS];
    load_angles<INTERLEAVED, N>(p.table + static_cast<long long>(u.count > 0 ? position(p, u.token, u.token_in_row, false) : 0) * p.d, p.d, lane, cs);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      widen<T, N>(raw_x[h], f[h]), widen<T, N>(raw_dy[h], g[h]);
      if (AFTER) turn<INTERLEAVED, false, N>(f[h], cs);
      else turn<INTERLEAVED, true, N>(g[h], cs);
      float sum = 0.f, dot = 0.f;
#pragma unroll
      for (int j = 0; j < 2 * N; ++j) sum += f[h][j] * f[h][j], dot += g[h][j] * w[j] * f[h][j];
      sums_of[2 * h] = sum, sums_of[2 * h + 1] = dot;
    }
    group_sums<2 * HEADS, G>(sums_of);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      const float r = h < u.count ? rsqrtf(sums_of[2 * h] * p.per_d + p.eps) : 0.f;
      const float mean = sums_of[2 * h + 1] * p.per_d * r;  // of dn n
#pragma unroll
      for (int j = 0; j < 2 * N; ++j) {
        const float n = f[h][j] * r;
        dw[j] += g[h][j] * n;
        f[h][j] = r * (g[h][j] * w[j] - n * mean);
      }
      if (AFTER) turn<INTERLEAVED, true, N>(f[h], cs);
      Run<T, N> out[2];
      narrow<T, N>(f[h], out);
      if (h < u.count) out[0].store(dx + h * part.y_h), out[1].store(dx + h * part.y_h + p.d / 2);
    }
  }
  if (p.work == nullptr) return;
  // groups of a warp, then warps, in a fixed order
#pragma unroll
  for (int j = 0; j < 2 * N; ++j) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
  }
  if ((threadIdx.x & 31) < G) {
#pragma unroll
    for (int j = 0; j < 2 * N; ++j) sums[threadIdx.x >> 5][j * G + v] = dw[j];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.d; c += kThreads) {
    const int half = c >= p.d / 2, in = c - half * (p.d / 2);
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kThreads / 32; ++k) t += sums[k][(half * N + in % N) * G + in / N];
    p.work[static_cast<long long>(blockIdx.x) * p.d + c] = t;
  }
}

// Adds up the rows of the workspace: grid (d / 16, 2), 16 columns of one gain per CTA.
static constexpr int kSumRows = 64;
template <typename T>
__global__ void __launch_bounds__(16 * kSumRows) gain_kernel(const float* __restrict__ work, int rows_q, int rows, int d, void* gq, void* gk, int wide) {
  __shared__ float part[kSumRows][17];
  const int c = threadIdx.x & 15, r0 = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  const int from = blockIdx.y ? rows_q : 0, to = blockIdx.y ? rows : rows_q;
  void* out = blockIdx.y ? gk : gq;
  if (out == nullptr) return;
  float t = 0.f;
  for (int r = from + r0; r < to; r += kSumRows) t += work[static_cast<long long>(r) * d + col];
  part[r0][c] = t;
  __syncthreads();
  for (int o = kSumRows / 2; o > 0; o >>= 1) {
    if (r0 < o) part[r0][c] += part[r0 + o][c];
    __syncthreads();
  }
  if (r0 == 0) {
    if (wide) static_cast<float*>(out)[col] = part[0][c];
    else static_cast<T*>(out)[col] = narrowed<T>(part[0][c]);
  }
}

// What a call brings, packed by the host language in this order.
struct Call {
  long long x[3], y[3], dy[2], gain[2];
  long long x_step[3][3], y_step[3][3], dy_step[2][3];  // batch, token, head
  long long table, pos, slots, work, work_rows, d_gain[2];
  long long b, s, heads[3], d, table_len, slot_count, type, wide_gain, interleaved, after;
};

template <typename F>
static int by_type(long long type, F f) {
  if (type == 0) return f(__nv_bfloat16());
  if (type == 1) return f(__half());
  return f(0.f);
}
// Channels of a half per lane and lanes of a head row: four channels leave registers for the next heads; more than 256 channels need eight.
template <typename F>
static int by_size(int d, F f) {
  using Four = std::integral_constant<int, 4>;
  if (d <= 32) return f(Four(), std::integral_constant<int, 4>());
  if (d <= 64) return f(Four(), std::integral_constant<int, 8>());
  if (d <= 128) return f(Four(), std::integral_constant<int, 16>());
  if (d <= 256) return f(Four(), std::integral_constant<int, 32>());
  return f(std::integral_constant<int, 8>(), std::integral_constant<int, 32>());
}
template <typename F>
static int by_order(const Call& c, F f) {
  if (c.interleaved) return c.after ? f(std::true_type(), std::true_type()) : f(std::true_type(), std::false_type());
  return c.after ? f(std::false_type(), std::true_type()) : f(std::false_type(), std::false_type());
}

static int params_of(const Call& c, Params& p, int parts, int heads_of_unit) {
  if (c.b <= 0 || c.s <= 0 || c.d <= 0 || c.d % 16 || c.d > 512 || c.b > 0x7fffffff || c.s > 0x7fffffff || c.table_len <= 0) return kErrBadShape;
  if (c.b * c.s * (c.heads[0] + c.heads[1] + c.heads[2]) > 0x7fffffffll) return kErrTooLarge;
  if (c.table & 15) return kErrBadShape;
  p.table = reinterpret_cast<const float*>(c.table), p.pos = reinterpret_cast<const int*>(c.pos), p.slots = reinterpret_cast<const long long*>(c.slots);
  p.work = reinterpret_cast<float*>(c.work);
  p.b = static_cast<int>(c.b), p.s = static_cast<int>(c.s), p.d = static_cast<int>(c.d), p.table_len = static_cast<int>(c.table_len), p.slot_count = static_cast<int>(c.slot_count);
  p.wide_gain = static_cast<int>(c.wide_gain), p.chunks = 0, p.per_d = 1.f / static_cast<float>(c.d);
  for (int i = 0; i < parts; ++i) {
    Part& t = p.part[i];
    t.x = reinterpret_cast<const void*>(c.x[i]), t.y = reinterpret_cast<void*>(c.y[i]);
    t.x_b = c.x_step[i][0], t.x_s = c.x_step[i][1], t.x_h = c.x_step[i][2];
    t.y_b = c.y_step[i][0], t.y_s = c.y_step[i][1], t.y_h = c.y_step[i][2];
    if ((c.x[i] | c.y[i]) & 15) return kErrBadShape;
    for (int j = 0; j < 3; ++j)
      if ((c.x_step[i][j] | c.y_step[i][j]) & 7) return kErrBadShape;
    if (i < 2) {
      t.gain = reinterpret_cast<const void*>(c.gain[i]), t.dy = reinterpret_cast<const void*>(c.dy[i]);
      t.dy_b = c.dy_step[i][0], t.dy_s = c.dy_step[i][1], t.dy_h = c.dy_step[i][2];
      if ((c.gain[i] | c.dy[i]) & 15) return kErrBadShape;
      for (int j = 0; j < 3; ++j)
        if (c.dy_step[i][j] & 7) return kErrBadShape;
    }
    t.heads = static_cast<int>(c.heads[i]);
    t.chunks = (t.heads + heads_of_unit - 1) / heads_of_unit;
    p.chunks += t.chunks;
  }
  return p.chunks > 0 ? kOk : kErrBadShape;
}

// Backward: CTAs, at most three to an SM, dealt to queries and keys by their heads.
static void ctas_of(const Call& c, int groups, int heads_of_unit, int& q, int& k) {
  const long long uq = c.b * c.s * ((c.heads[0] + heads_of_unit - 1) / heads_of_unit), uk = c.b * c.s * ((c.heads[1] + heads_of_unit - 1) / heads_of_unit);
  const long long nq = (uq + groups - 1) / groups, nk = (uk + groups - 1) / groups, most = 3ll * sm_count();
  if (nq + nk <= most) {
    q = static_cast<int>(nq), k = static_cast<int>(nk);
    return;
  }
  k = nk == 0 ? 0 : static_cast<int>(most * nk / (nq + nk));
  if (nk > 0 && k == 0) k = 1;
  q = static_cast<int>(most) - k;
}
static constexpr int kBackHeads = 2;

}  // namespace qkn
}  // namespace ttb

// y = norm and rotation of x for queries and keys (heads[0], heads[1]), with heads[2] > 0 values copied as well; call: a qkn::Call.
extern "C" int ttb_qk_norm_rope(const char* call, float eps, void* stream) {
  using namespace ttb;
  using namespace ttb::qkn;
  const Call& c = *reinterpret_cast<const Call*>(call);
  auto st = static_cast<cudaStream_t>(stream);
  const int parts = c.heads[2] > 0 ? 3 : 2;
  return by_type(c.type, [&](auto t) {
    using T = decltype(t);
    return by_size(static_cast<int>(c.d), [&](auto n, auto g) {
      constexpr int N = decltype(n)::value, G = decltype(g)::value;
      return by_order(c, [&](auto interleaved, auto after) {
        auto go = [&](auto heads) {
          constexpr int H = decltype(heads)::value;
          Params p{};
          p.eps = eps;
          const int rc = params_of(c, p, parts, H);
          if (rc != kOk) return rc;
          const long long units = c.b * c.s * p.chunks, ctas = (units * G + kThreads - 1) / kThreads;  // fewer than 2^31 of the former
          TTB_COUNT_LAUNCH(1);
          forward_kernel<T, decltype(interleaved)::value, decltype(after)::value, N, G, H><<<static_cast<unsigned>(ctas), kThreads, 0, st>>>(p);
          return cudaGetLastError() == cudaSuccess ? static_cast<int>(kOk) : static_cast<int>(kErrDriver);
        };
        // several heads to a group once there is work for all SMs
        const long long rows = c.b * c.s * (c.heads[0] + c.heads[1] + c.heads[2]);
        return rows * G < 2048ll * sm_count() ? go(std::integral_constant<int, 1>()) : go(std::integral_constant<int, 4>());
      });
    });
  });
}

// Rows of d floats that suffice as a workspace of the backward pass where a gain has a gradient: one for each CTA.
extern "C" long long ttb_qk_norm_rope_rows() { return 3ll * ttb::sm_count(); }

extern "C" int ttb_qk_norm_rope_bwd(const char* call, float eps, void* stream) {
  using namespace ttb;
  using namespace ttb::qkn;
  const Call& c = *reinterpret_cast<const Call*>(call);
  auto st = static_cast<cudaStream_t>(stream);
  return by_type(c.type, [&](auto t) {
    using T = decltype(t);
    return by_size(static_cast<int>(c.d), [&](auto n, auto g) {
      constexpr int N = decltype(n)::value, G = decltype(g)::value;
      return by_order(c, [&](auto interleaved, auto after) {
        Params p{};
        p.eps = eps;
        const int rc = params_of(c, p, 2, kBackHeads);
        if (rc != kOk) return rc;
        int q = 0, k = 0;
        ctas_of(c, kThreads / G, kBackHeads, q, k);
        p.ctas_q = q;
        if (p.work != nullptr && c.work_rows < q + k) return static_cast<int>(kErrBadShape);
        TTB_COUNT_LAUNCH(1);
        backward_kernel<T, decltype(interleaved)::value, decltype(after)::value, N, G, kBackHeads><<<q + k, kThreads, 0, st>>>(p);
        if (cudaGetLastError() != cudaSuccess) return static_cast<int>(kErrDriver);
        if (p.work != nullptr) {
          TTB_COUNT_LAUNCH(1);
          gain_kernel<T><<<dim3(static_cast<unsigned>(c.d / 16), 2), 16 * kSumRows, 0, st>>>(p.work, q, q + k, static_cast<int>(c.d), reinterpret_cast<void*>(c.d_gain[0]),
                                                                                             reinterpret_cast<void*>(c.d_gain[1]), static_cast<int>(c.wide_gain));
          if (cudaGetLastError() != cudaSuccess) return static_cast<int>(kErrDriver);
        }
        return static_cast<int>(kOk);
      });
    });
  });
}
