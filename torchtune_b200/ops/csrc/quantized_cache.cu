// A key/value cache in 4 or 8 bits: rows are quantised as they are written, and read back.
//
// A row is what one token and head leave: d codes and d / 32 bf16 scales.  Seen as [4, d / 32, 8] its channels with the same middle index j are a group: four runs of eight, a quarter
// of the row apart, so that the quarter of a row which one lane of the attention kernel loads (quantized_attention.cu) holds eight channels of every group and the scales can be
// applied to sums over whole groups.  Of a group with m its value of largest magnitude (the first of equals) and h = 2^(bits - 1)
//   scale = bf16(-m / h)        code = clamp(rint(x / scale), -h, h - 1)        stored: code + h, of 4 bits two to a byte, the even channel in the low half,
// so that all 2 h codes are used: m itself is -h.  Of bf16 values -m / h is exact (underflow aside), and x / scale is a quotient of two 8-bit numbers, which is a tie or at least 2^-10 away from
// one; with an IEEE division the codes therefore are those of exact arithmetic.  A group of zeros (or one whose scale underflows) has code 0 and reads as 0; a group with an infinity or
// a NaN reads as NaN: nothing non-finite is lost on the way.
//
// Rows come as bf16, fp16 or fp32 (the scale of the latter two is rounded, and codes are those of the scale that is stored).
//
// Rows lie [batch, head, slot]: a head's rows are one stream for the attention kernel.  A thread has 8 channels, 16 bytes of bf16.  Measured (4 bits, 8 heads of 128 channels, cold L2): 2 x 8000
// tokens 25 us written, 17.5 us read (83.5 MB: 3.4 and 4.8 TB/s); 1 x 65 000 tokens 86 and 60 us (4.0 and 5.7); one token of 16 rows 4 and 3.3 us, a launch.  Reading is bound by its bytes; writing
// by issue: 151 instructions per 8 channels (unpacking, the two extrema, codes and their packing) at 0.74 of the rate, two fifths of them in the integer unit, which takes one every other cycle (59 %).  With one token to a
// thread and divisions instead of products with the reciprocal the first took 55 and 34 us; with eight tokens to a thread it takes 27.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common/ptx.cuh"
#include "common/tmap.h"

TTB_DEFINE_VIOLATION_COUNTER(quantized)

namespace ttb {
namespace qkv {

static constexpr int kThreads = 256;

struct Rows {  // one operand of a cache; strides in bytes
  uint8_t* codes;
  uint8_t* scales;
  long long codes_b, codes_h, codes_s, scales_b, scales_h, scales_s;
};
struct AppendParams {
  const void* x[2];
  long long x_b[2], x_s[2], x_h[2];  // elements
  Rows to[2];
  const long long* slots;
  int s, h, slot_count;
};
struct ReadParams {
  Rows from[2];
  void* y[2];
  int first, n, h;
};

__device__ __forceinline__ float widened(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widened(__half x) { return __half2float(x); }
__device__ __forceinline__ float widened(float x) { return x; }
template <typename T>
static constexpr bool kHalfPrecision = false;
template <>
constexpr bool kHalfPrecision<__half> = true;

// How a CTA's threads lie over the rows of a token and several tokens: `lanes` units (a quad of threads for a group when writing, a thread for eight channels when reading) have one token each, `sub`
// tokens at a time; a thread goes through kRun tokens, `sub` apart, with its addresses moving by constants.  grid (runs of tokens, parts of a token, 2 * batch: keys and values)
static constexpr int kRun = 4;
struct Spread {
  int units, lanes, sub;
  uint32_t per_lane;  // 2^20 / lanes, rounded up: a CTA's thread over `lanes` without a division
};
static Spread spread_of(long long units, int per_cta) {
  Spread sp;
  sp.units = static_cast<int>(units), sp.lanes = static_cast<int>(units < per_cta ? units : per_cta), sp.sub = per_cta / sp.lanes, sp.per_lane = ((1u << 20) + sp.lanes - 1) / sp.lanes;
  return sp;
}

// The largest and the smallest of three; a NaN stays.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A quad of threads per group: thread t has run t of it.
template <int BITS, typename T, bool WIDE, int GROUPS>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendParams p, const __grid_constant__ Spread sp, int some_groups) {
  constexpr int kHalf = 1 << (BITS - 1);
  const int groups = GROUPS > 0 ? GROUPS : some_groups;
  const int which = blockIdx.z & 1, bi = blockIdx.z >> 1;
  const int lane = threadIdx.x & 31, t = lane & 3, quad = threadIdx.x >> 2;
  const int sub = static_cast<int>(quad * sp.per_lane >> 20), unit = blockIdx.y * sp.lanes + (quad - sub * sp.lanes);
  const bool live = sub < sp.sub && unit < sp.units;
  const int head = live ? unit / groups : 0, j = live ? unit - head * groups : 0;
  const int run = t * groups + j;  // runs of eight channels
  const int i0 = blockIdx.x * (kRun * sp.sub) + sub;
  const long long first = p.slots[0];
  // tokens whose slot is in the cache
  const int from_i = first >= 0 ? 0 : first <= -p.s ? p.s : static_cast<int>(-first), to_i = first >= p.slot_count ? 0 : first <= p.slot_count - p.s ? p.s : static_cast<int>(p.slot_count - first);
  const T* row = static_cast<const T*>(p.x[which]) + bi * p.x_b[which] + head * p.x_h[which] + run * 8 + (live && i0 < p.s ? i0 : 0) * p.x_s[which];
  const long long step = sp.sub * p.x_s[which];
  T from[kRun][8];
  bool ours[kRun];  // whether a token takes the slot behind the one before it
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = i0 + k * sp.sub;
    const bool there = live && i < p.s;
    ours[k] = there && i >= from_i && i < to_i && p.slots[i] == first + i;
    if (k > 0 && there) row += step;
    if (WIDE) {
#pragma unroll
      for (int e = 0; e < static_cast<int>(sizeof(T)) / 2; ++e) reinterpret_cast<uint4*>(from[k])[e] = reinterpret_cast<const uint4*>(row)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) from[k][e] = row[e];
    }
  }
  const Rows& to = p.to[which];
  uint8_t* codes = to.codes + bi * to.codes_b + head * to.codes_h + run * BITS + (first + i0) * to.codes_s;
  uint8_t* scales = to.scales + bi * to.scales_b + head * to.scales_h + j * 2 + (first + i0) * to.scales_s;
  const long long codes_step = sp.sub * to.codes_s, scales_step = sp.sub * to.scales_s;
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    if (static_cast<int>(blockIdx.x) * (kRun * sp.sub) + k * sp.sub >= p.s) break;  // for the whole CTA
    const int i = i0 + k * sp.sub;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = widened(from[k][e]);
    // The value of largest magnitude: the largest or the smallest one, and where they are opposites the one that comes first.
    float high = max3_nan(max3_nan(v[0], v[1], v[2]), max3_nan(v[3], v[4], v[5]), v[6]), low = min3_nan(min3_nan(v[0], v[1], v[2]), min3_nan(v[3], v[4], v[5]), v[6]);
    high = max3_nan(high, v[7], v[7]), low = min3_nan(low, v[7], v[7]);
    const float h1 = __shfl_xor_sync(0xffffffffu, high, 1), l1 = __shfl_xor_sync(0xffffffffu, low, 1);
    high = max3_nan(high, h1, h1), low = min3_nan(low, l1, l1);
    const float h2 = __shfl_xor_sync(0xffffffffu, high, 2), l2 = __shfl_xor_sync(0xffffffffu, low, 2);
    high = max3_nan(high, h2, h2), low = min3_nan(low, l2, l2);
    float m = high > -low ? high : low;
    if (__any_sync(0xffffffffu, high == -low)) {
      float own = 0.f;  // the first of this thread's channels that has the magnitude
      bool has = false;
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (fabsf(v[e]) == high) own = v[e], has = true;
      const uint32_t with = __ballot_sync(0xffffffffu, has) >> (lane & 28) & 15u;
      own = __shfl_sync(0xffffffffu, own, (lane & 28) + (with != 0u ? __ffs(with) - 1 : 0));
      if (high == -low) m = own;
    }
    const __nv_bfloat16 scale = __float2bfloat16_rn(m * (-1.f / kHalf));
    const float s = __bfloat162float(scale);
    const bool usable = s != 0.f && fabsf(s) <= 3.4e38f;
    uint32_t code[2] = {0u, 0u};  // 4 bits: one word; 8 bits: two
    constexpr int kPer = 32 / BITS;
    auto put = [&](int e, uint32_t c) {
      asm("mad.lo.u32 %0, %1, %2, %0;" : "+r"(code[e / kPer]) : "r"(c), "r"(1u << (BITS * (e % kPer))));  // the integer unit is what bounds this kernel; this is not on it
    };
    if (sizeof(T) == 2 && !kHalfPrecision<T> && fabsf(s) >= 1e-30f && usable) {
      // bf16: a quotient is a tie or at least 2^-10 away from one (see above).  The product with the reciprocal (off by at most 2^-22 of itself) is off by at most 2^-15, so that on a grid of 2^-10 it lies on the same side, and a tie
      // on itself: 1.5 x 2^13 + quotient has that grid.  The sum that brings it to 1.5 x 2^23 + h is rounded to a whole number, ties to even, whose low bits are the code; what the exponents add up to in a word of
      // codes is taken off beforehand.  A tenth of the instructions of a division.
      constexpr uint32_t kBase = 0x4b400000u;  // 1.5 x 2^23
      code[0] = code[1] = 0u - kBase * (BITS == 4 ? 0x11111111u : 0x01010101u);
      float inv;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t c = __float_as_uint(__fadd_rn(__fmaf_rn(v[e], inv, 12288.f), 12582912.f - 12288.f + kHalf));
        put(e, min(c, kBase + 2u * kHalf - 1u));  // no quotient is below -h: m itself gives that
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = usable ? __float2int_rn(__fdiv_rn(v[e], s)) : 0;
        put(e, static_cast<uint32_t>(min(max(c, -kHalf), kHalf - 1) + kHalf));
      }
    }
    // Tokens take consecutive slots, so that no two of them meet in one: anything else, and what does not fit, is counted and not written.
    if (ours[k]) {
      if (BITS == 4)
        *reinterpret_cast<uint32_t*>(codes) = code[0];
      else
        *reinterpret_cast<uint2*>(codes) = make_uint2(code[0], code[1]);
      if (t == 0) *reinterpret_cast<__nv_bfloat16*>(scales) = scale;
    } else if (live && i < p.s && t == 0 && unit == 0 && which == 0) {
      TTB_NOTE_VIOLATION(quantized);
    }
    codes += codes_step, scales += scales_step;
  }
}

// A thread has eight channels of a row.  bf16 results are rounded once, fp32 ones are exact.
template <int BITS, typename T, int GROUPS>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadParams p, const __grid_constant__ Spread sp, int some_groups) {
  constexpr float kHalf = 1 << (BITS - 1);
  const int groups = GROUPS > 0 ? GROUPS : some_groups;
  const int which = blockIdx.z & 1, bi = blockIdx.z >> 1;
  const int sub = static_cast<int>(threadIdx.x * sp.per_lane >> 20), unit = blockIdx.y * sp.lanes + (threadIdx.x - sub * sp.lanes);
  if (sub >= sp.sub || unit >= sp.units) return;
  const int runs = 4 * groups, head = unit / runs, run = unit - head * runs;
  const int i0 = blockIdx.x * (kRun * sp.sub) + sub;
  const Rows& from = p.from[which];
  const uint8_t* codes = from.codes + bi * from.codes_b + head * from.codes_h + run * BITS + static_cast<long long>(p.first) * from.codes_s;
  const uint8_t* scales = from.scales + bi * from.scales_b + head * from.scales_h + (run % groups) * 2 + static_cast<long long>(p.first) * from.scales_s;
  uint32_t w[kRun][2];
  float s[kRun];
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const long long i = min(i0 + k * sp.sub, p.n - 1);
    const uint8_t* at = codes + i * from.codes_s;
    if (BITS == 4) {
      w[k][0] = *reinterpret_cast<const uint32_t*>(at);
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(at);
      w[k][0] = u.x, w[k][1] = u.y;
    }
    s[k] = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(scales + i * from.scales_s));
  }
  T* y = static_cast<T*>(p.y[which]) + static_cast<long long>(bi) * p.n * sp.units * 8 + unit * 8;
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = i0 + k * sp.sub;
    if (i >= p.n) return;
    float v[8];
    // 2^23 + (code << n) is exact, and so is the sum that leaves code - h of it
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (BITS == 4) {
        const uint32_t part = e < 4 ? w[k][0] : w[k][0] >> 16;
        const int n = 4 * (e & 3);
        v[e] = fmaf(__uint_as_float(0x4b000000u | (part & (15u << n))), 1.f / (1 << n), -(8388608.f / (1 << n) + kHalf)) * s[k];
      } else {
        v[e] = (__uint_as_float(0x4b000000u | (w[k][e >> 2] >> (8 * (e & 3)) & 255u)) - (8388608.f + kHalf)) * s[k];
      }
    }
    T* to = y + static_cast<long long>(i) * sp.units * 8;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
      *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
}

static Rows rows_of(void* codes, void* scales, const long long* strides) {
  Rows r;
  r.codes = static_cast<uint8_t*>(codes), r.scales = static_cast<uint8_t*>(scales);
  r.codes_b = strides[0], r.codes_h = strides[1], r.codes_s = strides[2];
  r.scales_b = strides[3] * 2, r.scales_h = strides[4] * 2, r.scales_s = strides[5] * 2;
  return r;
}
static bool aligned(const Rows& r) {  // eight codes are one access
  return ((reinterpret_cast<uintptr_t>(r.codes) | r.codes_b | r.codes_h | r.codes_s) & 7) == 0 && (reinterpret_cast<uintptr_t>(r.scales) & 1) == 0;
}

// Tokens and parts of a token as a grid; 0 CTAs where a dimension is too large.
static dim3 grid_of(const Spread& sp, long long tokens, int b) {
  const long long runs = (tokens + kRun * sp.sub - 1) / (kRun * sp.sub), parts = (sp.units + sp.lanes - 1) / sp.lanes;
  return runs > 0x7fffffff - kRun || parts > 65535 || 2ll * b > 65535 ? dim3(0) : dim3(static_cast<unsigned>(runs), static_cast<unsigned>(parts), 2u * b);
}

template <typename T, int GROUPS>
static void append_of(const AppendParams& p, const Spread& sp, bool wide, dim3 grid, int groups, int bits, cudaStream_t st) {
  auto kern = bits == 4 ? (wide ? append_kernel<4, T, true, GROUPS> : append_kernel<4, T, false, GROUPS>) : (wide ? append_kernel<8, T, true, GROUPS> : append_kernel<8, T, false, GROUPS>);
  kern<<<grid, kThreads, 0, st>>>(p, sp, groups);
}

template <typename T>
static int launch_append(const AppendParams& p, bool wide, int b, int groups, int bits, cudaStream_t st) {
  const Spread sp = spread_of(static_cast<long long>(p.h) * groups, kThreads / 4);
  const dim3 grid = grid_of(sp, p.s, b);
  if (grid.x == 0) return kErrTooLarge;
  TTB_COUNT_LAUNCH(1);
  if (groups == 4)
    append_of<T, 4>(p, sp, wide, grid, groups, bits, st);
  else if (groups == 2)
    append_of<T, 2>(p, sp, wide, grid, groups, bits, st);
  else
    append_of<T, 0>(p, sp, wide, grid, groups, bits, st);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrDriver;
}

template <int GROUPS>
static void read_of(const ReadParams& p, const Spread& sp, dim3 grid, int groups, int bits, int wide, cudaStream_t st) {
  auto kern = bits == 4 ? (wide ? read_kernel<4, float, GROUPS> : read_kernel<4, __nv_bfloat16, GROUPS>) : (wide ? read_kernel<8, float, GROUPS> : read_kernel<8, __nv_bfloat16, GROUPS>);
  kern<<<grid, kThreads, 0, st>>>(p, sp, groups);
}

}  // namespace qkv
}  // namespace ttb

// A call's arguments, 8 bytes each: handed over as one piece, which takes the caller less time than as many arguments.
struct QuantizedAppendCall {
  const void *k, *v;
  void *k_codes, *k_scales, *v_codes, *v_scales;
  long long strides[18];
  const long long* slots;
  long long type, b, s, h, d, bits, slot_count;
};
struct QuantizedReadCall {
  const void *k_codes, *k_scales, *v_codes, *v_scales;
  long long strides[12];
  void *k, *v;
  long long b, first, n, h, d, bits, wide;
};

// Quantises k, v [b, s, h, d] (type 0: bf16, 1: fp16, 2: fp32; strides[0..5]: batch, token, head of k, then of v, in elements) into slots slots[0] ... slots[0] + s - 1 (int64 on the device,
// consecutive) of the caches: codes [b, h, slot, d * bits / 8] bytes, scales [b, h, slot, d / 32] bf16; strides[6..11]: batch, head, slot of k's codes, then of its scales (elements), [12..17] of v's.
extern "C" int ttb_quantized_append(const QuantizedAppendCall* call, void* stream) {
  using namespace ttb;
  const QuantizedAppendCall& c = *call;
  const long long most = 0x7fffffff;
  if (c.b <= 0 || c.b > most || c.s <= 0 || c.s > most - qkv::kRun * qkv::kThreads || c.h <= 0 || c.h > most || c.d <= 0 || c.d > most || c.d % 32 || c.h * c.d > most ||
      (c.bits != 4 && c.bits != 8) || c.slot_count <= 0 || c.slot_count > most)
    return kErrBadShape;
  qkv::AppendParams p;
  p.x[0] = c.k, p.x[1] = c.v;
  const int per = c.type == 2 ? 3 : 7;  // elements of 16 bytes, less one
  bool wide = true;
  for (int w = 0; w < 2; ++w) {
    p.x_b[w] = c.strides[3 * w], p.x_s[w] = c.strides[3 * w + 1], p.x_h[w] = c.strides[3 * w + 2];
    wide = wide && (reinterpret_cast<uintptr_t>(p.x[w]) & 15) == 0 && ((p.x_b[w] | p.x_s[w] | p.x_h[w]) & per) == 0;
  }
  p.to[0] = qkv::rows_of(c.k_codes, c.k_scales, c.strides + 6), p.to[1] = qkv::rows_of(c.v_codes, c.v_scales, c.strides + 12);
  if (!qkv::aligned(p.to[0]) || !qkv::aligned(p.to[1])) return kErrBadShape;
  p.slots = c.slots, p.s = static_cast<int>(c.s), p.h = static_cast<int>(c.h), p.slot_count = static_cast<int>(c.slot_count);
  const int b = static_cast<int>(c.b), groups = static_cast<int>(c.d / 32), bits = static_cast<int>(c.bits);
  auto st = static_cast<cudaStream_t>(stream);
  switch (c.type) {
    case 0: return qkv::launch_append<__nv_bfloat16>(p, wide, b, groups, bits, st);
    case 1: return qkv::launch_append<__half>(p, wide, b, groups, bits, st);
    case 2: return qkv::launch_append<float>(p, wide, b, groups, bits, st);
  }
  return kErrBadShape;
}

// Slots first ... first + n - 1 of both caches as k, v [b, n, h, d], contiguous, bf16 or (wide) fp32; strides[0..5] of k's rows, [6..11] of v's, as above.
extern "C" int ttb_quantized_read(const QuantizedReadCall* call, void* stream) {
  using namespace ttb;
  const QuantizedReadCall& c = *call;
  const long long most = 0x7fffffff;
  if (c.b <= 0 || c.b > most || c.first < 0 || c.first > most || c.n <= 0 || c.n > most || c.h <= 0 || c.h > most || c.d <= 0 || c.d > most || c.d % 32 || c.h * c.d > most ||
      (c.bits != 4 && c.bits != 8))
    return kErrBadShape;
  if ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15) return kErrBadShape;
  qkv::ReadParams p;
  p.from[0] = qkv::rows_of(const_cast<void*>(c.k_codes), const_cast<void*>(c.k_scales), c.strides);
  p.from[1] = qkv::rows_of(const_cast<void*>(c.v_codes), const_cast<void*>(c.v_scales), c.strides + 6);
  if (!qkv::aligned(p.from[0]) || !qkv::aligned(p.from[1])) return kErrBadShape;
  p.y[0] = c.k, p.y[1] = c.v, p.first = static_cast<int>(c.first), p.n = static_cast<int>(c.n), p.h = static_cast<int>(c.h);
  const int groups = static_cast<int>(c.d / 32), bits = static_cast<int>(c.bits), wide = c.wide != 0;
  const qkv::Spread sp = qkv::spread_of(c.h * groups * 4, qkv::kThreads);
  const dim3 grid = qkv::grid_of(sp, c.n, static_cast<int>(c.b));
  if (grid.x == 0 || c.n > most - qkv::kRun * qkv::kThreads) return kErrTooLarge;
  auto st = static_cast<cudaStream_t>(stream);
  TTB_COUNT_LAUNCH(1);
  if (groups == 4)
    qkv::read_of<4>(p, sp, grid, groups, bits, wide, st);
  else if (groups == 2)
    qkv::read_of<2>(p, sp, grid, groups, bits, wide, st);
  else
    qkv::read_of<0>(p, sp, grid, groups, bits, wide, st);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrDriver;
}
