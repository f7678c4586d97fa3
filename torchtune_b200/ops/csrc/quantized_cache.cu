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
// Both kernels are bound by bytes: 8 channels per thread, 16-byte accesses on the wide side.  Rows lie [batch, head, slot]: a head's rows are one stream for the attention kernel.
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

// grid (units / 256, batch, keys and values), 4 threads per group: thread t has run t of it.
template <int BITS, typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendParams p, int groups) {
  constexpr int kHalf = 1 << (BITS - 1);
  const int which = blockIdx.z, bi = blockIdx.y;
  const long long unit = static_cast<long long>(blockIdx.x) * (kThreads / 4) + (threadIdx.x >> 2);
  const int t = threadIdx.x & 3;
  const bool live = unit < static_cast<long long>(p.s) * p.h * groups;
  const long long at = live ? unit : 0;
  const int j = static_cast<int>(at % groups);
  const long long row = at / groups;
  const int head = static_cast<int>(row % p.h), i = static_cast<int>(row / p.h);
  const int run = t * groups + j;  // runs of eight channels
  const T* x = static_cast<const T*>(p.x[which]) + bi * p.x_b[which] + i * p.x_s[which] + head * p.x_h[which] + run * 8;
  T from[8];
  if (WIDE) {
#pragma unroll
    for (int e = 0; e < static_cast<int>(sizeof(T)) / 2; ++e) reinterpret_cast<uint4*>(from)[e] = reinterpret_cast<const uint4*>(x)[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) from[e] = x[e];
  }
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = widened(from[e]);
  // The value of largest magnitude (its bits; NaN is above infinity), then the first channel that has it, with its sign.
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  uint32_t place = 0xffffffffu;
#pragma unroll
  for (int e = 7; e >= 0; --e)
    if ((__float_as_uint(v[e]) & 0x7fffffffu) == top) place = static_cast<uint32_t>(t * 8 + e) << 1 | __float_as_uint(v[e]) >> 31;
  place = min(place, __shfl_xor_sync(0xffffffffu, place, 1));
  place = min(place, __shfl_xor_sync(0xffffffffu, place, 2));
  const float m = __uint_as_float(top | place << 31);
  const __nv_bfloat16 scale = __float2bfloat16_rn(m * (-1.f / kHalf));
  const float s = __bfloat162float(scale);
  const bool usable = s != 0.f && fabsf(s) <= 3.4e38f;
  uint32_t code[2] = {0u, 0u};  // 4 bits: one word; 8 bits: two
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    int c = usable ? __float2int_rn(__fdiv_rn(v[e], s)) : 0;
    c = min(max(c, -kHalf), kHalf - 1) + kHalf;
    if (BITS == 4)
      code[0] |= static_cast<uint32_t>(c) << (4 * e);
    else
      code[e >> 2] |= static_cast<uint32_t>(c) << (8 * (e & 3));
  }
  if (!live) return;
  // Tokens take consecutive slots, so that no two of them meet in one: anything else, and what does not fit, is counted and not written.
  const long long slot = p.slots[0] + i;
  if (slot < 0 || slot >= p.slot_count || p.slots[i] != slot) {
    if (t == 0 && j == 0 && head == 0 && which == 0) TTB_NOTE_VIOLATION(quantized);
    return;
  }
  const Rows& to = p.to[which];
  uint8_t* codes = to.codes + bi * to.codes_b + head * to.codes_h + slot * to.codes_s + run * BITS;
  if (BITS == 4)
    *reinterpret_cast<uint32_t*>(codes) = code[0];
  else
    *reinterpret_cast<uint2*>(codes) = make_uint2(code[0], code[1]);
  if (t == 0) *reinterpret_cast<__nv_bfloat16*>(to.scales + bi * to.scales_b + head * to.scales_h + slot * to.scales_s + j * 2) = scale;
}

// grid (units / 256, batch, keys and values); a thread has eight channels of one row.  bf16 results are rounded once, fp32 ones are exact.
template <int BITS, typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadParams p, int groups) {
  constexpr int kHalf = 1 << (BITS - 1);
  const int which = blockIdx.z, bi = blockIdx.y;
  const int runs = 4 * groups;
  const long long unit = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  if (unit >= static_cast<long long>(p.n) * p.h * runs) return;
  const int run = static_cast<int>(unit % runs);
  const long long row = unit / runs;
  const int head = static_cast<int>(row % p.h), i = static_cast<int>(row / p.h);
  const Rows& from = p.from[which];
  const long long slot = p.first + i;
  const uint8_t* codes = from.codes + bi * from.codes_b + head * from.codes_h + slot * from.codes_s + run * BITS;
  const float s = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(from.scales + bi * from.scales_b + head * from.scales_h + slot * from.scales_s + (run % groups) * 2));
  uint32_t w[2];
  if (BITS == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(codes);
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(codes);
    w[0] = u.x, w[1] = u.y;
  }
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t c = BITS == 4 ? w[0] >> (4 * e) & 15u : w[e >> 2] >> (8 * (e & 3)) & 255u;
    v[e] = static_cast<float>(static_cast<int>(c) - kHalf) * s;
  }
  T* y = static_cast<T*>(p.y[which]) + ((static_cast<long long>(bi) * p.n + i) * p.h + head) * (runs * 8) + run * 8;
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(y) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
    *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(y + 4) = make_float4(v[4], v[5], v[6], v[7]);
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

template <typename T>
static int launch_append(const AppendParams& p, bool wide, int b, int groups, int bits, cudaStream_t st) {
  const long long blocks = (static_cast<long long>(p.s) * p.h * groups + kThreads / 4 - 1) / (kThreads / 4);
  if (blocks > 0x7fffffff) return kErrTooLarge;
  auto kern = bits == 4 ? (wide ? append_kernel<4, T, true> : append_kernel<4, T, false>) : (wide ? append_kernel<8, T, true> : append_kernel<8, T, false>);
  TTB_COUNT_LAUNCH(1);
  kern<<<dim3(static_cast<unsigned>(blocks), b, 2), kThreads, 0, st>>>(p, groups);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrDriver;
}

}  // namespace qkv
}  // namespace ttb

// Quantises k, v [b, s, h, d] (type 0: bf16, 1: fp16, 2: fp32; strides[0..5]: batch, token, head of k, then of v, in elements) into slots slots[0] ... slots[0] + s - 1 (int64 on the device,
// consecutive) of the caches: codes [b, h, slot, d * bits / 8] bytes, scales [b, h, slot, d / 32] bf16; strides[6..11]: batch, head, slot of k's codes, then of its scales (elements), [12..17] of v's.
extern "C" int ttb_quantized_append(const void* k, const void* v, void* k_codes, void* k_scales, void* v_codes, void* v_scales, const long long* strides, const long long* slots, int type, int b,
                                    int s, int h, int d, int bits, int slot_count, void* stream) {
  using namespace ttb;
  if (b <= 0 || b > 65535 || s <= 0 || h <= 0 || d <= 0 || d % 32 || (bits != 4 && bits != 8) || slot_count <= 0) return kErrBadShape;
  qkv::AppendParams p;
  p.x[0] = k, p.x[1] = v;
  const int per = type == 2 ? 3 : 7;  // elements of 16 bytes, less one
  bool wide = true;
  for (int w = 0; w < 2; ++w) {
    p.x_b[w] = strides[3 * w], p.x_s[w] = strides[3 * w + 1], p.x_h[w] = strides[3 * w + 2];
    wide = wide && (reinterpret_cast<uintptr_t>(p.x[w]) & 15) == 0 && ((p.x_b[w] | p.x_s[w] | p.x_h[w]) & per) == 0;
  }
  p.to[0] = qkv::rows_of(k_codes, k_scales, strides + 6), p.to[1] = qkv::rows_of(v_codes, v_scales, strides + 12);
  if (!qkv::aligned(p.to[0]) || !qkv::aligned(p.to[1])) return kErrBadShape;
  p.slots = slots, p.s = s, p.h = h, p.slot_count = slot_count;
  auto st = static_cast<cudaStream_t>(stream);
  switch (type) {
    case 0: return qkv::launch_append<__nv_bfloat16>(p, wide, b, d / 32, bits, st);
    case 1: return qkv::launch_append<__half>(p, wide, b, d / 32, bits, st);
    case 2: return qkv::launch_append<float>(p, wide, b, d / 32, bits, st);
  }
  return kErrBadShape;
}

// Slots first ... first + n - 1 of both caches as k, v [b, n, h, d], contiguous, bf16 or (wide) fp32; strides[0..5] of k's rows, [6..11] of v's, as above.
extern "C" int ttb_quantized_read(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, const long long* strides, void* k, void* v, int b, int first, int n, int h,
                                  int d, int bits, int wide, void* stream) {
  using namespace ttb;
  if (b <= 0 || b > 65535 || first < 0 || n <= 0 || h <= 0 || d <= 0 || d % 32 || (bits != 4 && bits != 8)) return kErrBadShape;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return kErrBadShape;
  qkv::ReadParams p;
  p.from[0] = qkv::rows_of(const_cast<void*>(k_codes), const_cast<void*>(k_scales), strides);
  p.from[1] = qkv::rows_of(const_cast<void*>(v_codes), const_cast<void*>(v_scales), strides + 6);
  if (!qkv::aligned(p.from[0]) || !qkv::aligned(p.from[1])) return kErrBadShape;
  p.y[0] = k, p.y[1] = v, p.first = first, p.n = n, p.h = h;
  const int groups = d / 32;
  const long long blocks = (static_cast<long long>(n) * h * groups * 4 + qkv::kThreads - 1) / qkv::kThreads;
  if (blocks > 0x7fffffff) return kErrTooLarge;
  const dim3 grid(static_cast<unsigned>(blocks), b, 2);
  auto kern = bits == 4 ? (wide ? qkv::read_kernel<4, float> : qkv::read_kernel<4, __nv_bfloat16>) : (wide ? qkv::read_kernel<8, float> : qkv::read_kernel<8, __nv_bfloat16>);
  TTB_COUNT_LAUNCH(1);
  kern<<<grid, qkv::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p, groups);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrDriver;
}
