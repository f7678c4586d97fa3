// Log-probabilities of given tokens with the entropy and the likeliest alternatives, from one pass over the logits, and their gradient in one more.
//
// Of z = x / T, in units of log2 (c = log2(e) / T):  d = (x - base) c,  s = sum 2^d,  t = sum 2^d d,  with a base less than some four powers of two from the maximum, so that
//   log p = ln2 (d - log2 s)        H = -sum p log p = ln2 (log2 s - t / s)
// are differences of numbers that are small where the results are.  Near certainty what is left of them is their roundings: up to 1e-6 of log p and 3e-6 of H (400 x 128256 with one token 14 above the
// others' maximum; with a base up to 2^24 away 2e-6 and 1e-5), neither of which crosses 0.  When the base moves up by a / c, s' = s 2^-a and t' = (t - a s) 2^-a.  A base that followed every new
// maximum would move in nearly all steps of a warp, since one of its 32 lanes has a new one; so it begins four powers of two above the maximum of the warp's first 256 elements, and a lane whose elements
// go four above it moves its own.  Rows in rising order, whose lanes move it all the time, take 1.1 to 1.35 times as long (8192 x 8000 bf16 41 -> 55 us).  Differences are taken before they are
// scaled: a row of a type's lowest values is one of equal logits.
// With g, h and k_j the gradients of the token's log-probability, of the entropy and of the alternatives' log-probabilities:
//   dx_v = ([v = token] g + sum_j [v = alternative j] k_j - p_v (g + sum_j k_j + h (log p_v + H))) / T.
//
// The alternatives are the `top` largest logits, of equal ones those with the lower index.  The pass leaves the largest value of every segment of 256 elements (what a warp reads at once) in shared
// memory; the `top` segments with the largest ones (of equal ones the first) hold all alternatives, since an element outside is beaten by `top` maxima.  Of their elements those count that reach the
// least of these maxima: hardly more than `top` as a rule, whose ranks one warp finds by comparing each with each.  Rows of no more segments than alternatives take the maxima of the lanes' elements
// instead, of which there are 32.  Where candidates are too many (logits in order, ties), the choice is a search: for the `top`-th largest key bit by bit among the segments, their lanes and the lanes'
// elements, or, where a warp has a row of its own, for one alternative after the other.  So it is there for ordinary logits too, where more than 32 alternatives come from hardly more segments than that, or
// some 30 from as many: 8192 x 8000 bf16 94 us with 20, 770 with 32, 3000 with 33, 5800 with 64; 8192 x 16000 123, 147, 152 and 12 200; 8192 x 20000 133, 160, 164 and 254.
//
// Three ways through the rows.  Long ones: CTAs go from row to row; warps that stream take runs of a row and go on to the next one without waiting for each other, and a warp of its own ends the row
// before, from sums and segments that lie in shared memory twice.  Many that are not long: a warp streams and ends rows of its own, since the end of a row, some 5 us of instructions that wait for one
// another, takes longer than its stream, and there it lies beside the streams of 23 other warps.  Few rows: split over clusters of up to eight CTAs, which meet in the shared memory of the first.
// In all of them a lane copies its vectors two runs ahead, over the ends of rows too, to slots of its own.
//
// Bound by bytes in 32 bits, in 16 bits by issue and the exponentials' unit (16 a cycle and SM: 64 % busy, and 66 % of the cycles issue), and with alternatives by the maxima beside them.
// Measured (cold L2, out of a graph): 4096 x 151936 bf16 forward 248 us (5.0 TB/s), gradient 446 us (5.6 TB/s); 4136 x 128256 bf16 with 5 alternatives 262 us (4.1 TB/s); 8192 x 32000 fp32 184 us
// (5.7 TB/s), its gradient 309 us; 8192 x 8000 bf16 41 us; 16 x 128256 fp32 with 20 alternatives 17 us (kernels behind one another).
//
// Rows begin at any address: vectors lie on 16 bytes, and the first and last of a row are read element by element.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common/attn_math.cuh"
#include "common/tmap.h"

TTB_DEFINE_VIOLATION_COUNTER(token_stats)

namespace ttb {
namespace tstat {

namespace cg = cooperative_groups;
using attn::add_f32x2;
using attn::fma_f32x2;
using attn::mul_f32x2;
using attn::pack_f32x2;
using attn::unpack_f32x2;

static constexpr int kWarps = 16;      // that stream
static constexpr int kThreads = (kWarps + 1) * 32;
static constexpr int kCtas = 2;        // of an SM
template <typename T, bool TOP>
static constexpr int kEach = sizeof(T) == 4 ? (TOP ? 1 : 2) : (TOP ? 3 : 4);  // vectors that a lane takes at once; alternatives need room of their own in shared memory
template <typename T, bool TOP>
static constexpr int kRun = 32 * kEach<T, TOP>;
template <typename T, bool TOP>
static constexpr int kSlotBytes = kWarps * kRun<T, TOP> * 8 * sizeof(T);
static constexpr int kSlots = 3;
static constexpr int kGradThreads = 256;
static constexpr int kMaxTop = 64;
static constexpr int kMaxSegments = 1024;  // of a CTA
static constexpr int kMaxCluster = 8;
static constexpr float kLn2 = 0.6931471805599453f;
static constexpr float kLowest = -200.f;  // 2^kLowest is 0 in fp32
static constexpr float kMostAllowed = 16.f;  // sum of the exponentials of eight elements: eight equal to the base leave as much room again
static constexpr float kLift = 4.f;         // powers of two from a warp's first maximum up to its first base

struct Params {
  const void* x;  // row r at x + (r / inner) * step_outer + (r % inner) * step_inner, in elements
  long long step_outer, step_inner;
  const long long* tokens;
  float* logprobs;
  float* entropy;
  float* stats;          // [rows, 2]: base and log2 s, or nullptr
  float* top_logprobs;   // [rows, top]
  long long* top_tokens;
  long long ignore, rows;
  int inner, vocab, top;
  float c, rate, lift;  // log2(e) / T, 1 / T and kLift / c
};
struct GradParams {
  const void* x;
  long long step_outer, step_inner;
  const long long* tokens;
  const float *stats, *entropy;
  const long long* top_tokens;
  const float *g, *h, *k;  // gradients of log-probabilities, entropy and alternatives; nullptr: none
  void* dx;                // [rows, vocab]
  long long ignore, rows;
  int inner, vocab, top, parts;  // parts: of a row
  float c, rate;           // rate = 1 / T
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
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float warp_max_nan(float x) {
  float d;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(x));
  return d;
}
// Order of logits as whole numbers: NaN above all, zeros of both signs equal, nothing below 1 (0 stands for no element); bits that the type does not have are left out.
template <typename T>
static constexpr int kSpareBits = std::is_same_v<T, float> ? 0 : std::is_same_v<T, __half> ? 13 : 16;
template <typename T>
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (x != x ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u)) >> kSpareBits<T>;
}

template <typename T>
__device__ __forceinline__ float value_of(uint32_t key) {
  const uint32_t u = key << kSpareBits<T>;
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~(u | ((1u << kSpareBits<T>) - 1)));
}

// A row as eight-element vectors on 16 bytes, the first of which may begin before it.
template <typename T>
struct Row {
  struct alignas(16) Vector {
    T v[8];
  };
  const T* x;
  int vocab, off;  // off: elements of vector 0 in front of the row
  __device__ __forceinline__ Row(const T* row, int n) : x(row), vocab(n), off(static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T))) {}
  __device__ __forceinline__ int vectors() const { return static_cast<int>((static_cast<long long>(vocab) + off + 7) / 8); }
  // vectors [whole_from(), whole_to()) hold no element outside the row
  __device__ __forceinline__ int whole_from() const { return off != 0; }
  __device__ __forceinline__ int whole_to() const { return static_cast<int>((static_cast<long long>(vocab) + off) / 8); }
  __device__ __forceinline__ const Vector* vector(int j) const { return reinterpret_cast<const Vector*>(x - off) + j; }
  __device__ __forceinline__ static Vector whole(const Vector* at) {
    Vector r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(r.v)[i] = reinterpret_cast<const uint4*>(at)[i];
    return r;
  }
  __device__ __forceinline__ Vector load(int j) const {  // elements outside the row: the lowest value
    if (j >= whole_from() && j < whole_to()) return whole(vector(j));
    Vector r;
    const long long e = j * 8ll - off;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = e + i >= 0 && e + i < vocab ? x[e + i] : narrowed<T>(-INFINITY);
    return r;
  }
  __device__ __forceinline__ uint32_t key(long long e) const { return e >= 0 && e < vocab ? key_of<T>(widened(x[e])) : 0u; }
};
// Eight values in 32 bits.
template <typename Vector>
__device__ __forceinline__ void widen8(const Vector& raw, float (&f)[8]) {
  if constexpr (std::is_same_v<decltype(+raw.v), const __nv_bfloat16*>) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = widened(raw.v[i]);
  }
}
__device__ __forceinline__ float most_of(const float (&f)[8]) { return max3_nan(max3_nan(f[0], f[1], f[2]), max3_nan(f[3], f[4], f[5]), max3_nan(f[6], f[7], f[7])); }

// x - base of elements i and i + 1
template <typename T, typename Vector>
__device__ __forceinline__ uint64_t minus(const Vector& raw, int i, float base) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {  // the conversion is part of the sum
    const uint32_t w = reinterpret_cast<const uint32_t*>(raw.v)[i >> 1];
    float d0, d1;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tadd.rn.f32.bf16 %0, lo, %3;\n\tadd.rn.f32.bf16 %1, hi, %3;\n\t}" : "=f"(d0), "=f"(d1) : "r"(w), "f"(-base));
    return pack_f32x2(d0, d1);
  } else {
    return add_f32x2(pack_f32x2(widened(raw.v[i]), widened(raw.v[i + 1])), pack_f32x2(-base, -base));
  }
}
template <typename T, typename Vector>
__device__ __forceinline__ float most_of_vector(const Vector& raw) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(raw.v);
    uint32_t a, b;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(w[0]), "r"(w[1]));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(w[2]), "r"(w[3]));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(b));
    const float lo = __uint_as_float(a << 16), hi = __uint_as_float(a & 0xffff0000u);
    return max3_nan(lo, hi, hi);
  } else {
    float f[8];
    widen8(raw, f);
    return most_of(f);
  }
}

// base, s and t of a part of a row
struct Sums {
  float base, s, t;
};
// The sums of a thread as it goes along its part.
struct Running {
  float c;
  float most_allowed = -1.f, base = 0.f;  // there is no base until there is a logit above the infinitely low ones
  uint64_t s2 = 0, t2 = 0;
  __device__ __forceinline__ void begin(float most) {  // of the whole warp; a row that begins with NaN or infinitely low logits leaves its lanes to themselves
    if (most > -INFINITY) base = most, most_allowed = kMostAllowed;
  }
  __device__ __forceinline__ Sums sums() const {
    float s0, s1, t0, t1;
    unpack_f32x2(s2, s0, s1), unpack_f32x2(t2, t0, t1);
    return {base, s0 + s1, t0 + t1};
  }
  __device__ __forceinline__ void careful(const float (&f)[8]) {  // moves the base, and takes what is infinitely low to have no share (0 * -inf)
    const float most = most_of(f);
    if (!(most <= (most_allowed < 0.f ? -INFINITY : base))) {  // NaN too
      const float d = fminf(fmaxf((base - most) * c, kLowest), 0.f), g = fast_exp2(d);
      const Sums now = sums();
      s2 = pack_f32x2(now.s * g, 0.f), t2 = pack_f32x2((now.t + now.s * d) * g, 0.f);
      base = most, most_allowed = kMostAllowed;
    }
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = (f[i] - base) * c, e = fast_exp2(d);
      s += e, t += e * (d < kLowest ? kLowest : d);
    }
    s2 = add_f32x2(s2, pack_f32x2(s, 0.f)), t2 = add_f32x2(t2, pack_f32x2(t, 0.f));
  }
  template <typename T, typename Vector>
  __device__ __forceinline__ void take(const Vector& raw, uint64_t c2) {  // c2: c twice
    uint64_t sv = 0, tv = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint64_t d = mul_f32x2(minus<T>(raw, i, base), c2);
      float d0, d1;
      unpack_f32x2(d, d0, d1);
      const uint64_t e = pack_f32x2(fast_exp2(d0), fast_exp2(d1));
      sv = i == 0 ? e : add_f32x2(sv, e);
      tv = i == 0 ? mul_f32x2(e, d) : fma_f32x2(e, d, tv);
    }
    float s0, s1, t0, t1;
    unpack_f32x2(sv, s0, s1), unpack_f32x2(tv, t0, t1);
    const float sum = s0 + s1, t = t0 + t1;
    if (!(sum <= most_allowed) || t != t) {
      float f[8];
      widen8(raw, f);
      careful(f);
    } else {
      s2 = add_f32x2(s2, sv), t2 = add_f32x2(t2, tv);
    }
  }
};
// The sums of all lanes of a warp, over the highest of their bases; one without a finite logit (s = 0) has none.  NaN goes on.
__device__ __forceinline__ Sums joined_lanes(const Sums& mine, float c) {
  float s = mine.s, t = mine.t;
  const float highest = warp_max_nan(s == 0.f ? -INFINITY : mine.base);
  if (s != 0.f) {
    const float d = fmaxf((mine.base - highest) * c, kLowest), f = fast_exp2(d);
    t = (t + s * d) * f, s *= f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), t += __shfl_xor_sync(0xffffffffu, t, o);
  return {highest == -INFINITY ? 0.f : highest, s, t};
}

// The `want` largest of n keys, of equal ones the first, in order of their place: to[0 ...]; by one warp.  Returns how many (n, if there are no more).  The keys lie on 16 bytes and have room for zeros
// up to the next multiple of 128.
__device__ __forceinline__ int choose(uint32_t* keys, int n, int want, uint16_t* to) {
  const int lane = threadIdx.x & 31;
  if (n <= want) {
    for (int i = lane; i < n; i += 32) to[i] = static_cast<uint16_t>(i);
    __syncwarp();
    return n;
  }
  uint32_t high = 0, low = 0xffffffffu;
  for (int i = lane; i < n; i += 32) high = max(high, keys[i]), low = min(low, keys[i]);
  high = __reduce_max_sync(0xffffffffu, high), low = __reduce_min_sync(0xffffffffu, low);
  const int groups = (n + 127) / 128;
  for (int i = n + lane; i < groups * 128; i += 32) keys[i] = 0;
  __syncwarp();
  const uint4* fours = reinterpret_cast<const uint4*>(keys);
  auto count = [&](uint32_t least) {  // least > 0
    int c = 0;
#pragma unroll 4
    for (int g = 0; g < groups; ++g) {
      const uint4 k = fours[g * 32 + lane];
      c += (k.x >= least) + (k.y >= least) + (k.z >= least) + (k.w >= least);
    }
    return static_cast<int>(__reduce_add_sync(0xffffffffu, c));
  };
  // at least `want` keys reach the level; all share the bits above the first in which the highest and the lowest differ
  const int differ = 32 - __clz(high ^ low);
  uint32_t level = differ == 32 ? 0u : high >> differ << differ;
  for (int bit = differ - 1; bit >= 0; --bit) {
    const int c = count(level | 1u << bit);
    if (c >= want) level |= 1u << bit;
    if (c == want) break;
  }
  int equal = level == 0xffffffffu ? want : want - count(level + 1);  // of those that just reach it so many are taken
  int at = 0;
  for (int g = 0; g < groups; ++g) {
    const uint4 four = fours[g * 32 + lane];
    const uint32_t k[4] = {four.x, four.y, four.z, four.w};
    const int place = g * 128 + lane * 4;
    if (!__any_sync(0xffffffffu, max(max(k[0], k[1]), max(k[2], k[3])) >= level)) continue;
    const uint32_t below = (1u << lane) - 1;
    int same_before = 0, same_all = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t same = __ballot_sync(0xffffffffu, place + c < n && k[c] == level);
      same_before += __popc(same & below), same_all += __popc(same);
    }
    bool taken[4];
    int taken_before = 0, taken_all = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bool same = place + c < n && k[c] == level;
      taken[c] = place + c < n && (k[c] > level || (same && same_before < equal));
      same_before += same;
      const uint32_t all = __ballot_sync(0xffffffffu, taken[c]);
      taken_before += __popc(all & below), taken_all += __popc(all);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (taken[c]) to[at + taken_before++] = static_cast<uint16_t>(place + c);
    at += taken_all;
    equal -= min(equal, same_all);
  }
  __syncwarp();
  return at;
}

// An alternative, or a segment: its key above, and below it the complement of its index, so that the larger number comes first.  0: none.
using Entry = unsigned long long;
__device__ __forceinline__ Entry entry_of(uint32_t key, int index) { return static_cast<Entry>(key) << 32 | ~static_cast<uint32_t>(index); }
__device__ __forceinline__ uint32_t key_in(Entry e) { return static_cast<uint32_t>(e >> 32); }
__device__ __forceinline__ int index_in(Entry e) { return static_cast<int>(~static_cast<uint32_t>(e)); }
static constexpr int kMostCandidates = 512;  // all entries of a cluster

// The `want` largest of `count` candidates, in their order, to `to`; by one warp.
__device__ __forceinline__ void rank(const Entry* list, int count, int want, Entry* to) {
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < want; i += 32) to[i] = 0;
  __syncwarp();
  for (int i = lane; i < count; i += 64) {  // two per lane
    const Entry a = list[i], b = i + 32 < count ? list[i + 32] : 0;
    int rank_a = 0, rank_b = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) {
      const Entry e = list[j];
      rank_a += e > a, rank_b += e > b;
    }
    if (rank_a < want) to[rank_a] = a;
    if (i + 32 < count && rank_b < want) to[rank_b] = b;
  }
  __syncwarp();
}
// Entries go to the list's next places, as far as there is room, those of lower lanes first; by a whole warp.
__device__ __forceinline__ void append(Entry* list, int& count, bool mine, Entry e) {
  const uint32_t all = __ballot_sync(0xffffffffu, mine);
  const int at = count + __popc(all & ((1u << (threadIdx.x & 31)) - 1));
  if (mine && at < kMostCandidates) list[at] = e;
  count += __popc(all);
}
// The `want` (up to 64) largest of n > want values, of equal ones the first, with their places as indices and in order, to `to`; false, if there are too many candidates.  Values, which lie on 16 bytes
// with room up to the next multiple of 128, become keys where they are.  At least `want` keys reach the want-th largest of the maxima of 32 or 64 sets, and hardly more than twice as many if keys
// are in no order.  One warp does this alone, so that its time is that of what waits for what: it takes four keys at a time.
template <typename T>
__device__ __forceinline__ bool choose_few(uint32_t* keys, int n, int want, Entry* list, int room, Entry* to) {
  const int lane = threadIdx.x & 31, groups = (n + 127) / 128;
  uint4* fours = reinterpret_cast<uint4*>(keys) + lane;
  uint32_t most[2] = {0, 0};
#pragma unroll 1
  for (int g = 0; g < groups; ++g) {
    uint4 k = fours[g * 32];
    const int left = n - g * 128 - lane * 4;
    k.x = left > 0 ? key_of<T>(__uint_as_float(k.x)) : 0u, k.y = left > 1 ? key_of<T>(__uint_as_float(k.y)) : 0u;
    k.z = left > 2 ? key_of<T>(__uint_as_float(k.z)) : 0u, k.w = left > 3 ? key_of<T>(__uint_as_float(k.w)) : 0u;
    fours[g * 32] = k;
    most[0] = max(most[0], max(k.x, k.y)), most[1] = max(most[1], max(k.z, k.w));
  }
  const bool two = want > 12;  // 64 sets leave fewer candidates than 32; to rank them takes twice as long
  if (!two) most[0] = max(most[0], most[1]);
  int above[2] = {0, 0};
#pragma unroll 8
  for (int x = 0; x < 32; ++x) {
    const uint32_t other = __shfl_sync(0xffffffffu, most[0], x);
    above[0] += (other > most[0]) | ((other == most[0]) & (x < lane));
    if (two) {
      const uint32_t second = __shfl_sync(0xffffffffu, most[1], x);
      above[0] += second > most[0];
      above[1] += (other >= most[1]) + ((second > most[1]) | ((second == most[1]) & (x < lane)));
    }
  }
  const uint32_t first = __ballot_sync(0xffffffffu, above[0] == want - 1), other = __ballot_sync(0xffffffffu, two && above[1] == want - 1);
  const uint32_t least = max(1u, __shfl_sync(0xffffffffu, first != 0 ? most[0] : most[1], __ffs(first | other) - 1));  // of few keys, sets may be empty
  const uint32_t below = (1u << lane) - 1;
  int found = 0;
#pragma unroll 1
  for (int g = 0; g < groups; ++g) {
    const uint4 four = fours[g * 32];
    const uint32_t k[4] = {four.x, four.y, four.z, four.w};
    uint32_t all[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) all[c] = __ballot_sync(0xffffffffu, k[c] >= least);
    if ((all[0] | all[1] | all[2] | all[3]) == 0) continue;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int at = found + __popc(all[c] & below);
      if (k[c] >= least && at < room) list[at] = entry_of(k[c], g * 128 + lane * 4 + c);
      found += __popc(all[c]);
    }
  }
  __syncwarp();
  if (found <= room) rank(list, found, want, to);
  return found <= room;
}

// The elements of two vectors, the first of which are elements e[0] and e[1], that reach the least; by one warp.  `count`: entries so far, which lie in
// `shared_count` where warps share the list.  Two at a time, since one warp waits for most of its instructions.
template <typename T>
__device__ __forceinline__ void gather_from(const typename Row<T>::Vector& raw0, const typename Row<T>::Vector& raw1, const int (&e)[2], int vocab, float least, Entry* list, int room, int& count,
                                          int* shared_count) {
  const int lane = threadIdx.x & 31;
  float f[2][8];
  widen8(raw0, f[0]), widen8(raw1, f[1]);
  uint32_t mine = 0;
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    uint32_t bit[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) bit[k] = f[y][k] < least ? 0u : 1u << k;  // NaN is among them
    uint32_t m = ((bit[0] | bit[1]) | (bit[2] | bit[3])) | ((bit[4] | bit[5]) | (bit[6] | bit[7]));
    if (e[y] < 0) m &= 0xffu << -e[y];
    if (e[y] > vocab - 8) m &= e[y] < vocab ? 0xffu >> (e[y] + 8 - vocab) : 0u;
    mine |= m << 8 * y;
  }
  for (uint32_t all; (all = __ballot_sync(0xffffffffu, mine != 0)) != 0; mine &= mine - 1) {
    const int k = __ffs(mine) - 1;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = k & 8 ? f[1][i] : f[0][i];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = k & 4 ? x[i + 4] : x[i];
    x[0] = k & 2 ? x[2] : x[0], x[1] = k & 2 ? x[3] : x[1];
    const Entry entry = entry_of(key_of<T>(k & 1 ? x[1] : x[0]), (k & 8 ? e[1] : e[0]) + (k & 7));
    if (shared_count != nullptr) {
      count = lane == 0 ? atomicAdd(shared_count, __popc(all)) : 0;
      count = __shfl_sync(0xffffffffu, count, 0);
    }
    const int at = count + __popc(all & ((1u << lane) - 1));
    if (mine != 0 && at < room) list[at] = entry;
    count += __popc(all);
  }
}

// What cannot be above 0 but for roundings; NaN stays.
__device__ __forceinline__ float at_most_0(float x) { return x > 0.f ? 0.f : x; }
// The results of a row, by one warp, with its alternatives in order.
template <typename T, bool TOP>
__device__ __forceinline__ void finish(const Params& p, long long r, long long token, float logit, const Sums& sum, const Entry* entries) {
  const int lane = threadIdx.x & 31;
  const float log_s = log2f(sum.s);
  if constexpr (TOP) {
    for (int x = lane; x < p.top; x += 32) {
      const Entry e = entries[x];
      p.top_tokens[r * p.top + x] = index_in(e);
      p.top_logprobs[r * p.top + x] = at_most_0((value_of<T>(key_in(e)) - sum.base) * p.rate - log_s * kLn2);
    }
    __syncwarp();
  }
  if (lane == 0) {
    float lp = 0.f;
    if (token >= 0 && token < p.vocab) lp = at_most_0((logit - sum.base) * p.rate - log_s * kLn2);
    else if (token != p.ignore) TTB_NOTE_VIOLATION(token_stats);  // as a row that is ignored
    p.logprobs[r] = token == p.ignore ? 0.f : lp;
    const float entropy = (log_s - sum.t / sum.s) * kLn2;
    p.entropy[r] = entropy < 0.f ? 0.f : entropy;
    if (p.stats != nullptr) p.stats[2 * r] = sum.base, p.stats[2 * r + 1] = log_s;
  }
}

struct Shared {
  Sums warp[2][kWarps];
  Sums part[kMaxCluster];
};
struct SharedTop : Shared {
  alignas(16) uint32_t segments[2][kMaxSegments];
  alignas(16) uint32_t lanes[kMaxTop * 32];
  alignas(16) uint32_t elements[kMaxTop * 8];
  uint16_t chosen[3][kMaxTop];
  Entry candidates[kMostCandidates];
  Entry found[kMaxTop];                 // segments
  Entry entries[kMaxCluster][kMaxTop];  // in their order; the first CTA's are those of all
  int count, few;                       // candidates; whether `found` holds the segments to be looked at
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void wait_at(int barrier) { asm volatile("barrier.cta.sync %0, %1;" ::"r"(barrier), "n"(kThreads) : "memory"); }
__device__ __forceinline__ void wait_for_all() { asm volatile("barrier.cta.sync 5, %0;" ::"n"(kThreads) : "memory"); }
__device__ __forceinline__ void arrive_at(int barrier) { asm volatile("barrier.cta.arrive %0, %1;" ::"r"(barrier), "n"(kThreads) : "memory"); }

// Many rows that are not long: a warp streams and ends rows of its own, so that the ends of some lie beside the streams of others.
static constexpr int kOwnSegments = 256;  // of a row at most
static constexpr int kOwnCandidates = 256;
template <bool TOP>
static constexpr int kOwnWarps = TOP ? 12 : 16;  // of a CTA; what the ends of rows take in shared memory leaves room for twelve
struct OwnTop {
  alignas(16) uint32_t segments[kOwnSegments];
  Entry candidates[kOwnCandidates], found[kMaxTop], entries[kMaxTop];
  uint16_t chosen[kMaxTop];
};
template <typename T, bool TOP>
static constexpr int kOwnSlots = kSlots * kRun<T, TOP> * 8 * sizeof(T);
template <typename T, bool TOP>
static constexpr int kOwnBytes = kOwnSlots<T, TOP> + (TOP ? (sizeof(OwnTop) + 15) / 16 * 16 : 0);

// The want-th largest (want <= 32) of the lanes' keys, at least 1.
__device__ __forceinline__ uint32_t nth_of_lanes(uint32_t key, int want) {
  const int lane = threadIdx.x & 31;
  int above = 0;
#pragma unroll 8
  for (int x = 0; x < 32; ++x) {
    const uint32_t other = __shfl_sync(0xffffffffu, key, x);
    above += (other > key) | ((other == key) & (x < lane));
  }
  return max(1u, __shfl_sync(0xffffffffu, key, __ffs(__ballot_sync(0xffffffffu, above == want - 1)) - 1));
}

// The alternatives of a row, in order, from the maxima of its segments and of the lanes' elements; by one warp.
template <typename T>
__device__ __forceinline__ void choose_alone(const Row<T>& row, int want, float lane_most, OwnTop& sh) {
  const int lane = threadIdx.x & 31, segments = (row.vectors() + 31) / 32;
  const bool by_segments = segments > want;
  bool few = true;
  uint32_t least = 1;
  if (by_segments) {
    few = choose_few<T>(sh.segments, segments, want, sh.candidates, kOwnCandidates, sh.found);
    if (few) least = key_in(sh.found[want - 1]);
  } else {
    for (int i = lane; i < segments; i += 32) sh.segments[i] = key_of<T>(__uint_as_float(sh.segments[i]));
    if (want <= 32) least = nth_of_lanes(key_of<T>(lane_most), want);  // as many elements at least reach it
    else few = row.vocab <= kOwnCandidates;
  }
  __syncwarp();
  if (few) {
    const int n = by_segments ? want : segments;
    const float limit = least == 1 ? -INFINITY : value_of<T>(least);  // that of the lowest key is none
    int count = 0;
#pragma unroll 1
    for (int i = 0; i < n; i += 2) {
      typename Row<T>::Vector raw[2];
      int e[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int segment = i + y >= n ? segments : by_segments ? index_in(sh.found[i + y]) : i + y;
        e[y] = (segment * 32 + lane) * 8 - row.off;
        raw[y] = row.load(segment * 32 + lane);
      }
      gather_from<T>(raw[0], raw[1], e, row.vocab, limit, sh.candidates, kOwnCandidates, count, nullptr);
    }
    __syncwarp();
    if (count <= kOwnCandidates) {
      rank(sh.candidates, count, want, sh.entries);
      return;
    }
  }
  // many equal or ordered logits: one alternative after the other
  const int n = choose(sh.segments, segments, want, sh.chosen);
  Entry last = 0;
  for (int x = 0; x < want; ++x) {
    Entry best = 0;
    for (int i = 0; i < n; ++i) {
      const int j = sh.chosen[i] * 32 + lane;
      const typename Row<T>::Vector raw = row.load(j);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = j * 8 - row.off + k;
        const Entry entry = e >= 0 && e < row.vocab ? entry_of(key_of<T>(widened(raw.v[k])), e) : 0;
        if ((x == 0 || entry < last) && entry > best) best = entry;  // nothing bounds the first: a NaN of 32 bits at index 0 is the largest number
      }
    }
    const uint32_t high = __reduce_max_sync(0xffffffffu, key_in(best));
    const uint32_t low = __reduce_max_sync(0xffffffffu, key_in(best) == high ? static_cast<uint32_t>(best) : 0u);
    last = static_cast<Entry>(high) << 32 | low;
    if (lane == 0) sh.entries[x] = last;
  }
  __syncwarp();
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kOwnWarps<TOP> * 32, kCtas) row_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t slots[];
  using Vector = typename Row<T>::Vector;
  constexpr int kMine = kEach<T, TOP>, kVectors = kRun<T, TOP>, kPieces = sizeof(T) / 2, kPieceBytes = kVectors * 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* my_slots = slots + warp * kOwnBytes<T, TOP> + lane * 16;
  [[maybe_unused]] OwnTop& sh = *reinterpret_cast<OwnTop*>(slots + warp * kOwnBytes<T, TOP> + kOwnSlots<T, TOP>);
  const uint32_t rows = p.rows, step = gridDim.x * kOwnWarps<TOP>, first = warp * gridDim.x + blockIdx.x;
  auto row_of = [&](uint32_t r) {
    const uint32_t outer = static_cast<uint32_t>(p.inner) >= rows ? 0u : r / p.inner;
    return Row<T>(static_cast<const T*>(p.x) + outer * p.step_outer + static_cast<long long>(r - outer * p.inner) * p.step_inner, p.vocab);
  };
  if (first >= rows) return;
  uint32_t ahead_r = first;
  Row<T> ahead_row = row_of(first);
  int ahead_j = 0, ahead_slot = 0;
  auto whole = [](const Row<T>& row, int j0) { return j0 >= row.whole_from() && j0 + kVectors <= row.whole_to(); };  // the same for a warp
  auto copy_ahead = [&]() {
    if (ahead_r < rows) {
      if (whole(ahead_row, ahead_j)) {
        const uint4* from = reinterpret_cast<const uint4*>(ahead_row.vector(ahead_j)) + lane;
        const uint32_t to = smem_u32(my_slots) + ahead_slot * kPieces * kPieceBytes;
#pragma unroll
        for (int a = 0; a < kMine; ++a)
#pragma unroll
          for (int x = 0; x < kPieces; ++x) copy16(to + x * kPieceBytes + a * 512, from + (a * kPieces + x) * 32);
      }
      ahead_slot = ahead_slot + 1 == kSlots ? 0 : ahead_slot + 1;
      ahead_j += kVectors;
      if (ahead_j >= ahead_row.vectors()) {
        ahead_r += step, ahead_j = 0;
        if (ahead_r < rows) ahead_row = row_of(ahead_r);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  copy_ahead(), copy_ahead();
  const uint64_t c2 = pack_f32x2(p.c, p.c);
  int slot = 0;
  for (uint32_t r = first; r < rows; r += step) {
    const Row<T> row = row_of(r);
    const int vectors = row.vectors();
    const long long token = p.tokens[r];
    Running run{p.c};
    const float lift = vectors > 32 ? p.lift : 0.f;  // the first vectors are the row: their maximum is the base
    float lane_most = -INFINITY;
    auto note = [&](int j, float most) {  // the maximum of a segment
      if constexpr (TOP) {
        lane_most = max_nan(lane_most, most);
        const float m = warp_max_nan(most);
        if (lane == 0) sh.segments[j >> 5] = __float_as_uint(m);
      }
    };
    for (int j0 = 0; j0 < vectors; j0 += kVectors) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      copy_ahead();  // to the slot before this one
      if (whole(row, j0)) {
        const uint8_t* at = my_slots + slot * kPieces * kPieceBytes;
#pragma unroll
        for (int a = 0; a < kMine; ++a) {
          Vector raw;
#pragma unroll
          for (int x = 0; x < kPieces; ++x) reinterpret_cast<uint4*>(raw.v)[x] = *reinterpret_cast<const uint4*>(at + x * kPieceBytes + a * 512);
          if constexpr (TOP) note(j0 + a * 32, most_of_vector<T>(raw));
          if (a == 0 && j0 == 0) run.begin(warp_max_nan(most_of_vector<T>(raw)) + lift);
          run.take<T>(raw, c2);
        }
      } else {
#pragma unroll 1
        for (int a = 0; a < kMine && j0 + a * 32 < vectors; ++a) {
          float f[8];
          widen8(row.load(j0 + a * 32 + lane), f);
          note(j0 + a * 32, most_of(f));
          if (a == 0 && j0 == 0) run.begin(warp_max_nan(most_of(f)) + lift);
          run.careful(f);
        }
      }
      slot = slot + 1 == kSlots ? 0 : slot + 1;
    }
    const T logit = token >= 0 && token < p.vocab ? row.x[token] : T();
    const Sums sum = joined_lanes(run.sums(), p.c);
    __syncwarp();
    if constexpr (TOP) {
      choose_alone<T>(row, p.top, lane_most, sh);
      finish<T, TOP>(p, r, token, widened(logit), sum, sh.entries);
    } else {
      finish<T, TOP>(p, r, token, widened(logit), sum, nullptr);
    }
    __syncwarp();
  }
}

// grid: CTAs that take rows in turn, or for few rows a cluster for each
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, kCtas) stats_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t slots[];
  __shared__ std::conditional_t<TOP, SharedTop, Shared> sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = cluster.num_blocks(), split = cluster.block_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t step = gridDim.x / splits, rows = p.rows;  // below 2^31
  auto row_of = [&](uint32_t r) {
    const uint32_t outer = static_cast<uint32_t>(p.inner) >= rows ? 0u : r / p.inner;
    return Row<T>(static_cast<const T*>(p.x) + outer * p.step_outer + static_cast<long long>(r - outer * p.inner) * p.step_inner, p.vocab);
  };
  struct Part {  // of a row, in vectors and segments of 32 of them
    int first, end, segments;
  };
  auto part_of = [&](const Row<T>& row) {
    const int vectors = row.vectors(), all = (vectors + 31) / 32, per = splits == 1 ? all : (all + splits - 1) / splits, from = min(per * split, all), count = min(all - from, per);
    return Part{from * 32, min(vectors, (from + count) * 32), count};
  };

  [[maybe_unused]] auto keys_of = [&](const Row<T>& row, const Part& part, int j, uint32_t (&key)[8]) {  // of a vector's elements
    if (j >= row.whole_from() && j < min(part.end, row.whole_to())) {
      float f[8];
      widen8(Row<T>::whole(row.vector(j)), f);
#pragma unroll
      for (int k = 0; k < 8; ++k) key[k] = key_of<T>(f[k]);
    } else {
      const long long e = j * 8ll - row.off;
#pragma unroll
      for (int k = 0; k < 8; ++k) key[k] = j < part.end ? row.key(e + k) : 0u;
    }
  };
  // The elements of the segments that were found which reach the least of their maxima; by one warp, or by all, `member` of which this is
  [[maybe_unused]] auto gather = [&](const Row<T>& row, const Part& part, int member) {
    if constexpr (TOP) {
    const float least = value_of<T>(key_in(sh.found[p.top - 1]));
    int count = 0;
    if (splits > 1) {
#pragma unroll 1
      for (int i0 = member; i0 < p.top; i0 += 2 * (kWarps + 1)) {
        typename Row<T>::Vector raw[2];
        int e[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int i = i0 + y * (kWarps + 1), j = i < p.top ? part.first + index_in(sh.found[i]) * 32 + lane : part.end;
          e[y] = j < part.end ? j * 8 - row.off : p.vocab;
#pragma unroll
          for (int k = 0; k < 8; ++k) raw[y].v[k] = narrowed<T>(-INFINITY);
          if (j < part.end) raw[y] = row.load(j);
        }
        gather_from<T>(raw[0], raw[1], e, p.vocab, least, sh.candidates, kMostCandidates, count, &sh.count);
      }
    } else {
      // a ring of pairs of segments: every lane copies its vectors and reads them, so that no other lane has to be waited for
      constexpr int kPairs = 4, kVectorBytes = 8 * sizeof(T);
      static_assert(kPairs * 64 * kVectorBytes <= sizeof(sh.lanes), "the ring lies where lanes do");
      uint8_t* ring = reinterpret_cast<uint8_t*>(sh.lanes) + lane * kVectorBytes;
      const int pairs = (p.top + 1) / 2;
      auto first_of = [&](int i) { return i < p.top ? (part.first + index_in(sh.found[i]) * 32 + lane) * 8 - row.off : p.vocab; };  // element; vocabularies with alternatives are below 2^21
#pragma unroll 1
      for (int i = 0; i < pairs + kPairs - 1; ++i) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int e = i < pairs ? first_of(2 * i + y) : p.vocab;
          uint8_t* to = ring + ((i % kPairs) * 2 + y) * 32 * kVectorBytes;
          if (e >= 0 && e <= p.vocab - 8) {
#pragma unroll
            for (int x = 0; x < kVectorBytes / 16; ++x) copy16(smem_u32(to) + x * 16, reinterpret_cast<const uint4*>(row.x + e) + x);
          } else if (e < p.vocab) {
#pragma unroll 1
            for (int k = 0; k < 8; ++k) reinterpret_cast<T*>(to)[k] = e + k >= 0 && e + k < p.vocab ? row.x[e + k] : narrowed<T>(-INFINITY);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (i < kPairs - 1) continue;
        asm volatile("cp.async.wait_group %0;" ::"n"(kPairs - 1) : "memory");
        const int at = i - (kPairs - 1), e[2] = {first_of(2 * at), first_of(2 * at + 1)};
        const auto* from = reinterpret_cast<const typename Row<T>::Vector*>(ring + (at % kPairs) * 64 * kVectorBytes);
        gather_from<T>(Row<T>::whole(from), Row<T>::whole(from + 32), e, p.vocab, least, sh.candidates, kMostCandidates, count, nullptr);
      }
      if (lane == 0) sh.count = count;
    }
    __syncwarp();
    }
  };
  if constexpr (TOP) {
    if (threadIdx.x == kWarps * 32) sh.count = 0;
  }

  if (warp < kWarps) {
    const uint64_t c2 = pack_f32x2(p.c, p.c);
    constexpr int kMine = kEach<T, TOP>, kPieces = sizeof(T) / 2;  // 16-byte pieces of a vector; a lane's are 512 bytes apart, since a copy that leaves out every other piece costs as much as all
    using Vector = typename Row<T>::Vector;
    uint8_t* my_slots = slots + (warp * kRun<T, TOP> + lane) * 16;  // piece x of vector a of slot s: (s * kPieces + x) slots' pieces and a * 32 vectors further on
    constexpr int kPieceBytes = kWarps * kRun<T, TOP> * 16;
    // the next run to be copied
    uint32_t ahead_r = blockIdx.x / splits;
    Row<T> ahead_row = row_of(ahead_r < rows ? ahead_r : 0);
    Part ahead_part = part_of(ahead_row);
    int ahead_j = ahead_part.first + warp * kRun<T, TOP>, ahead_slot = 0;
    auto whole = [](const Row<T>& row, const Part& part, int j0) { return j0 >= row.whole_from() && j0 + kRun<T, TOP> <= min(part.end, row.whole_to()); };  // the same for a warp
    auto copy_ahead = [&]() {
      while (ahead_r < rows && ahead_j >= ahead_part.end) {
        ahead_r += step;
        if (ahead_r < rows) ahead_row = row_of(ahead_r), ahead_part = part_of(ahead_row), ahead_j = ahead_part.first + warp * kRun<T, TOP>;
      }
      if (ahead_r < rows) {
        if (whole(ahead_row, ahead_part, ahead_j)) {
          const uint4* from = reinterpret_cast<const uint4*>(ahead_row.vector(ahead_j)) + lane;
          const uint32_t to = smem_u32(my_slots) + ahead_slot * kPieces * kPieceBytes;
#pragma unroll
          for (int a = 0; a < kMine; ++a)
#pragma unroll
            for (int x = 0; x < kPieces; ++x) copy16(to + x * kPieceBytes + a * 512, from + (a * kPieces + x) * 32);
        }
        ahead_j += kWarps * kRun<T, TOP>;
        ahead_slot = ahead_slot + 1 == kSlots ? 0 : ahead_slot + 1;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    copy_ahead(), copy_ahead();
    int buffer = 0, turn = 0, slot = 0;
    for (uint32_t r = blockIdx.x / splits; r < rows; r += step, buffer ^= 1, ++turn) {
      const Row<T> row = row_of(r);
      const Part part = part_of(row);
      if (turn > 1) wait_at(3 + buffer);  // what lies in this buffer has been used
      Running run{p.c};
      auto note = [&](int j, float most) {  // the maximum of a segment
        if constexpr (TOP) {
          const float m = warp_max_nan(most);
          if (lane == 0) sh.segments[buffer][(j - part.first) >> 5] = __float_as_uint(m);  // the warp that ends the row makes a key of it
        }
      };
      const int first = part.first + warp * kRun<T, TOP>;
      for (int j0 = first; j0 < part.end; j0 += kWarps * kRun<T, TOP>) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        copy_ahead();  // to the slot before this one
        if (whole(row, part, j0)) {
          const uint8_t* at = my_slots + slot * kPieces * kPieceBytes;
#pragma unroll
          for (int a = 0; a < kMine; ++a) {
            Vector raw;
#pragma unroll
            for (int x = 0; x < kPieces; ++x) reinterpret_cast<uint4*>(raw.v)[x] = *reinterpret_cast<const uint4*>(at + x * kPieceBytes + a * 512);
            if constexpr (TOP) note(j0 + a * 32, most_of_vector<T>(raw));
            if (a == 0 && j0 == first) run.begin(warp_max_nan(most_of_vector<T>(raw)) + p.lift);
            run.take<T>(raw, c2);
          }
        } else {
#pragma unroll 1
          for (int a = 0; a < kMine && j0 + a * 32 < part.end; ++a) {
            const int j = j0 + a * 32 + lane;
            float f[8];
            if (j < part.end) {
              widen8(row.load(j), f);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = -INFINITY;
            }
            note(j0 + a * 32, most_of(f));
            if (a == 0 && j0 == first) run.begin(warp_max_nan(most_of(f)) + p.lift);
            run.careful(f);
          }
        }
        slot = slot + 1 == kSlots ? 0 : slot + 1;
      }
      const Sums mine = joined_lanes(run.sums(), p.c);
      if (lane == 0) sh.warp[buffer][warp] = mine;
      __syncwarp();
      arrive_at(1 + buffer);
    }
    if (splits > 1) {
      if constexpr (TOP) {
        wait_for_all();
        const Row<T> row = row_of(blockIdx.x / splits);
        if (sh.few) gather(row, part_of(row), warp);
        wait_for_all();
      }
      cluster.sync(), cluster.sync();
    }
    return;
  }

  // ------------------------------------------------------------------------------------------------ the warp that ends rows
  auto choose_segments = [&](const Part& part, uint32_t* segments) {  // sh.few: whether it went without a search
    if constexpr (TOP) {
    const bool few = part.segments > p.top && choose_few<T>(segments, part.segments, p.top, sh.candidates, kMostCandidates, sh.found);
    if (part.segments <= p.top)
      for (int i = lane; i < part.segments; i += 32) segments[i] = key_of<T>(__uint_as_float(segments[i]));
    __syncwarp();
    if (lane == 0) sh.few = few;
    __syncwarp();
    }
  };
  auto select = [&](const Row<T>& row, const Part& part, uint32_t* segments, Entry* to) {  // the alternatives of a part, in their order, behind gather()
    if constexpr (TOP) {
    const int count = sh.few ? sh.count : kMostCandidates + 1;
    __syncwarp();
    if (lane == 0) sh.count = 0;
    if (count <= kMostCandidates) {
      rank(sh.candidates, count, p.top, to);
      return;
    }
    const int n_segments = choose(segments, part.segments, p.top, sh.chosen[0]);
    for (int i = 0; i < n_segments; ++i) {
      uint32_t key[8], most = 0;
      keys_of(row, part, part.first + sh.chosen[0][i] * 32 + lane, key);
#pragma unroll
      for (int k = 0; k < 8; ++k) most = max(most, key[k]);
      sh.lanes[i * 32 + lane] = most;
    }
    __syncwarp();
    const int n_lanes = choose(sh.lanes, n_segments * 32, p.top, sh.chosen[1]);
    auto index_of = [&](int i) {  // of element i of the chosen lanes
      const int at = sh.chosen[1][i >> 3];
      return (part.first + sh.chosen[0][at >> 5] * 32ll + (at & 31)) * 8 - row.off + (i & 7);
    };
    for (int i = lane; i < n_lanes * 8; i += 32) sh.elements[i] = row.key(index_of(i));
    __syncwarp();
    const int n = choose(sh.elements, n_lanes * 8, p.top, sh.chosen[2]);
    for (int i = lane; i < n; i += 32) {
      const uint32_t key = sh.elements[sh.chosen[2][i]];
      sh.candidates[i] = key != 0 ? entry_of(key, static_cast<int>(index_of(sh.chosen[2][i]))) : 0;
    }
    __syncwarp();
    rank(sh.candidates, n, p.top, to);
    }
  };
  auto first_entries = [&]() -> const Entry* {
    if constexpr (TOP) return sh.entries[0];
    else return nullptr;
  };
  auto sum_of = [&](int buffer) {  // of the warps
    return joined_lanes(lane < kWarps ? sh.warp[buffer][lane] : Sums{0.f, 0.f, 0.f}, p.c);
  };
  if (splits == 1) {
    int buffer = 0;
    auto logit_of = [&](uint32_t r, long long token) { return token >= 0 && token < p.vocab ? row_of(r).x[token] : T(); };
    long long next_token = p.tokens[blockIdx.x];  // a row ahead
    T next_logit = logit_of(blockIdx.x, next_token);
    for (uint32_t r = blockIdx.x; r < rows; r += step, buffer ^= 1) {
      const Row<T> row = row_of(r);
      const long long token = next_token;
      const T logit = next_logit;
      wait_at(1 + buffer);
      if (r + step < rows) next_token = p.tokens[r + step];
      const Sums sum = sum_of(buffer);
      if constexpr (TOP) {
        const Part part = part_of(row);
        choose_segments(part, sh.segments[buffer]);
        if (sh.few) gather(row, part, 0);
        select(row, part, sh.segments[buffer], sh.entries[0]);
      }
      __syncwarp();
      if (r + 2 * step < rows) arrive_at(3 + buffer);
      if (r + step < rows) next_logit = logit_of(r + step, next_token);
      finish<T, TOP>(p, r, token, widened(logit), sum, first_entries());
    }
    return;
  }
  const uint32_t r = blockIdx.x / splits;
  const Row<T> row = row_of(r);
  const long long token = p.tokens[r];
  const T logit = token >= 0 && token < p.vocab ? row.x[token] : T();
  wait_at(1);
  if constexpr (TOP) {
    const Part part = part_of(row);
    choose_segments(part, sh.segments[0]);
    wait_for_all();
    if (sh.few) gather(row, part, kWarps);
    wait_for_all();
  }
  cluster.sync();  // all CTAs have started: their shared memory may be written
  auto* home = cluster.map_shared_rank(&sh, 0);
  const Sums mine = sum_of(0);
  if (lane == 0) home->part[split] = mine;
  if constexpr (TOP) select(row, part_of(row), sh.segments[0], home->entries[split]);
  cluster.sync();
  if (split != 0) return;
  const Sums sum = joined_lanes(lane < splits ? sh.part[lane] : Sums{0.f, 0.f, 0.f}, p.c);
  if constexpr (TOP) {
    uint32_t least = 1;  // a part with as many entries has nothing lower to give
    for (int i = 0; i < splits; ++i) least = max(least, key_in(sh.entries[i][p.top - 1]));
    int count = 0;
    for (int i = lane; i < splits * kMaxTop; i += 32) {  // kMaxTop is a multiple of 32
      const Entry e = i % kMaxTop < p.top ? sh.entries[i / kMaxTop][i % kMaxTop] : 0;
      append(sh.candidates, count, key_in(e) >= least, e);
    }
    __syncwarp();
    rank(sh.candidates, count, p.top, sh.entries[0]);
  }
  finish<T, TOP>(p, r, token, widened(logit), sum, first_entries());
}

static constexpr int kGradVectors = 4;  // of a thread
// Vectors of a row, up to which a warp takes a part: a CTA's part is filled badly by short rows, and its threads wait for the row's numbers together.  us with CTAs -> warps of 8192 rows: bf16 x 800
// 44 -> 12, x 8000 78 -> 51, x 32003 220 -> 186 (with 21 alternatives 259 -> 256), fp32 x 4000 57 -> 44 (73 -> 61); on the other side fp32 x 8000 87 -> 83 (100 -> 115), bf16 2048 x 151936 203 -> 205.
template <typename T>
static constexpr int kGradByWarp = sizeof(T) == 2 ? 4096 : 512;
// G threads, those of a CTA or of a warp, take a part of a row.
template <typename T, int G>
__global__ void __launch_bounds__(kGradThreads, 4) grad_kernel(const __grid_constant__ GradParams p) {
  constexpr int kBlock = G * kGradVectors;
  const int thread = G == kGradThreads ? threadIdx.x : threadIdx.x % G, unit = G == kGradThreads ? blockIdx.x : blockIdx.x * (kGradThreads / G) + threadIdx.x / G;  // units are below 2^31 - 8
  const int r = unit / p.parts, part = unit - r * p.parts;
  if (G != kGradThreads && r >= p.rows) return;
  const Row<T> row(static_cast<const T*>(p.x) + r / p.inner * p.step_outer + r % p.inner * p.step_inner, p.vocab);
  T* out = static_cast<T*>(p.dx) + static_cast<long long>(r) * p.vocab;
  const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(row.x)) & 15) == 0;  // whole vectors of the row are such of the gradient
  const int vectors = row.vectors(), j0 = part * kBlock;
  const bool whole = same && j0 >= row.whole_from() && j0 + kBlock <= row.whole_to();
  typename Row<T>::Vector raw[kGradVectors];
  constexpr int kPieces = sizeof(T) / 2;
  const int mine = (thread & ~31) * kPieces + (thread & 31);  // first of 16-byte pieces that lie 512 bytes apart: a warp's loads and stores leave no gaps
  if (whole) {
    const uint4* at = reinterpret_cast<const uint4*>(row.vector(j0)) + mine;
#pragma unroll
    for (int a = 0; a < kGradVectors; ++a)
#pragma unroll
      for (int i = 0; i < kPieces; ++i) reinterpret_cast<uint4*>(raw[a].v)[i] = __ldcs(at + a * G * kPieces + i * 32);
  } else if constexpr (G == 32) {  // rows that are all ends, as a rule
#pragma unroll
    for (int a = 0; a < kGradVectors; ++a) raw[a] = row.load(j0 + a * G + thread);
  }
  const long long token = p.tokens[r];
  const bool counts = token != p.ignore && token >= 0 && token < p.vocab;
  const float base = p.stats[2ll * r], log_s = p.stats[2ll * r + 1];
  const float g = p.g != nullptr && counts ? p.g[r] : 0.f, h = p.h != nullptr ? p.h[r] : 0.f;
  float all = 0.f, any = 0.f;
  if (p.k != nullptr) {  // a lane for each
    for (int i = threadIdx.x & 31; i < p.top; i += 32) {
      const float k = p.k[static_cast<long long>(r) * p.top + i];
      all += k, any += fabsf(k);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o), any += __shfl_xor_sync(0xffffffffu, any, o);
  }
  all += g, any += fabsf(g) + fabsf(h);
  const bool none = any == 0.f;  // zeros then, whatever the logits are; else what is NaN in a row reaches its gradient
  // -p (all + h (H + ln2 q)) / T with q = log2 p
  const float offset = -(all + (h != 0.f ? h * p.entropy[r] : 0.f)) * p.rate, slope = -h * kLn2 * p.rate;
  const uint64_t base2 = pack_f32x2(-base, -base), c2 = pack_f32x2(p.c, p.c), log2s = pack_f32x2(-log_s, -log_s), offset2 = pack_f32x2(offset, offset), slope2 = pack_f32x2(slope, slope);
  auto two = [&](float x0, float x1, float& d0, float& d1) {
    float q0, q1;
    unpack_f32x2(fma_f32x2(add_f32x2(pack_f32x2(x0, x1), base2), c2, log2s), q0, q1);
    q0 = max_nan(q0, kLowest), q1 = max_nan(q1, kLowest);
    unpack_f32x2(mul_f32x2(pack_f32x2(fast_exp2(q0), fast_exp2(q1)), fma_f32x2(slope2, pack_f32x2(q0, q1), offset2)), d0, d1);
  };
  auto eight = [&](const typename Row<T>::Vector& x) {
    typename Row<T>::Vector d;
    if (none) {
#pragma unroll
      for (int i = 0; i < 8; ++i) d.v[i] = narrowed<T>(0.f);
      return d;
    }
    float f[8];
    widen8(x, f);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float d0, d1;
      two(f[i], f[i + 1], d0, d1);
      d.v[i] = narrowed<T>(d0), d.v[i + 1] = narrowed<T>(d1);
    }
    return d;
  };
  if (whole) {
    uint4* to = reinterpret_cast<uint4*>(reinterpret_cast<typename Row<T>::Vector*>(out - row.off) + j0) + mine;
#pragma unroll
    for (int a = 0; a < kGradVectors; ++a) {
      const typename Row<T>::Vector d = eight(raw[a]);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) __stcs(to + a * G * kPieces + i * 32, reinterpret_cast<const uint4*>(d.v)[i]);
    }
  } else {
#pragma unroll G == 32 ? kGradVectors : 1
    for (int a = 0; a < kGradVectors; ++a) {
      const int j = j0 + a * G + thread;
      if (j >= vectors) break;
      typename Row<T>::Vector at_j;
      if constexpr (G == 32) at_j = raw[a];
      else at_j = row.load(j);
      const typename Row<T>::Vector d = eight(at_j);
      const long long e = j * 8ll - row.off;
      if (same && j >= row.whole_from() && j < row.whole_to()) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) __stcs(reinterpret_cast<uint4*>(out + e) + i, reinterpret_cast<const uint4*>(d.v)[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i >= 0 && e + i < p.vocab) out[e + i] = d.v[i];
      }
    }
  }
  // the token and the alternatives again, with what is theirs; of two equal ones both write the same
  const int targets = (p.k != nullptr ? p.top : 0) + 1;
  if constexpr (G == kGradThreads) __syncthreads();
  else __syncwarp();
  const long long* best = p.top_tokens + static_cast<long long>(r) * p.top;
  const float* of_best = p.k + static_cast<long long>(r) * p.top;
  auto put = [&](int x) {
    const long long target = x == 0 ? (counts ? token : -1) : best[x - 1];
    if (target >= 0 && (target + row.off) / 8 / kBlock == part) {
      float extra = counts && token == target ? g : 0.f, d, unused;
      for (int i = 0; i + 1 < targets; ++i) extra += best[i] == target ? of_best[i] : 0.f;
      two(widened(row.x[target]), 0.f, d, unused);
      out[target] = narrowed<T>(fmaf(extra, p.rate, d));
    }
  };
  if constexpr (G == kGradThreads) {
    if (!none && thread < targets) put(thread);
  } else {
    for (int x = none ? targets : thread; x < targets; x += G) put(x);
  }
}

// What a call brings, packed by the host language in this order.
struct Call {
  long long x, step_outer, step_inner, inner, rows, vocab, type, top, ignore;
  long long tokens, logprobs, entropy, stats, top_logprobs, top_tokens;
  long long g, h, k, dx;
};

static int shape_of(const Call& c) {
  if (c.rows <= 0 || c.vocab <= 0 || c.vocab > 0x7fffff00ll || c.inner <= 0 || c.inner > 0x7fffffff || c.top < 0 || c.top > kMaxTop || c.top > c.vocab || c.type < 0 || c.type > 2)
    return kErrBadShape;
  return kOk;
}

template <typename T, bool TOP>
static int launch(const Call& c, float log2_rate, float rate, cudaStream_t st) {
  Params p{};
  p.x = reinterpret_cast<const void*>(c.x), p.step_outer = c.step_outer, p.step_inner = c.step_inner, p.tokens = reinterpret_cast<const long long*>(c.tokens);
  p.logprobs = reinterpret_cast<float*>(c.logprobs), p.entropy = reinterpret_cast<float*>(c.entropy), p.stats = reinterpret_cast<float*>(c.stats);
  p.top_logprobs = reinterpret_cast<float*>(c.top_logprobs), p.top_tokens = reinterpret_cast<long long*>(c.top_tokens);
  p.ignore = c.ignore, p.rows = c.rows, p.inner = static_cast<int>(c.inner), p.vocab = static_cast<int>(c.vocab), p.top = static_cast<int>(c.top), p.c = log2_rate, p.rate = rate, p.lift = kLift / log2_rate;
  const long long segments = (c.vocab + 7 + 255) / 256;
  // A warp for a row, where there are rows for a good part of all warps.  us with CTAs for rows -> with warps, without / with 20 alternatives: bf16 600 x 2000 18 -> 12 / 51 -> 16, 8192 x 8000
  // 121 -> 43 / 317 -> 96, 8192 x 32000 141 -> 117 / 352 -> 180, fp32 8192 x 32000 184 -> 184 / 377 -> 240; on the other side bf16 600 x 32000 19 -> 29 / 47 -> 45, 333 x 50257 25 -> 41 / 39 -> 59,
  // fp32 1200 x 32000 43 -> 47 / 76 -> 68.
  const bool own = segments <= kOwnSegments && (segments <= (c.top > 4 ? c.top : 4) || c.rows * (32 / static_cast<int>(sizeof(T))) >= segments * sm_count());
  // few rows: a cluster to a row, while each of its CTAs has a run for every warp, as long as all are on an SM at once
  const long long at_once = static_cast<long long>(kCtas) * sm_count();
  int splits = 1;
  // and, with alternatives, has more segments than those (the last one too): their choice needs a search otherwise, 20 -> 45 us of 4 rows of 50257 with 29
  auto enough = [&](long long n) { return segments >= n * kWarps && (!TOP || segments - (n - 1) * ((segments + n - 1) / n) > c.top); };
  while (splits < kMaxCluster && ((c.rows * splits * 2 <= at_once && enough(splits * 2)) || (TOP && segments > static_cast<long long>(splits) * kMaxSegments))) splits *= 2;
  if ((TOP && segments > static_cast<long long>(splits) * kMaxSegments) || c.rows * splits > 0x7fffffffll) return kErrTooLarge;
  if (own) {
    constexpr int own_bytes = kOwnWarps<TOP> * kOwnBytes<T, TOP>;
    static bool own_attr[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return kErrDriver;
    if (!own_attr[device]) {
      if (cudaFuncSetAttribute(row_kernel<T, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, own_bytes) != cudaSuccess) return kErrDriver;
      own_attr[device] = true;
    }
    TTB_COUNT_LAUNCH(1);
    row_kernel<T, TOP><<<static_cast<unsigned>(c.rows < at_once ? c.rows : at_once), kOwnWarps<TOP> * 32, own_bytes, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? kOk : kErrDriver;
  }
  constexpr int bytes = kSlots * kSlotBytes<T, TOP>;
  static bool attr[64] = {};  // an attribute of the kernel on one device
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return kErrDriver;
  if (!attr[device]) {
    if (cudaFuncSetAttribute(stats_kernel<T, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return kErrDriver;
    attr[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = bytes;
  cfg.gridDim = dim3(static_cast<unsigned>(splits > 1 || c.rows < at_once ? c.rows * splits : at_once));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  TTB_COUNT_LAUNCH(1);
  return cudaLaunchKernelEx(&cfg, stats_kernel<T, TOP>, p) == cudaSuccess ? kOk : kErrDriver;
}
template <typename T>
static int launch_grad(const Call& c, float log2_rate, float rate, cudaStream_t st) {
  GradParams p{};
  p.x = reinterpret_cast<const void*>(c.x), p.step_outer = c.step_outer, p.step_inner = c.step_inner, p.tokens = reinterpret_cast<const long long*>(c.tokens);
  p.stats = reinterpret_cast<const float*>(c.stats), p.entropy = reinterpret_cast<const float*>(c.entropy), p.top_tokens = reinterpret_cast<const long long*>(c.top_tokens);
  p.g = reinterpret_cast<const float*>(c.g), p.h = reinterpret_cast<const float*>(c.h), p.k = reinterpret_cast<const float*>(c.k), p.dx = reinterpret_cast<void*>(c.dx);
  p.ignore = c.ignore, p.rows = c.rows, p.inner = static_cast<int>(c.inner), p.vocab = static_cast<int>(c.vocab), p.top = static_cast<int>(c.top), p.c = log2_rate, p.rate = rate;
  const long long vectors = (c.vocab + 7 + 7) / 8;
  const bool by_warp = vectors <= kGradByWarp<T>;
  const int each = (by_warp ? 32 : kGradThreads) * kGradVectors;
  p.parts = static_cast<int>((vectors + each - 1) / each);
  if (c.rows * p.parts > 0x7ffffff0ll) return kErrTooLarge;
  TTB_COUNT_LAUNCH(1);
  if (by_warp) grad_kernel<T, 32><<<static_cast<unsigned>((c.rows * p.parts * 32 + kGradThreads - 1) / kGradThreads), kGradThreads, 0, st>>>(p);
  else grad_kernel<T, kGradThreads><<<static_cast<unsigned>(c.rows * p.parts), kGradThreads, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrDriver;
}

}  // namespace tstat
}  // namespace ttb

// call: a tstat::Call; log2_rate = log2(e) / T, rate = 1 / T.
extern "C" int ttb_token_stats(const char* call, float log2_rate, float rate, void* stream) {
  using namespace ttb;
  using namespace ttb::tstat;
  const Call& c = *reinterpret_cast<const Call*>(call);
  const int rc = shape_of(c);
  if (rc != kOk) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto t) { return c.top > 0 ? launch<decltype(t), true>(c, log2_rate, rate, st) : launch<decltype(t), false>(c, log2_rate, rate, st); };
  return c.type == 0 ? go(__nv_bfloat16()) : c.type == 1 ? go(__half()) : go(0.f);
}
extern "C" int ttb_token_stats_bwd(const char* call, float log2_rate, float rate, void* stream) {
  using namespace ttb;
  using namespace ttb::tstat;
  const Call& c = *reinterpret_cast<const Call*>(call);
  const int rc = shape_of(c);
  if (rc != kOk) return rc;
  auto st = static_cast<cudaStream_t>(stream);
  return c.type == 0 ? launch_grad<__nv_bfloat16>(c, log2_rate, rate, st) : c.type == 1 ? launch_grad<__half>(c, log2_rate, rate, st) : launch_grad<float>(c, log2_rate, rate, st);
}
