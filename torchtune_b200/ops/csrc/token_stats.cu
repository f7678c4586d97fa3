// Log-probabilities of given tokens with the entropy and the likeliest alternatives, from one pass over the logits, and their gradient in one more.
//
// Of z = x / T, in units of log2 (c = log2(e) / T):  d = (x - base) c,  s = sum 2^d,  t = sum 2^d d,  base within 2^24 of the largest 2^z so far, so that
//   log p = ln2 (d - log2 s)        H = -sum p log p = ln2 (log2 s - t / s),
// where both terms stay below some 40: little cancels.  When the base moves up by a / c, s' = s 2^-a and t' = (t - a s) 2^-a.  A base that followed every new maximum would move in nearly all
// steps of a warp, since one of its 32 lanes has a new one; so it hardly ever moves after a thread's first elements.  Differences are taken before they are scaled: a row of a type's lowest values is
// one of equal logits.
// With g, h and k_j the gradients of the token's log-probability, of the entropy and of the alternatives' log-probabilities:
//   dx_v = ([v = token] g + sum_j [v = alternative j] k_j - p_v (g + sum_j k_j + h (log p_v + H))) / T.
//
// The alternatives are the `top` largest logits, of equal ones those with the lower index.  The pass leaves the largest value of every segment of 256 elements (what a warp reads at once) in shared
// memory; the `top` segments with the largest ones (of equal ones the first) hold all alternatives, since an element outside is beaten by `top` maxima.  The same choice among the 32 lanes of those
// segments and then among their eight elements leaves the alternatives, whatever the order of the logits, with a few hundred reads.  A choice is a search for the `top`-th largest key,
// bit by bit, by one warp, while the other CTAs of the SM stream.
//
// Rows begin at any address: vectors lie on 16 bytes, and the first and last of a row are read element by element.  Few rows are split over clusters of up to eight CTAs, which meet in the shared
// memory of the first.
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

static constexpr int kThreads = 256, kWarps = kThreads / 32;
static constexpr int kAhead = 4;  // vectors in flight per thread
static constexpr int kBlock = kThreads * kAhead;
static constexpr int kMaxTop = 64;
static constexpr int kMaxSegments = 2048;  // of a CTA
static constexpr int kMaxCluster = 8;
static constexpr float kLn2 = 0.6931471805599453f;
static constexpr float kLowest = -200.f;  // 2^kLowest is 0 in fp32
static constexpr float kReach = 24.f;     // log2 of how far exponentials may be above 1

struct Params {
  const void* x;  // row r at x + (r / inner) * step_outer + (r % inner) * step_inner, in elements
  long long step_outer, step_inner;
  const long long* tokens;
  float* logprobs;
  float* entropy;
  float* stats;          // [rows, 2]: base and log2 s, or nullptr
  float* top_logprobs;   // [rows, top]
  long long* top_tokens;
  long long ignore;
  int inner, vocab, top;
  float c, rate;  // log2(e) / T and 1 / T
};
struct GradParams {
  const void* x;
  long long step_outer, step_inner;
  const long long* tokens;
  const float *stats, *entropy;
  const long long* top_tokens;
  const float *g, *h, *k;  // gradients of log-probabilities, entropy and alternatives; nullptr: none
  void* dx;                // [rows, vocab]
  long long ignore;
  int inner, vocab, top, parts;  // parts: CTAs of a row
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

// base, s and t of a part of a row
struct Sums {
  float base, s, t;
};
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b, float c) {
  if (b.s == 0.f) return a;  // NaN goes on
  if (a.s == 0.f) return b;
  const Sums &hi = a.base >= b.base ? a : b, &lo = a.base >= b.base ? b : a;
  const float d = fmaxf((lo.base - hi.base) * c, kLowest), f = exp2f(d);
  return {hi.base, hi.s + lo.s * f, hi.t + (lo.t + lo.s * d) * f};
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

struct Entry {  // an alternative; index -1: none
  uint32_t key;
  int index;
};
struct Shared {
  Sums warp[kWarps];
  Sums part[kMaxCluster];
};
struct SharedTop : Shared {
  alignas(16) uint32_t segments[kMaxSegments];
  alignas(16) uint32_t lanes[kMaxTop * 32];  // also keys of the cluster's entries
  alignas(16) uint32_t elements[kMaxTop * 8];
  uint16_t chosen[3][kMaxTop];
  int counts[3];
  Entry entries[kMaxCluster][kMaxTop];  // in order of their index; the first CTA's are those of all
};

// grid: rows, each of `cluster` CTAs
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) stats_kernel(const __grid_constant__ Params p) {
  __shared__ std::conditional_t<TOP, SharedTop, Shared> sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int splits = cluster.num_blocks(), split = cluster.block_rank();
  const long long r = blockIdx.x / splits;
  const Row<T> row(static_cast<const T*>(p.x) + r / p.inner * p.step_outer + r % p.inner * p.step_inner, p.vocab);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int vectors = row.vectors(), all_segments = (vectors + 31) / 32, per = (all_segments + splits - 1) / splits;
  const int first = min(per * split, all_segments) * 32, segments = min(all_segments - first / 32, per), end = min(vectors, first + segments * 32);

  const uint64_t c2 = pack_f32x2(p.c, p.c);
  float limit = -INFINITY, base = 0.f;  // 0 until there is a logit above the infinitely low ones
  const float reach = kReach / p.c;
  uint64_t s2 = 0, t2 = 0;
  auto raise = [&](float most) {
    if (!(most <= limit)) {  // NaN too
      const float d = fminf(fmaxf((base - most) * p.c, kLowest), 0.f), g = fast_exp2(d);
      float s0, s1, t0, t1;
      unpack_f32x2(s2, s0, s1), unpack_f32x2(t2, t0, t1);
      const float s = s0 + s1, t = t0 + t1;
      s2 = pack_f32x2(s * g, 0.f), t2 = pack_f32x2((t + s * d) * g, 0.f);
      base = most, limit = most + reach;
    }
  };
  auto take = [&](const float (&f)[8]) {
    const uint64_t b2 = pack_f32x2(-base, -base);
    uint64_t sv = 0, tv = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint64_t d = mul_f32x2(add_f32x2(pack_f32x2(f[i], f[i + 1]), b2), c2);
      float d0, d1;
      unpack_f32x2(d, d0, d1);
      const uint64_t e = pack_f32x2(fast_exp2(d0), fast_exp2(d1));
      sv = add_f32x2(sv, e);
      tv = fma_f32x2(e, d, tv);
    }
    float t0, t1;
    unpack_f32x2(tv, t0, t1);
    if (t0 + t1 != t0 + t1) {  // an infinitely low logit (0 * -inf); its share is 0
      t0 = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = (f[i] - base) * p.c;
        t0 += fast_exp2(d) * (d < kLowest ? kLowest : d);
      }
      tv = pack_f32x2(t0, 0.f);
    }
    s2 = add_f32x2(s2, sv), t2 = add_f32x2(t2, tv);
  };
  auto note = [&](int j, float most) {  // the maximum of a segment
    if constexpr (TOP) {
      const float m = warp_max_nan(most);
      if (lane == 0) sh.segments[(j - first) >> 5] = key_of<T>(m);
    }
  };
  for (int j0 = first; j0 < end; j0 += kBlock) {
    if (j0 >= row.whole_from() && j0 + kBlock <= min(end, row.whole_to())) {  // the same for the CTA
      const typename Row<T>::Vector* at = row.vector(j0 + threadIdx.x);
      typename Row<T>::Vector raw[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) raw[a] = Row<T>::whole(at + a * kThreads);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        float f[8];
        widen8(raw[a], f);
        const float most = most_of(f);
        note(j0 + a * kThreads + threadIdx.x, most);
        raise(most);
        take(f);
      }
    } else {
#pragma unroll 1
      for (int a = 0; a < kAhead; ++a) {
        const int j = j0 + a * kThreads + threadIdx.x;
        if (j - lane >= end) break;  // the same for a warp
        float f[8];
        if (j < end) {
          widen8(row.load(j), f);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = -INFINITY;
        }
        const float most = most_of(f);
        note(j, most);
        raise(most);
        take(f);
      }
    }
  }
  Sums mine;
  {
    float a, b;
    mine.base = base;
    unpack_f32x2(s2, a, b), mine.s = a + b;
    unpack_f32x2(t2, a, b), mine.t = a + b;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums other = {__shfl_xor_sync(0xffffffffu, mine.base, o), __shfl_xor_sync(0xffffffffu, mine.s, o), __shfl_xor_sync(0xffffffffu, mine.t, o)};
    mine = lane & o ? joined(other, mine, p.c) : joined(mine, other, p.c);
  }
  if (lane == 0) sh.warp[warp] = mine;
  if (splits > 1) cluster.sync();  // all CTAs have started: their shared memory may be written
  else __syncthreads();
  auto* home = cluster.map_shared_rank(&sh, 0);
  if (threadIdx.x == 0) {
    mine = sh.warp[0];
    for (int w = 1; w < kWarps; ++w) mine = joined(mine, sh.warp[w], p.c);
    home->part[split] = mine;
  }

  if constexpr (TOP) {
    if (warp == 0) {
      const int n = choose(sh.segments, segments, p.top, sh.chosen[0]);
      if (lane == 0) sh.counts[0] = n;
    }
    __syncthreads();
    const int n_segments = sh.counts[0];
    for (int i = warp; i < n_segments; i += kWarps) {
      const int j = first + sh.chosen[0][i] * 32 + lane;
      uint32_t best = 0;
      if (j < end) {
        const typename Row<T>::Vector v = row.load(j);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const long long e = j * 8ll - row.off + k;
          const uint32_t key = e >= 0 && e < p.vocab ? key_of<T>(widened(v.v[k])) : 0u;
          best = max(best, key);
        }
      }
      sh.lanes[i * 32 + lane] = best;
    }
    __syncthreads();
    if (warp == 0) {
      const int n = choose(sh.lanes, n_segments * 32, p.top, sh.chosen[1]);
      if (lane == 0) sh.counts[1] = n;
    }
    __syncthreads();
    const int n_lanes = sh.counts[1];
    auto index_of = [&](int i) {  // of element i of the chosen lanes
      const int at = sh.chosen[1][i >> 3];
      return (first + sh.chosen[0][at >> 5] * 32ll + (at & 31)) * 8 - row.off + (i & 7);
    };
    for (int i = threadIdx.x; i < n_lanes * 8; i += kThreads) sh.elements[i] = row.key(index_of(i));
    __syncthreads();
    if (warp == 0) {
      const int n = choose(sh.elements, n_lanes * 8, p.top, sh.chosen[2]);
      for (int i = lane; i < p.top; i += 32) {
        Entry e = {0u, -1};
        if (i < n && sh.elements[sh.chosen[2][i]] != 0) e = {sh.elements[sh.chosen[2][i]], static_cast<int>(index_of(sh.chosen[2][i]))};
        home->entries[split][i] = e;
      }
    }
  }
  if (splits > 1) {
    cluster.sync();
    if (split != 0) return;
  } else {
    __syncthreads();
  }
  Sums sum = sh.part[0];
  for (int i = 1; i < splits; ++i) sum = joined(sum, sh.part[i], p.c);
  const float log_s = log2f(sum.s);
  if constexpr (TOP) {
    Entry* best = sh.entries[0];
    if (splits > 1) {
      for (int i = threadIdx.x; i < splits * p.top; i += kThreads) sh.lanes[i] = sh.entries[i / p.top][i % p.top].key;
      __syncthreads();
      Entry mine_too = {0u, -1};
      if (warp == 0) choose(sh.lanes, splits * p.top, p.top, sh.chosen[0]);
      __syncthreads();
      if (threadIdx.x < p.top) mine_too = sh.entries[sh.chosen[0][threadIdx.x] / p.top][sh.chosen[0][threadIdx.x] % p.top];
      __syncthreads();
      if (threadIdx.x < p.top) best[threadIdx.x] = mine_too;
      __syncthreads();
    }
    if (threadIdx.x < p.top) {
      const Entry e = best[threadIdx.x];
      int rank = 0;  // entries lie in order of their index
      for (int i = 0; i < p.top; ++i) rank += best[i].key > e.key || (best[i].key == e.key && i < static_cast<int>(threadIdx.x));
      p.top_tokens[r * p.top + rank] = e.index;
      p.top_logprobs[r * p.top + rank] = (widened(row.x[e.index]) - sum.base) * p.rate - log_s * kLn2;
    }
  }
  if (threadIdx.x == 0) {
    const long long token = p.tokens[r];
    float lp = 0.f;
    if (token >= 0 && token < p.vocab) lp = (widened(row.x[token]) - sum.base) * p.rate - log_s * kLn2;
    else if (token != p.ignore) TTB_NOTE_VIOLATION(token_stats);  // as a row that is ignored
    p.logprobs[r] = token == p.ignore ? 0.f : lp;
    p.entropy[r] = (log_s - sum.t / sum.s) * kLn2;
    if (p.stats != nullptr) p.stats[2 * r] = sum.base, p.stats[2 * r + 1] = log_s;
  }
}

static constexpr int kGradVectors = 4;  // of a thread
// grid: rows * parts
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) grad_kernel(const __grid_constant__ GradParams p) {
  constexpr int kBlock = kThreads * kGradVectors;
  const int r = blockIdx.x / p.parts, part = blockIdx.x - r * p.parts;
  const Row<T> row(static_cast<const T*>(p.x) + r / p.inner * p.step_outer + r % p.inner * p.step_inner, p.vocab);
  T* out = static_cast<T*>(p.dx) + static_cast<long long>(r) * p.vocab;
  const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(row.x)) & 15) == 0;  // whole vectors of the row are such of the gradient
  const int vectors = row.vectors(), j0 = part * kBlock;
  const bool whole = same && j0 >= row.whole_from() && j0 + kBlock <= row.whole_to();
  typename Row<T>::Vector raw[kGradVectors];
  if (whole) {
    const typename Row<T>::Vector* at = row.vector(j0 + threadIdx.x);
#pragma unroll
    for (int a = 0; a < kGradVectors; ++a)
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(raw[a].v)[i] = __ldcs(reinterpret_cast<const uint4*>(at + a * kThreads) + i);
  }
  const long long token = p.tokens[r];
  const bool counts = token != p.ignore && token >= 0 && token < p.vocab;
  const float base = p.stats[2ll * r], log_s = p.stats[2ll * r + 1];
  const float g = p.g != nullptr && counts ? p.g[r] : 0.f, h = p.h != nullptr ? p.h[r] : 0.f;
  float all = g;
  if (p.k != nullptr)
    for (int i = 0; i < p.top; ++i) all += p.k[static_cast<long long>(r) * p.top + i];
  // -p (all + h (H + ln2 q)) / T with q = log2 p
  const float offset = -(all + (h != 0.f ? h * p.entropy[r] : 0.f)) * p.rate, slope = -h * kLn2 * p.rate;
  const uint64_t base2 = pack_f32x2(-base, -base), c2 = pack_f32x2(p.c, p.c), log2s = pack_f32x2(-log_s, -log_s), offset2 = pack_f32x2(offset, offset), slope2 = pack_f32x2(slope, slope);
  auto two = [&](float x0, float x1, float& d0, float& d1) {
    float q0, q1;
    unpack_f32x2(fma_f32x2(add_f32x2(pack_f32x2(x0, x1), base2), c2, log2s), q0, q1);
    q0 = fmaxf(q0, kLowest), q1 = fmaxf(q1, kLowest);
    unpack_f32x2(mul_f32x2(pack_f32x2(fast_exp2(q0), fast_exp2(q1)), fma_f32x2(slope2, pack_f32x2(q0, q1), offset2)), d0, d1);
  };
  auto eight = [&](const typename Row<T>::Vector& x) {
    typename Row<T>::Vector d;
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
    typename Row<T>::Vector* to = reinterpret_cast<typename Row<T>::Vector*>(out - row.off) + j0 + threadIdx.x;
#pragma unroll
    for (int a = 0; a < kGradVectors; ++a) {
      const typename Row<T>::Vector d = eight(raw[a]);
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) __stcs(reinterpret_cast<uint4*>(to + a * kThreads) + i, reinterpret_cast<const uint4*>(d.v)[i]);
    }
  } else {
#pragma unroll 1
    for (int a = 0; a < kGradVectors; ++a) {
      const int j = j0 + a * kThreads + threadIdx.x;
      if (j >= vectors) break;
      const typename Row<T>::Vector d = eight(row.load(j));
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
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < targets) {
    const long long* best = p.top_tokens + static_cast<long long>(r) * p.top;
    const float* of_best = p.k + static_cast<long long>(r) * p.top;
    const long long mine = threadIdx.x == 0 ? (counts ? token : -1) : best[threadIdx.x - 1];
    if (mine >= 0 && (mine + row.off) / 8 / kBlock == part) {
      float extra = counts && token == mine ? g : 0.f, d, unused;
      for (int i = 0; i + 1 < targets; ++i) extra += best[i] == mine ? of_best[i] : 0.f;
      two(widened(row.x[mine]), 0.f, d, unused);
      out[mine] = narrowed<T>(fmaf(extra, p.rate, d));
    }
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
  p.ignore = c.ignore, p.inner = static_cast<int>(c.inner), p.vocab = static_cast<int>(c.vocab), p.top = static_cast<int>(c.top), p.c = log2_rate, p.rate = rate;
  const long long segments = (c.vocab + 7 + 255) / 256;
  // few rows: more CTAs to a row, up to two for an SM, while each has eight segments (one for every warp)
  int splits = 1;
  while (splits < kMaxCluster && ((c.rows * splits * 2 <= 2ll * sm_count() && segments >= splits * 2 * kWarps) || (TOP && segments > static_cast<long long>(splits) * kMaxSegments))) splits *= 2;
  if ((TOP && segments > static_cast<long long>(splits) * kMaxSegments) || c.rows * splits > 0x7fffffffll) return kErrTooLarge;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(c.rows * splits));
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
  p.ignore = c.ignore, p.inner = static_cast<int>(c.inner), p.vocab = static_cast<int>(c.vocab), p.top = static_cast<int>(c.top), p.c = log2_rate, p.rate = rate;
  const long long vectors = (c.vocab + 7 + 7) / 8;
  p.parts = static_cast<int>((vectors + kThreads * kGradVectors - 1) / (kThreads * kGradVectors));
  if (c.rows * p.parts > 0x7fffffffll) return kErrTooLarge;
  TTB_COUNT_LAUNCH(1);
  grad_kernel<T><<<static_cast<unsigned>(c.rows * p.parts), kThreads, 0, st>>>(p);
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
