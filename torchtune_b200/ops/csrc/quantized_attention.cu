// Attention of a few queries over a key/value cache held in 4 or 8 bits (rows as quantized_cache.cu writes them).
//
//   score[r, k] = c sum_j ks[k, j] sum_{d in j} q[r, d] (kc[k, d] - h)          j: groups of 32 channels, h = 2^(bits - 1)
//   out[r, d]   = sum_k (p[r, k] vs[k, j(d)]) (vc[k, d] - h) / sum_k p[r, k]    p: exponentials of the scores
//
// A small integer i in the low bits of a 16-bit word is the subnormal bf16 number i * 2^-133 (up to 255: the exponents 0 and 1 have the same step), and the tensor cores take subnormal operands
// as they are.  So the codes, masked out of their words, are matrix operands without a conversion, and exact; a nibble in the upper half of a byte is 16 times its code, which the
// operand on the other side or the result makes up for.  Queries and probabilities are scaled by powers of two (2^110 over the largest query value; 2^90) to meet them in the middle of fp32's range.
// h is taken off by a sum that starts at -h sum q, and of values by a product of its own with a matrix of -h, so that the running sum never holds it.  Scales are applied in fp32, to the scores
// of a group and to the probabilities in front of a group's product; nothing is rounded but the probabilities times their scale (to bf16, as in the other attention kernels; their sum is
// fp32) and the result.
//
// Decoding is bound by the bytes of the cache as long as turning codes into operands keeps up: at 6.5 TB/s an SM takes in 41 4-bit codes per cycle and issues 128 lane instructions, half of them to the
// integer unit.  So keys (and channels) are the 16 rows of an m16n8k16 tile and a key head's query rows its 8 columns: no code is turned twice, and few rows do not pay for 16.  A lane holds a
// quarter of a row of keys (with eight channels of every group) and, for the second product, half a word of every group of four rows of values, whose nibbles meet in one register as
// the pairs of keys that the operand wants.
// Measured (4 bits, 32 query on 8 key heads of 128 channels, cold L2, replayed from a graph): 64 x 4096 slots 66 us (4.5 TB/s), in 8 bits 102 us (5.6 TB/s); 16 x 732 9.3 us; 1 x 65 000 25 us.  The same
// from bf16 rows: 176, 29 and 117 us.  The large ones issue 590 instructions per tile at 0.58 per cycle and scheduler (integer unit 54 % busy, tensor cores 37 %): 16 warps per SM (128
// registers each) do not hide the latency of the chains from load to product, and with 12, 20 or 24 it is no better.  The small ones are latency.
//
// A warp takes tiles of 32 keys through a cp.async ring of its own, with its own running maximum (moved only when a score exceeds it by 2^8), sum and output.  Tiles are dealt round-robin to
// the warps of a CTA and the CTAs of a cluster, which meet once at the end in distributed shared memory in a fixed order; of few and long rows to more CTAs, which meet in a workspace, also in a
// fixed order, in a second launch.  Tiles without a visible key are not read, and only tiles that some query does not see whole pay for visibility.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "common/ptx.cuh"
#include "common/tmap.h"

namespace ttb {
namespace qattn {

namespace cg = cooperative_groups;

static constexpr int kWarps = 4;
static constexpr int kTileKeys = 32;
static constexpr int kMaxCluster = 8;        // portable; the CTAs of larger ones share SMs while others idle (8 heads of 65 003 slots, 16 splits: 45 us as clusters, 37 in a workspace)
static constexpr int kMaxSpread = 128;       // splits that meet in a workspace
static constexpr int kMaxBitBytes = 16384;   // visibility words of one CTA
static constexpr float kLog2e = 1.4426950408889634f;
static constexpr float kRescale = 8.f;       // log2 units
static constexpr int kMaxDevices = 64;
static constexpr uint32_t kWhole = 0x80000000u, kSeen = 0x40000000u, kIndex = 0x3fffffffu;  // of an entry of the list of tiles: all queries see all of it; some see some

struct Params {
  const __nv_bfloat16* q;  // [b, s, hq, D]
  const uint8_t *kc, *vc;  // rows of one head one behind the other
  const uint8_t *ks, *vs;
  long long kc_b, kc_h, ks_b, ks_h, vc_b, vc_h, vs_b, vs_h;  // bytes
  __nv_bfloat16* o;        // [b, s, hq, D]
  const uint8_t* mask;     // row (b, i) at mask + b * mask_b + i * mask_r, nonzero = visible; or nullptr
  long long mask_b, mask_r;
  const int* key_start;    // [b] or nullptr
  int offset;              // >= 0: query i sits in slot offset + i and sees no later one
  int window, sinks;       // window > 0: of the slots up to its own it sees the last `window` and the first `sinks`
  int s, sk, hq, hkv, group;
  int per_query;           // 65536 / group + 1: query of a row (below 16) without a division
  int tiles;               // to be dealt
  int skip_from, skipped;  // tiles skip_from ... skip_from + skipped - 1 lie between the first tokens and every window
  float scale;
  float* work;  // results of splits that are no cluster
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t x;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
  return x;
}
template <int WORDS>  // consecutive words of one 16-byte piece
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t* x) {
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(a) : "memory");
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(a) : "memory");
  else
    x[0] = lds32(a);
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

template <int D, int BITS>
struct Layout {
  static constexpr int kGroups = D / 32;
  static constexpr int kRow = D * BITS / 8;           // bytes of a row's codes
  static constexpr int kPieces = kRow / 16;
  static constexpr int kQuarter = kRow / 4;           // bytes that one lane loads
  static constexpr int kWords = kQuarter / 4;
  static constexpr int kPerLoad = kQuarter % 16 == 0 ? 4 : (kQuarter % 8 == 0 ? 2 : 1);
  static constexpr int kCodes = kTileKeys * kRow;
  static constexpr int kScales = kTileKeys * kGroups * 2;
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kStages = 2;                   // a third takes room from other CTAs (8 bits, 16 x 4111 slots of 128 channels, 16 query rows: 47 us, with three 51; 1 x 65 000, one: 38.7 and 42.0)
  static constexpr int kWarpRing = kStages * kStage;
  // where 16-byte piece `piece` of key `key` lies: the four rows of values that a quarter of a warp reads at once (even keys) are spread over the banks
  __device__ static __forceinline__ int place(int key, int piece) {
    if constexpr (kPieces == 2) return key * kRow + ((piece ^ ((key >> 2) & 1)) << 4);
    if constexpr ((kPieces & (kPieces - 1)) == 0) return key * kRow + ((piece ^ ((key >> 1) & 3)) << 4);
    return key * kRow + (piece << 4);
  }
};

template <int D>
static constexpr int kPitch = D + 4;  // fp32 numbers of a row in the workspace

template <int D, int BITS, int NT>
struct Shared {
  using L = Layout<D, BITS>;
  static constexpr int kRows = 8 * NT;
  static constexpr int kPart = kRows * D * 4;  // fp32 output of one warp; reuses the warp's ring
  static constexpr int kWarp = L::kWarpRing > kPart ? L::kWarpRing : kPart;
  static constexpr int kLess = kWarps * kWarp;                      // [NT][groups][4] float4: what the score sums of a group start at, for the columns 2t and 2t + 1, twice
  static constexpr int kStats = kLess + NT * L::kGroups * 4 * 16;   // [warps + 1][rows]: maximum and sum of a warp, and of the CTA
  static constexpr int kInbox = kStats + (kWarps + 1) * kRows * 8;  // what the CTAs of a cluster send one another: outputs, then maxima and sums
  static constexpr int kInboxStats = kInbox + kPart + kMaxCluster * 16;
  static constexpr int kFixed = kInboxStats + kMaxCluster * kRows * 8;
};

// A lane's quarter of a row.
template <typename L>
__device__ __forceinline__ void load_quarter(uint32_t base, int key, int quarter, uint32_t (&w)[L::kWords]) {
#pragma unroll
  for (int x = 0; x < L::kWords; x += L::kPerLoad) {
    const int off = quarter * L::kQuarter + x * 4;
    lds_words<L::kPerLoad>(base + L::place(key, off >> 4) + (off & 15), w + x);
  }
}
// The scales of a row, two to a word.
template <int G>
__device__ __forceinline__ void load_scales(uint32_t base, int key, uint32_t (&w)[(G + 1) / 2]) {
  const uint32_t a = base + key * G * 2;
  if constexpr (G % 2 == 0) {
    constexpr int kPer = G % 8 == 0 ? 4 : (G % 4 == 0 ? 2 : 1);
#pragma unroll
    for (int x = 0; x < G / 2; x += kPer) lds_words<kPer>(a + x * 4, w + x);
  } else {
#pragma unroll
    for (int x = 0; x < (G + 1) / 2; ++x) w[x] = 0u;
#pragma unroll
    for (int x = 0; x < G; ++x) {
      uint16_t v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a + x * 2) : "memory");
      w[x / 2] |= static_cast<uint32_t>(v) << (16 * (x & 1));
    }
  }
}
template <int N>
__device__ __forceinline__ float scale_of(const uint32_t (&w)[N], int j) { return j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]); }

// Bits of the keys first ... last among the 32 from j0 on.
__device__ __forceinline__ uint32_t keys_between(int j0, int first, int last) {
  const int a = max(first - j0, 0), b = min(last - j0, 31);
  return b >= a ? (0xffffffffu << a) & (0xffffffffu >> (31 - b)) : 0u;
}

// grid (splits, key heads, batch); the splits of a key head are a cluster, or (SPREAD) leave their results in the workspace for combine_kernel.
template <int D, int BITS, int NT, bool SPREAD>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 && D <= 128 ? 4 : 1)
attention_kernel(const __grid_constant__ Params p) {
  using L = Layout<D, BITS>;
  using S = Shared<D, BITS, NT>;
  constexpr int G = L::kGroups, kRows = S::kRows, kScaleWords = (G + 1) / 2;
  constexpr uint32_t kLow = BITS == 4 ? 0x000f000fu : 0x00ff00ffu, kHigh = 0x00f000f0u;
  constexpr float kHalf = BITS == 4 ? 8.f : 128.f;
  // -h of the codes that a lane's rows g and g + 8 of an operand hold (of 4 bits the latter are 16 times their code); out of sight of the compiler, which else makes them anew for each product
  uint32_t minus_h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) asm volatile("mov.b32 %0, %1;" : "=r"(minus_h[i]) : "r"(BITS == 4 && !(i & 1) ? 0x80088008u : 0x80808080u));
  extern __shared__ __align__(1024) uint8_t smem[];
  float4* less = reinterpret_cast<float4*>(smem + S::kLess);
  float2* stats = reinterpret_cast<float2*>(smem + S::kStats);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, splits = gridDim.x, hk = blockIdx.y, bi = blockIdx.z;
  const int rows = p.s * p.group;
  const int own = p.tiles > split ? (p.tiles - split + splits - 1) / splits : 0;
  const int words = p.s + 1;
  const bool joins = !SPREAD && splits > 1;
  if (joins) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // waited for before the first word goes to another CTA
  auto query_of = [&](int r) { return (r * p.per_query) >> 16; };
  uint32_t* list = reinterpret_cast<uint32_t*>(smem + S::kFixed);  // the own tiles that some query sees, and how many they are
  uint32_t* bits = list + own + 1;                                 // [own tiles][s + 1]: one word per query, and their union
  auto first_key = [&](int i) {  // of own tile i
    int tile = split + i * splits;
    if (tile >= p.skip_from) tile += p.skipped;
    return tile * kTileKeys;
  };

  // Query rows: column g of tile n is row 8n + g (query r / group, head r % group of the key head); this lane has its quarter t.  Their loads are under way while the tiles are looked through.
  uint4 raw[NT][G];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 8 + g;
    const int qi = query_of(r);
    const __nv_bfloat16* q = p.q + ((static_cast<long long>(bi) * p.s + qi) * p.hq + hk * p.group + (r - qi * p.group)) * D + t * (D / 4);
#pragma unroll
    for (int j = 0; j < G; ++j) raw[n][j] = r < rows ? *reinterpret_cast<const uint4*>(q + 8 * j) : make_uint4(0u, 0u, 0u, 0u);
  }

  // Which keys of the own tiles each query sees, one bit per key.
  const int start = p.key_start != nullptr ? p.key_start[bi] : 0;
  if (p.mask != nullptr) {  // a warp per tile, a lane per key
    for (int i = warp; i < own; i += kWarps) {
      const int j = first_key(i) + lane;
      uint32_t any = 0u, all = 0xffffffffu;
      for (int qi = 0; qi < p.s; ++qi) {
        const uint32_t word = __ballot_sync(0xffffffffu, j < p.sk && p.mask[bi * p.mask_b + qi * p.mask_r + j] != 0);
        any |= word, all &= word;
        if (lane == 0) bits[i * words + qi] = word;
      }
      if (lane == 0) bits[i * words + p.s] = any, list[i] = static_cast<uint32_t>(i) | (any != 0u ? kSeen : 0u) | (all == 0xffffffffu ? kWhole : 0u);
    }
  } else {  // a thread per tile
    for (int i = threadIdx.x; i < own; i += kWarps * 32) {
      const int j0 = first_key(i);
      uint32_t any = 0u, all = 0xffffffffu;
      for (int qi = 0; qi < p.s; ++qi) {
        const int last = p.offset >= 0 ? min(p.sk - 1, p.offset + qi) : p.sk - 1;
        uint32_t word = keys_between(j0, p.window > 0 ? max(start, p.offset + qi - p.window + 1) : start, last);
        if (p.window > 0) word |= keys_between(j0, start, min(last, p.sinks - 1));
        any |= word, all &= word;
        bits[i * words + qi] = word;
      }
      bits[i * words + p.s] = any, list[i] = static_cast<uint32_t>(i) | (any != 0u ? kSeen : 0u) | (all == 0xffffffffu ? kWhole : 0u);
    }
  }
  __syncthreads();
  if (warp == 0) {  // the tiles that are seen move to the front
    int kept = 0;
    for (int i0 = 0; i0 < own; i0 += 32) {
      const uint32_t entry = i0 + lane < own ? list[i0 + lane] : 0u;
      const uint32_t with = __ballot_sync(0xffffffffu, (entry & kSeen) != 0u);
      if (entry & kSeen) list[kept + __popc(with & ((1u << lane) - 1u))] = entry;
      kept += __popc(with);
      __syncwarp();
    }
    if (lane == 0) list[own] = static_cast<uint32_t>(kept);
  }
  __syncthreads();

  const uint32_t ring = smem_u32(smem) + warp * S::kWarp, less_lane = smem_u32(less) + t * 16;
  const uint8_t* kc = p.kc + bi * p.kc_b + hk * p.kc_h;
  const uint8_t* vc = p.vc + bi * p.vc_b + hk * p.vc_h;
  const uint8_t* ks = p.ks + bi * p.ks_b + hk * p.ks_h;
  const uint8_t* vs = p.vs + bi * p.vs_b + hk * p.vs_h;
  // A tile is one contiguous piece of each of the four arrays; lanes copy 16 bytes each, 512 apart.
  constexpr int kPieces = kTileKeys * L::kPieces, kScalePieces = L::kScales / 16;
  const uint8_t *k_lane = kc + lane * 16, *v_lane = vc + lane * 16;
  const uint8_t* s_lane = lane < kScalePieces ? ks + lane * 16 : vs - L::kScales + lane * 16;
  auto load = [&](uint32_t entry, uint32_t to) {
    const int j0 = first_key(static_cast<int>(entry & kIndex));
    if (j0 + kTileKeys <= p.sk) {
      const uint8_t *k = k_lane + static_cast<long long>(j0) * L::kRow, *v = v_lane + static_cast<long long>(j0) * L::kRow;
#pragma unroll
      for (int x = 0; x < kPieces; x += 32) {
        const uint32_t dst = to + L::place((x + lane) / L::kPieces, (x + lane) % L::kPieces);
        cp16(dst, k + x * 16, 16);
        cp16(dst + L::kCodes, v + x * 16, 16);
      }
      const long long scales_from = static_cast<long long>(j0) * G * 2;
      if constexpr (2 * kScalePieces <= 32) {
        if (lane < 2 * kScalePieces) cp16(to + 2 * L::kCodes + lane * 16, s_lane + scales_from, 16);
      } else {
#pragma unroll
        for (int piece = lane; piece < 2 * kScalePieces; piece += 32) cp16(to + 2 * L::kCodes + piece * 16, (piece < kScalePieces ? ks : vs - L::kScales) + scales_from + piece * 16, 16);
      }
    } else {  // what lies behind the last slot is not read
#pragma unroll 1
      for (int x = lane; x < kPieces; x += 32) {
        const int key = x / L::kPieces;
        const bool keep = j0 + key < p.sk;
        const long long off = keep ? static_cast<long long>(j0) * L::kRow + x * 16 : 0;
        const uint32_t dst = to + L::place(key, x % L::kPieces);
        cp16(dst, kc + off, keep ? 16 : 0);
        cp16(dst + L::kCodes, vc + off, keep ? 16 : 0);
      }
#pragma unroll 1
      for (int x = lane; x < 2 * kScalePieces; x += 32) {
        const int which = x >= kScalePieces ? 1 : 0, piece = x - which * kScalePieces;
        const int left = min(16, max(0, (p.sk - j0) * G * 2 - piece * 16));
        cp16(to + 2 * L::kCodes + x * 16, (which ? vs : ks) + (left > 0 ? static_cast<long long>(j0) * G * 2 + piece * 16 : 0), left);
      }
    }
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };

  const int kept = static_cast<int>(list[own]);
  uint32_t fill = ring, drain = ring;  // stages
  const uint32_t ring_end = ring + L::kWarpRing;
  auto step = [&](uint32_t& at) {
    at += L::kStage;
    if (at == ring_end) at = ring;
  };
#pragma unroll
  for (int st = 0; st < L::kStages - 1; ++st) {
    if (warp + st * kWarps < kept) load(list[warp + st * kWarps], fill);
    commit();
    step(fill);
  }

  // Queries as the B operand.  The scale is positive from here on: another sign (or 0) goes into the queries, which is exact, as is the power of two.
  const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
  uint32_t qf[NT][G][2][2];
  uint32_t largest = 0u;  // exponent of the largest finite query value
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < G; ++j) {
      uint4 u = raw[n][j];
      u.x ^= flip, u.y ^= flip, u.z ^= flip, u.w ^= flip;
      if (p.scale == 0.f) u = make_uint4(0u, 0u, 0u, 0u);
      for (uint32_t x : {u.x, u.y, u.z, u.w})
        for (uint32_t e : {(x >> 7) & 255u, (x >> 23) & 255u}) largest = max(largest, e == 255u ? 0u : e);
      // the channels that meet in a register of codes: e and e + 4 (4 bits), e and e + 2 (8 bits)
      if constexpr (BITS == 4) {
        qf[n][j][0][0] = __byte_perm(u.x, u.z, 0x5410), qf[n][j][0][1] = __byte_perm(u.x, u.z, 0x7632);
        qf[n][j][1][0] = __byte_perm(u.y, u.w, 0x5410), qf[n][j][1][1] = __byte_perm(u.y, u.w, 0x7632);
      } else {
        qf[n][j][0][0] = __byte_perm(u.x, u.y, 0x5410), qf[n][j][0][1] = __byte_perm(u.x, u.y, 0x7632);
        qf[n][j][1][0] = __byte_perm(u.z, u.w, 0x5410), qf[n][j][1][1] = __byte_perm(u.z, u.w, 0x7632);
      }
    }
  }
  const int lift_q = min(127, max(20, 110 - (static_cast<int>(__reduce_max_sync(0xffffffffu, largest)) - 127)));
  const float c = (p.scale == 0.f ? 1.f : fabsf(p.scale)) * kLog2e * power_of_two(64) * power_of_two(69 - lift_q);  // of scores in units of 2^(lift_q - 133)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < G; ++j) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t& x = qf[n][j][i >> 1][i & 1];
        const float lo = bf16_lo(x) * power_of_two(lift_q), hi = bf16_hi(x) * power_of_two(lift_q);
        sum += lo + hi;
        x = BITS == 4 && (i & 1) ? pack_bf16x2(lo * 0.0625f, hi * 0.0625f) : pack_bf16x2(lo, hi);  // the second register of codes holds upper nibbles
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= -kHalf * power_of_two(-67);
      const float even = __shfl_sync(0xffffffffu, sum, 8 * t) * power_of_two(-66), odd = __shfl_sync(0xffffffffu, sum, 8 * t + 4) * power_of_two(-66);
      if (warp == 0 && g == 0) less[(n * G + j) * 4 + t] = make_float4(even, odd, even, odd);
    }
    __syncthreads();  // less

  float acc[NT][G][2][4];  // [tile of columns][group][channels 2u, 2u + 1 of a lane's four]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][u][e] = 0.f;
  float m[NT][2], l[NT][2];  // m in log2 units; l and acc in units of 2^-lift and 2^(133 - lift)
#pragma unroll
  for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
  int lift = 90;
  const uint32_t half_sel = (g & 1) ? 0x7632u : 0x5410u;

  auto tile = [&](auto masked, uint32_t tk, int cur) {
    const uint32_t tv = tk + L::kCodes, tks = tv + L::kCodes, tvs = tks + L::kScales;
    float y[2][NT][4];  // scores of keys 16x + g and + 8, columns 2t and 2t + 1
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t w0[L::kWords], w1[L::kWords], s0[kScaleWords], s1[kScaleWords];
      load_quarter<L>(tk, x * 16 + g, t, w0);
      load_quarter<L>(tk, x * 16 + g + 8, t, w1);
      load_scales<G>(tks, x * 16 + g, s0);
      load_scales<G>(tks, x * 16 + g + 8, s1);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        uint32_t lo[4], hi[4];  // keys g and g + 8 by turns
        if constexpr (BITS == 4) {
          const uint32_t v0 = w0[j] >> 8, v1 = w1[j] >> 8;
          lo[0] = w0[j] & kLow, lo[1] = w1[j] & kLow, lo[2] = w0[j] & kHigh, lo[3] = w1[j] & kHigh;
          hi[0] = v0 & kLow, hi[1] = v1 & kLow, hi[2] = v0 & kHigh, hi[3] = v1 & kHigh;
        } else {
          lo[0] = w0[2 * j] & kLow, lo[1] = w1[2 * j] & kLow, lo[2] = (w0[2 * j] >> 8) & kLow, lo[3] = (w1[2 * j] >> 8) & kLow;
          hi[0] = w0[2 * j + 1] & kLow, hi[1] = w1[2 * j + 1] & kLow, hi[2] = (w0[2 * j + 1] >> 8) & kLow, hi[3] = (w1[2 * j + 1] >> 8) & kLow;
        }
        const float f0 = scale_of(s0, j), f1 = scale_of(s1, j);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float z[4];
          lds_words<4>(less_lane + (n * G + j) * 64, reinterpret_cast<uint32_t*>(z));
          mma16816(z, lo, qf[n][j][0][0], qf[n][j][0][1], z);
          mma16816(z, hi, qf[n][j][1][0], qf[n][j][1][1], z);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[x][n][e] = j == 0 ? (e < 2 ? f0 : f1) * z[e] : fmaf(e < 2 ? f0 : f1, z[e], y[x][n][e]);
        }
      }
    }
    uint32_t vsw[2][2][kScaleWords], some = 0u;  // scales of the values of the same keys
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        load_scales<G>(tvs, x * 16 + g + 8 * i, vsw[x][i]);
#pragma unroll
        for (int j = 0; j < kScaleWords; ++j) some |= vsw[x][i][j];
      }
    uint32_t seen[NT][2];
    if constexpr (masked.value) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = n * 8 + 2 * t + e;
          seen[n][e] = (r < rows ? bits[cur * words + query_of(r)] : 0xffffffffu) >> g;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (!((seen[n][e] >> (x * 16)) & 1u)) y[x][n][e] = -INFINITY;
            if (!((seen[n][e] >> (x * 16 + 8)) & 1u)) y[x][n][e + 2] = -INFINITY;
          }
        }
    }
    float top[NT][2];
    bool special = (some & 0x40004000u) != 0u;  // a scale of 2 or more: 2^lift may be too much
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[n][e] = fmaxf(max3(y[0][n][e], y[0][n][e + 2], y[1][n][e]), y[1][n][e + 2]) * c;
        special = special || top[n][e] > m[n][e] + kRescale;
      }
    if (__any_sync(0xffffffffu, special)) {
      uint32_t exponent = 0u;  // the largest of a finite scale
      const uint32_t keys = bits[cur * words + p.s] >> g;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < kScaleWords; ++j)
            for (uint32_t e : {(vsw[x][i][j] >> 7) & 255u, (vsw[x][i][j] >> 23) & 255u})
              if (e != 255u && ((keys >> (x * 16 + i * 8)) & 1u)) exponent = max(exponent, e);
      // probabilities up to 2^8 times a scale below 2^(exponent - 126) stay below 2^127
      const int lower = min(lift, 244 - static_cast<int>(__reduce_max_sync(0xffffffffu, exponent)));
      const float fall = power_of_two(lower - lift);
      lift = lower;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = top[n][e];
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = x > m[n][e] + kRescale ? x : m[n][e];
          f[e] = (x == -INFINITY ? 1.f : fast_exp2(m[n][e] - x)) * fall;
          m[n][e] = x;
          l[n][e] *= f[e];
        }
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][j][u][e] *= f[e & 1];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float base[2] = {(m[n][0] == -INFINITY ? 0.f : -m[n][0]) + lift, (m[n][1] == -INFINITY ? 0.f : -m[n][1]) + lift};
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[x][n][e] = fast_exp2(fmaf(y[x][n][e], c, base[e & 1]));
          l[n][e & 1] += y[x][n][e];
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t w[4][L::kWords];  // rows of values 2t, 2t + 1, 2t + 8, 2t + 9 of the sixteen
#pragma unroll
      for (int i = 0; i < 4; ++i) load_quarter<L>(tv, x * 16 + 2 * t + (i & 1) + (i >> 1) * 8, g >> 1, w[i]);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        uint32_t lo[4], hi[4];  // channels 0 and 1, 2 and 3 of this lane's four of the group, pairs of keys
        if constexpr (BITS == 4) {
          const uint32_t x01 = __byte_perm(w[0][j], w[1][j], half_sel), x23 = __byte_perm(w[2][j], w[3][j], half_sel);
          const uint32_t y01 = x01 >> 8, y23 = x23 >> 8;
          lo[0] = x01 & kLow, lo[1] = x01 & kHigh, lo[2] = x23 & kLow, lo[3] = x23 & kHigh;
          hi[0] = y01 & kLow, hi[1] = y01 & kHigh, hi[2] = y23 & kLow, hi[3] = y23 & kHigh;
        } else {
          uint32_t h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = (g & 1) ? w[i][2 * j + 1] : w[i][2 * j];
          const uint32_t x01 = __byte_perm(h[0], h[1], 0x5410), x23 = __byte_perm(h[2], h[3], 0x5410);
          const uint32_t y01 = __byte_perm(h[0], h[1], 0x7632), y23 = __byte_perm(h[2], h[3], 0x7632);
          lo[0] = x01 & kLow, lo[1] = (x01 >> 8) & kLow, lo[2] = x23 & kLow, lo[3] = (x23 >> 8) & kLow;
          hi[0] = y01 & kLow, hi[1] = (y01 >> 8) & kLow, hi[2] = y23 & kLow, hi[3] = (y23 >> 8) & kLow;
        }
        const float f0 = scale_of(vsw[x][0], j), f1 = scale_of(vsw[x][1], j);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w0 = y[x][n][0] * f0, w1 = y[x][n][1] * f0, w2 = y[x][n][2] * f1, w3 = y[x][n][3] * f1;
          if constexpr (masked.value) {  // the scales of a slot that is not visible may be anything
            const uint32_t b0 = seen[n][0] >> (x * 16), b1 = seen[n][1] >> (x * 16);
            w0 = b0 & 1u ? w0 : 0.f, w1 = b1 & 1u ? w1 : 0.f;
            w2 = b0 & 256u ? w2 : 0.f, w3 = b1 & 256u ? w3 : 0.f;
          }
          const uint32_t p0 = transpose8x8(pack_bf16x2(w0, w1)), p1 = transpose8x8(pack_bf16x2(w2, w3));
          mma16816(acc[n][j][0], lo, p0, p1, acc[n][j][0]);
          mma16816(acc[n][j][1], hi, p0, p1, acc[n][j][1]);
          mma16816(acc[n][j][0], minus_h, p0, p1, acc[n][j][0]);
          mma16816(acc[n][j][1], minus_h, p0, p1, acc[n][j][1]);
        }
      }
    }
  };

#pragma unroll 1
  for (int i = warp; i < kept; i += kWarps) {
    if (i + (L::kStages - 1) * kWarps < kept) load(list[i + (L::kStages - 1) * kWarps], fill);
    commit();
    step(fill);
    asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 1) : "memory");
    __syncwarp();
    const uint32_t entry = list[i];
    if (entry & kWhole)
      tile(std::false_type{}, drain, static_cast<int>(entry & kIndex));
    else
      tile(std::true_type{}, drain, static_cast<int>(entry & kIndex));
    step(drain);
    __syncwarp();  // the next iteration refills this stage: no lane may still read it
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();

  // The warps meet in shared memory (each in its own ring), then the CTAs of the cluster.
  float* part = reinterpret_cast<float*>(smem + warp * S::kWarp);
  const float even = power_of_two(69 - lift), odd = BITS == 4 ? even * 0.0625f : even;  // times 2^64
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = n * 8 + 2 * t + e;
      float sum = l[n][e] * power_of_two(-lift);
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (g == 0) stats[warp * kRows + r] = make_float2(m[n][e], sum);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const int d = (g >> 1) * (D / 4) + 8 * j + 4 * (g & 1);
        constexpr float kUp = 18446744073709551616.f;  // 2^64
        *reinterpret_cast<float4*>(part + r * D + d) = make_float4(acc[n][j][0][e] * kUp * even, acc[n][j][0][e + 2] * kUp * odd, acc[n][j][1][e] * kUp * even, acc[n][j][1][e + 2] * kUp * odd);
      }
    }
  }
  __syncthreads();
  float2* total = stats + kWarps * kRows;  // maximum and sum of the CTA; the warps' maxima become their weights
  if (threadIdx.x < rows) {
    const int r = threadIdx.x;
    float high = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) high = fmaxf(high, stats[w * kRows + r].x);
    const float base = high == -INFINITY ? 0.f : high;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = fast_exp2(stats[w * kRows + r].x - base);
      sum += f * stats[w * kRows + r].y;
      stats[w * kRows + r].x = f;
    }
    total[r] = make_float2(high, sum);
  }
  __syncthreads();
  // A query that sees nothing gives 0; a NaN stays one.
  auto put = [&](int r, int d, const float4& x, float sum) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int qi = query_of(r);
    *reinterpret_cast<uint2*>(p.o + ((static_cast<long long>(bi) * p.s + qi) * p.hq + hk * p.group + (r - qi * p.group)) * D + d) =
        make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
  };
  cg::cluster_group cluster = cg::this_cluster();
  if (joins) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    float2* inbox = reinterpret_cast<float2*>(smem + S::kInboxStats);  // [split][row]
    for (int i = threadIdx.x; i < rows * splits; i += kWarps * 32) {
      const int to = i / rows, r = i - to * rows;
      cluster.map_shared_rank(inbox, to)[split * rows + r] = total[r];
    }
  }
  float4* inbox = reinterpret_cast<float4*>(smem + S::kInbox);  // [element of this CTA's share][split]
  const int pieces = rows * (D / 4);
  for (int i = threadIdx.x; i < pieces; i += kWarps * 32) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = stats[w * kRows + r].x;
      const float4 v = *reinterpret_cast<const float4*>(smem + w * S::kWarp + (r * D + d) * 4);
      x.x = fmaf(f, v.x, x.x), x.y = fmaf(f, v.y, x.y), x.z = fmaf(f, v.z, x.z), x.w = fmaf(f, v.w, x.w);
    }
    if (SPREAD) {
      float* to = p.work + ((static_cast<long long>(bi) * p.hkv + hk) * splits + split) * rows * kPitch<D> + r * kPitch<D>;  // D sums, the maximum and the sum of the row
      *reinterpret_cast<float4*>(to + d) = x;
      if (d == 0) *reinterpret_cast<float2*>(to + D) = total[r];
    } else if (!joins) {
      put(r, d, x, total[r].y);
    } else {
      const int share = i / splits;
      cluster.map_shared_rank(inbox, i - share * splits)[share * splits + split] = x;
    }
  }
  if (!joins) return;
  cluster.sync();  // everything has arrived; from here on a CTA reads its own memory only
  const float2* heads = reinterpret_cast<const float2*>(smem + S::kInboxStats);
  for (int i = threadIdx.x * splits + split; i < pieces; i += kWarps * 32 * splits) {
    const int r = i / (D / 4), d = (i % (D / 4)) * 4;
    const float4* from = inbox + (i - split);
    float high = -INFINITY, sum = 0.f;
    for (int x = 0; x < splits; ++x) high = fmaxf(high, heads[x * rows + r].x);
    const float base = high == -INFINITY ? 0.f : high;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = 0; x < splits; ++x) {
      const float f = fast_exp2(heads[x * rows + r].x - base);
      const float4 v = from[x];
      sum = fmaf(f, heads[x * rows + r].y, sum);
      o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
    }
    put(r, d, o, sum);
  }
}

// Joins the results of the splits, in their order: grid (query rows of a key head, key heads, batch).
static constexpr int kCombine = 256;
template <int D>
__global__ void __launch_bounds__(kCombine)
combine_kernel(const __grid_constant__ Params p, int splits) {
  constexpr int kLanes = D / 4, kSlices = kCombine / kLanes;
  __shared__ float weight[kMaxSpread], high[kCombine / 32], sums[kCombine / 32];
  __shared__ float4 part[kSlices][kLanes];
  const int r = blockIdx.x, rows = gridDim.x, hk = blockIdx.y, bi = blockIdx.z;
  const long long pitch = static_cast<long long>(rows) * kPitch<D>;
  const float* from = p.work + ((static_cast<long long>(bi) * p.hkv + hk) * splits * rows + r) * kPitch<D>;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  static_assert(kMaxSpread <= kCombine, "a thread per split");
  const float2 own = static_cast<int>(threadIdx.x) < splits ? *reinterpret_cast<const float2*>(from + threadIdx.x * pitch + D) : make_float2(-INFINITY, 0.f);
  float top = own.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) high[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kCombine / 32; ++w) top = fmaxf(top, high[w]);
  const float f = fast_exp2(own.x - (top == -INFINITY ? 0.f : top));
  if (threadIdx.x < kMaxSpread) weight[threadIdx.x] = f;
  float sum = f * own.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  const int slice = threadIdx.x / kLanes, d = threadIdx.x % kLanes;
  if (slice < kSlices) {
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int x = slice; x < splits; x += kSlices) {
      const float4 v = *reinterpret_cast<const float4*>(from + x * pitch + d * 4);
      const float w = weight[x];
      o.x = fmaf(w, v.x, o.x), o.y = fmaf(w, v.y, o.y), o.z = fmaf(w, v.z, o.z), o.w = fmaf(w, v.w, o.w);
    }
    part[slice][d] = o;
  }
  __syncthreads();
  if (slice != 0) return;
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kCombine / 32; ++w) sum += sums[w];
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int x = 0; x < kSlices; ++x) o.x += part[x][d].x, o.y += part[x][d].y, o.z += part[x][d].z, o.w += part[x][d].w;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int qi = (r * p.per_query) >> 16;
  *reinterpret_cast<uint2*>(p.o + ((static_cast<long long>(bi) * p.s + qi) * p.hq + hk * p.group + (r - qi * p.group)) * D + d * 4) =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
}

static long long bit_bytes(int tiles, int s, int splits) { return (static_cast<long long>((tiles + splits - 1) / splits) * (s + 2) + 1) * 4; }

// Splits of a key head's tiles, by a model of the time in units of what an SM needs for one round of tiles of a CTA's warps when it is full (0.57 us at 4 bits and 128 channels): an SM works off
// its share of the CTAs in waves of those that it holds, a wave costs 8 units of latency in front of and behind its tiles and at least 1.4 per round, and a join in the workspace another 8.
// Measured (without a graph) and modelled us (4 bits, 128 channels): 64 x 4096 slots, 1 split 74 / 73, 2 74 / 73, 8 96 / 96; 16 x 732, 1 11 / 9, 8 17 / 18; 1 x 65 003, 8 54 / 56, 32 in the workspace 30 / 30.
// Of equal ones it takes the larger if its CTAs have fewer rounds, since two stages of a tile hide less latency than a wave of more CTAs (32 x 4096 of 64 channels, 1 and 2 splits: 33 and 31 us in 4
// bits, 41 and 37 in 8).
static int splits_of(long long pairs, int tiles, int s, int per_sm, bool spread) {
  int best = 0;
  long long least = 0, least_waves = 0, least_rounds = 0;
  for (int n = 1; n <= (spread ? kMaxSpread : kMaxCluster); n += n < kMaxCluster ? n : 1) {  // clusters of 3, 5 or 7 are placed worse
    if (bit_bytes(tiles, s, n) > kMaxBitBytes) continue;
    const long long ctas = (pairs * n + sm_count() - 1) / sm_count(), waves = (ctas + per_sm - 1) / per_sm, rounds = (tiles + n * kWarps - 1) / (n * kWarps);
    const long long cost = max(10 * ctas * rounds, 14 * waves * rounds) + 80 * waves + (n > kMaxCluster ? 80 : 0);
    if (best == 0 || cost < least || (cost == least && waves == least_waves && rounds < least_rounds)) best = n, least = cost, least_waves = waves, least_rounds = rounds;
  }
  return best;
}

template <int D, int BITS, int NT>
static int launch(const Params& p, int b, long long work_floats, cudaStream_t st) {
  using S = Shared<D, BITS, NT>;
  const int tiles = p.tiles;
  const void* kerns[2] = {reinterpret_cast<const void*>(attention_kernel<D, BITS, NT, false>), reinterpret_cast<const void*>(attention_kernel<D, BITS, NT, true>)};
  static int resident[kMaxDevices] = {};  // CTAs that an SM holds
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices) return kErrDriver;
  if (resident[device] == 0) {
    for (const void* k : kerns)
      if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kFixed + kMaxBitBytes) != cudaSuccess) return kErrDriver;
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kerns[0], kWarps * 32, S::kFixed + 1024) != cudaSuccess || per_sm <= 0) return kErrDriver;
    resident[device] = per_sm;
  }
  const int rows = p.s * (p.hq / p.hkv);
  const long long pairs = static_cast<long long>(b) * p.hkv;
  const int splits = splits_of(pairs, tiles, p.s, resident[device], work_floats >= kMaxSpread * pairs * rows * kPitch<D>);
  if (splits == 0) return kErrTooLarge;
  const int spread = splits > kMaxCluster ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, p.hkv, b);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = S::kFixed + static_cast<int>(bit_bytes(tiles, p.s, splits));
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = spread ? 0 : 1;
  void* args[1] = {const_cast<Params*>(&p)};
  TTB_COUNT_LAUNCH(1);
  if (cudaLaunchKernelExC(&cfg, kerns[spread], args) != cudaSuccess) return kErrDriver;
  if (spread) {
    TTB_COUNT_LAUNCH(1);
    cudaLaunchConfig_t next = {};
    next.gridDim = dim3(rows, p.hkv, b);
    next.blockDim = dim3(kCombine);
    next.stream = st;
    cudaLaunchAttribute early[1];
    early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // its CTAs are there when the last of the other kernel's have written
    early[0].val.programmaticStreamSerializationAllowed = 1;
    next.attrs = early, next.numAttrs = 1;
    if (cudaLaunchKernelEx(&next, combine_kernel<D>, p, splits) != cudaSuccess) return kErrDriver;
  }
  return cudaGetLastError() == cudaSuccess ? kOk : kErrDriver;
}

template <int D, int BITS>
static int by_rows(const Params& p, int b, long long work_floats, cudaStream_t st) {
  if (p.s * (p.hq / p.hkv) <= 8) return launch<D, BITS, 1>(p, b, work_floats, st);
  if constexpr (D <= 128) return launch<D, BITS, 2>(p, b, work_floats, st);
  return kErrTooLarge;
}

}  // namespace qattn
}  // namespace ttb

// A call's arguments, 8 bytes each: handed over as one piece, which takes the caller less time than as many arguments.
struct QuantizedAttentionCall {
  const void *q, *k_codes, *k_scales, *v_codes, *v_scales;
  long long strides[8];
  void* o;
  const void* mask;
  long long mask_b, mask_r;
  const int* key_start;
  long long offset, window, sinks, b, s, sk, hq, hkv, d, bits;
  void* work;
  long long work_floats;
};

// Attention of s queries over the first sk slots of a quantised cache: q, o [b, s, hq, d] contiguous, s * (hq / hkv) <= 16 (d 256: 8) query rows per key head, d 64, 96, 128 or 256, bits 4 or 8.
// Rows as ttb_quantized_append writes them, those of one head one behind the other; strides[0..1]: batch and head of k's codes (bytes), [2..3] of its scales (elements), [4..7] of v's; all starts on
// 16 bytes.  mask (nullable): nonzero byte = visible, row (b, i) at mask + b * mask_b + i * mask_r.  key_start (nullable) int32 [b]: first visible slot.  offset >= 0: query i sits in slot
// offset + i and sees no later one, with window > 0 only the last `window` of them and the first `sinks`.  A query that sees nothing gives 0.
// work (nullable): work_floats fp32 numbers, used where few and long rows are split further than a cluster reaches, if they are at least 128 * b * hq * s * (d + 4).
extern "C" int ttb_quantized_attention(const QuantizedAttentionCall* call, float scale, void* stream) {
  using namespace ttb;
  const QuantizedAttentionCall& x = *call;
  const long long most = 0x7fffffff - 64;
  if (x.b <= 0 || x.b > 65535 || x.s <= 0 || x.s > 16 || x.sk <= 0 || x.sk > most || x.hkv <= 0 || x.hkv > 65535 || x.hq <= 0 || x.hq % x.hkv || x.hq / x.hkv > 16 ||
      x.s * (x.hq / x.hkv) > (x.d == 256 ? 8 : 16) || x.d > 256)
    return kErrBadShape;
  if (x.offset > most || x.window < 0 || x.window > most || x.sinks < 0 || x.sinks > most || (x.window > 0 && x.offset < 0)) return kErrBadShape;
  qattn::Params p{};
  p.q = static_cast<const __nv_bfloat16*>(x.q), p.o = static_cast<__nv_bfloat16*>(x.o);
  p.kc = static_cast<const uint8_t*>(x.k_codes), p.vc = static_cast<const uint8_t*>(x.v_codes);
  p.ks = static_cast<const uint8_t*>(x.k_scales), p.vs = static_cast<const uint8_t*>(x.v_scales);
  p.kc_b = x.strides[0], p.kc_h = x.strides[1], p.ks_b = x.strides[2] * 2, p.ks_h = x.strides[3] * 2;
  p.vc_b = x.strides[4], p.vc_h = x.strides[5], p.vs_b = x.strides[6] * 2, p.vs_h = x.strides[7] * 2;
  for (const void* t : {x.q, x.k_codes, x.k_scales, x.v_codes, x.v_scales, static_cast<const void*>(x.o), static_cast<const void*>(x.work)})
    if (reinterpret_cast<uintptr_t>(t) & 15) return kErrBadShape;
  if ((p.kc_b | p.kc_h | p.ks_b | p.ks_h | p.vc_b | p.vc_h | p.vs_b | p.vs_h) & 15) return kErrBadShape;
  const int b = static_cast<int>(x.b), s = static_cast<int>(x.s), sk = static_cast<int>(x.sk), hq = static_cast<int>(x.hq), hkv = static_cast<int>(x.hkv);
  const int offset = x.offset < 0 ? -1 : static_cast<int>(x.offset), window = static_cast<int>(x.window), sinks = static_cast<int>(x.sinks);
  const long long work_floats = x.work != nullptr ? x.work_floats : 0;
  p.mask = static_cast<const uint8_t*>(x.mask), p.mask_b = x.mask_b, p.mask_r = x.mask_r, p.key_start = x.key_start;
  p.offset = offset, p.window = window, p.sinks = sinks;
  p.s = s, p.sk = sk, p.hq = hq, p.hkv = hkv, p.scale = scale, p.work = static_cast<float*>(x.work);
  p.group = hq / hkv, p.per_query = 65536 / p.group + 1;
  p.skip_from = 0x7fffffff;
  if (window > 0) {  // the first query's window begins first
    const int from = (sinks + qattn::kTileKeys - 1) / qattn::kTileKeys, to = max(0, offset - window + 1) / qattn::kTileKeys;
    const int tiles = (sk + qattn::kTileKeys - 1) / qattn::kTileKeys;
    if (min(to, tiles) > from) p.skip_from = from, p.skipped = min(to, tiles) - from;
  }
  p.tiles = (sk + qattn::kTileKeys - 1) / qattn::kTileKeys - p.skipped;
  auto st = static_cast<cudaStream_t>(stream);
  switch (x.d * 16 + x.bits) {
    case 64 * 16 + 4: return qattn::by_rows<64, 4>(p, b, work_floats, st);
    case 64 * 16 + 8: return qattn::by_rows<64, 8>(p, b, work_floats, st);
    case 96 * 16 + 4: return qattn::by_rows<96, 4>(p, b, work_floats, st);
    case 96 * 16 + 8: return qattn::by_rows<96, 8>(p, b, work_floats, st);
    case 128 * 16 + 4: return qattn::by_rows<128, 4>(p, b, work_floats, st);
    case 128 * 16 + 8: return qattn::by_rows<128, 8>(p, b, work_floats, st);
    case 256 * 16 + 4: return qattn::by_rows<256, 4>(p, b, work_floats, st);
    case 256 * 16 + 8: return qattn::by_rows<256, 8>(p, b, work_floats, st);
  }
  return kErrBadShape;
}
