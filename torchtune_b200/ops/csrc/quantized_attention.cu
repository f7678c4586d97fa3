// Attention of a few queries over a key/value cache held in 4 or 8 bits (rows as quantized_cache.cu writes them).
//
//   score[r, k] = c sum_j ks[k, j] sum_{d in j} q[r, d] (kc[k, d] - h)          j: groups of 32 channels, h = 2^(bits - 1)
//   out[r, d]   = sum_k (p[r, k] vs[k, j(d)]) (vc[k, d] - h) / sum_k p[r, k]    p: exponentials of the scores
//
// Codes are small integers and as such exact bf16 numbers, so they are the matrix operands as they are: scales are applied in fp32, to the scores of a group and to the probabilities in front
// of a group's product, and nothing is rounded but the probabilities times their scale (to bf16, as in the other attention kernels; their sum is fp32) and the result.
//
// Decoding is bound by the bytes of the cache as long as turning codes into operands keeps up: at 6.5 TB/s an SM takes in 41 4-bit codes per cycle and issues 128 lane instructions.  So keys
// (and channels) are the 16 rows of an m16n8k16 tile and a key head's query rows its 8 columns: no code is turned twice, and few rows do not pay for 16.  A lane holds a quarter of a row of keys
// (with eight channels of every group) and, for the second product, half a word of every group of four rows of values, whose nibbles meet in one register as the pairs of keys that the operand
// wants: about one instruction per code and operand.  4-bit codes become bf16 by or-ing them into 128.0 (128 + code); of keys the 128 + h is taken off by starting the sum at
// -(128 + h) sum q, of values by one packed subtraction, since there the sum runs over the whole cache and would lose its low bits.
//
// A warp takes tiles of 32 keys through a cp.async ring of its own, with its own running maximum (moved only when a score exceeds it by 2^8), sum and output.  Tiles are dealt round-robin to
// the warps of a CTA and the CTAs of a cluster, which meet once at the end in distributed shared memory in a fixed order: no workspace and no second launch.  Tiles without a visible key are not read.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common/ptx.cuh"
#include "common/tmap.h"

namespace ttb {
namespace qattn {

namespace cg = cooperative_groups;

static constexpr int kWarps = 4;
static constexpr int kTileKeys = 32;
static constexpr int kMaxSplit = 16;         // non-portable cluster size
static constexpr int kMaxBitBytes = 16384;   // visibility words of one CTA
static constexpr float kLog2e = 1.4426950408889634f;
static constexpr float kRescale = 8.f;       // log2 units
static constexpr int kMaxDevices = 64;

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
  int s, sk, hq, hkv;
  int skip_from, skipped;  // tiles skip_from ... skip_from + skipped - 1 lie between the first tokens and every window
  float scale;
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
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
__device__ __forceinline__ float byte_minus_128(uint32_t word, uint32_t which) {  // 2^23 + byte as an fp32 number, less 2^23 + 128
  return __uint_as_float(__byte_perm(word, 0x4b000000u, 0x7540u | which)) - 8388736.f;
}
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
  static constexpr int kStages = 3;
  static constexpr int kWarpRing = kStages * kStage;
  // where 16-byte piece `piece` of key `key` lies: the four rows of values that a quarter of a warp reads at once (even keys) are spread over the banks
  __device__ static __forceinline__ int place(int key, int piece) {
    if constexpr (kPieces == 2) return key * kRow + ((piece ^ ((key >> 2) & 1)) << 4);
    if constexpr ((kPieces & (kPieces - 1)) == 0) return key * kRow + ((piece ^ ((key >> 1) & (kPieces - 1))) << 4);
    return key * kRow + (piece << 4);
  }
};

template <int D, int BITS, int NT>
struct Shared {
  using L = Layout<D, BITS>;
  static constexpr int kRows = 8 * NT;
  static constexpr int kPart = kRows * D * 4;  // fp32 output of one warp; reuses the warp's ring
  static constexpr int kWarp = L::kWarpRing > kPart ? L::kWarpRing : kPart;
  static constexpr int kStats = (kWarps + 1) * kRows * 2 * 4;
  static constexpr int kFixed = kWarps * kWarp + kStats;
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
template <int G>
__device__ __forceinline__ void load_scales(uint32_t base, int key, float (&s)[G]) {
  const uint32_t a = base + key * G * 2;
  if constexpr (G % 2 == 0) {
    constexpr int kPer = G % 8 == 0 ? 4 : (G % 4 == 0 ? 2 : 1);
    uint32_t w[G / 2];
#pragma unroll
    for (int x = 0; x < G / 2; x += kPer) lds_words<kPer>(a + x * 4, w + x);
#pragma unroll
    for (int x = 0; x < G / 2; ++x) s[2 * x] = bf16_lo(w[x]), s[2 * x + 1] = bf16_hi(w[x]);
  } else {
#pragma unroll
    for (int x = 0; x < G; ++x) {
      uint16_t v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a + x * 2) : "memory");
      s[x] = __uint_as_float(static_cast<uint32_t>(v) << 16);
    }
  }
}

// grid (splits = cluster, key heads, batch)
template <int D, int BITS, int NT>
__global__ void __launch_bounds__(kWarps * 32)
attention_kernel(const __grid_constant__ Params p) {
  using L = Layout<D, BITS>;
  using S = Shared<D, BITS, NT>;
  constexpr int G = L::kGroups, kRows = S::kRows;
  constexpr uint32_t kMagic = 0x43004300u, kNibbles = 0x000f000fu;  // 128.0 twice
  extern __shared__ __align__(1024) uint8_t smem[];
  float* stats = reinterpret_cast<float*>(smem + kWarps * S::kWarp);
  uint32_t* bits = reinterpret_cast<uint32_t*>(smem + S::kFixed);  // [own tiles][s + 1]: one word per query, then their union
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, splits = gridDim.x, hk = blockIdx.y, bi = blockIdx.z;
  const int group = p.hq / p.hkv, rows = p.s * group;
  const int tiles = (p.sk + kTileKeys - 1) / kTileKeys - p.skipped;
  const int own = tiles > split ? (tiles - split + splits - 1) / splits : 0;
  const int words = p.s + 1;
  auto first_key = [&](int i) {  // of own tile i
    int tile = split + i * splits;
    if (tile >= p.skip_from) tile += p.skipped;
    return tile * kTileKeys;
  };

  // Which keys of the own tiles each query sees, one bit per key.
  const int start = p.key_start != nullptr ? p.key_start[bi] : 0;
  for (int w = warp; w < own * p.s; w += kWarps) {
    const int i = w / p.s, qi = w % p.s;
    const int j = first_key(i) + lane;
    bool seen = j < p.sk && j >= start;
    if (p.offset >= 0) {
      const int at = p.offset + qi;
      seen = seen && j <= at && (p.window == 0 || at - j < p.window || j < p.sinks);
    }
    if (seen && p.mask != nullptr) seen = p.mask[bi * p.mask_b + qi * p.mask_r + j] != 0;
    const uint32_t word = __ballot_sync(0xffffffffu, seen);
    if (lane == 0) bits[i * words + qi] = word;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < own; i += kWarps * 32) {
    uint32_t any = 0;
    for (int qi = 0; qi < p.s; ++qi) any |= bits[i * words + qi];
    bits[i * words + p.s] = any;
  }

  // Queries as the B operand: column g of tile n is query row 8n + g (query r / group, head r % group of this key head); this lane has its quarter t.
  uint32_t qf[NT][G][2][2];
  float less[NT][G][2];  // -(128 + h) times the sum of a group's query values, for the columns 2t and 2t + 1 of the result
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 8 + g;
    const __nv_bfloat16* q = p.q + ((static_cast<long long>(bi) * p.s + r / group) * p.hq + hk * group + r % group) * D + t * (D / 4);
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const uint4 u = r < rows ? *reinterpret_cast<const uint4*>(q + 8 * j) : make_uint4(0u, 0u, 0u, 0u);
      // channels e and e + 4 are a pair, as the nibbles of a word leave them
      qf[n][j][0][0] = __byte_perm(u.x, u.z, 0x5410), qf[n][j][0][1] = __byte_perm(u.x, u.z, 0x7632);
      qf[n][j][1][0] = __byte_perm(u.y, u.w, 0x5410), qf[n][j][1][1] = __byte_perm(u.y, u.w, 0x7632);
      if constexpr (BITS == 4) {
        float sum = 0.f;
        for (uint32_t x : {u.x, u.y, u.z, u.w}) sum += bf16_lo(x) + bf16_hi(x);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        less[n][j][0] = -136.f * __shfl_sync(0xffffffffu, sum, 8 * t);
        less[n][j][1] = -136.f * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      }
    }
  }
  __syncthreads();

  const uint32_t ring = smem_u32(smem) + warp * S::kWarp;
  const uint8_t* kc = p.kc + bi * p.kc_b + hk * p.kc_h;
  const uint8_t* vc = p.vc + bi * p.vc_b + hk * p.vc_h;
  const uint8_t* ks = p.ks + bi * p.ks_b + hk * p.ks_h;
  const uint8_t* vs = p.vs + bi * p.vs_b + hk * p.vs_h;
  auto next = [&](int i) {  // next tile of this warp with a visible key
    while (i < own && bits[i * words + p.s] == 0) i += kWarps;
    return i;
  };
  auto load = [&](int i, int stage) {
    if (i < own) {
      const int j0 = first_key(i);
      const uint32_t to = ring + stage * L::kStage;
#pragma unroll
      for (int c = lane; c < kTileKeys * L::kPieces; c += 32) {
        const int key = c / L::kPieces, piece = c % L::kPieces;
        const bool keep = j0 + key < p.sk;  // what lies behind the last slot is not read
        const long long off = keep ? static_cast<long long>(j0 + key) * L::kRow + piece * 16 : 0;
        const uint32_t dst = to + L::place(key, piece);
        cp16(dst, kc + off, keep ? 16 : 0);
        cp16(dst + L::kCodes, vc + off, keep ? 16 : 0);
      }
      constexpr int kScalePieces = L::kScales / 16;
#pragma unroll
      for (int c = lane; c < 2 * kScalePieces; c += 32) {
        const int which = c >= kScalePieces ? 1 : 0, piece = c - which * kScalePieces;
        const long long off = static_cast<long long>(j0) * G * 2 + piece * 16;
        const int left = static_cast<int>(min(16ll, max(0ll, static_cast<long long>(p.sk) * G * 2 - off)));
        cp16(to + 2 * L::kCodes + which * L::kScales + piece * 16, (which ? vs : ks) + (left > 0 ? off : 0), left);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  float acc[NT][G][2][4];  // [tile of columns][group][channels 2u, 2u + 1 of a lane's four]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][u][e] = 0.f;
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
  const float c = p.scale * kLog2e;
  const uint32_t half_sel = (g & 1) ? 0x7632u : 0x5410u;

  int cur = next(warp), ahead = cur;
#pragma unroll
  for (int st = 0; st < L::kStages - 1; ++st) {
    load(ahead, st);
    if (ahead < own) ahead = next(ahead + kWarps);
  }
  for (int it = 0; cur < own; ++it) {
    load(ahead, (it + L::kStages - 1) % L::kStages);
    if (ahead < own) ahead = next(ahead + kWarps);
    asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 1) : "memory");
    __syncwarp();
    const uint32_t tk = ring + (it % L::kStages) * L::kStage, tv = tk + L::kCodes, tks = tv + L::kCodes, tvs = tks + L::kScales;

    float y[2][NT][4];  // scores of keys 16x + g and + 8, columns 2t and 2t + 1
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint32_t w0[L::kWords], w1[L::kWords];
      load_quarter<L>(tk, x * 16 + g, t, w0);
      load_quarter<L>(tk, x * 16 + g + 8, t, w1);
      float s0[G], s1[G];
      load_scales<G>(tks, x * 16 + g, s0);
      load_scales<G>(tks, x * 16 + g + 8, s1);
#pragma unroll
      for (int n = 0; n < NT; ++n) y[x][n][0] = y[x][n][1] = y[x][n][2] = y[x][n][3] = 0.f;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        uint32_t a0[4], a1[4];  // pairs of channels (e, e + 4) of the two keys
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BITS == 4) {
            a0[e] = ((w0[j] >> (4 * e)) & kNibbles) | kMagic;
            a1[e] = ((w1[j] >> (4 * e)) & kNibbles) | kMagic;
          } else {
            a0[e] = pack_bf16x2(byte_minus_128(w0[2 * j], e), byte_minus_128(w0[2 * j + 1], e));
            a1[e] = pack_bf16x2(byte_minus_128(w1[2 * j], e), byte_minus_128(w1[2 * j + 1], e));
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float z[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (BITS == 4) z[0] = z[2] = less[n][j][0], z[1] = z[3] = less[n][j][1];
          const uint32_t lo[4] = {a0[0], a1[0], a0[1], a1[1]}, hi[4] = {a0[2], a1[2], a0[3], a1[3]};
          mma16816(z, lo, qf[n][j][0][0], qf[n][j][0][1]);
          mma16816(z, hi, qf[n][j][1][0], qf[n][j][1][1]);
          y[x][n][0] += s0[j] * z[0], y[x][n][1] += s0[j] * z[1];
          y[x][n][2] += s1[j] * z[2], y[x][n][3] += s1[j] * z[3];
        }
      }
    }
    // Visibility; the words of the two columns differ only between queries.
    uint32_t seen[NT][2];
    bool whole = true;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = n * 8 + 2 * t + e;
        seen[n][e] = r < rows ? bits[cur * words + r / group] : 0xffffffffu;
        whole = whole && seen[n][e] == 0xffffffffu;
      }
    }
    whole = __all_sync(0xffffffffu, whole);
    bool higher = false;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[x][n][e] *= c;
          if (!whole && !((seen[n][e & 1] >> (x * 16 + g + (e >> 1) * 8)) & 1u)) y[x][n][e] = -INFINITY;
          higher = higher || y[x][n][e] > m[n][e & 1] + kRescale;
        }
    if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(fmaxf(y[0][n][e], y[0][n][e + 2]), fmaxf(y[1][n][e], y[1][n][e + 2]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          top = fmaxf(top, m[n][e]);
          f[e] = top == -INFINITY ? 1.f : fast_exp2(m[n][e] - top);
          m[n][e] = top;
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
      const float base[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[x][n][e] = fast_exp2(y[x][n][e] - base[e & 1]);
          l[n][e & 1] += y[x][n][e];
        }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float s0[G], s1[G];
      load_scales<G>(tvs, x * 16 + g, s0);
      load_scales<G>(tvs, x * 16 + g + 8, s1);
      uint32_t w[4][L::kWords];  // rows of values 2t, 2t + 1, 2t + 8, 2t + 9 of the sixteen
#pragma unroll
      for (int i = 0; i < 4; ++i) load_quarter<L>(tv, x * 16 + 2 * t + (i & 1) + (i >> 1) * 8, g >> 1, w[i]);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        uint32_t v01[4], v23[4];  // this lane's channels 0 - 3 of the group, pairs of keys
        if constexpr (BITS == 4) {
          const uint32_t x01 = __byte_perm(w[0][j], w[1][j], half_sel), x23 = __byte_perm(w[2][j], w[3][j], half_sel);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v01[e] = sub_bf16x2(((x01 >> (4 * e)) & kNibbles) | kMagic, 0x43084308u);  // 136.0 twice
            v23[e] = sub_bf16x2(((x23 >> (4 * e)) & kNibbles) | kMagic, 0x43084308u);
          }
        } else {
          uint32_t h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = (g & 1) ? w[i][2 * j + 1] : w[i][2 * j];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v01[e] = pack_bf16x2(byte_minus_128(h[0], e), byte_minus_128(h[1], e));
            v23[e] = pack_bf16x2(byte_minus_128(h[2], e), byte_minus_128(h[3], e));
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w0 = y[x][n][0] * s0[j], w1 = y[x][n][1] * s0[j], w2 = y[x][n][2] * s1[j], w3 = y[x][n][3] * s1[j];
          if (!whole) {  // the scales of a slot that is not visible may be anything
            const uint32_t b0 = seen[n][0] >> (x * 16 + g), b1 = seen[n][1] >> (x * 16 + g);
            w0 = b0 & 1u ? w0 : 0.f, w1 = b1 & 1u ? w1 : 0.f;
            w2 = b0 & 256u ? w2 : 0.f, w3 = b1 & 256u ? w3 : 0.f;
          }
          const uint32_t p0 = transpose8x8(pack_bf16x2(w0, w1)), p1 = transpose8x8(pack_bf16x2(w2, w3));
          const uint32_t lo[4] = {v01[0], v01[1], v23[0], v23[1]}, hi[4] = {v01[2], v01[3], v23[2], v23[3]};
          mma16816(acc[n][j][0], lo, p0, p1);
          mma16816(acc[n][j][1], hi, p0, p1);
        }
      }
    }
    __syncwarp();  // the stage is refilled two iterations on
    cur = next(cur + kWarps);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();

  // The warps meet in shared memory (each in its own ring), then the CTAs of the cluster.
  float* part = reinterpret_cast<float*>(smem + warp * S::kWarp);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = n * 8 + 2 * t + e;
      float sum = l[n][e];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      if (g == 0) stats[(warp * kRows + r) * 2] = m[n][e], stats[(warp * kRows + r) * 2 + 1] = sum;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const int d = (g >> 1) * (D / 4) + 8 * j + 4 * (g & 1);
        *reinterpret_cast<float4*>(part + r * D + d) = make_float4(acc[n][j][0][e], acc[n][j][0][e + 2], acc[n][j][1][e], acc[n][j][1][e + 2]);
      }
    }
  }
  __syncthreads();
  float* total = stats + kWarps * kRows * 2;  // maximum and sum of the CTA
  auto out = [&](int r, int d) { return p.o + ((static_cast<long long>(bi) * p.s + r / group) * p.hq + hk * group + r % group) * D + d; };
  for (int idx = threadIdx.x; idx < rows * D; idx += kWarps * 32) {
    const int r = idx / D, d = idx % D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[(w * kRows + r) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = fast_exp2(stats[(w * kRows + r) * 2] - base);
      sum += f * stats[(w * kRows + r) * 2 + 1];
      x += f * reinterpret_cast<const float*>(smem + w * S::kWarp)[r * D + d];
    }
    if (splits == 1) {
      *out(r, d) = __float2bfloat16_rn(sum == 0.f ? 0.f : x / sum);  // a query that sees nothing gives 0; a NaN stays one
    } else {
      reinterpret_cast<float*>(smem)[r * D + d] = x;  // the slot of warp 0, read by this thread alone
      if (d == 0) total[r * 2] = top, total[r * 2 + 1] = sum;
    }
  }
  if (splits == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int idx = split * kWarps * 32 + threadIdx.x; idx < rows * D; idx += splits * kWarps * 32) {
    const int r = idx / D, d = idx % D;
    float top = -INFINITY;
    for (int x = 0; x < splits; ++x) top = fmaxf(top, cluster.map_shared_rank(total, x)[r * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o = 0.f;
    for (int x = 0; x < splits; ++x) {
      const float* st = cluster.map_shared_rank(total, x);
      const float f = fast_exp2(st[r * 2] - base);
      sum += f * st[r * 2 + 1];
      o += f * cluster.map_shared_rank(reinterpret_cast<float*>(smem), x)[r * D + d];
    }
    *out(r, d) = __float2bfloat16_rn(sum == 0.f ? 0.f : o / sum);
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

template <int D, int BITS, int NT>
static int launch(const Params& p, int b, cudaStream_t st) {
  using S = Shared<D, BITS, NT>;
  const int tiles = (p.sk + kTileKeys - 1) / kTileKeys - p.skipped;
  auto bit_bytes = [&](int splits) { return static_cast<long long>((tiles + splits - 1) / splits) * (p.s + 1) * 4; };
  int splits = 1;  // four CTAs per SM as long as every warp has a tile of its own, and as many as the visibility words need
  while (splits < kMaxSplit && ((static_cast<long long>(b) * p.hkv * splits < 4ll * sm_count() && tiles >= 2 * kWarps * splits) || bit_bytes(splits) > kMaxBitBytes)) splits *= 2;
  if (bit_bytes(splits) > kMaxBitBytes) return kErrTooLarge;
  const int smem = S::kFixed + static_cast<int>(bit_bytes(splits));
  auto kern = attention_kernel<D, BITS, NT>;
  static bool ready[kMaxDevices] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= kMaxDevices) return kErrDriver;
  if (!ready[device]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kFixed + kMaxBitBytes) != cudaSuccess) return kErrDriver;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return kErrDriver;
    ready[device] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, p.hkv, b);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at, cfg.numAttrs = 1;
  TTB_COUNT_LAUNCH(1);
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? kOk : kErrDriver;
}

template <int D, int BITS>
static int by_rows(const Params& p, int b, cudaStream_t st) {
  if (p.s * (p.hq / p.hkv) <= 8) return launch<D, BITS, 1>(p, b, st);
  if constexpr (D <= 128) return launch<D, BITS, 2>(p, b, st);
  return kErrTooLarge;
}

}  // namespace qattn
}  // namespace ttb

// Attention of s queries over the first sk slots of a quantised cache: q, o [b, s, hq, d] contiguous, s * (hq / hkv) <= 16 (d 256: 8) query rows per key head, d 64, 96, 128 or 256, bits 4 or 8.
// Rows as ttb_quantized_append writes them, those of one head one behind the other; strides[0..1]: batch and head of k's codes (bytes), [2..3] of its scales (elements), [4..7] of v's; all starts on
// 16 bytes.  mask (nullable): nonzero byte = visible, row (b, i) at mask + b * mask_b + i * mask_r.  key_start (nullable) int32 [b]: first visible slot.  offset >= 0: query i sits in slot
// offset + i and sees no later one, with window > 0 only the last `window` of them and the first `sinks`.  A query that sees nothing gives 0.
extern "C" int ttb_quantized_attention(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, const long long* strides, void* o, const void* mask,
                                       long long mask_b, long long mask_r, const int* key_start, int offset, int window, int sinks, int b, int s, int sk, int hq, int hkv, int d, int bits,
                                       float scale, void* stream) {
  using namespace ttb;
  if (b <= 0 || b > 65535 || s <= 0 || sk <= 0 || hkv <= 0 || hkv > 65535 || hq <= 0 || hq % hkv || s > 16 || hq / hkv > 16 || s * (hq / hkv) > (d == 256 ? 8 : 16)) return kErrBadShape;
  if (sk > 0x7fffffff - 64 || offset > 0x7fffffff - 64 || window < 0 || sinks < 0 || (window > 0 && offset < 0)) return kErrBadShape;
  qattn::Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q), p.o = static_cast<__nv_bfloat16*>(o);
  p.kc = static_cast<const uint8_t*>(k_codes), p.vc = static_cast<const uint8_t*>(v_codes);
  p.ks = static_cast<const uint8_t*>(k_scales), p.vs = static_cast<const uint8_t*>(v_scales);
  p.kc_b = strides[0], p.kc_h = strides[1], p.ks_b = strides[2] * 2, p.ks_h = strides[3] * 2;
  p.vc_b = strides[4], p.vc_h = strides[5], p.vs_b = strides[6] * 2, p.vs_h = strides[7] * 2;
  for (const void* x : {q, k_codes, k_scales, v_codes, v_scales, static_cast<const void*>(o)})
    if (reinterpret_cast<uintptr_t>(x) & 15) return kErrBadShape;
  if ((p.kc_b | p.kc_h | p.ks_b | p.ks_h | p.vc_b | p.vc_h | p.vs_b | p.vs_h) & 15) return kErrBadShape;
  p.mask = static_cast<const uint8_t*>(mask), p.mask_b = mask_b, p.mask_r = mask_r, p.key_start = key_start;
  p.offset = offset, p.window = window, p.sinks = sinks;
  p.s = s, p.sk = sk, p.hq = hq, p.hkv = hkv, p.scale = scale;
  p.skip_from = 0x7fffffff;
  if (window > 0) {  // the first query's window begins first
    const int from = (sinks + qattn::kTileKeys - 1) / qattn::kTileKeys, to = max(0, offset - window + 1) / qattn::kTileKeys;
    const int tiles = (sk + qattn::kTileKeys - 1) / qattn::kTileKeys;
    if (min(to, tiles) > from) p.skip_from = from, p.skipped = min(to, tiles) - from;
  }
  auto st = static_cast<cudaStream_t>(stream);
  switch (d * 16 + bits) {
    case 64 * 16 + 4: return qattn::by_rows<64, 4>(p, b, st);
    case 64 * 16 + 8: return qattn::by_rows<64, 8>(p, b, st);
    case 96 * 16 + 4: return qattn::by_rows<96, 4>(p, b, st);
    case 96 * 16 + 8: return qattn::by_rows<96, 8>(p, b, st);
    case 128 * 16 + 4: return qattn::by_rows<128, 4>(p, b, st);
    case 128 * 16 + 8: return qattn::by_rows<128, 8>(p, b, st);
    case 256 * 16 + 4: return qattn::by_rows<256, 4>(p, b, st);
    case 256 * 16 + 8: return qattn::by_rows<256, 8>(p, b, st);
  }
  return kErrBadShape;
}
