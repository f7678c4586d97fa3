// Attention of rows that share a long prefix: a prompt's keys and values are read once for all rows (answers) of the prompt, a row's own keys once for the row.
//
//   o = sum_k e^(c q.k) v / sum_k e^(c q.k),   k over keys [start, stop) of the row's prompt and over the row's own keys up to the query's position.
//
// A softmax over pieces: each piece leaves m = max, l = sum 2^(x - m) and O = sum 2^(x - m) v, and o = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i.  A piece is a run of keys of one key head with up
// to 128 query rows: those of all rows of a prompt (answers x tokens x query heads that share the key head) on a run of the prefix, or those of one row on a run of its own keys.  Both are the
// same work: scores of 128 rows and 64 keys on tcgen05 tensor cores, a thread per row for the softmax, probabilities in the scores' place in tensor memory as the A operand of the second
// product, its accumulator next to them.  A tile of 64 keys and values is 32 KB: an SM's share of the memory's rate brings it in 1400 cycles, and 128 rows keep the tensor cores busy for 260 of them and the
// exponentials' unit for 512, so that padding a single token's four rows to 128 costs nothing that is not idle; warps without rows have no part in the softmax.
// Two CTAs to an SM take pieces in turn, a fixed share each.  A ring of slots that K and V fill in turn runs on over the end of a piece, so that the keys of the next one arrive while the output of the
// last is written; the scores of a tile are computed while the softmax of the one before is.  Pieces are as long as a model of their number and overhead says (plan_of), and lie in a
// workspace that a second launch joins in a fixed order.
//
// What lies behind the last visible key may be anything: scores are masked by selection, and the values of a piece's last tile that nobody sees are overwritten with zeros before they are
// multiplied.  Every wait is bounded and reports through the error word.
#include "common/attn_math.cuh"
#include "common/ptx.cuh"
#include "common/tmap.h"

namespace ttb {
namespace sprefix {

using namespace attn;

static constexpr int kThreads = 192;  // four warps of softmax, one that loads, one that multiplies
static constexpr int kRows = 128;     // query rows of a piece
static constexpr int kKeys = 64;      // keys of a tile
static constexpr int kPanel = kKeys * 128;  // 64 columns of a tile of keys

struct Params {
  const __nv_bfloat16* q;   // [rows, s, hq, D]
  __nv_bfloat16* o;
  const int *start, *stop;  // [prompts] or nullptr: 0, prefix
  const int* lengths;       // [rows] or nullptr: own
  float* part;              // pieces' outputs: rows of D floats
  float2* ml;               // their maxima (log2) and sums
  int prompts, rows, s, hq, hkv, group;
  int prefix, own;          // slots
  int rows_p, rows_o;       // query rows of a prompt and of a row, per key head
  int tiles_p, tiles_o;     // of 128 of them
  int run_p, run_o;         // keys of a piece
  int cuts_p, cuts_o;       // pieces of a key head's keys
  int pieces_p, pieces;     // of all prompts; with those of rows, which follow
  float scale;
  int* err;
};

template <int D>
struct Layout {
  static constexpr int kPanels = D / 64;
  static constexpr int kQuery = kPanels * kPanelBytes;  // queries; between two pieces the output on its way out
  static constexpr int kSlot = kPanels * kPanel;
  static constexpr int kSlots = D == 128 ? 4 : 8;
  static constexpr int kBars = kQuery + kSlots * kSlot;
  static constexpr int kBytes = kBars + (2 * kSlots + 6) * 8 + 16 + 1024;
  static constexpr int kColumns = 256;  // of tensor memory: outputs, then two tiles of scores
  static_assert(4 * 32 * 32 * 4 <= kQuery, "four warps' 32 x 32 outputs take the queries' place");
};

// The keys of a piece: [first, last) of the prompt's or row's slots.
__device__ __forceinline__ void range_of(const Params& p, bool prefix, int owner, int cut, int& first, int& last) {
  int lo = 0, hi;
  if (prefix) {
    lo = p.start != nullptr ? p.start[owner] : 0;
    hi = p.stop != nullptr ? p.stop[owner] : p.prefix;
    lo = max(lo, 0), hi = min(hi, p.prefix);
  } else {
    hi = p.lengths != nullptr ? p.lengths[owner] : p.own;
    hi = min(hi, p.own);
  }
  const int run = prefix ? p.run_p : p.run_o;
  first = max(lo, cut * run);
  last = min(static_cast<long long>(hi), (cut + 1ll) * run);
}

// Which piece: tiles of query rows are neighbours, so that the second of them finds the keys in L2.
struct Piece {
  bool prefix;
  int tile, head, cut, owner, first, last;
  __device__ __forceinline__ Piece(const Params& p, int at) {
    prefix = at < p.pieces_p;
    at -= prefix ? 0 : p.pieces_p;
    const int tiles = prefix ? p.tiles_p : p.tiles_o, cuts = prefix ? p.cuts_p : p.cuts_o;
    tile = at % tiles, at /= tiles;
    head = at % p.hkv, at /= p.hkv;
    cut = at % cuts, owner = at / cuts;
    range_of(p, prefix, owner, cut, first, last);
  }
  __device__ __forceinline__ int key_tiles() const { return first < last ? (last - first + kKeys - 1) / kKeys : 0; }  // 0: nothing to see; whoever joins the pieces knows that too
};

// A barrier of the four warps of the softmax; whether any of them says yes.
__device__ __forceinline__ bool any_of_four(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(mine))
      : "memory");
  return any != 0;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2)
piece_kernel(const __grid_constant__ CUtensorMap tm_kp, const __grid_constant__ CUtensorMap tm_vp, const __grid_constant__ CUtensorMap tm_ko, const __grid_constant__ CUtensorMap tm_vo,
             const __grid_constant__ Params p) {
  using L = Layout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* ring = smem + L::kQuery;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* empty = full + L::kSlots;
  uint64_t* q_full = empty + L::kSlots;
  uint64_t* s_full = q_full + 1;   // [2] scores of a tile are there
  uint64_t* p_full = q_full + 3;   // [2] its probabilities are
  uint64_t* pv_done = q_full + 5;  // its second product is
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 6);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;");  // the joining launch may take its place; it waits for the end of this one
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kSlots; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    mbar_init(q_full, 4);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4);
    mbar_init(pv_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, L::kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tO = *tmem_slot, tS = tO + D;

  if (warp == 4) {
    // ---------------------------------------------------------------- loads: K and V of a tile in turn
    if (lane == 0) prefetch_tmap(&tm_kp), prefetch_tmap(&tm_vp), prefetch_tmap(&tm_ko), prefetch_tmap(&tm_vo);
    int slot = 0, n = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int at = blockIdx.x; at < p.pieces && ok; at += gridDim.x) {
      const Piece c(p, at);
      const CUtensorMap *map_k = c.prefix ? &tm_kp : &tm_ko, *map_v = c.prefix ? &tm_vp : &tm_vo;
      for (int x = 0; x < 2 * c.key_tiles() && !*abort_flag; ++x, ++n) {
        if (!(ok = mbar_wait(&empty[slot], phase ^ 1))) {
          fail(abort_flag, p.err, 301);
          break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[slot], L::kSlot);
          for (int y = 0; y < L::kPanels; ++y) tma_load_4d(ring + slot * L::kSlot + y * kPanel, x & 1 ? map_v : map_k, &full[slot], y * 64, c.head, c.first + (x >> 1) * kKeys, c.owner);
        }
        __syncwarp();
        if (++slot == L::kSlots) slot = 0, phase ^= 1;
      }
    }
    if (*abort_flag)  // no copy is in flight when the shared memory goes
      for (int x = max(0, n - L::kSlots); x < n; ++x) mbar_wait(&full[x % L::kSlots], (x / L::kSlots) & 1);
  } else if (warp == 5) {
    // ---------------------------------------------------------------- products
    constexpr uint32_t idesc_s = make_idesc_bf16(kRows, kKeys, false, false);
    constexpr uint32_t idesc_o = make_idesc_bf16(kRows, D, false, true);
    const uint32_t aQ = smem_u32(sQ), aR = smem_u32(ring);
    bool ok = true;
    uint32_t pieces = 0, done = 0;  // pieces and tiles so far
    auto issue_s = [&](uint32_t t) {  // scores of tile t of all
      const uint32_t slot = 2 * t % L::kSlots;
      if (!mbar_wait(&full[slot], (2 * t / L::kSlots) & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t k_base = aR + slot * L::kSlot, to = tS + (t & 1) * kKeys;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16(to, desc_kmajor(aQ, k), make_smem_desc_sw128(k_base + (k >> 2) * kPanel + (k & 3) * 32, 16, 1024), idesc_s, k != 0);
        umma_commit(&s_full[t & 1]);
        umma_commit(&empty[slot]);
      }
      __syncwarp();
      return true;
    };
    for (int at = blockIdx.x; at < p.pieces && ok && !*abort_flag; at += gridDim.x) {
      const int n = Piece(p, at).key_tiles();
      if (n == 0) continue;
      ok = mbar_wait(q_full, pieces++ & 1) && issue_s(done);
      for (int j = 0; j < n && ok && !*abort_flag; ++j, ++done) {
        if (j + 1 < n && !(ok = issue_s(done + 1))) break;  // while the softmax of this tile runs
        const uint32_t slot = (2 * done + 1) % L::kSlots;
        ok = mbar_wait(&p_full[done & 1], (done >> 1) & 1) && mbar_wait(&full[slot], ((2 * done + 1) / L::kSlots) & 1);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t v_base = aR + slot * L::kSlot, from = tS + (done & 1) * kKeys;
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) umma_f16_ts(tO, from + k * 8, make_smem_desc_sw128(v_base + k * 2048, kPanel, 1024), idesc_o, (j | k) != 0);
          umma_commit(&empty[slot]);
          umma_commit(pv_done);
        }
        __syncwarp();
      }
    }
    if (!ok) fail(abort_flag, p.err, 302);
  } else {
    // ---------------------------------------------------------------- queries, softmax, output
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const float c = p.scale * kLog2e;
    const bool turned = !(c > 0.f);
    const float cc = turned ? 1.f : c;
    const uint64_t c2 = pack_f32x2(cc, cc);
    bool ok = true, stop = false;
    uint32_t done = 0;  // tiles so far
    for (int at = blockIdx.x; at < p.pieces && !stop; at += gridDim.x) {
      const Piece piece(p, at);
      const int n_tiles = piece.key_tiles(), first = piece.first, last = piece.last;
      if (n_tiles == 0) continue;
      const int rows = piece.prefix ? p.rows_p : p.rows_o, row0 = piece.tile * kRows, live = min(kRows, rows - row0), live_warps = (live + 31) / 32;
      const long long token0 = static_cast<long long>(piece.owner) * (piece.prefix ? p.rows / p.prompts * p.s : p.s);
      for (int x = threadIdx.x; x < live * (D / 8); x += 128) {
        const int r = x / (D / 8), ch = x % (D / 8), row = row0 + r, token = row / p.group;
        const uint4 v = *reinterpret_cast<const uint4*>(p.q + ((token0 + token) * p.hq + piece.head * p.group + row - token * p.group) * D + ch * 8);
        *reinterpret_cast<uint4*>(sQ + (ch >> 3) * kPanelBytes + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      const int r = warp * 32 + lane;
      int mine = r < live ? last : first;  // keys of this row end here
      if (!piece.prefix && r < live) {
        const int length = min(p.lengths != nullptr ? p.lengths[piece.owner] : p.own, p.own);
        mine = min(last, length - p.s + (row0 + r) / p.group + 1);
      }
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < n_tiles && !*abort_flag; ++j, ++done) {
        const int k0 = first + j * kKeys, seen = mine - k0;
        if (!(ok = mbar_wait(&s_full[done & 1], (done >> 1) & 1))) break;
        if (warp < live_warps) {
          const uint32_t tile = tS + (done & 1) * kKeys + lanes;
          tc_fence_after();
          uint32_t sv[2][32];
          tmem_ld_32x32(tile, sv[0]);
          tmem_ld_32x32(tile + 32, sv[1]);
          tmem_ld_wait();
          if (turned) {  // the maximum is taken of raw scores, which a negative scale would turn around, and 0 times a masked one is NaN
#pragma unroll
            for (int i = 0; i < 64; ++i) sv[i >> 5][i & 31] = __float_as_uint(__uint_as_float(sv[i >> 5][i & 31]) * c);
          }
          if (seen < kKeys) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (i >= seen) sv[i >> 5][i & 31] = 0xff800000u;  // -inf
          }
          float mx2[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            mx2[0] = max3(mx2[0], __uint_as_float(sv[i >> 5][i & 31]), __uint_as_float(sv[i >> 5][(i & 31) + 1]));
            mx2[1] = max3(mx2[1], __uint_as_float(sv[i >> 5][(i & 31) + 2]), __uint_as_float(sv[i >> 5][(i & 31) + 3]));
          }
          const float m_new = fmaxf(m_used, fmaxf(mx2[0], mx2[1]) * cc);
          float alpha = 1.f;
          bool rescale = false;
          if ((m_new > m_used + kRescaleThreshold || m_used == -INFINITY) && m_new != -INFINITY) {
            rescale = m_used != -INFINITY;
            alpha = rescale ? fast_exp2(m_used - m_new) : 0.f;
            m_used = m_new;
          }
          const float neg_m = m_used == -INFINITY ? 0.f : -m_used;
          const uint64_t nm2 = pack_f32x2(neg_m, neg_m);
          uint64_t sum2[2] = {0ull, 0ull};
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const uint64_t t = fma_f32x2(pack_u32x2(sv[i >> 5][i & 31], sv[i >> 5][(i & 31) + 1]), c2, nm2);
            float t0, t1;
            unpack_f32x2(t, t0, t1);
            const float e0 = fast_exp2(t0), e1 = fast_exp2(t1);
            sum2[(i >> 1) & 1] = add_f32x2(sum2[(i >> 1) & 1], pack_f32x2(e0, e1));
            pk[i >> 1] = pack_bf16x2(e0, e1);  // the second product's operand; the sum keeps 32 bits
          }
          float s0, s1, s2, s3;
          unpack_f32x2(sum2[0], s0, s1);
          unpack_f32x2(sum2[1], s2, s3);
          l = l * alpha + (s0 + s1) + (s2 + s3);
          tmem_st_32x32(tile, pk);
          if (j > 0 && __any_sync(0xffffffffu, rescale)) {
            if (!(ok = mbar_wait(pv_done, (done - 1) & 1))) break;  // the second product before this one has left the output
            tc_fence_after();
#pragma unroll 1
            for (int ch = 0; ch < D / 32; ++ch) {
              uint32_t v[32];
              tmem_ld_32x32(tO + lanes + ch * 32, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
              tmem_st_32x32(tO + lanes + ch * 32, v);
            }
          }
          tmem_st_wait();
          if (last - k0 < kKeys) {  // the last tile: values that nobody sees may be anything, and 0 * NaN is NaN
            const uint32_t slot = (2 * done + 1) % L::kSlots;
            if (!(ok = mbar_wait(&full[slot], ((2 * done + 1) / L::kSlots) & 1))) break;
            uint8_t* v = ring + slot * L::kSlot;
            const int dead = kKeys - (last - k0);
            for (int x = threadIdx.x; x < dead * L::kPanels * 8; x += live_warps * 32) {
              const int key = kKeys - dead + x / (L::kPanels * 8), y = x % (L::kPanels * 8);
              *reinterpret_cast<uint4*>(v + (y >> 3) * kPanel + key * 128 + (y & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[done & 1]);
      }
      if (ok && !*abort_flag) ok = mbar_wait(pv_done, (done - 1) & 1);
      if (ok && !*abort_flag && warp < live_warps) {
        tc_fence_after();
        // the output, unnormalised, by way of shared memory, where the queries are no longer needed, so that a row's values are written side by side
        const long long base = piece.prefix ? ((static_cast<long long>(piece.owner) * p.cuts_p + piece.cut) * p.hkv + piece.head) * p.rows_p + row0
                                            : static_cast<long long>(p.prompts) * p.cuts_p * p.hkv * p.rows_p +
                                                  ((static_cast<long long>(piece.owner) * p.cuts_o + piece.cut) * p.hkv + piece.head) * p.rows_o + row0;
        float* stage = reinterpret_cast<float*>(sQ) + warp * 1024;
        const int count = min(32, live - warp * 32);
#pragma unroll 1
        for (int ch = 0; ch < D / 32; ++ch) {
          uint32_t v[32];
          tmem_ld_32x32(tO + lanes + ch * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) stage[lane * 32 + (i ^ lane)] = __uint_as_float(v[i]);
          __syncwarp();
          float* to = p.part + (base + warp * 32) * D + ch * 32 + lane;
#pragma unroll 4
          for (int i = 0; i < count; ++i) to[static_cast<long long>(i) * D] = stage[i * 32 + (lane ^ i)];
          __syncwarp();
        }
        if (r < live) p.ml[base + r] = make_float2(m_used, l);
        tc_fence_before();
      }
      if (!ok) fail(abort_flag, p.err, 303);
      stop = any_of_four(!ok || *abort_flag);  // all outputs are out of the queries' place; the four warps go on together or not at all
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tO, L::kColumns);
}

// A warp per token and query head joins its pieces, those of the prefix and then its own: a lane per piece finds where it lies, its maximum and sum, and the weights go around, so that all loads but
// the first two are independent.  32 pieces at a time.
static constexpr int kJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ Params p) {
  const uint32_t w = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const uint32_t token = w / p.hq;
  if (token >= static_cast<uint32_t>(p.rows) * p.s) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the pieces are written
  const int h = static_cast<int>(w - token * p.hq), head = h / p.group, a = h - head * p.group;
  const int row = static_cast<int>(token / p.s), i = static_cast<int>(token - static_cast<uint32_t>(row) * p.s);
  const int per = p.rows / p.prompts, prompt = row / per;
  constexpr int kMine = D / 32;
  float m = -INFINITY, l = 0.f, o[kMine];
#pragma unroll
  for (int x = 0; x < kMine; ++x) o[x] = 0.f;
  const int pieces = p.cuts_p + p.cuts_o;
  for (int first_piece = 0; first_piece < pieces; first_piece += 32) {
    const int piece = first_piece + lane;
    long long at = 0;
    float2 t = make_float2(-INFINITY, 0.f);
    if (piece < pieces) {
      const bool prefix = piece < p.cuts_p;
      const int cut = prefix ? piece : piece - p.cuts_p, owner = prefix ? prompt : row;
      int first, last;
      range_of(p, prefix, owner, cut, first, last);
      if (first < last) {  // otherwise nobody has written it
        at = prefix ? ((static_cast<long long>(prompt) * p.cuts_p + cut) * p.hkv + head) * p.rows_p + ((row - prompt * per) * p.s + i) * p.group + a
                    : static_cast<long long>(p.prompts) * p.cuts_p * p.hkv * p.rows_p + ((static_cast<long long>(row) * p.cuts_o + cut) * p.hkv + head) * p.rows_o + i * p.group + a;
        t = p.ml[at];
      }
    }
    float top = fmaxf(m, t.x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float base = top == -INFINITY ? 0.f : top, f = exp2f(m - base), weight = exp2f(t.x - base);
    float sum = t.y * weight;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * f + sum;
    m = top;
#pragma unroll
    for (int y = 0; y < kMine; ++y) o[y] *= f;
    const int n = min(32, pieces - first_piece);
    for (int x0 = 0; x0 < n; x0 += 4) {
      float v[4][kMine], g[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        g[x] = __shfl_sync(0xffffffffu, weight, x0 + x);  // 0 where no key is seen
        const float* from = p.part + __shfl_sync(0xffffffffu, at, x0 + x) * D + lane * kMine;
        if (g[x] != 0.f) {
          if constexpr (kMine == 4) *reinterpret_cast<float4*>(v[x]) = *reinterpret_cast<const float4*>(from);
          else *reinterpret_cast<float2*>(v[x]) = *reinterpret_cast<const float2*>(from);
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (g[x] != 0.f) {
#pragma unroll
          for (int y = 0; y < kMine; ++y) o[y] += v[x][y] * g[x];
        }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a query without a key gives 0
  uint32_t out[kMine / 2];
#pragma unroll
  for (int y = 0; y < kMine / 2; ++y) out[y] = pack_bf16x2(o[2 * y] * inv, o[2 * y + 1] * inv);
  __nv_bfloat16* to = p.o + (static_cast<long long>(token) * p.hq + h) * D + lane * kMine;
  if constexpr (kMine == 4) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
  else *reinterpret_cast<uint32_t*>(to) = out[0];
}

// What a call brings, packed by the host language in this order.
struct Call {
  long long q, o, kp, vp, k, v, start, stop, lengths, work, work_floats;
  long long kp_step[3], vp_step[3], k_step[3], v_step[3];  // batch, slot, head; elements
  long long prompts, rows, s, hq, hkv, d, prefix, own;
};

// How long pieces are.  CTAs (two to an SM) take pieces in turn, those of the prefix first: the one with the most of both is done last.  A piece costs its tiles and an overhead that grows with its
// rows, whose queries and outputs move between the pieces: in tiles, 0.3 and one for each 64 rows.
static double overhead_of(int rows) { return 0.3 + (rows < kRows ? rows : kRows) / 64.0; }
static int plan_of(const Call& c, Params& p) {
  if (c.prompts <= 0 || c.rows <= 0 || c.rows % c.prompts || c.s <= 0 || c.hkv <= 0 || c.hq <= 0 || c.hq % c.hkv || (c.d != 64 && c.d != 128) || c.prefix < 0 || c.own < 0) return kErrBadShape;
  if (c.rows > 0x7fffffff || c.prefix > 0x3fffffff || c.own > 0x3fffffff || c.rows * c.s > 0x7fffffff / c.hq) return kErrTooLarge;
  p.prompts = static_cast<int>(c.prompts), p.rows = static_cast<int>(c.rows), p.s = static_cast<int>(c.s), p.hq = static_cast<int>(c.hq), p.hkv = static_cast<int>(c.hkv);
  p.group = p.hq / p.hkv, p.prefix = static_cast<int>(c.prefix), p.own = static_cast<int>(c.own);
  p.rows_p = static_cast<int>(c.rows / c.prompts * c.s * p.group), p.rows_o = static_cast<int>(c.s * p.group);
  p.tiles_p = (p.rows_p + kRows - 1) / kRows, p.tiles_o = (p.rows_o + kRows - 1) / kRows;
  const long long np = (c.prefix + kKeys - 1) / kKeys, no = (c.own + kKeys - 1) / kKeys;  // tiles of keys
  const long long heads_p = c.prompts * c.hkv * p.tiles_p, heads_o = c.rows * c.hkv * p.tiles_o, ctas = 2ll * sm_count();
  const double over_p = overhead_of(p.rows_p), over_o = overhead_of(p.rows_o);
  double best = 0;
  long long run = 1;
  for (long long t = 2; t <= 4096; t += t < 32 ? 1 : t / 8) {
    const long long cuts_p = (np + t - 1) / t, cuts_o = (no + t - 1) / t;
    const double each_p = cuts_p ? (np + cuts_p - 1) / cuts_p + over_p : 0, each_o = cuts_o ? (no + cuts_o - 1) / cuts_o + over_o : 0;
    const long long pieces_p = heads_p * cuts_p, pieces = pieces_p + heads_o * cuts_o;
    auto of = [&](long long cta) {  // what a CTA has to do
      const long long first = pieces_p > cta ? (pieces_p - cta + ctas - 1) / ctas : 0, all = pieces > cta ? (pieces - cta + ctas - 1) / ctas : 0;
      return first * each_p + (all - first) * each_o;
    };
    double time = of(0);
    for (long long cta : {pieces_p % ctas, (pieces_p + ctas - 1) % ctas, (pieces + ctas - 1) % ctas}) time = of(cta) > time ? of(cta) : time;
    if (best == 0 || time < best) best = time, run = t;
    if (t > np && t > no) break;
  }
  auto cut = [&](long long n, int& cuts, int& keys) {
    cuts = static_cast<int>((n + run - 1) / run);
    keys = cuts == 0 ? kKeys : static_cast<int>((n + cuts - 1) / cuts) * kKeys;
  };
  cut(np, p.cuts_p, p.run_p), cut(no, p.cuts_o, p.run_o);
  const double pieces_p = static_cast<double>(heads_p) * p.cuts_p, pieces_o = static_cast<double>(heads_o) * p.cuts_o;
  if (pieces_p + pieces_o > 2e9) return kErrTooLarge;
  p.pieces_p = static_cast<int>(pieces_p), p.pieces = static_cast<int>(pieces_p + pieces_o);
  return kOk;
}
static long long piece_rows(const Params& p) {
  return static_cast<long long>(p.prompts) * p.cuts_p * p.hkv * p.rows_p + static_cast<long long>(p.rows) * p.cuts_o * p.hkv * p.rows_o;
}

template <int D>
static int launch(const Call& c, Params& p, cudaStream_t st) {
  using L = Layout<D>;
  CUtensorMap maps[4];
  const long long at[4] = {c.kp, c.vp, c.k, c.v};
  const long long* steps[4] = {c.kp_step, c.vp_step, c.k_step, c.v_step};
  for (int i = 0; i < 4; ++i) {
    const uint64_t n = i < 2 ? c.prefix : c.own;
    if (n == 0) continue;  // no piece reads through it
    const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(c.hkv), n, static_cast<uint64_t>(i < 2 ? c.prompts : c.rows)};
    const uint64_t bytes[3] = {static_cast<uint64_t>(steps[i][2]) * 2, static_cast<uint64_t>(steps[i][1]) * 2, static_cast<uint64_t>(steps[i][0]) * 2};
    const int rc = make_tmap_4d(&maps[i], reinterpret_cast<const void*>(at[i]), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, bytes, {64, 1, kKeys, 1}, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != kOk) return rc;
  }
  if (c.prefix == 0) maps[0] = maps[2], maps[1] = maps[3];
  if (c.own == 0) maps[2] = maps[0], maps[3] = maps[1];
  static bool attr[64] = {};  // an attribute of the kernel on one device
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= 64) return kErrDriver;
  if (!attr[device]) {
    if (cudaFuncSetAttribute(piece_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess) return kErrDriver;
    attr[device] = true;
  }
  if (p.pieces > 0) {
    const int ctas = 2 * sm_count();
    TTB_COUNT_LAUNCH(1);
    piece_kernel<D><<<p.pieces < ctas ? p.pieces : ctas, kThreads, L::kBytes, st>>>(maps[0], maps[1], maps[2], maps[3], p);
    if (cudaGetLastError() != cudaSuccess) return kErrDriver;
  }
  const long long warps = static_cast<long long>(p.rows) * p.s * p.hq;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((warps + kJoinWarps - 1) / kJoinWarps));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early, cfg.numAttrs = p.pieces > 0 ? 1 : 0;
  TTB_COUNT_LAUNCH(1);
  return cudaLaunchKernelEx(&cfg, join_kernel<D>, p) == cudaSuccess ? kOk : kErrDriver;
}

}  // namespace sprefix
}  // namespace ttb

// Floats of the workspace of a call (an sprefix::Call), or a negative error.
extern "C" long long ttb_shared_prefix_floats(const char* call, void*) {
  using namespace ttb::sprefix;
  const Call& c = *reinterpret_cast<const Call*>(call);
  Params p{};
  const int rc = plan_of(c, p);
  return rc != ttb::kOk ? rc : piece_rows(p) * (c.d + 2);
}

extern "C" int ttb_shared_prefix_attention(const char* call, float scale, int* err, void* stream) {
  using namespace ttb;
  using namespace ttb::sprefix;
  const Call& c = *reinterpret_cast<const Call*>(call);
  Params p{};
  const int rc = plan_of(c, p);
  if (rc != kOk) return rc;
  if ((c.q | c.o | c.kp | c.vp | c.k | c.v | c.work) & 15) return kErrBadShape;
  const long long rows = piece_rows(p);
  if (c.work_floats < rows * (c.d + 2)) return kErrBadShape;
  p.q = reinterpret_cast<const __nv_bfloat16*>(c.q), p.o = reinterpret_cast<__nv_bfloat16*>(c.o);
  p.start = reinterpret_cast<const int*>(c.start), p.stop = reinterpret_cast<const int*>(c.stop), p.lengths = reinterpret_cast<const int*>(c.lengths);
  p.part = reinterpret_cast<float*>(c.work), p.ml = reinterpret_cast<float2*>(p.part + rows * c.d);
  p.scale = scale, p.err = err;
  auto st = static_cast<cudaStream_t>(stream);
  return c.d == 128 ? launch<128>(c, p, st) : launch<64>(c, p, st);
}
