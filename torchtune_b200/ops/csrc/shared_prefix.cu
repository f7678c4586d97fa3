// Attention of rows that share a long prefix: a prompt's keys and values are read once for all rows (answers) of the prompt, a row's own keys once for the row.
//
//   o = sum_k e^(c q.k) v / sum_k e^(c q.k),   k over keys [start, stop) of the row's prompt and over the row's own keys up to the query's position.
//
// A softmax over pieces: each piece leaves m = max, l = sum 2^(x - m) and O = sum 2^(x - m) v, and o = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i.  A piece is a run of keys of one key head with up
// to 128 query rows: those of all rows of a prompt (answers x tokens x query heads that share the key head) on a run of the prefix, or those of one row on a run of its own keys.  Both are the
// same work: scores of 128 rows and 64 keys on tcgen05 tensor cores, a thread per row for the softmax, probabilities in the scores' place in tensor memory as the A operand of the second
// product, its accumulator next to them.  They are two bf16 numbers each, a rounded one and the rest, which take the 32 bits of a score: rounded once, they are off
// by more than the output's own rounding (outputs 0.0023 from exact ones, of which the latter is 0.0017; now it is all there is).  The second product takes twice as long, which shows where several
// tiles of rows meet the same keys and the tensor cores bound (256 rows of three tokens: 200 -> 216 us; one token of 4 to 64 rows: 1 % at most).
// A tile of 64 keys and values is 32 KB: an SM's share of the memory's rate brings it in 1400 cycles, and 128 rows keep the tensor cores busy for 770 of them and the
// exponentials' unit for 512, so that padding a single token's four rows to 128 costs nothing that is not idle; warps without rows have no part in the softmax.
// Two CTAs to an SM share the tiles of all key heads out evenly, as they are: tiles of the prefixes in their order are one line, those of the rows another, CTAs get a stretch of one of them each
// (with more than 128 query rows to a head, as many CTAs next to each other as there are tiles of rows, so that all but one find the keys in L2), and a piece ends where a head or a
// stretch does.  Lengths are read on the device, so a recorded launch follows them.  A ring of slots that K and V fill in turn runs on over the end of a piece, so that the keys of the next one
// arrive while the output of the last is written; the scores of a tile are computed while the softmax of the one before is.  Pieces lie in a workspace that a second launch joins in a fixed order.
//
// What lies behind the last visible key may be anything: scores are masked by selection, and the values of a piece's last tile that nobody sees are overwritten with zeros before they are
// multiplied.  A value that is seen and infinite times a rest of 0 is NaN, as it is times a probability of 0.  Every wait is bounded and reports through the error word.
//
// Bound by bytes on long rows, else by what a piece does one after the other (products, softmax, products, output: 3 to 5 us, which the two CTAs of an SM hide from each other in part) and by the
// start (finding the shares, first loads: 5 us) and the joining launch.  Measured (32 query on 8 key heads of 128 channels, kernels behind one another in a graph): 16 rows on 32003 shared keys and
// 300 of their own 39 us (3.7 TB/s); 64 rows of 4 prompts of 613 and 391 own 30 us; 256 rows of three tokens, 8 prompts of 4096 and 1001 own 216 us (4.3 TB/s; tensor cores 63 % busy); one prompt of 61
// 11 us.
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
  int* shared_out;          // what the CTAs have agreed on: groups of the prefix and of rows, tiles in front of every prompt and of all, of every row and of all
  float* part;              // pieces' outputs: rows of D floats
  float2* ml;               // their maxima (log2) and sums
  int prompts, rows, s, hq, hkv, group;
  int prefix, own;          // slots
  int rows_p, rows_o;       // query rows of a prompt and of a row, per key head
  int pieces_p;             // most pieces of the prefix: those of rows lie behind them
  uint32_t per_group;       // 2^32 / group, rounded up: the high word of a row times that is row / group, for rows below 2^32 / group
  float scale;
  int* err;
};
static constexpr int kSide = 8;  // CTAs next to each other for the tiles of rows of a head; more tiles than that are a CTA's one after the other
__host__ __device__ __forceinline__ int tiles_of(int rows) { return (rows + kRows - 1) / kRows; }
__host__ __device__ __forceinline__ int side_of(int rows) { return tiles_of(rows) < kSide ? tiles_of(rows) : kSide; }

// Token of a query row.
__device__ __forceinline__ int token_of(const Params& p, int row) { return p.group == 1 ? row : static_cast<int>(__umulhi(row, p.per_group)); }

// Visible slots [lo, hi) of a prompt or a row.
__device__ __forceinline__ void slots_of(const Params& p, bool prefix, int owner, int& lo, int& hi) {
  if (prefix) {
    lo = p.start != nullptr ? max(p.start[owner], 0) : 0;
    hi = p.stop != nullptr ? min(p.stop[owner], p.prefix) : p.prefix;
  } else {
    lo = 0;
    hi = p.lengths != nullptr ? min(p.lengths[owner], p.own) : p.own;
  }
}
__device__ __forceinline__ int key_tiles(const Params& p, bool prefix, int owner) {
  int lo, hi;
  slots_of(p, prefix, owner, lo, hi);
  return lo < hi ? (hi - lo + kKeys - 1) / kKeys : 0;
}

// n tiles over g groups: group i has [i n / g, (i + 1) n / g).  The check of sizes keeps n below 2^31, and g is a number of CTAs, below 2^11: quotients are below 2^31 and those that are no whole number
// at least 2^-11 from one (border), or below 2^11 and 2^-31 (group_of), further than a double's rounding of 2^-53 of them, and the others are exact; a division of doubles is a tenth of one of 64-bit integers.
__device__ __forceinline__ long long border(long long n, int g, int i) { return static_cast<long long>(static_cast<double>(n * i) / g); }
__device__ __forceinline__ int group_of(long long n, int g, long long tile) { return static_cast<int>(static_cast<double>((tile + 1) * g - 1) / static_cast<double>(n)); }

// A CTA's part: a stretch of the tiles of the prefixes or of the rows.
struct Share {
  bool prefix;
  int group, side, sides, owner, head, tile;  // where it begins
  int count;                                  // tiles of keys
};
// The pieces of a share, for each of its tiles of query rows.
struct Walk {
  int owner, head, tile, left;  // left: of the stretch
  int row_tile;
  int lo, hi, n;                // of the owner
  __device__ __forceinline__ Walk(const Params& p, const Share& s) : row_tile(s.side) { restart(p, s); }
  __device__ __forceinline__ void restart(const Params& p, const Share& s) {
    owner = s.owner, head = s.head, tile = s.tile, left = s.count;
    if (left > 0) enter(p, s.prefix);
  }
  __device__ __forceinline__ void enter(const Params& p, bool prefix) {
    slots_of(p, prefix, owner, lo, hi);
    n = lo < hi ? (hi - lo + kKeys - 1) / kKeys : 0;
  }
  __device__ __forceinline__ int count() const { return min(n - tile, left); }  // tiles of the piece
  __device__ __forceinline__ int first() const { return lo + tile * kKeys; }
  __device__ __forceinline__ int last() const { return min(hi, lo + (tile + count()) * kKeys); }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next(const Params& p, const Share& s) {
    left -= count();
    tile = 0;
    if (left > 0) {
      if (++head == p.hkv) {
        head = 0;
        n = 0;
        while (n == 0 && ++owner < (s.prefix ? p.prompts : p.rows)) enter(p, s.prefix);
        if (n == 0) left = 0;  // not unless the lengths have changed meanwhile
      }
    } else if ((row_tile += s.sides) < tiles_of(s.prefix ? p.rows_p : p.rows_o)) {
      restart(p, s);
    }
  }
  // first row of the piece in the workspace
  __device__ __forceinline__ long long base(const Params& p, const Share& s) const {
    const long long piece = static_cast<long long>(owner) * p.hkv + head + s.group;  // pieces are one for every head and one for every border within a head
    return (s.prefix ? piece * p.rows_p : static_cast<long long>(p.pieces_p) * p.rows_p + piece * p.rows_o) + row_tile * kRows;
  }
};

template <int D>
struct Layout {
  static constexpr int kPanels = D / 64;
  static constexpr int kQuery = kPanels * kPanelBytes;  // queries; between two pieces the output on its way out
  static constexpr int kSlot = kPanels * kPanel;
  static constexpr int kSlots = D == 128 ? 4 : 8;
  static constexpr int kBars = kQuery + kSlots * kSlot;
  static constexpr int kBytes = kBars + (2 * kSlots + 7) * 8 + 16 + 1024;
  static constexpr int kColumns = 256;  // of tensor memory: outputs, then two tiles of scores
  static_assert(4 * 32 * 32 * 4 <= kQuery, "four warps' 32 x 32 outputs take the queries' place");
};

// Every CTA adds up the tiles of all prompts and rows, a run of them to a thread, and finds its share; the first one leaves the sums for the joining launch.
__device__ __forceinline__ void add_tiles(const Params& p, int (&mine)[2]) {
  const int t = threadIdx.x, run_p = (p.prompts + kThreads - 1) / kThreads, run_o = (p.rows + kThreads - 1) / kThreads;
  mine[0] = t * run_p < p.prompts ? key_tiles(p, true, t * run_p) : 0;  // the loads of these two go out together
  mine[1] = t * run_o < p.rows ? key_tiles(p, false, t * run_o) : 0;
  for (int i = t * run_p + 1; i < min(p.prompts, (t + 1) * run_p); ++i) mine[0] += key_tiles(p, true, i);
  for (int i = t * run_o + 1; i < min(p.rows, (t + 1) * run_o); ++i) mine[1] += key_tiles(p, false, i);
}
__device__ __forceinline__ void find_share(const Params& p, const int (&mine)[2], Share& share, int (*sums)[2]) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int run_p = (p.prompts + kThreads - 1) / kThreads, run_o = (p.rows + kThreads - 1) / kThreads;
  int upto[2] = {mine[0], mine[1]};
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int up = __shfl_up_sync(0xffffffffu, upto[k], x);
      if (lane >= x) upto[k] += up;
    }
  }
  if (lane == 31) sums[warp][0] = upto[0], sums[warp][1] = upto[1];
  __syncthreads();
  int before[2] = {upto[0] - mine[0], upto[1] - mine[1]}, all[2] = {0, 0};
  for (int w = 0; w < kThreads / 32; ++w)
#pragma unroll
    for (int k = 0; k < 2; ++k) before[k] += w < warp ? sums[w][k] : 0, all[k] += sums[w][k];
  // CTAs in proportion to the tiles, at most one to a tile of few rows or to two of 64 and more
  const int ctas = gridDim.x, side_p = side_of(p.rows_p), side_o = side_of(p.rows_o);
  const long long n_p = static_cast<long long>(all[0]) * p.hkv, n_o = static_cast<long long>(all[1]) * p.hkv;
  // the end of a piece costs about 1.5 tiles, and a head is one piece at least
  const long long work_p = (n_p + 3ll * p.prompts * p.hkv / 2) * tiles_of(p.rows_p), work_o = (n_o + 3ll * p.rows * p.hkv / 2) * tiles_of(p.rows_o);
  int ctas_p = n_p == 0 ? 0 : n_o == 0 ? ctas : static_cast<int>(static_cast<float>(work_p) / static_cast<float>(work_p + work_o) * ctas / side_p + 0.5f) * side_p;
  if (n_p > 0 && n_o > 0) ctas_p = max(side_p, min(ctas_p, (ctas - side_o) / side_p * side_p));
  auto groups_of = [](long long n, int room, int rows) { return n == 0 ? 0 : static_cast<int>(max(1ll, min(static_cast<long long>(room), n >> (rows >= 64)))); };
  const int groups[2] = {groups_of(n_p, ctas_p / side_p, p.rows_p), groups_of(n_o, (ctas - ctas_p) / side_o, p.rows_o)};
  const int cta = blockIdx.x, which = cta >= ctas_p, side = which ? side_o : side_p, at = which ? cta - ctas_p : cta;
  share.prefix = !which, share.group = at / side, share.side = at % side, share.sides = side, share.count = 0;
  __shared__ int found[3];
  if (share.group < groups[which]) {
    const long long n = which ? n_o : n_p, from = border(n, groups[which], share.group);
    share.count = static_cast<int>(border(n, groups[which], share.group + 1) - from);
    if (from >= static_cast<long long>(before[which]) * p.hkv && from < static_cast<long long>(before[which] + mine[which]) * p.hkv) {  // in this thread's run
      long long at_owner = static_cast<long long>(before[which]) * p.hkv;
      int owner = t * (which ? run_o : run_p), tiles = key_tiles(p, share.prefix, owner);
      const int owners = which ? p.rows : p.prompts;
      while (owner + 1 < owners && from >= at_owner + static_cast<long long>(tiles) * p.hkv) at_owner += static_cast<long long>(tiles) * p.hkv, tiles = key_tiles(p, share.prefix, ++owner);
      const int in = static_cast<int>(from - at_owner);  // of all tiles, below 2^31
      found[0] = owner, found[1] = in / tiles, found[2] = in % tiles;
    }
  }
  if (cta == 0) {
    if (t == 0) p.shared_out[0] = groups[0], p.shared_out[1] = groups[1], p.shared_out[2 + p.prompts] = all[0], p.shared_out[3 + p.prompts + p.rows] = all[1];
    for (int i = t * run_p; i < min(p.prompts, (t + 1) * run_p); ++i) p.shared_out[2 + i] = before[0], before[0] += key_tiles(p, true, i);
    for (int i = t * run_o; i < min(p.rows, (t + 1) * run_o); ++i) p.shared_out[3 + p.prompts + i] = before[1], before[1] += key_tiles(p, false, i);
  }
  __syncthreads();
  share.owner = found[0], share.head = found[1], share.tile = found[2];
}

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

// What two values' rounding to bf16 leaves over, rounded itself; the widening of the former is part of the difference.
__device__ __forceinline__ uint32_t rest_of(float a, float b, uint32_t rounded) {
  float x, y;
  asm("{\n\t.reg .b16 lo, hi, one;\n\tmov.b32 {lo, hi}, %2;\n\tmov.b16 one, 0xbf80;\n\tfma.rn.f32.bf16 %0, lo, one, %3;\n\tfma.rn.f32.bf16 %1, hi, one, %4;\n\t}" : "=f"(x), "=f"(y) : "r"(rounded), "f"(a), "f"(b));
  return pack_bf16x2(x, y);
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
  uint64_t* pv_done = q_full + 5;  // [2] its second product is done: one for odd and one for even tiles, since who waits knows only that the tile before the last is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 7);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;");  // the joining launch may take its place; it waits for the end of this one
  int my_tiles[2];
  add_tiles(p, my_tiles);
  if (threadIdx.x == 128) prefetch_tmap(&tm_kp), prefetch_tmap(&tm_vp), prefetch_tmap(&tm_ko), prefetch_tmap(&tm_vo);
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kSlots; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    mbar_init(q_full, 4);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 4), mbar_init(&pv_done[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, L::kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __shared__ int sums[kThreads / 32][2];
  Share share;
  find_share(p, my_tiles, share, sums);  // with two barriers
  tc_fence_after();
  const uint32_t tO = *tmem_slot, tS = tO + D;

  if (warp == 4) {
    // ---------------------------------------------------------------- loads: K and V of a tile in turn
    int slot = 0, n = 0;
    uint32_t phase = 0;
    bool ok = true;
    const CUtensorMap *map_k = share.prefix ? &tm_kp : &tm_ko, *map_v = share.prefix ? &tm_vp : &tm_vo;
    for (Walk w(p, share); w.more() && ok && !*abort_flag; w.next(p, share)) {
      const int first = w.first(), loads = 2 * w.count();
      for (int x = 0; x < loads && !*abort_flag; ++x, ++n) {
        if (!(ok = mbar_wait(&empty[slot], phase ^ 1))) {
          fail(abort_flag, p.err, 301);
          break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[slot], L::kSlot);
          for (int y = 0; y < L::kPanels; ++y) tma_load_4d(ring + slot * L::kSlot + y * kPanel, x & 1 ? map_v : map_k, &full[slot], y * 64, w.head, first + (x >> 1) * kKeys, w.owner);
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
    for (Walk w(p, share); w.more() && ok && !*abort_flag; w.next(p, share)) {
      const int n = w.count();
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
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) umma_f16_ts(tO, from + kKeys / 2 + k * 8, make_smem_desc_sw128(v_base + k * 2048, kPanel, 1024), idesc_o, 1);
          umma_commit(&empty[slot]);
          umma_commit(&pv_done[done & 1]);
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
    // Queries are on their way while the output of the piece before is written: eight 16-byte parts per thread, which for 128 channels are 64 rows; more rows follow when their piece begins.
    constexpr int kParts = D / 8, kStep = 128 / kParts;  // parts of a row; rows at a time
    const int q_part = threadIdx.x % kParts, q_row = threadIdx.x / kParts;
    const int rows = share.prefix ? p.rows_p : p.rows_o;
    auto fetch = [&](const Walk& w, int r0, uint4 (&v)[8]) {
      const int row0 = w.row_tile * kRows + r0, end = min(rows - w.row_tile * kRows, kRows) - r0;
      const long long token0 = static_cast<long long>(w.owner) * (share.prefix ? p.rows / p.prompts * p.s : p.s);
      const __nv_bfloat16* from = p.q + (token0 * p.hq + w.head * p.group) * D + q_part * 8;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int r = q_row + x * kStep;
        if (r < end) {
          const uint32_t row = row0 + r, token = token_of(p, row);
          v[x] = *reinterpret_cast<const uint4*>(from + static_cast<long long>(token * p.hq + row - token * p.group) * D);
        }
      }
    };
    auto put = [&](int r0, int live, const uint4 (&v)[8]) {
      uint8_t* to = sQ + (q_part >> 3) * kPanelBytes;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int r = r0 + q_row + x * kStep;
        if (r < live) *reinterpret_cast<uint4*>(to + r * 128 + (((q_part & 7) ^ (r & 7)) << 4)) = v[x];
      }
    };
    Walk w(p, share);
    uint4 queries[8];
    if (w.more()) fetch(w, 0, queries);
    while (w.more() && !stop) {
      const int n_tiles = w.count(), first = w.first(), last = w.last();
      const int row0 = w.row_tile * kRows, live = min(kRows, rows - row0), live_warps = (live + 31) / 32;
      put(0, live, queries);
      if (live > 8 * kStep) {
        fetch(w, 8 * kStep, queries);
        put(8 * kStep, live, queries);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      const int r = warp * 32 + lane;
      int mine = r < live ? last : first;  // keys of this row end here
      if (!share.prefix && r < live) mine = min(last, w.hi - p.s + token_of(p, row0 + r) + 1);
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
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t hi[16], lo[16];  // the second product's operand: probabilities rounded to 8 bits, and what that leaves over, so that it has 16
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t t = fma_f32x2(pack_u32x2(sv[half][i], sv[half][i + 1]), c2, nm2);
              float t0, t1;
              unpack_f32x2(t, t0, t1);
              const float e0 = fast_exp2(t0), e1 = fast_exp2(t1);
              sum2[(i >> 1) & 1] = add_f32x2(sum2[(i >> 1) & 1], pack_f32x2(e0, e1));
              hi[i >> 1] = pack_bf16x2(e0, e1);
              lo[i >> 1] = rest_of(e0, e1, hi[i >> 1]);
            }
            tmem_st_32x16(tile + half * 16, hi);
            tmem_st_32x16(tile + 32 + half * 16, lo);
          }
          float s0, s1, s2, s3;
          unpack_f32x2(sum2[0], s0, s1);
          unpack_f32x2(sum2[1], s2, s3);
          l = l * alpha + (s0 + s1) + (s2 + s3);
          if (j > 0 && __any_sync(0xffffffffu, rescale)) {
            if (!(ok = mbar_wait(&pv_done[(done - 1) & 1], ((done - 1) >> 1) & 1))) break;  // the second product before this one has left the output
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
          tc_fence_before();
        }
        if (last - k0 < kKeys && (warp >= live_warps || live_warps == 4)) {  // the last tile: values that nobody sees may be anything, and 0 * NaN is NaN; warps without rows see to it, if there are any
          const uint32_t slot = (2 * done + 1) % L::kSlots;
          if (!(ok = mbar_wait(&full[slot], ((2 * done + 1) / L::kSlots) & 1))) break;
          uint8_t* v = ring + slot * L::kSlot;
          const int dead = kKeys - (last - k0), from = live_warps == 4 ? 0 : live_warps * 32;
          for (int x = threadIdx.x - from; x < dead * L::kPanels * 8; x += 128 - from) {
            const int key = kKeys - dead + x / (L::kPanels * 8), y = x % (L::kPanels * 8);
            *reinterpret_cast<uint4*>(v + (y >> 3) * kPanel + key * 128 + (y & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[done & 1]);
      }
      Walk after = w;
      after.next(p, share);
      if (after.more()) fetch(after, 0, queries);
      if (ok && !*abort_flag) ok = mbar_wait(&pv_done[(done - 1) & 1], ((done - 1) >> 1) & 1);
      if (ok && !*abort_flag && warp < live_warps) {
        tc_fence_after();
        // the output, unnormalised, by way of shared memory, where the queries are no longer needed, so that a row's values are written side by side
        const long long base = w.base(p, share);
        float4* stage = reinterpret_cast<float4*>(sQ) + warp * 256;
        const int count = live - warp * 32;
        float* to = p.part + (base + warp * 32 + (lane >> 3)) * D + (lane & 7) * 4;
#pragma unroll 1
        for (int ch = 0; ch < D / 32; ++ch) {
          uint32_t v[32];
          tmem_ld_32x32(tO + lanes + ch * 32, v);
          tmem_ld_wait();
          if (count <= 16) {  // few rows: straight from the registers (12 rows to a piece: 4 % of the time in all; where pieces have 128, the same from there 50 -> 54)
            if (lane < count) {
              float4* at = reinterpret_cast<float4*>(p.part + (base + r) * D + ch * 32);
#pragma unroll
              for (int i = 0; i < 8; ++i) at[i] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
            }
            continue;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) stage[lane * 8 + (i ^ (lane & 7))] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // four rows at a time
            const int y = i * 4 + (lane >> 3);
            if (y < count) *reinterpret_cast<float4*>(to + i * 4 * D + ch * 32) = stage[y * 8 + ((lane & 7) ^ (y & 7))];
          }
          __syncwarp();
        }
        if (r < live) p.ml[base + r] = make_float2(m_used, l);
        tc_fence_before();
      }
      if (!ok) fail(abort_flag, p.err, 303);
      stop = any_of_four(!ok || *abort_flag);  // all outputs are out of the queries' place; the four warps go on together or not at all
      w = after;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tO, L::kColumns);
}

// Joins the pieces of Q query rows of one row and key head, those of the prefix and then their own.  Where Q is 1, a warp of `wide` (a power of two up to 8) takes every wide-th run of 32 pieces or, of
// fewer, its part of them; warps meet in shared memory, in their order.  A lane per piece finds where it lies, its maxima and sums, and the weights go around, so that all loads but the first two are
// independent.  With many results it is the finding that takes the time, so that four of them share it (59 136 results of 3 to 4 pieces, 64 channels: 48 -> 27 us after the last piece).
static constexpr int kJoinWarps = 8;
template <int D, int Q>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ Params p, int wide, int chunks) {
  __shared__ float outputs[kJoinWarps][Q == 1 ? D : 1];
  __shared__ float2 sums[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, member = Q == 1 ? warp & (wide - 1) : 0;
  const uint32_t w = Q == 1 ? (blockIdx.x * kJoinWarps + warp) / wide : blockIdx.x * kJoinWarps + warp;  // of rows, key heads and chunks of query rows
  const uint32_t owner = w / chunks;
  const int row = static_cast<int>(owner / p.hkv), head = static_cast<int>(owner - row * static_cast<uint32_t>(p.hkv)), q0 = static_cast<int>(w - owner * chunks) * Q;
  const bool live = row < p.rows;
  const int per = p.rows / p.prompts, prompt = row / per, mine = min(Q, p.rows_o - q0);  // query rows
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the pieces are written
  constexpr int kMine = D / 32;
  float m[Q], l[Q], o[Q][kMine];
#pragma unroll
  for (int y = 0; y < Q; ++y) {
    m[y] = -INFINITY, l[y] = 0.f;
#pragma unroll
    for (int x = 0; x < kMine; ++x) o[y][x] = 0.f;
  }
  if (live) {
    // pieces of the prompt's head, then of the row's own: those of all groups of CTAs with a tile of it
    const int* before_p = p.shared_out + 2;
    const int* before_o = before_p + p.prompts + 1;
    const int owners[2] = {prompt, row}, groups[2] = {p.shared_out[0], p.shared_out[1]}, at[2] = {before_p[prompt], before_o[row]}, next[2] = {before_p[prompt + 1], before_o[row + 1]};
    const int all[2] = {before_p[p.prompts], before_o[p.rows]};
    int from[2], count[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int n = next[k] - at[k];
      const long long total = static_cast<long long>(all[k]) * p.hkv, first = static_cast<long long>(at[k]) * p.hkv + static_cast<long long>(head) * n;
      from[k] = n > 0 ? group_of(total, groups[k], first) : 0;
      count[k] = n > 0 ? group_of(total, groups[k], first + n - 1) - from[k] + 1 : 0;
    }
    const int pieces = count[0] + count[1], run = min(32, (pieces + wide - 1) / wide);
    for (int first_piece = member * run; first_piece < pieces; first_piece += wide * run) {
      const int piece = first_piece + lane, n = min(run, pieces - first_piece);
      long long place = 0;
      float2 t[Q];
#pragma unroll
      for (int y = 0; y < Q; ++y) t[y] = make_float2(-INFINITY, 0.f);
      if (lane < n) {
        place = piece < count[0] ? (static_cast<long long>(owners[0]) * p.hkv + head + from[0] + piece) * p.rows_p + (row - prompt * per) * p.rows_o + q0
                                 : static_cast<long long>(p.pieces_p) * p.rows_p + (static_cast<long long>(owners[1]) * p.hkv + head + from[1] + piece - count[0]) * p.rows_o + q0;
#pragma unroll
        for (int y = 0; y < Q; ++y)
          if (y < mine) t[y] = p.ml[place + y];
      }
      float weight[Q];
#pragma unroll
      for (int y = 0; y < Q; ++y) {
        float top = fmaxf(m[y], t[y].x);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float base = top == -INFINITY ? 0.f : top, f = exp2f(m[y] - base);
        weight[y] = exp2f(t[y].x - base);
        float sum = t[y].y * weight[y];
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        l[y] = l[y] * f + sum;
        m[y] = top;
#pragma unroll
        for (int c = 0; c < kMine; ++c) o[y][c] *= f;
      }
      constexpr int kAtOnce = Q == 1 ? 8 : 2;
      for (int x0 = 0; x0 < n; x0 += kAtOnce) {
        float v[kAtOnce][Q][kMine], g[kAtOnce][Q];
        const float* of[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
          of[x] = p.part + __shfl_sync(0xffffffffu, place, x0 + x) * D + lane * kMine;
#pragma unroll
          for (int y = 0; y < Q; ++y) g[x][y] = __shfl_sync(0xffffffffu, weight[y], x0 + x);  // 0 where no key is seen
        }
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
#pragma unroll
          for (int y = 0; y < Q; ++y)
            if (g[x][y] != 0.f) {
              if constexpr (kMine == 4) *reinterpret_cast<float4*>(v[x][y]) = *reinterpret_cast<const float4*>(of[x] + y * D);
              else *reinterpret_cast<float2*>(v[x][y]) = *reinterpret_cast<const float2*>(of[x] + y * D);
            }
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x)
#pragma unroll
          for (int y = 0; y < Q; ++y)
            if (g[x][y] != 0.f) {
#pragma unroll
              for (int c = 0; c < kMine; ++c) o[y][c] += v[x][y][c] * g[x][y];
            }
      }
    }
  }
  if constexpr (Q == 1) {
    if (wide > 1) {
      if (lane == 0) sums[warp] = make_float2(m[0], l[0]);
#pragma unroll
      for (int y = 0; y < kMine; ++y) outputs[warp][lane * kMine + y] = o[0][y];
      __syncthreads();
      if (member != 0) return;
      for (int x = 1; x < wide; ++x) {
        const float2 t = sums[warp + x];
        const float top = fmaxf(m[0], t.x), base = top == -INFINITY ? 0.f : top, f = exp2f(m[0] - base), g = exp2f(t.x - base);
        l[0] = l[0] * f + t.y * g;
        m[0] = top;
#pragma unroll
        for (int y = 0; y < kMine; ++y) o[0][y] = o[0][y] * f + outputs[warp + x][lane * kMine + y] * g;
      }
    }
  }
  if (!live) return;
#pragma unroll
  for (int x = 0; x < Q; ++x) {
    if (x >= mine) break;
    const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];  // a query without a key gives 0
    uint32_t out[kMine / 2];
#pragma unroll
    for (int y = 0; y < kMine / 2; ++y) out[y] = pack_bf16x2(o[x][2 * y] * inv, o[x][2 * y + 1] * inv);
    const int i = token_of(p, q0 + x);
    __nv_bfloat16* to = p.o + ((static_cast<long long>(row) * p.s + i) * p.hq + head * p.group + q0 + x - i * p.group) * D + lane * kMine;
    if constexpr (kMine == 4) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
    else *reinterpret_cast<uint32_t*>(to) = out[0];
  }
}

// What a call brings, packed by the host language in this order.
struct Call {
  long long q, o, kp, vp, k, v, start, stop, lengths, work, work_floats;
  long long kp_step[3], vp_step[3], k_step[3], v_step[3];  // batch, slot, head; elements
  long long prompts, rows, s, hq, hkv, d, prefix, own;
};

// Sizes, and rows of the workspace: a piece for every head and one for every group of CTAs, of the prefixes and of the rows.
static int plan_of(const Call& c, Params& p, long long& rows, long long& head_floats, int& ctas) {
  if (c.prompts <= 0 || c.rows <= 0 || c.rows % c.prompts || c.s <= 0 || c.hkv <= 0 || c.hq <= 0 || c.hq % c.hkv || (c.d != 64 && c.d != 128) || c.prefix < 0 || c.own < 0) return kErrBadShape;
  if (c.rows > 0x3fffffff || c.prefix > 0x3fffffff || c.own > 0x3fffffff || c.rows * c.s > 0x7fffffff / c.hq || c.hkv > 256 || c.rows * (c.own / kKeys + 1) > 0x3fffffff ||
      c.prompts * (c.prefix / kKeys + 1) > 0x3fffffff)
    return kErrTooLarge;
  const long long np = (c.prefix + kKeys - 1) / kKeys, no = (c.own + kKeys - 1) / kKeys;  // tiles of keys
  if (c.prompts * np * c.hkv > 0x7fffffff || c.rows * no * c.hkv > 0x7fffffff) return kErrTooLarge;  // those of all heads are counted in 32 bits
  p.prompts = static_cast<int>(c.prompts), p.rows = static_cast<int>(c.rows), p.s = static_cast<int>(c.s), p.hq = static_cast<int>(c.hq), p.hkv = static_cast<int>(c.hkv);
  p.group = p.hq / p.hkv, p.prefix = static_cast<int>(c.prefix), p.own = static_cast<int>(c.own);
  p.per_group = p.group == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + p.group - 1) / p.group);
  if (c.rows / c.prompts * c.s * p.group * p.group > 0xffffffffll) return kErrTooLarge;
  p.rows_p = static_cast<int>(c.rows / c.prompts * c.s * p.group), p.rows_o = static_cast<int>(c.s * p.group);
  const long long most = c.prompts * c.hkv * np * tiles_of(p.rows_p) + c.rows * c.hkv * no * tiles_of(p.rows_o);
  const int all = 2 * sm_count();
  ctas = most < 2 * kSide ? 2 * kSide : most < all ? static_cast<int>(most) : all;
  const long long pieces_p = np > 0 ? c.prompts * c.hkv + ctas / side_of(p.rows_p) : 0, pieces_o = no > 0 ? c.rows * c.hkv + ctas / side_of(p.rows_o) : 0;
  if (pieces_p > 0x7fffffff) return kErrTooLarge;
  p.pieces_p = static_cast<int>(pieces_p);
  rows = pieces_p * p.rows_p + pieces_o * p.rows_o;
  head_floats = (4 + c.prompts + c.rows + 3) / 4 * 4;
  return kOk;
}

template <int D>
static int launch(const Call& c, Params& p, int ctas, cudaStream_t st) {
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
  TTB_COUNT_LAUNCH(2);
  piece_kernel<D><<<ctas, kThreads, L::kBytes, st>>>(maps[0], maps[1], maps[2], maps[3], p);
  if (cudaGetLastError() != cudaSuccess) return kErrDriver;
  const long long results = static_cast<long long>(p.rows) * p.s * p.hq;
  const bool four = p.rows_o > 2 && results >= 64ll * sm_count();  // to a warp, where that leaves sixteen to an SM
  const int chunks = four ? (p.rows_o + 3) / 4 : p.rows_o;
  const long long warps = static_cast<long long>(p.rows) * p.hkv * chunks;
  int wide = 1;  // few results are joined by more warps each, until there are sixteen to an SM
  while (!four && wide < kJoinWarps && warps * wide * 2 <= 16ll * sm_count()) wide *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((warps * wide + kJoinWarps - 1) / kJoinWarps));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute early[1];
  early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = early, cfg.numAttrs = 1;
  return (four ? cudaLaunchKernelEx(&cfg, join_kernel<D, 4>, p, wide, chunks) : cudaLaunchKernelEx(&cfg, join_kernel<D, 1>, p, wide, chunks)) == cudaSuccess ? kOk : kErrDriver;
}

}  // namespace sprefix
}  // namespace ttb

// Floats of the workspace of a call (an sprefix::Call), or a negative error.
extern "C" long long ttb_shared_prefix_floats(const char* call, void*) {
  using namespace ttb::sprefix;
  const Call& c = *reinterpret_cast<const Call*>(call);
  Params p{};
  long long rows = 0, head = 0;
  int ctas = 0;
  const int rc = plan_of(c, p, rows, head, ctas);
  return rc != ttb::kOk ? rc : head + rows * (c.d + 2);
}

extern "C" int ttb_shared_prefix_attention(const char* call, float scale, int* err, void* stream) {
  using namespace ttb;
  using namespace ttb::sprefix;
  const Call& c = *reinterpret_cast<const Call*>(call);
  Params p{};
  long long rows = 0, head = 0;
  int ctas = 0;
  const int rc = plan_of(c, p, rows, head, ctas);
  if (rc != kOk) return rc;
  if ((c.q | c.o | c.kp | c.vp | c.k | c.v | c.work) & 15) return kErrBadShape;
  if (c.work_floats < head + rows * (c.d + 2)) return kErrBadShape;
  p.q = reinterpret_cast<const __nv_bfloat16*>(c.q), p.o = reinterpret_cast<__nv_bfloat16*>(c.o);
  p.start = reinterpret_cast<const int*>(c.start), p.stop = reinterpret_cast<const int*>(c.stop), p.lengths = reinterpret_cast<const int*>(c.lengths);
  p.shared_out = reinterpret_cast<int*>(c.work);
  p.part = reinterpret_cast<float*>(c.work) + head, p.ml = reinterpret_cast<float2*>(p.part + rows * c.d);
  p.scale = scale, p.err = err;
  auto st = static_cast<cudaStream_t>(stream);
  if (c.prefix == 0 && c.own == 0) return cudaMemsetAsync(p.o, 0, c.rows * c.s * c.hq * c.d * 2, st) == cudaSuccess ? kOk : kErrDriver;
  return c.d == 128 ? launch<128>(c, p, ctas, st) : launch<64>(c, p, ctas, st);
}
