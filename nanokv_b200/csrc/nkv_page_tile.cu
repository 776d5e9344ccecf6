// Attention over the paged 16-bit cache, on tcgen05.
//
// The rows of a kv head (its group's heads of all pending tokens) are the left operand of both products: S = Q K^T of a tile
// of 128 tokens goes to tensor memory, eight warps take the softmax (a thread per row), P replaces S as the operand of O += P V.  One
// warp brings K and V as they lie, page by page, into a ring of swizzled tiles.  Two forms, by the rows a kv head has:
//
//   wide    more than 128: units of 256 rows, two query tiles that share every K and V tile, four warps each.
//   narrow  up to 128, one query tile; the two groups of four warps take the even and the odd tiles of its tokens, each with sums of
//           its own.  Up to 32 rows stand in the query tile four times, one below the other, and every copy takes a share of a tile's
//           tokens or of its weights' bits: the weights of the others are stored as zeros.  The copies' sums are joined in shared memory.
//
// Softmax: P' = 2^(s - m) with a reference m that follows the running maximum of the scaled scores, s; it moves when P' would pass
// 2^8 times what it was set to.  bf16: set so that the sum of a row's P' stays below 1, O = sum P' V then below the largest |V|, any
// number of bf16.  fp16: set to 2^7, up to 2^15 from there: weights down to 2^-21 of the largest keep all their bits (2^-29 at
// best), smaller ones have half a step of 2^-25 where the largest has at least 2^7.  The row sum, the maximum and O
// stay in fp32.  P' enters the product with V in 16 bits: fp16 rounded to nearest; bf16 as the upper half of its fp32 bits, a byte
// permutation instead of a conversion.  What is cut off is up to 2^-7 of a weight and, where many weights are alike, the same for all of
// them: so rows of O are divided by the sum of the weights as they entered the product, two additions more a pair of scores, and lse
// takes the sum of the weights in full.  (4,680 queries x 24 heads over 24,960 tokens 1,413 us, 32 trees of 16 nodes x 40 heads 232, cases in
// turn; divided by the full sum, cut off / rounded to nearest: 1,370 / 1,389 and 226 / 227, and results up to 2^-8 off as a whole, row by row.
// The second sum behind the weights' handing over: 1,411 and 238; from halves unpacked by shifts and masks 1,455 and 239.)  With four
// copies, two of them take the upper half of P' and two the rest (2^-15 of it is left): few rows have few results, and no average to hide an
// unlucky weight in.  A token's row is therefore rounded otherwise alone than as one of more than 32 rows.
//
// Pending tokens that some row does not see, and whatever lies in a page behind a sequence's last token, are masked in the scores.  A weight
// of 0 times a value that is not finite would be NaN, so two warps look at the V tiles with such tokens: values behind the
// last token become 0 in shared memory, and so do values that are not finite; rows that see them get them added at the end, from memory.
//
// A page of K or V comes as one copy, whatever its size: the tensor map has the eight rows of a swizzle group, the 64-element chunks of a
// row and the groups of a page as dimensions, so that a tile is its groups one behind the other, each with its chunks side by side.
//
// Measured (kernel and join; over three states in turn, a quarter of a second long / six calls after a second's rest: the difference is the
// clock that the power limit leaves, one state or several are alike): one query token over 99,840 tokens x 40 heads 336 / 311 us (2.04 GB, 6.1 /
// 6.6 TB/s: memory); 32 trees of 16 nodes x 40 heads over up to 16,411 tokens x 8 heads 233 / 199 us (4.6 / 5.4 TB/s; as many bytes of one
// sequence 225 / 191, in pages of 64 for 16 tokens 205 / 186); 4,680 queries x 24 heads over 24,960 tokens 1.43 / 1.26 ms (1,000 / 1,140 TFLOP/s),
// 2 x 4,095 causal queries x 32 heads 352 / 337 us.  What bounds the wide form: the MMA warp, whose six batches a tile pair (S and two
// halves of PV for both query tiles, 2,048 tensor cycles) take about 3,400 cycles with the waits between them, and power: reading K and V from L2
// instead of memory gave 10 % (rounds, below).  Small calls: two launches, the plan, and a chain of table, tile, two products, rows.
// Tried and dropped (4,680 queries, us, kept form first, before the weights' second sum): exponentials ahead of the row's maximum (1,333 /
// 1,390; with straight code and a fallback 1,345 / 1,368); K awaited with the weights (1,333 / 1,362); two barriers per wait (1,339 / 1,393); waits without parking (no change); P
// beside S in tensor memory for 64-wide heads (no change); two more copies' bits by a second product (batch of trees 238 / 324).
//
// Table, lengths and counts are read by the kernel: every thread block makes the plan (nkv_page_plan.h) for itself.  The tiles of all
// units form one list that the SMs take in equal runs; a unit that a run's end cuts leaves fp32 parts, joined by a second launch.
// Warps: 0-7 softmax, 8-9 queries and masked values, 10 MMA issue, 11 pages: 384 threads, whose registers are dealt out
// so that a softmax thread holds a row's 128 scores at once.
#include "nkv_internal.h"
#include "nkv_page.cuh"
#include "nkv_tile.cuh"

namespace nkv {
namespace {

using namespace tc;
using page::Piece;
using page::Plan;
using page::Shape;
using page::TOK;
using page::Tour;

constexpr int QT = 128;                           // rows of a query tile
constexpr int SUB = 128 * 128;                    // bytes of a [128 rows x 64 elements] swizzled tile
constexpr int SOFTMAX_WARPS = 8, OPERAND_WARPS = 2, MMA_WARP = 10, THREADS = 384;
constexpr float RESCALE_THRESHOLD = 8.0f;
// Rounds that there is scratch for, and places of a run that a cut more is worth.  us in 1 / 2 / 3 / 4 / 5 / 6 / 8 rounds, heads of 128, quarters
// of a second of each in shuffled order over three states, at the power limit; queries x heads over tokens x kv heads (MB of them, units):
//   4,680 x 24 over 24,960 x 24 (307, 456)           1,632 1,603 1,424 1,472 1,483 1,451 1,486   5.06 GB read from memory in one, 0.58 in three
//   1,560 x 40 over 100,120 x 8 (410, 248)           3,509 3,512 3,402 3,249 3,054 3,215 3,097
//   6,000 x 8 over 66,000 x 8 (270, 192)             1,805 1,793 1,672 1,579 1,653 1,626 1,615
//   2,048 x 40 over 18,432 x 40, causal (377, 320)     838   815   811   802   824   819   835
//   4 x 512 x 32 over 32,768 x 8, causal (537, 256)  1,225 1,232 1,222 1,169 1,192 1,155 1,166
//   1,560 x 24 over 24,960 x 24 (307, 168)             604   583   577   571   594   592   626
//   4,095 x 32 over 24,095 x 8, causal (99, 512)     1,411 1,396 1,427 1,457 1,477 1,484 1,567
//   2 x 1,024 x 24 over 13,312 x 24 (327, 192)         402   387   408   400   419   428   456   140 places a run in one round
//   600 x 40 over 30,600 x 40 (627, 120)               515   523   532   518   531   538   571   200 places
//   8 x 333 x 16 over 8,500 x 16, causal (557, 256)    303   312   329   338   353   354   367   120 places
// The rule takes 3, 5, 4, 4, 5, 3, 2, 2, 3 and 1.
constexpr int MOST_ROUNDS = 5, LEAST_RUN = 64;
constexpr float NOTHING = -3e38f;                 // the reference before the first score: below all, and a number

// (P_READY: chain i, half h of a tile's tokens at 2 i + h)
enum Bar { Q_FULL = 0, Q_FREE = 1, S_FULL = 2, P_READY = 4, O_DONE = 8, O_FREE = 10, DRAINED = 12, FULL = 13, FREE = 23, LOOK = 33, CLEAN = 43, NUM_BARS = 53 };
constexpr int M_SLOT = NUM_BARS * 8, M_ABORT = M_SLOT + 4, M_STRAY = M_SLOT + 8, M_ROUNDS = M_SLOT + 12, M_EXTENTS = 448;
constexpr int M_START = M_EXTENTS + page::MOST_SEQUENCES * static_cast<int>(sizeof(page::Extent)), META = 2048;
static_assert(M_ROUNDS + 4 <= M_EXTENTS && M_START + 4 * (page::MOST_SEQUENCES + 1) <= META && page::MOST_SEQUENCES < 128, "meta block");

// COPIES 0: the wide form
template <int D, int COPIES> struct Layout {
  static constexpr bool NARROW = COPIES > 0;
  static constexpr int QTILES = NARROW ? 1 : 2, UNIT = QTILES * QT;
  static constexpr int DCH = D / 64;
  static constexpr int STAGE = DCH * SUB, STAGES = D == 128 ? 5 : 10;
  static constexpr int LEAD = NARROW ? 2 : 1;      // K tiles ahead of the first V tile in the ring
  static constexpr int Q_OFF = META;
  static constexpr int RING_OFF = Q_OFF + QTILES * DCH * SUB;
  static constexpr int ML_OFF = RING_OFF + STAGES * STAGE;             // narrow: references and sums of 256 threads, of two pieces
  static constexpr int JOIN_OFF = ML_OFF + (NARROW ? 2 * 256 * 8 : 0);     // narrow: columns of O of all copies of the rows; of one copy what
                                                                            // cut weights are short of, as the references
  static constexpr int JOIN_WORDS = D == 128 ? 6912 : 11264;
  static constexpr int BYTES = JOIN_OFF + (NARROW ? JOIN_WORDS * 4 : 0);
  static constexpr int DYNAMIC = BYTES + 1024;     // room to start on 1,024 bytes
  static constexpr int GROUP = DCH * 1024;         // eight rows of a K or V tile: their chunks of 64 elements side by side
};
static_assert(Layout<128, 0>::DYNAMIC <= 232448 && Layout<64, 0>::DYNAMIC <= 232448 && Layout<128, 1>::DYNAMIC <= 232448 &&
                  Layout<64, 1>::DYNAMIC <= 232448,
              "shared memory");
static_assert(Layout<128, 1>::JOIN_WORDS >= 256 * 20, "16 columns of all rows and copies");

// copies of the query rows: SLICES of a tile's tokens times PARTS of a weight's bits
template <int DT, int COPIES> constexpr int PARTS = DT == NKV_BF16 && COPIES == 4 ? 2 : 1;
template <int DT, int COPIES> constexpr int SLICES = COPIES > 1 ? COPIES / PARTS<DT, COPIES> : 1;

// The n-th tile of a piece in the ring, which holds them in the order in which they are used: LEAD tiles of K, then a tile of V and
// one of K in turn.
template <class L> __device__ __forceinline__ int ring_tile(int n, int nt, bool& value) {
  const int lead = min(nt, L::LEAD), k = n - lead, pairs = max(0, nt - L::LEAD);   // K ahead; V 0, K lead, V 1, ...; then V alone
  value = k >= 0 && (k >= 2 * pairs || (k & 1) == 0);
  return k < 0 ? n : k >= 2 * pairs ? k - pairs : value ? k / 2 : k / 2 + L::LEAD;
}
template <class L> __device__ __forceinline__ uint32_t place_of_v(int t, int nt) { return t + min(nt, L::LEAD + t); }

// steps of chain i of a piece, and the tile of a step: query tile i over the tiles it sees, or every other tile
template <class L> __device__ __forceinline__ int steps_of(const Shape& s, const Extent& e, const Piece& p, int i) {
  if (L::NARROW) return (p.nt - i + 1) / 2;
  return max(0, min(p.nt, page::tiles_seen(s, e, p.unit * L::UNIT + i * QT, QT) - p.tile0));
}
template <class L> __device__ __forceinline__ int tile_of(int i, int step) { return L::NARROW ? 2 * step + i : step; }

// the first tile of a piece (or one before it) with tokens that some row does not see
__device__ __forceinline__ int first_masked(const Shape& s, const Extent& e, const Piece& p) {
  return page::sees_all_before(s.sight, e, p.unit * s.unit / s.group) / TOK - p.tile0;
}

// A run holds at most one piece that starts inside a unit and one that starts with it and is cut: two places each.  The second launch
// finds the latter in `cut`, with the run that has the unit's last tile.
struct Cut { int b, h, unit, last; };   // last 0: none (a cut unit never ends in the first run)
struct Parts {
  float* o;             // [2 runs][unit rows][D], relative to 2^m
  float2* ml;           // [2 runs][unit rows] m, row sum
  Cut* cut;             // [runs]
};

struct TileCall : PageCall {
  Shape shape;
  int sequences, most_rounds;
};

__device__ __forceinline__ int plan_rounds(const uint8_t* smem) { return *reinterpret_cast<const volatile int*>(smem + M_ROUNDS); }

// ---- warp 11: pages ------------------------------------------------------------------------------------------------
template <int D, int COPIES>
__device__ __forceinline__ void page_role(uint8_t* smem, uint64_t* bars, const CUtensorMap* map_k, const CUtensorMap* map_v, const PageArrays& c,
                                          const TileCall& a, const Plan& plan, const Ctx& ctx, int32_t* status) {
  using L = Layout<D, COPIES>;
  const int lane = threadIdx.x & 31, rows = 1 << c.shift, per_tile = TOK >> c.shift;
  const int groups = rows / 8, nowhere = c.pages * c.kv_heads * groups;   // groups of a page; behind the last one of the pool: read as zeros
  Tour tour(plan, a.shape, blockIdx.x, gridDim.x, plan_rounds(smem));
  Piece p;
  bool ok = true, bad = false;
  Ring at;
  int round = 0;        // times round the ring
  while (ok && tour.next(plan, a.shape, p)) {
    const Extent e = plan.extents[p.b];
    const int total = e.length + e.there;
    const int32_t* const entries = c.table + static_cast<size_t>(p.b) * c.row_pages;
    // lane l knows entry 32 w + l of the table: of K's window, the one before (V lags behind) and the next
    auto window = [&](int w) {
      const int entry = 32 * w + lane;
      return entry < c.row_pages && entry << c.shift < total ? __ldg(entries + entry) : -1;
    };
    int now = p.tile0 * per_tile / 32, before = -1, here = window(now), after = window(now + 1);
    const int masked = first_masked(a.shape, e, p);
    for (int n = 0; n < 2 * p.nt && ok; ++n) {
      bool value;
      const int t = ring_tile<L>(n, p.nt, value);
      const int entry = (p.tile0 + t) * per_tile, w = entry / 32;
      if (w > now) {
        before = here;
        here = after;
        now = w;
        after = window(now + 1);
      }
      const int id = __shfl_sync(0xffffffffu, w == now ? here : before, (entry + lane) & 31);
      const int first = (p.tile0 + t) * TOK, pages = min(per_tile, (total - first + rows - 1) >> c.shift);
      if (round > 0) ok = wait(&bars[FREE + at.stage], at.phase ^ 1, ctx, 930);
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars[FULL + at.stage], static_cast<uint32_t>(pages << c.shift) * D * 2);
        if (value && t >= masked) mbar_arrive(&bars[LOOK + at.stage]);
      }
      __syncwarp();
      if (lane < pages) {
        const bool in = static_cast<unsigned>(id) < static_cast<unsigned>(c.pages);
        bad |= !in;
        tma_load_4d(smem + L::RING_OFF + at.stage * L::STAGE + lane * groups * L::GROUP, value ? map_v : map_k,
                    in ? (id * c.kv_heads + p.h) * groups : nowhere, &bars[FULL + at.stage]);
      }
      __syncwarp();
      at.advance(L::STAGES);
      round += at.stage == 0;
    }
  }
  if (bad) report(status, STATUS_PAGE);
  if (!ok) {   // copies in flight land before the block goes away
    const long long begin = clock64();
    while (clock64() - begin < (1ll << 21)) {}
  }
}

// ---- warps 8-9: queries, and values that rows do not see ---------------------------------------------------------------
template <int DT> __device__ __forceinline__ bool not_finite(uint32_t bits16) {
  constexpr uint32_t E = DT == NKV_BF16 ? 0x7F80u : 0x7C00u;
  return (bits16 & E) == E;
}

// lo + the lower half of two bf16 numbers, hi + the upper one, in fp32
__device__ __forceinline__ void add_bf16x2(float& lo, float& hi, uint32_t two) {
  asm("{\n\t.reg .b16 x, y;\n\t"
      "mov.b32 {x, y}, %2;\n\t"
      "add.rn.f32.bf16 %0, x, %0;\n\t"
      "add.rn.f32.bf16 %1, y, %1;\n\t}"
      : "+f"(lo), "+f"(hi)
      : "r"(two));
}

// 16 bytes from memory to shared memory, or zeros
__device__ __forceinline__ void copy16_async(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

template <int DT, int D, int COPIES>
__device__ __forceinline__ void operand_role(uint8_t* smem, uint64_t* bars, const PageArrays& c, const TileCall& a, const Plan& plan, const Ctx& ctx) {
  using L = Layout<D, COPIES>;
  const int tid = threadIdx.x - 32 * SOFTMAX_WARPS, lane = tid & 31;
  const uint32_t base = smem_u32(smem);
  // queries: a thread has one 16-byte column of every ROWS-th row of the unit
  constexpr int PER_ROW = D / 8, ROWS = 32 * OPERAND_WARPS / PER_ROW, APART = QT / (COPIES > 0 ? COPIES : 1);
  const int q_row = tid / PER_ROW, q_col = tid % PER_ROW * 8;
  const uint32_t q_to = base + L::Q_OFF + (q_col / 64) * SUB;
  const bool negative = a.scale_log2 < 0.f;   // a negative scale is the queries' sign
  const int token_step = ROWS / a.group, head_step = ROWS - token_step * a.group;
  volatile int* const stray = reinterpret_cast<volatile int*>(smem + M_STRAY);
  Tour tour(plan, a.shape, blockIdx.x, gridDim.x, plan_rounds(smem));
  Piece p;
  bool ok = true;
  int pieces = 0;
  uint32_t items = 0, looked = 0;   // tiles in the ring of the pieces before; phases of LOOK, a bit per stage
  while (ok && tour.next(plan, a.shape, p)) {
    const Extent e = plan.extents[p.b];
    const uint16_t* const q_head = a.q + p.b * a.q_batch + static_cast<long long>(p.h) * a.group * a.q_head + q_col;
    if (pieces > 0) ok = wait(&bars[Q_FREE], (pieces - 1) & 1, ctx, 931);
    if (!ok) break;
    // rows of a narrow unit are the same ones every time: behind the last of them zeros stay
    const int rows = !L::NARROW ? L::UNIT : pieces > 0 ? min(APART, a.rows) : APART;
    auto q_place = [&](int row) { return q_to + (row / QT) * L::DCH * SUB + sw128_offset(row % QT, q_col % 64); };
    int r = p.unit * L::UNIT + q_row, token = r / a.group, head = r - token * a.group;
#pragma unroll 4
    for (int row = q_row; row < rows; row += ROWS) {
      const uint16_t* const src = q_head + token * a.q_token + head * a.q_head;
      const bool there = r < a.rows;
#pragma unroll
      for (int copy = 0; copy < (COPIES > 0 ? COPIES : 1); ++copy) {
        const uint32_t to = q_place(row + copy * APART);
        if (a.q_vector) copy16_async(to, there ? src : a.q, there);
        else sts128(to, there ? gather16(src) : make_uint4(0, 0, 0, 0));
      }
      r += ROWS;
      token += token_step;
      head += head_step;
      if (head >= a.group) { head -= a.group; ++token; }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (negative)
      for (int row = q_row; row < rows; row += ROWS)
#pragma unroll 1
        for (int copy = 0; copy < (COPIES > 0 ? COPIES : 1); ++copy) {
          const uint4 v = lds128(q_place(row + copy * APART));
          sts128(q_place(row + copy * APART), make_uint4(v.x ^ 0x80008000u, v.y ^ 0x80008000u, v.z ^ 0x80008000u, v.w ^ 0x80008000u));
        }
    ++pieces;
    fence_proxy_async();
    warp_arrive(&bars[Q_FULL], lane);
    // ---- V tiles with tokens that some row does not see: two tokens a thread.  LOOK tells that a stage waits for such a tile: a
    // wait for FULL alone, by warps that skip all other tiles, could not tell this phase of it from an earlier one.
    const int total = e.length + e.there;
    for (int t = max(0, first_masked(a.shape, e, p)); t < p.nt; ++t) {
      const uint32_t item = items + place_of_v<L>(t, p.nt), stage = item % L::STAGES;
      ok = wait(&bars[LOOK + stage], (looked >> stage) & 1, ctx, 932) && wait(&bars[FULL + stage], (item / L::STAGES) & 1, ctx, 942);
      if (!ok) break;
      looked ^= 1u << stage;
#pragma unroll 1
      for (int row = tid; row < TOK; row += 32 * OPERAND_WARPS) {
        const bool behind = (p.tile0 + t) * TOK + row >= total;
        const uint32_t first = base + L::RING_OFF + stage * L::STAGE + (row / 8) * L::GROUP + (row & 7) * 128;
#pragma unroll 4
        for (int k = 0; k < L::DCH * 8; ++k) {
          const uint32_t place = first + (k / 8) * 1024 + (((k & 7) ^ (row & 7)) << 4);   // (lanes of a row group take different banks)
          if (behind) {
            sts128(place, make_uint4(0, 0, 0, 0));
            continue;
          }
          const uint4 v = lds128(place);
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          bool found = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool lo = not_finite<DT>(w[i]), hi = not_finite<DT>(w[i] >> 16);
            found |= lo || hi;
            w[i] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
          }
          if (found) {
            sts128(place, make_uint4(w[0], w[1], w[2], w[3]));
            *stray = 1;
          }
        }
      }
      fence_proxy_async();
      warp_arrive(&bars[CLEAN + stage], lane);
    }
    items += 2 * p.nt;
  }
  // ---- rows of units without tiles: they see nothing
  const int units = a.shape.units, heads = a.shape.kv_heads;
  for (int i = blockIdx.x; i < a.sequences * units * heads; i += gridDim.x) {
    const int h = i % heads, u = i / heads % units, b = i / heads / units, r0 = u * L::UNIT, rows = min(L::UNIT, a.rows - r0);
    if (page::tiles_seen(a.shape, plan.extents[b], r0, L::UNIT) > 0) continue;
    for (int k = tid; k < rows * PER_ROW; k += 32 * OPERAND_WARPS) {
      const int r = r0 + k / PER_ROW, col = k % PER_ROW * 8, token = r / a.group;
      const size_t at = (static_cast<size_t>(b) * a.tokens + token) * a.heads + h * a.group + r - token * a.group;
      *reinterpret_cast<uint4*>(a.out + at * D + col) = make_uint4(0, 0, 0, 0);
      if (col == 0) a.lse[at] = -INFINITY;
    }
  }
}

// ---- warp 10: MMA issue -----------------------------------------------------------------------------------------
// Descriptor of a K tile (K-major) or, read along its rows, of a V tile (MN-major; `leading`: from one chunk of 64 columns to the next, in
// 16 bytes): groups of eight rows `group` bytes apart, 128-byte swizzle.
__device__ __forceinline__ uint64_t tile_desc(uint32_t smem_addr, uint32_t leading, uint32_t group) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFF) | (static_cast<uint64_t>(leading) << 16) | (static_cast<uint64_t>(group / 16) << 32) |
         (1ull << 46) | (2ull << 61);
}

template <int DT, int D, int COPIES>
__device__ __forceinline__ void mma_role(uint8_t* smem, uint64_t* bars, uint32_t tmem, const TileCall& a, const Plan& plan, const Ctx& ctx) {
  using L = Layout<D, COPIES>;
  constexpr int DCH = L::DCH;
  const bool leader = elect_one();   // the whole warp runs the (uniform) control flow; one elected lane issues
  const uint32_t base = smem_u32(smem);
  const uint64_t q_desc = make_smem_desc_sw128(base + L::Q_OFF);
  const uint64_t k_desc = tile_desc(base + L::RING_OFF, 1, L::GROUP), v_desc = tile_desc(base + L::RING_OFF, 1024 / 16, L::GROUP);
  auto issue_s = [&](int i, uint32_t stage) {
    const uint64_t qd = q_desc + (L::NARROW ? 0u : static_cast<uint32_t>(i * (DCH * SUB / 16))), kd = k_desc + stage * static_cast<uint32_t>(L::STAGE / 16);
    const uint32_t d = tmem + i * 128;
#pragma unroll
    for (int ch = 0; ch < DCH; ++ch)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (leader) mma_bf16(d, qd + ch * (SUB / 16) + 2 * k, kd + ch * (1024 / 16) + 2 * k, idesc<DT>(TOK), ch + k > 0);
    if (leader) mma_commit(&bars[S_FULL + i]);
  };
  // weights of half a tile's tokens times V of them: V's rows are tokens, its columns the result's
  auto issue_pv = [&](int i, uint32_t stage, int half, bool accumulate) {
    const uint64_t vd = v_desc + stage * static_cast<uint32_t>(L::STAGE / 16) + half * static_cast<uint32_t>(8 * L::GROUP / 16);
    const uint32_t d = tmem + 256 + i * 128, w = tmem + i * 128 + half * 32;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (leader) mma_bf16_ts(d, w + 8 * k, vd + k * (2 * L::GROUP / 16), idesc<DT>(D) | (1u << 16), accumulate || k > 0);
  };
  Tour tour(plan, a.shape, blockIdx.x, gridDim.x, plan_rounds(smem));
  Piece p;
  bool ok = true;
  Ring at;                                         // tiles are used in the order in which they lie in the ring
  uint32_t cleaned = 0;                            // phases of CLEAN, a bit per stage
  int pieces = 0, done[2] = {0, 0}, used[2] = {0, 0};   // steps and pieces of each chain so far
  while (ok && tour.next(plan, a.shape, p)) {
    const Extent e = plan.extents[p.b];
    const int n[2] = {steps_of<L>(a.shape, e, p, 0), steps_of<L>(a.shape, e, p, 1)};
    const int longest = max(n[0], n[1]), masked = first_masked(a.shape, e, p);   // V tiles from here on are looked at
    ok = wait(&bars[Q_FULL], pieces & 1, ctx, 933);
    ++pieces;
    // the first and the last chain to use a tile: each stage is waited for once and given back once
    auto is_first = [&](int i, int step) { return L::NARROW || i == (step < n[0] ? 0 : 1); };
    auto is_last = [&](int i, int step) { return L::NARROW || i == (step < n[1] ? 1 : 0); };
    uint32_t k_stage = 0, v_stage = 0;
#pragma unroll 1
    for (int j = 0; j <= longest && ok; ++j) {
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int steps = i ? n[1] : n[0];
        if (j > 0 && j - 1 < steps) {
          const uint32_t phase = ((i ? done[1] : done[0]) + j - 1) & 1;
          if (is_first(i, j - 1)) {
            v_stage = at.stage;
            if (tile_of<L>(i, j - 1) >= masked) {
              ok = wait(&bars[CLEAN + v_stage], (cleaned >> v_stage) & 1, ctx, 934);
              cleaned ^= 1u << v_stage;
            } else {
              ok = wait(&bars[FULL + v_stage], at.phase, ctx, 935);
            }
            at.advance(L::STAGES);
          }
          if (j == 1) {   // the first PV of a piece overwrites O: the rows of the piece before must have been read
            const int before = i ? used[1] : used[0];
            if (ok && before > 0) ok = wait(&bars[O_FREE + i], (before - 1) & 1, ctx, 936);
          }
          ok = ok && wait(&bars[P_READY + 2 * i], phase, ctx, 937);
          if (!ok) break;
          tc_fence_after();
          issue_pv(i, v_stage, 0, j > 1);
          if (COPIES <= 1) {
            ok = wait(&bars[P_READY + 2 * i + 1], phase, ctx, 938);
            if (!ok) break;
            tc_fence_after();
          }
          issue_pv(i, v_stage, 1, true);
          if (j == steps && leader) mma_commit(&bars[O_DONE + i]);
          if (is_last(i, j - 1) && leader) mma_commit(&bars[FREE + v_stage]);
        }
        if (j < steps) {
          // S of the next step overwrites P of this one, right behind the PV that reads it: the tensor core executes one
          // thread's MMAs in order
          if (is_first(i, j)) {
            k_stage = at.stage;
            ok = wait(&bars[FULL + k_stage], at.phase, ctx, 939);
            if (!ok) break;
            at.advance(L::STAGES);
            tc_fence_after();
          }
          issue_s(i, k_stage);
          if (is_last(i, j) && leader) mma_commit(&bars[FREE + k_stage]);
        }
      }
    }
    if (!ok) break;
    if (leader) mma_commit(&bars[Q_FREE]);
    for (int i = 0; i < 2; ++i) {
      done[i] += n[i];
      used[i] += n[i] > 0 ? 1 : 0;
    }
  }
  if (!ok) {   // MMAs in flight end before tensor memory is given back (nobody looks at how: the launch has given up)
    if (leader) mma_commit(&bars[DRAINED]);
#pragma unroll 1
    for (int i = 0; i < MOST_PARKED && !mbar_try_wait_parked(&bars[DRAINED], 0, 1000u); ++i) {}
  }
  __syncwarp();
}

// ---- warps 0-7: softmax -------------------------------------------------------------------------------------------

// Values of column `col` that are not finite, of the tokens of a piece that were looked at and that query t sees.
template <int DT>
__device__ __noinline__ float strays(const PageArrays& c, const TileCall& a, Extent e, Piece p, int t, int col, int d) {
  float sum = 0.f;
  if (t >= e.count) return sum;
  const int total = e.length + e.there, from = (p.tile0 + max(0, first_masked(a.shape, e, p))) * TOK, to = min((p.tile0 + p.nt) * TOK, total);
  for (int first = from; first < to; first += 32) {
    const uint32_t sees = sight_of(a, e, p.b, t, first);
    for (int i = 0; i < 32 && first + i < to; ++i) {
      if (!(sees >> i & 1)) continue;
      const int at = page_of(c, p.b, first + i);
      if (at < 0) continue;
      const uint16_t bits = c.v[row_at(c, at, p.h, first + i, d) + col];
      if (not_finite<DT>(bits)) sum += load_float(&bits, DT, 0);
    }
  }
  return sum;
}

// barrier of the softmax warps; whether any of them passes `fails`
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool softmax_any(bool fails) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(fails))
      : "memory");
  return any != 0;
}

template <int DT, int D, int COPIES>
__device__ __forceinline__ void softmax_role(uint8_t* smem, uint64_t* bars, uint32_t tmem, const PageArrays& c, const TileCall& a, const Plan& plan,
                                             const Parts& parts, const Ctx& ctx) {
  using L = Layout<D, COPIES>;
  constexpr int WIDTH = TOK / SLICES<DT, COPIES>, GROUPS = WIDTH / 32, SOURCES = 2 * (COPIES > 0 ? COPIES : 1), APART = 2 * QT / SOURCES;
  constexpr bool TWO = PARTS<DT, COPIES> == 2, CUT = DT == NKV_BF16 && !TWO;   // CUT: O is divided by the sum of the weights as they are stored
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const int wg = warp / 4, row = tid & 127;
  const int slice = COPIES > 1 ? row / APART % SLICES<DT, COPIES> : 0;   // (the same in all of a warp, as is whether it takes the rest)
  const bool rest = TWO && row / APART >= SLICES<DT, COPIES>;
  const uint32_t s_addr = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + wg * 128, o_addr = s_addr + 256;
  const float scale = fabsf(a.scale_log2);
  volatile int* const stray = reinterpret_cast<volatile int*>(smem + M_STRAY);
  float* const join = reinterpret_cast<float*>(smem + L::JOIN_OFF);
  Tour tour(plan, a.shape, blockIdx.x, gridDim.x, plan_rounds(smem));
  Piece p = {};
  bool ok = true, more = true;
  int ci = 0, pieces = 0;   // steps and pieces of this chain
  int odd = 0;
  if (tid == 0)
    for (int run = blockIdx.x; run < static_cast<int>(gridDim.x) * a.most_rounds; run += gridDim.x) parts.cut[run] = Cut{0, 0, 0, 0};
  auto note_cut = [&]() {   // (the last piece of a run, where there is one)
    if (tid == 0 && !p.whole && p.tile0 == 0) parts.cut[tour.run] = Cut{p.b, p.h, p.unit, tour.last_run(plan)};
  };
  const bool wide_out = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0, wide_part = (reinterpret_cast<uintptr_t>(parts.o) & 31) == 0;
  auto place_of = [&](const Piece& pc) { return (2 * static_cast<size_t>(tour.run) + (pc.tile0 == 0 ? 1 : 0)) * L::UNIT; };
  // the row of the results that row r of a piece's kv head is
  auto at_of = [&](const Piece& pc, int r) {
    const int token = r / a.group;
    return (static_cast<size_t>(pc.b) * a.tokens + token) * a.heads + pc.h * a.group + r - token * a.group;
  };
  while (ok && (more = tour.next(plan, a.shape, p))) {
    const Extent e = plan.extents[p.b];
    const int r = L::NARROW ? row % APART : p.unit * L::UNIT + wg * QT + row, token = r / a.group;
    const bool real = r < a.rows;
    const int clear = real ? page::sees_all_before(a.sight, e, token) : 0x7FFFFFFF;   // (rows of nobody are not masked)
    const int clear_least = __reduce_min_sync(0xffffffffu, clear);
    const int steps = steps_of<L>(a.shape, e, p, wg);
    // where P' stands when the reference is set: see the top of the file
    const float raise = DT == NKV_F16 ? 7.0f : -(RESCALE_THRESHOLD + 32 - __clz(e.length + e.there));
    float m = NOTHING, l = 0.f, stored = 0.f;   // (stored: CUT)
#pragma unroll 1
    for (int n = 0; n < steps; ++n, ++ci) {
      const int first = (p.tile0 + tile_of<L>(wg, n)) * TOK + slice * WIDTH;
      ok = wait(&bars[S_FULL + wg], ci & 1, ctx, 940);
      if (!ok) break;
      tc_fence_after();
      uint32_t raw[GROUPS][32];
#pragma unroll
      for (int k = 0; k < GROUPS; ++k) tmem_ld32_issue(s_addr + slice * WIDTH + 32 * k, raw[k]);
      if constexpr (GROUPS == 4) {
        tmem_ld128_wait(raw[0], raw[1], raw[2], raw[3]);
      } else {
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) tmem_ld32_wait(raw[k]);
      }
      float f = scale;
      if (first + WIDTH > clear_least) {   // some row of the warp does not see all of it
        // scaled before they are masked: -inf times a scale of 0 would be NaN
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
          const uint32_t sees = !real ? 0xFFFFFFFFu : token < e.count ? sight_of(a, e, p.b, token, first + 32 * k) : 0u;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            raw[k][j] = sees >> j & 1 ? __float_as_uint(__uint_as_float(raw[k][j]) * f) : 0xFF800000u;
        }
        f = 1.f;
      }
      float top = max32(raw[0]);
#pragma unroll
      for (int k = 1; k < GROUPS; ++k) top = fmaxf(top, max32(raw[k]));
      top *= f;
      if (__any_sync(0xffffffffu, top - m > raise + RESCALE_THRESHOLD)) {
        // Move the reference: O and the sum are scaled by 2^(old - new).  S was issued behind PV of the step before and its commit
        // covers both.
        const float m_new = fmaxf(m, top - raise), alpha = exp2f(m - m_new);
        if (n > 0) {
#pragma unroll 1
          for (int cc = 0; cc < D / 16; ++cc) {
            uint32_t v[16];
            tmem_ld16(o_addr + cc * 16, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
            tmem_st16(o_addr + cc * 16, v);
          }
          tmem_wait_st();
        }
        l *= alpha;
        stored *= alpha;
        m = m_new;
      }
      // P' replaces S, eight scores at a time in a software pipeline: exponentials of one block beside the arguments of the next and the
      // sums and stores of the one before.  The first half of the weights is handed over as soon as it is stored.
      const uint64_t scale2 = pair_f32(f, f), off2 = pair_f32(-m, -m);
      uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull}, arg[2][4];
      float w[2][8];
      float held[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      uint32_t packed[16];
      auto args = [&](int b) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          arg[b & 1][i] = fma_f32x2(pair_bits(raw[b / 4][(b & 3) * 8 + 2 * i], raw[b / 4][(b & 3) * 8 + 2 * i + 1]), scale2, off2);
      };
      auto exps = [&](int b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x, y;
          split_f32(arg[b & 1][i], x, y);
          w[b & 1][2 * i] = exp2_fast(x);
          w[b & 1][2 * i + 1] = exp2_fast(y);
        }
      };
      auto finish = [&](int b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = w[b & 1][2 * i], y = w[b & 1][2 * i + 1];
          sum2[i] = add_f32x2(sum2[i], pair_f32(x, y));
          if (DT == NKV_F16) {
            packed[(b & 3) * 4 + i] = pack2<DT>(x, y);
          } else {
            uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
            if (rest) {
              xb = __float_as_uint(x - __uint_as_float(xb & 0xFFFF0000u));
              yb = __float_as_uint(y - __uint_as_float(yb & 0xFFFF0000u));
            }
            packed[(b & 3) * 4 + i] = __byte_perm(xb, yb, 0x7632);
            if (CUT) add_bf16x2(held[2 * i], held[2 * i + 1], packed[(b & 3) * 4 + i]);
          }
        }
        if ((b & 3) == 3) {
          tmem_st16(s_addr + slice * (WIDTH / 2) + b / 4 * 16, packed);
          if (COPIES <= 1 && b == 7) {
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(&bars[P_READY + 2 * wg], lane);
          }
        }
      };
      args(0);
#pragma unroll
      for (int b = 0; b < 4 * GROUPS; ++b) {
        exps(b);
        if (b + 1 < 4 * GROUPS) args(b + 1);
        if (b >= 1) finish(b - 1);
      }
      finish(4 * GROUPS - 1);
      if (COPIES > 1) {   // the other copies' tokens
        constexpr uint32_t zeros[16] = {};
#pragma unroll
        for (int k = GROUPS; k < 4; ++k) tmem_st16(s_addr + ((slice * GROUPS + k) & 3) * 16, zeros);
      }
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&bars[P_READY + 2 * wg + (COPIES <= 1 ? 1 : 0)], lane);
      float x, y;
      split_f32(add_f32x2(add_f32x2(sum2[0], sum2[1]), add_f32x2(sum2[2], sum2[3])), x, y);
      l += x + y;
      if (CUT) stored += ((held[0] + held[1]) + (held[2] + held[3])) + ((held[4] + held[5]) + (held[6] + held[7]));
    }
    const float raised = CUT && l != 0.f ? l / stored : 1.f;   // what O is short of by its weights' cut-off bits
    if (rest) l = 0.f;   // (the other part's)
    if (ok && steps > 0) {
      ok = wait(&bars[O_DONE + wg], pieces & 1, ctx, 941);
      ++pieces;
    }
    // ---- the rows: results, or a part of them
    note_cut();
    if (L::NARROW) {
      // (places in turn: a warp may still read those of the piece before, not of the one before that)
      float2* const mls = reinterpret_cast<float2*>(smem + L::ML_OFF) + odd * 256;
      odd ^= 1;
      mls[tid] = make_float2(m, l);
      float* const raises = join + (mls - reinterpret_cast<float2*>(smem + L::ML_OFF));
      if (CUT) raises[tid] = raised;
      tc_fence_before();
      if (softmax_any(!ok)) {   // (all of the warps take part in what follows, or none)
        ok = false;
        break;
      }
      tc_fence_after();
      // A row has the same lane of tensor memory in both chains: a thread takes both, of half the columns.
      const bool second = p.nt > 1;      // chain 1 had steps
      float top = NOTHING, sum = 0.f;
#pragma unroll
      for (int k = 0; k < SOURCES; ++k) top = fmaxf(top, mls[k * APART + row % APART].x);
#pragma unroll
      for (int k = 0; k < SOURCES; ++k) sum = fmaf(mls[k * APART + row % APART].y, exp2f(mls[k * APART + row % APART].x - top), sum);
      const bool any = sum != 0.f, look = *stray != 0;      // (NaN: any)
      const float inv = p.whole ? 1.f / sum : 1.f, f0 = exp2f(mls[row].x - top) * inv * (CUT ? raises[row] : 1.f),
                  f1 = exp2f(mls[128 + row].x - top) * inv * (CUT ? raises[128 + row] : 1.f);
      const uint32_t o0 = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + 256 + wg * (D / 2);
      // 16 columns of the row: both chains' together
      auto joined = [&](int at, float (&x)[16]) {
        uint32_t u[16], v[16];
        tmem_ld16_issue(o0 + at, u);
        if (second) tmem_ld16_issue(o0 + 128 + at, v);
        tmem_ld16_wait(u);
        if (second) tmem_ld16_wait(v);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          x[j] = __uint_as_float(u[j]) * f0;
          if (second) x[j] = fmaf(__uint_as_float(v[j]), f1, x[j]);
          if (!any) x[j] = 0.f;
        }
      };
      const size_t row_at = at_of(p, r);
      auto put = [&](int col, const float (&x)[16], size_t to, size_t part) {   // 16 columns of a row
        if (p.whole) {
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = pack2<DT>(x[2 * i], x[2 * i + 1]);
          store32(a.out + to * D + col, o, wide_out);
        } else {
#pragma unroll
          for (int j = 0; j < 16; j += 8) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(x[j + i]);
            store32(parts.o + part * D + col + j, o, wide_part);
          }
        }
      };
      auto add_strays = [&](int t, int col, float (&x)[16]) {
#pragma unroll 1
        for (int j = 0; j < 16; ++j) {
          const float y = strays<DT>(c, a, e, p, t, col + j, D);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i == j) x[i] += y;
        }
      };
      if (COPIES <= 1) {
#pragma unroll 1
        for (int cc = 0; cc < D / 2; cc += 16) {
          float x[16];
          joined(cc, x);
          if (!real) continue;
          const int col = wg * (D / 2) + cc;
          if (look) add_strays(token, col, x);
          put(col, x, row_at, place_of(p) + r);
        }
      } else {
        // The copies of a row are other warps': through shared memory, as many columns at a time as there is room for, a row of them
        // and four words apart.  Results are fetched 16 columns a thread.
        int bits = D == 128 ? 6 : 5;
        while (SOURCES * a.rows * ((1 << bits) + 4) > L::JOIN_WORDS) --bits;
        const int columns = 1 << bits, stride = columns + 4, here = row >> (bits - 4), col = (row & (columns / 16 - 1)) * 16;
        float* const ours = join + wg * (SOURCES / 2) * a.rows * stride;
#pragma unroll 1
        for (int c0 = 0; c0 < D / 2; c0 += columns) {
#pragma unroll 1
          for (int cc = 0; cc < columns; cc += 16) {
            float x[16];
            joined(c0 + cc, x);
            float* const to = ours + (row / APART * a.rows + r) * stride + cc;
            if (real)
#pragma unroll
              for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(to + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
          }
          softmax_sync();
#pragma unroll 1
          for (int from = here; from < a.rows; from += 2048 >> bits) {
            float x[16];
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
              const float* const at = ours + from * stride + col + j;
              float4 y = *reinterpret_cast<const float4*>(at);
#pragma unroll
              for (int k = 1; k < SOURCES / 2; ++k) {
                const float4 z = *reinterpret_cast<const float4*>(at + k * a.rows * stride);
                y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
              }
              x[j] = y.x;
              x[j + 1] = y.y;
              x[j + 2] = y.z;
              x[j + 3] = y.w;
            }
            const int first = wg * (D / 2) + c0 + col;
            if (look) add_strays(from / a.group, first, x);
            put(first, x, at_of(p, from), place_of(p) + from);
          }
          if (c0 + columns < D / 2) softmax_sync();
        }
      }
      if (tid < APART && real) {
        if (p.whole) a.lse[row_at] = any ? (top + log2f(sum)) * LN2 : -INFINITY;
        else parts.ml[place_of(p) + r] = make_float2(top, sum);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars[O_FREE]);
        if (second) mbar_arrive(&bars[O_FREE + 1]);
      }
    } else {
      if (!ok) break;
      tc_fence_after();
      const float inv = raised / l;
      const bool any = l != 0.f, look = *stray != 0;
      float* const part = parts.o + (place_of(p) + wg * QT + row) * D;
      const size_t at = at_of(p, r);
      uint16_t* const out = a.out + at * D;
#pragma unroll 1
      for (int cc = 0; cc < D; cc += 32) {
        uint32_t v[32];
        if (steps > 0) {
          tmem_ld32_issue(o_addr + cc, v);
          tmem_ld32_wait(v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0u;
        }
        if (!real) continue;
        if (look) {
#pragma unroll 1
          for (int j = 0; j < 32; ++j) {
            const float x = strays<DT>(c, a, e, p, token, cc + j, D);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i == j) v[i] = __float_as_uint(__uint_as_float(v[i]) + x);
          }
        }
        if (p.whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 16) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              o[i] = any ? pack2<DT>(__uint_as_float(v[j + 2 * i]) * inv, __uint_as_float(v[j + 2 * i + 1]) * inv) : 0u;
            store32(out + cc + j, o, wide_out);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(__uint_as_float(v[j + i]) * raised);
            store32(part + cc + j, o, wide_part);
          }
        }
      }
      if (real) {
        if (p.whole) a.lse[at] = any ? (m + log2f(l)) * LN2 : -INFINITY;
        else parts.ml[place_of(p) + wg * QT + row] = make_float2(m, l);
      }
      if (steps > 0) {
        tc_fence_before();
        warp_arrive(&bars[O_FREE + wg], lane);
      }
    }
  }
  // a launch that gave up: NaN for the piece it stopped in and all later ones
  if (!ok) {
    while (more) {
      const int r = L::NARROW ? tid : p.unit * L::UNIT + tid;
      if (r < a.rows && tid < L::UNIT) {
        if (p.whole) a.lse[at_of(p, r)] = CUDART_NAN_F;
        else parts.ml[place_of(p) + tid] = make_float2(0.f, CUDART_NAN_F);
      }
      note_cut();
      more = tour.next(plan, a.shape, p);
    }
  }
}

template <int DT, int D, int COPIES>
__global__ void __launch_bounds__(THREADS, 1)
page_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PageArrays c,
                 const __grid_constant__ TileCall a, Parts parts, int32_t* status) {
  using L = Layout<D, COPIES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + M_SLOT);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + M_ABORT);
  page::Extent* const extents = reinterpret_cast<page::Extent*>(smem + M_EXTENTS);
  uint32_t* const start = reinterpret_cast<uint32_t*>(smem + M_START);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&bars[Q_FULL], OPERAND_WARPS);
    mbar_init(&bars[Q_FREE], 1);
    mbar_init(&bars[DRAINED], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[S_FULL + i], 1);
      mbar_init(&bars[O_DONE + i], 1);
      mbar_init(&bars[O_FREE + i], L::NARROW ? SOFTMAX_WARPS : QT / 32);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bars[P_READY + i], QT / 32);
    for (int i = 0; i < L::STAGES; ++i) {
      mbar_init(&bars[FULL + i], 1);
      mbar_init(&bars[FREE + i], 1);
      mbar_init(&bars[LOOK + i], 1);
      mbar_init(&bars[CLEAN + i], OPERAND_WARPS);
    }
    *abort_flag = 0;
    *reinterpret_cast<volatile int*>(smem + M_STRAY) = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  // ---- the plan.  Few units a sequence: one warp makes it, ahead of the barrier that the others need anyway.
  if (warp == MMA_WARP) tmem_alloc(tmem_slot, 512);
  if (warp > MMA_WARP && lane == 0) {
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  const bool one_warp = a.shape.units <= 4;
  if (!one_warp) {
    if (tid < a.sequences) {
      bool bad;
      extents[tid] = extent_of(c, a.counts, a.tokens, tid, bad);
      if (bad) report(status, STATUS_PAGE);
      start[tid] = 0;
    }
    __syncthreads();
    for (int i = tid; i < a.sequences * a.shape.units; i += THREADS) {
      const int b = i / a.shape.units, u = i % a.shape.units;
      const uint32_t cost = page::cost_of(page::tiles_seen(a.shape, extents[b], u * L::UNIT, L::UNIT));
      if (cost) atomicAdd(&start[b], cost);
    }
    __syncthreads();
  }
  if (warp == 0) {
    uint32_t carry = 0, units = 0;
    uint64_t tokens = 0;
    for (int b0 = 0; b0 <= a.sequences; b0 += 32) {
      const int b = b0 + lane;
      uint32_t cost = 0;
      if (b < a.sequences) {
        if (one_warp) {
          bool bad;
          const Extent e = extent_of(c, a.counts, a.tokens, b, bad);
          if (bad) report(status, STATUS_PAGE);
          extents[b] = e;
          for (int u = 0; u < a.shape.units; ++u) cost += page::cost_of(page::tiles_seen(a.shape, e, u * L::UNIT, L::UNIT));
        } else {
          cost = start[b];
        }
        cost *= a.shape.kv_heads;
        if (cost) {
          tokens += extents[b].length + extents[b].there;
          units += a.shape.units * a.shape.kv_heads;
        }
      }
      uint32_t upto = cost;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const uint32_t other = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += other;
      }
      if (b <= a.sequences) start[b] = carry + upto - cost;
      carry += __shfl_sync(0xffffffffu, upto, 31);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) tokens += __shfl_xor_sync(0xffffffffu, tokens, x);
    units = __reduce_add_sync(0xffffffffu, units);
    if (lane == 0)
      *reinterpret_cast<volatile int*>(smem + M_ROUNDS) =
          page::rounds_for(tokens * (4ull * D * a.shape.kv_heads), carry, max(units, 1u), gridDim.x, LEAST_RUN, a.most_rounds);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Ctx ctx{abort_flag};
  Plan plan;
  plan.start = start;
  plan.extents = extents;
  plan.sequences = a.sequences;
  plan.deal(gridDim.x * plan_rounds(smem));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // registers: 12 warps of 168 at launch, 8 of 200 and 4 of 104 from here on
  if (warp < SOFTMAX_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    softmax_role<DT, D, COPIES>(smem, bars, tmem, c, a, plan, parts, ctx);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp < SOFTMAX_WARPS + OPERAND_WARPS) operand_role<DT, D, COPIES>(smem, bars, c, a, plan, ctx);
    else if (warp > MMA_WARP) page_role<D, COPIES>(smem, bars, &map_k, &map_v, c, a, plan, ctx, status);
    else mma_role<DT, D, COPIES>(smem, bars, tmem, a, plan, ctx);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
  if (tid == 0 && *abort_flag) atomicCAS(status, 0, *abort_flag);
}

// Joins the parts of cut units: a thread block per run in which a cut unit begins, and SLICE rows of the unit.
constexpr int SLICE = 16;
template <int DT, int D>
__global__ void __launch_bounds__(256)
join_parts_kernel(TileCall a, Parts parts) {
  __shared__ float shared[256][11];   // (rows of an odd number of words: no two of a warp's in one bank)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Shape& s = a.shape;
  const int r0 = blockIdx.x, row0 = blockIdx.y * SLICE;
  const int4 cut = __ldcg(reinterpret_cast<const int4*>(parts.cut) + r0);
  const int b = cut.x, h = cut.y, unit = cut.z, r1 = cut.w, rows = min(SLICE, min(s.unit, a.rows - unit * s.unit) - row0);
  if (r1 == 0 || rows <= 0) return;
  // a thread per row, 16 bytes of it and share of the parts: with few rows the threads that rows do not need share a row's parts
  constexpr int PER_ROW = D / 8, ROWS = 256 / PER_ROW;
  int shares = 1;
  while (shares * 2 * rows <= ROWS) shares *= 2;
  const int col = (threadIdx.x % PER_ROW) * 8, share = threadIdx.x / PER_ROW & (shares - 1);
  for (int i = threadIdx.x / PER_ROW / shares; i < (rows + ROWS / shares - 1) / (ROWS / shares) * (ROWS / shares); i += ROWS / shares) {
    const int row = row0 + i, r = unit * s.unit + row, token = r / a.group;
    float top = NOTHING, sum = 0.f, acc[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
    if (i < rows) {
#pragma unroll 4
      for (int run = r0 + share; run <= r1; run += shares) {
        // the run the unit starts in has it as a piece that starts with the unit, the others as one that starts inside
        const size_t place = (2 * static_cast<size_t>(run) + (run == r0 ? 1 : 0)) * s.unit + row;
        const float2 ml = __ldcg(&parts.ml[place]);
        const float4 lo = __ldcg(reinterpret_cast<const float4*>(parts.o + place * D + col));
        const float4 hi = __ldcg(reinterpret_cast<const float4*>(parts.o + place * D + col + 4));
        const float part[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        const float next = fmaxf(top, ml.x), old = exp2f(top - next), now = exp2f(ml.x - next);
        top = next;
        sum = fmaf(ml.y, now, sum * old);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] = fmaf(part[k], now, acc[k] * old);
      }
    }
    if (shares > 1) {   // (one round: rows <= ROWS / shares)
      float* const mine = shared[threadIdx.x];
      mine[0] = top;
      mine[1] = sum;
#pragma unroll
      for (int k = 0; k < 8; ++k) mine[2 + k] = acc[k];
      __syncthreads();
      if (share > 0) return;
      for (int k = 1; k < shares; ++k) {
        const float* const other = shared[threadIdx.x + k * PER_ROW];
        const float next = fmaxf(top, other[0]), old = exp2f(top - next), now = exp2f(other[0] - next);
        top = next;
        sum = fmaf(other[1], now, sum * old);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = fmaf(other[2 + j], now, acc[j] * old);
      }
    }
    if (i >= rows) continue;
    const bool any = sum != 0.f;
    const float inv = any ? 1.f / sum : 0.f;
    const size_t at = (static_cast<size_t>(b) * a.tokens + token) * a.heads + h * a.group + r - token * a.group;
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = any ? pack2<DT>(acc[2 * k] * inv, acc[2 * k + 1] * inv) : 0u;
    *reinterpret_cast<uint4*>(a.out + at * D + col) = make_uint4(o[0], o[1], o[2], o[3]);
    if (col == 0) a.lse[at] = any ? (top + log2f(sum)) * LN2 : -INFINITY;
  }
}

int unit_of(int rows) { return rows > QT ? 2 * QT : QT; }
// Units of a kv head that share its keys and values, in more of the pool than a round is to read.
int most_rounds_of(const PageArrays& c, int n, int rows, int d) {
  const uint64_t tokens = min(static_cast<uint64_t>(c.pages), static_cast<uint64_t>(c.row_pages) * n) << c.shift, bytes = tokens * c.kv_heads * 4 * d;
  return rows > unit_of(rows) ? static_cast<int>(min((bytes + page::FITS - 1) / page::FITS, static_cast<uint64_t>(MOST_ROUNDS))) : 1;
}

}  // namespace

size_t page_tile_bytes(const PageArrays& c, int n, int rows, int d) {
  return static_cast<size_t>(sm_count()) * most_rounds_of(c, n, rows, d) * (2 * unit_of(rows) * (d * sizeof(float) + sizeof(float2)) + sizeof(Cut));
}

int page_tile(const PageArrays& c, const PageCall& call, int n, int dtype, int d, void* workspace, int32_t* status, cudaStream_t stream) {
  TileCall a;
  static_cast<PageCall&>(a) = call;
  const int unit = unit_of(a.rows);
  a.sequences = n;
  a.shape = Shape{a.sight, a.group, a.rows, unit, ceil_div(a.rows, unit), c.kv_heads};
  // places of the list are counted in 32 bits
  const uint64_t tiles = (static_cast<uint64_t>(c.row_pages) << c.shift) / TOK + 1 + page::PIECE_TILES, most = tiles * a.shape.units * c.kv_heads * n;
  NKV_REQUIRE(most <= UINT32_MAX, NKV_ERR_TOO_LARGE, "page_attend: up to %llu tiles of %d x %d tokens are more than 32 bits count",
              static_cast<unsigned long long>(most), unit, TOK);
  const int runs = static_cast<int>(min(most, static_cast<uint64_t>(sm_count())));
  Parts parts;
  parts.o = static_cast<float*>(workspace);
  a.most_rounds = most_rounds_of(c, n, a.rows, d);
  const size_t places = static_cast<size_t>(sm_count()) * a.most_rounds * 2 * unit;
  parts.ml = reinterpret_cast<float2*>(parts.o + places * d);
  parts.cut = reinterpret_cast<Cut*>(parts.ml + places);
  CUtensorMap maps[2];
  for (int i = 0; i < 2; ++i) {
    // elements of a chunk, rows of a group, chunks of a row, groups
    const uint64_t dims[4] = {64, 8, static_cast<uint64_t>(d) / 64, (static_cast<uint64_t>(c.pages) * c.kv_heads << c.shift) / 8};
    const uint64_t strides[3] = {static_cast<uint64_t>(d) * 2, 128, static_cast<uint64_t>(d) * 16};
    const uint32_t box[4] = {64, 8, static_cast<uint32_t>(d) / 64, (1u << c.shift) / 8};
    const int rc = encode_tensor_map(&maps[i], 2, i ? c.v : c.k, 4, dims, strides, box, 128);
    if (rc != NKV_OK) return rc;
  }
  auto run = [&](auto kernel, int smem) {
    NKV_CUDA(allow_shared(reinterpret_cast<const void*>(kernel), smem));
    kernel<<<runs, THREADS, smem, stream>>>(maps[0], maps[1], c, a, parts, status);
    NKV_CUDA(cudaGetLastError());
    return NKV_OK;
  };
  int rc = NKV_OK;
#define NKV_PAGE_RUN(COPIES)                                                                                                             \
  rc = d == 128 ? (dtype == NKV_BF16 ? run(page_tile_kernel<NKV_BF16, 128, COPIES>, Layout<128, COPIES>::DYNAMIC)                         \
                                     : run(page_tile_kernel<NKV_F16, 128, COPIES>, Layout<128, COPIES>::DYNAMIC))                         \
                : (dtype == NKV_BF16 ? run(page_tile_kernel<NKV_BF16, 64, COPIES>, Layout<64, COPIES>::DYNAMIC)                           \
                                     : run(page_tile_kernel<NKV_F16, 64, COPIES>, Layout<64, COPIES>::DYNAMIC))
  // The forms by rows (32 sequences of up to 16,411 tokens, 8 kv heads of 128, bf16, short runs, before the weights' second sum): narrow against wide at 65 / 80 / 125 rows 198 / 200 /
  // 209 against 228 / 229 / 235 us.  Four copies are for what they add to the weights' bits, and cost 1 % (5 rows 188 us, 187 without; over
  // up to 700 tokens 32.2 and 30.1); two copies of up to 64 rows gained nothing (60 rows 199 us, 196 without).
  if (a.rows > QT) NKV_PAGE_RUN(0);
  else if (a.rows > QT / 4) NKV_PAGE_RUN(1);
  else NKV_PAGE_RUN(4);
#undef NKV_PAGE_RUN
  if (rc != NKV_OK) return rc;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(runs * a.most_rounds, ceil_div(min(unit, a.rows), SLICE));
  config.blockDim = dim3(256);
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  auto join = d == 128 ? (dtype == NKV_BF16 ? join_parts_kernel<NKV_BF16, 128> : join_parts_kernel<NKV_F16, 128>)
                       : (dtype == NKV_BF16 ? join_parts_kernel<NKV_BF16, 64> : join_parts_kernel<NKV_F16, 64>);
  NKV_CUDA(cudaLaunchKernelEx(&config, join, a, parts));
  return NKV_OK;
}

}  // namespace nkv
