// Attention of many query rows over the 8-bit block cache, on tcgen05.
//
// The rows of a kv head (its group's heads of all query tokens) are cut into units of 256: two 128-row tiles that share
// every K and V tile.  A tile is 128 tokens, two blocks of the cache.  A warp brings its codes into a ring by bulk
// copies; four warps turn them into the cache's 16-bit type (exactly: a code is an integer below 2^7) and store them as the
// swizzled operands the tensor cores read; no 16-bit copy of the cache exists in memory.  S = Q K^T goes to tensor memory,
// eight warps take the softmax (one thread per row), P replaces S as the operand of O += P V.  The block scales never touch
// an operand.  K's multiplies the scores.  V's goes into the exponent: the weight handed over is P' = 2^(s + log2 vs - m'),
// with m' a reference that follows the running maximum of s + log2 vs, so that a row's weights stay in their type's range however
// unlike the scales of its blocks are.  It lies below the maximum, in bf16 by 86, which leaves O the rest of fp32's exponents for
// values far below the largest (2^200 of them).  Values of the open block come to the codes' size by a power of two, which is
// its vs (bf16; fp16 values are taken as they are).  The row sum has a reference of its own, c, near the running maximum of s: a
// block's part is the sum of its P' times 2^(m' - log2 vs - c), or, where vs lies so far below the others that P' leaves fp32, the sum of
// 2^(s - c) itself.  P' is rounded to the cache's 16-bit type, as the tensor cores take it; sums, maxima and O stay in fp32.
//
// Measured: 4,680 queries x 24 heads of 128 over 24,960 tokens 1.43 ms (1,000 TFLOP/s) one call at a time, 1.52 to 1.57 without
// pause (the clock sinks); the MMAs alone, with weights that nothing computes, take 1.07.  Bound: the chain of one query tile,
// softmax of its 128 scores a row and the two products that wait for it, which the other tile's covers in part, beside the codes'
// conversion in the same issue slots (1,560 queries: tensor cores busy for 44 % of the cycles, half of the issue slots taken).
//
// The tiles of all units form one list that the SMs take in equal runs; a unit that a run's end cuts leaves fp32 parts,
// joined by a second launch.  Warps: 0-7 softmax, 8-11 operands, 12 MMA issue, 13 codes.
#include "nkv_block.cuh"
#include "nkv_internal.h"
#include "nkv_tc.cuh"

namespace nkv {
namespace {

using namespace tc;

constexpr int QT = 128, NQ = 2, UNIT = QT * NQ;   // rows of a query tile, tiles and rows of a unit
constexpr int TOK = 128;                          // tokens of a tile
constexpr int STAGES = 2;                         // K / V operand stages
constexpr int SOFTMAX_WARPS = 8, OPERAND_WARPS = 4, MMA_WARP = 12, THREADS = 448;
constexpr int SUB = 128 * 128;                    // bytes of a [128 rows x 64 elements] swizzled operand tile
// m' below the maximum when it is set, and how far the maximum may rise before it is set again.  bf16: P' up to 2^94 times codes
// times 2^26 tokens are fp32 numbers.  fp16: P' up to 2^15, so that 2^-21 of the largest keeps all its bits and 2^-32 is a number.
template <int DT> constexpr float RAISE = DT == NKV_BF16 ? 86.0f : 7.0f;
constexpr float RESCALE_THRESHOLD = 8.0f;
// c may lag the scores by this much (sums stay below 2^16 times the number of tokens), and P' is what counts in the sum as long
// as it stands for at most this power of two of 2^c: weights down to 2^-46 are numbers in it then
constexpr float SUM_THRESHOLD = 16.0f, MOST_APART = 80.0f;
constexpr float NOTHING = -3e38f;                 // either reference before the first score: below all, and a number

// (P_READY: query tile i, half h of its tokens at 2 i + h)
enum Bar { Q_FULL = 0, Q_FREE = 1, K_FULL = 2, K_FREE = 4, V_FULL = 6, V_FREE = 8, S_FULL = 10, P_READY = 12, PV_HALF = 16,
           O_DONE = 18, O_FREE = 20, RAW_FULL = 22, RAW_FREE = 26, NUM_BARS = 30 };
// scales are written up to four tiles ahead of the softmax (two operand stages, the ring of codes)
constexpr int NMETA = 8;
constexpr int M_SLOT = NUM_BARS * 8, M_ABORT = M_SLOT + 4, M_SCALES = 512;   // scales: [NMETA][2 blocks] float2 {ks, log2 vs}

template <int D> struct Layout {
  static constexpr int DCH = D / 64;
  static constexpr int Q_OFF = 1024;
  static constexpr int K_OFF = Q_OFF + NQ * DCH * SUB;
  static constexpr int V_OFF = K_OFF + STAGES * DCH * SUB;
  static constexpr int V_SUB = D * 128;            // [D rows x 64 tokens]
  static constexpr int RAW_OFF = V_OFF + STAGES * 2 * V_SUB;
  static constexpr int RAW = TOK * D;              // codes of a tile of K or V
  static constexpr int RAWS = D == 128 ? 2 : 4;    // ring of them
  static constexpr int BYTES = RAW_OFF + RAWS * RAW;
  static constexpr int DYNAMIC = BYTES + 1024;     // room to start on 1,024 bytes
};
static_assert(STAGES == 2, "the MMA warp's stages are told by a bit");
static_assert(M_SCALES + NMETA * 2 * 8 <= 1024, "meta block");

// A unit costs a run as much as PIECE_TILES tiles on top of its own: its queries' way in, the first softmax with nothing beside it,
// its rows' way out.  Causal units of a prompt's start have few tiles, and runs of equally many tiles would take up to twenty of them
// or three (2 x 4,095 queries x 32 heads over their own tokens, costs of 0 / 2 / 3 / 4 / 5: 474 / 412 / 409 / 418 / 422 us).
constexpr uint32_t PIECE_TILES = 3;
__host__ __device__ inline uint32_t cost_of(int tiles) { return tiles > 0 ? tiles + PIECE_TILES : 0; }

// The list of tiles: sequence by sequence, kv head by kv head, unit by unit, with PIECE_TILES places ahead of a unit's.
struct Plan {
  uint32_t start[MAX_SEQUENCES + 1];
  int sequences, runs, units;      // runs: thread blocks; units per kv head
  bool fits;                       // places are counted in 32 bits
  uint32_t run, longer;            // places of a run; the first `longer` have one more
  __host__ __device__ uint32_t first_of(uint32_t i) const { return i * run + min(i, longer); }
  __host__ __device__ uint32_t run_of(uint32_t g) const {
    const uint32_t edge = longer * (run + 1);
    return g < edge ? g / (run + 1) : longer + (g - edge) / run;
  }
};

// tokens that any of rows [0, r_end) ... of a query tile sees, as tiles: rows r0 .. r0 + n - 1 of `rows`
__host__ __device__ inline int tiles_seen(int length, int count, int group, int rows, bool causal, int r0, int n) {
  const int r1 = min(rows, r0 + n) - 1;
  if (r1 < r0 || r0 / group >= count) return 0;
  const int last = min(r1 / group, count - 1);
  const int seen = causal ? min(length, length - count + last + 1) : length;
  return seen > 0 ? (seen + TOK - 1) / TOK : 0;
}

struct Piece {                     // a unit, or a run's part of one
  int b, h, unit, tile0, nt, whole;   // tiles tile0 .. tile0 + nt - 1; whole: all the unit has
};

// The pieces of one run in order; every role walks the same list.
struct Walk {
  uint32_t g, end;
  int b, h, unit, tiles;           // the unit that g lies in, its tiles
  uint32_t at;                     // places of the unit before g
  __device__ __forceinline__ int tiles_of(const Call& a, const Sequences& s, int bb, int u) const {
    return tiles_seen(s.length[bb], s.count[bb], a.group, a.rows, a.causal, u * UNIT, UNIT);
  }
  __device__ __forceinline__ Walk(const Plan& p, const Call& a, const Sequences& s, int run, int kv_heads) {
    g = p.first_of(run);
    end = p.first_of(run + 1);
    int lo = 0, hi = p.sequences - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.start[mid] <= g) lo = mid; else hi = mid - 1;
    }
    b = lo;
    const uint32_t per_head = (p.start[b + 1] - p.start[b]) / kv_heads;
    at = g - p.start[b];
    h = static_cast<int>(at / per_head);
    at -= h * per_head;
    unit = 0;
    while (at >= cost_of(tiles = tiles_of(a, s, b, unit))) {
      at -= cost_of(tiles);
      ++unit;
    }
  }
  __device__ __forceinline__ bool next(const Plan& p, const Call& a, const Sequences& s, int kv_heads, Piece& out) {
    uint32_t from, to;
    do {
      if (g >= end) return false;
      while (at >= cost_of(tiles)) {   // on to the next unit that has tiles
        at = 0;
        if (++unit == p.units) {
          unit = 0;
          if (++h == kv_heads) {
            h = 0;
            ++b;
          }
        }
        tiles = tiles_of(a, s, b, unit);
      }
      from = at;
      to = min(cost_of(tiles), at + (end - g));
      g += to - from;
      at = to;
    } while (to <= PIECE_TILES);     // (the run's end, ahead of the unit's tiles)
    out.b = b;
    out.h = h;
    out.unit = unit;
    out.tile0 = static_cast<int>(max(from, PIECE_TILES) - PIECE_TILES);
    out.nt = static_cast<int>(to - PIECE_TILES) - out.tile0;
    out.whole = out.nt == tiles;
    return true;
  }
};

// tiles of a piece that query tile i takes part in (causal: the first tile sees less than the second)
__device__ __forceinline__ int tiles_for(const Call& a, const Sequences& s, const Piece& p, int i) {
  return max(0, min(p.nt, tiles_seen(s.length[p.b], s.count[p.b], a.group, a.rows, a.causal, p.unit * UNIT + i * QT, QT) - p.tile0));
}

// A run holds at most one piece that starts inside a unit and one that starts with it and is cut: two places each.
struct Parts {
  float* o;       // [2 runs][UNIT][D], relative to 2^m'
  float4* ml;     // [2 runs][UNIT] m', row sum relative to 2^c, c, -
};

struct Ctx { volatile int* abort_flag; };

// Bounded wait of a whole warp.  A phase that is over costs a few instructions; otherwise the warp parks in the barrier unit, a
// microsecond at most at a time, and leaves the issue slots to the others.  The bound is a count of those (seconds): every
// instruction here is fetched at two dozen sites by warps that share their cache.
constexpr int MOST_PARKED = 1 << 20;
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, const Ctx& c, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity) ? 1 : 0)) return true;
  bool ok = false;
#pragma unroll 1
  for (int n = 0; n < MOST_PARKED && !ok; ++n) {
    ok = mbar_try_wait_parked(bar, parity, 1000u);
    if (*c.abort_flag) break;
  }
  if (!ok) atomicCAS(const_cast<int*>(c.abort_flag), 0, code);
  return __all_sync(0xffffffffu, ok ? 1 : 0) != 0;
}
// The same for two barriers at once, a lane each: one trip to shared memory instead of two.
__device__ __forceinline__ bool wait_both(uint64_t* bar, uint32_t parity, bool want, const Ctx& c, int code) {
  bool ok = !want || mbar_try_wait(bar, parity);
  if (__all_sync(0xffffffffu, ok ? 1 : 0)) return true;
#pragma unroll 1
  for (int n = 0; n < MOST_PARKED && !ok; ++n) {
    ok = mbar_try_wait_parked(bar, parity, 1000u);
    if (*c.abort_flag) break;
  }
  if (!ok) atomicCAS(const_cast<int*>(c.abort_flag), 0, code);
  return __all_sync(0xffffffffu, ok ? 1 : 0) != 0;
}
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

template <int DT> __host__ __device__ constexpr uint32_t idesc(int n) {
  return (1u << 4) | (DT == NKV_BF16 ? (1u << 7) | (1u << 10) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}

// four codes (plus 128) as two 16-bit pairs, exactly.  fp16: 0x64 above a byte is 1024 + byte.  bf16 has room for seven
// bits: 0x43 above them is 128 + low bits, and the top bit decides whether 128 or 256 is subtracted.
template <int DT>
__device__ __forceinline__ void expand(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (DT == NKV_F16) {
    const __half2 off = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), off), hb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    const uint32_t low = w & 0x7F7F7F7Fu, top = ~w & 0x80808080u;
    const uint32_t a = __byte_perm(low, 0x43434343u, 0x4140), b = __byte_perm(low, 0x43434343u, 0x4342);
    const uint32_t c = __byte_perm(top, 0x43434343u, 0x4140), d = __byte_perm(top, 0x43434343u, 0x4342);
    const __nv_bfloat162 ha = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&c));
    const __nv_bfloat162 hb = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&d));
    lo = *reinterpret_cast<const uint32_t*>(&ha);
    hi = *reinterpret_cast<const uint32_t*>(&hb);
  }
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// 32 bytes of a result row, in one store where they start on as many: a warp's rows lie apart, and what its stores cost is the
// lines that each of them touches
__device__ __forceinline__ void store32(void* to, const uint32_t (&v)[8], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    static_cast<uint4*>(to)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    static_cast<uint4*>(to)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// 16 bytes of a row that may start anywhere
__device__ __forceinline__ uint4 gather16(const uint16_t* src) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = __ldg(src + 2 * e) | (static_cast<uint32_t>(__ldg(src + 2 * e + 1)) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float max32(const uint32_t (&r)[32]) {
  float x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])), y = fmaxf(__uint_as_float(r[2]), __uint_as_float(r[3]));
#pragma unroll
  for (int j = 4; j < 32; j += 4) {
    x = max3(x, __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
    y = max3(y, __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
  }
  return fmaxf(x, y);
}

// ---- warp 13: codes and scales ---------------------------------------------------------------------------------
// The open block's values as bf16 operands are multiplied by 2^-e, which takes the largest of its `held` tokens to [64, 128): e for
// a whole warp.  (fp16 has no exponents to spare for that, and no values that would need it.)  16 sequences of 500 tokens x 32 heads
// over their own: 147 us, 142 without it.
template <int D>
__device__ __forceinline__ float open_exponent(const uint16_t* tail, int held, int lane) {
  const int col = 8 * lane % NKV_BLOCK;   // the lane's eight tokens are the same in every row; behind the last one there may be anything
  uint32_t keep[4], tops[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e) keep[e] = (col + 2 * e < held ? 0x7FFFu : 0u) | (col + 2 * e + 1 < held ? 0x7FFF0000u : 0u);
#pragma unroll 8
  for (int at = 8 * lane; at < D * NKV_BLOCK; at += 256) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(tail + at));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) tops[e] = __vmaxu2(tops[e], w[e] & keep[e]);   // bits of magnitudes are ordered as these are
  }
  tops[0] = __vmaxu2(__vmaxu2(tops[0], tops[1]), __vmaxu2(tops[2], tops[3]));
  const uint32_t most = __reduce_max_sync(0xffffffffu, max(tops[0] & 0xFFFFu, tops[0] >> 16));
  const int exponent = most >= 0x80u ? static_cast<int>(most >> 7) - 127 : 31 - __clz(most) - 133;   // (subnormal numbers: by their bits)
  return most == 0 ? -60.f : static_cast<float>(min(121, max(-120, exponent - 6)));
}

template <int DT, int D>
__device__ __forceinline__ void codes_role(uint8_t* smem, uint64_t* bars, const BlockArrays& c, const Call& a, const Sequences& seqs,
                                           const Plan& plan, const Ctx& ctx) {
  using L = Layout<D>;
  constexpr uint32_t BLOCK_BYTES = NKV_BLOCK * D;
  const int lane = threadIdx.x & 31;
  float2* const scales = reinterpret_cast<float2*>(smem + M_SCALES);
  Walk walk(plan, a, seqs, blockIdx.x, c.kv_heads);
  Piece p;
  bool ok = true;
  int seq = 0, item = 0;
  while (ok && walk.next(plan, a, seqs, c.kv_heads, p)) {
    const size_t bh = static_cast<size_t>(p.b) * c.kv_heads + p.h;
    const int full = seqs.length[p.b] / NKV_BLOCK, held = seqs.length[p.b] - full * NKV_BLOCK;
    long long slot = 0;
    float2 sc = make_float2(1.f, 1.f);
    for (int t = 0; t < p.nt && ok; ++t, ++seq) {
      const int block0 = 2 * (p.tile0 + t), at = (2 * t) & 31;
      if (at == 0) {   // lane l knows block l of the next sixteen tiles: one trip to memory for all of them
        const int block = block0 + lane;
        sc = make_float2(1.f, 1.f);
        if (block < full) {
          slot = static_cast<long long>(slot_of(c, bh, block));
          sc = __ldg(reinterpret_cast<const float2*>(c.scales) + slot);
        }
      }
      if ((lane & ~1) == at) {
        // a block of scale 0 has only codes 0: any scale serves, and a small one leaves the reference to the others
        scales[(seq % NMETA) * 2 + (lane & 1)] = make_float2(sc.x == 0.f ? 1.f : sc.x, sc.y == 0.f ? -60.f : log2f(sc.y));
      }
      if (DT == NKV_BF16 && full - block0 <= 1 && held > 0) {
        const float e = open_exponent<D>(static_cast<const uint16_t*>(c.v_tail) + bh * NKV_BLOCK * D, held, lane);
        __syncwarp();
        if (lane == 0) scales[(seq % NMETA) * 2 + full - block0] = make_float2(1.f, e);
      }
      __syncwarp();   // ahead of the request whose completion lets S be computed
      const long long s0 = __shfl_sync(0xffffffffu, slot, at), s1 = __shfl_sync(0xffffffffu, slot, at + 1);
      const uint32_t blocks = min(2, max(0, full - block0));   // full ones: the open block is read where it is needed
      for (int tensor = 0; tensor < 2 && ok; ++tensor, ++item) {
        const int stage = item % L::RAWS;
        if (item >= L::RAWS) ok = wait(&bars[RAW_FREE + stage], (item / L::RAWS - 1) & 1, ctx, 975);
        if (!ok) break;
        if (lane == 0) {
          uint8_t* const to = smem + L::RAW_OFF + stage * L::RAW;
          const uint8_t* const from = tensor ? c.v_codes : c.k_codes;
          mbar_arrive_expect_tx(&bars[RAW_FULL + stage], blocks * BLOCK_BYTES);
          if (blocks > 0) bulk_load_1d(to, from + s0 * BLOCK_BYTES, BLOCK_BYTES, &bars[RAW_FULL + stage]);
          if (blocks > 1) bulk_load_1d(to + BLOCK_BYTES, from + s1 * BLOCK_BYTES, BLOCK_BYTES, &bars[RAW_FULL + stage]);
        }
        __syncwarp();
      }
    }
  }
  if (!ok) {   // copies in flight land before the block goes away
    const long long begin = clock64();
    while (clock64() - begin < (1ll << 21)) {}
  }
}

// ---- warps 8-11: queries, K and V as operands -----------------------------------------------------------------
template <int DT, int D>
__device__ __forceinline__ void operand_role(uint8_t* smem, uint64_t* bars, const BlockArrays& c, const Call& a, const Sequences& seqs,
                                             const Plan& plan, const Ctx& ctx) {
  using L = Layout<D>;
  constexpr int DCH = L::DCH, LOADS = D / 16;   // 16-byte pieces of a thread per tile and tensor, half of them of each block
  const int tid = threadIdx.x - 32 * SOFTMAX_WARPS, lane = tid & 31;
  const uint32_t base = smem_u32(smem);
  // queries: a thread has one 16-byte column of every ROWS-th row of the unit
  constexpr int PER_ROW = D / 8, ROWS = 32 * OPERAND_WARPS / PER_ROW, AHEAD = 16;
  const int q_row = tid / PER_ROW, q_col = tid % PER_ROW * 8;
  const uint32_t q_to = base + L::Q_OFF + (q_col / 64) * SUB;
  const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;   // a negative scale is the queries' sign
  Walk walk(plan, a, seqs, blockIdx.x, c.kv_heads);
  Piece p;
  bool ok = true;
  int seq = 0, pieces = 0, item = 0;
  // Where this thread's 16 codes of a tile go, as two 16-byte pieces of an operand row: K rows are tokens of D codes, V rows
  // columns of 64 per block.  Its next 16 codes lie 2,048 bytes on in the ring and a whole number of 8-row groups
  // on in the operand, so one step serves all of them.
  const int k_row = tid * 16 / D, k_col = tid * 16 % D, v_row = tid / 4, v_col = tid % 4 * 16;
  const uint32_t k_to = base + L::K_OFF + (k_col / 64) * SUB, v_to = base + L::V_OFF;
  const uint32_t k0 = k_to + sw128_offset(k_row, k_col % 64), k1 = k_to + sw128_offset(k_row, k_col % 64 + 8);
  const uint32_t v0 = v_to + sw128_offset(v_row, v_col), v1 = v_to + sw128_offset(v_row, v_col + 8);
  constexpr uint32_t K_STEP = 2048 / D * 128, V_STEP = 32 * 128;
  // The eight lanes that store together shall fill all banks: for K of 128-wide heads half of them take their second piece first.
  const uint32_t swap = D == 128 && (lane & 4) != 0 ? 8 : 0;
  const uint32_t kf = swap ? k1 : k0, ks = swap ? k0 : k1;
  // One loop for both, on purpose: a copy for each, unrolled, pushes the softmax warps' instructions out of the cache they share
  // (a quarter of the issue slots went to fetching, 2.5 ms against 1.8 at the time for 4,680 queries x 24 heads over 24,960 tokens;
  // unrolled by 1 / 2 / 4: 1.45 / 1.43 / 1.44).
  auto convert = [&](uint32_t to0, uint32_t to1, uint32_t step, uint32_t first) {
    uint32_t from = base + L::RAW_OFF + (item % L::RAWS) * L::RAW + tid * 16;
#pragma unroll 2
    for (int i = 0; i < LOADS; i += 2) {
      const uint2 a0 = lds64(from + first), a1 = lds64(from + (first ^ 8));
      const uint2 b0 = lds64(from + 2048 + first), b1 = lds64(from + 2048 + (first ^ 8));
      uint4 p0, p1, p2, p3;
      expand<DT>(a0.x, p0.x, p0.y);
      expand<DT>(a0.y, p0.z, p0.w);
      expand<DT>(a1.x, p1.x, p1.y);
      expand<DT>(a1.y, p1.z, p1.w);
      sts128(to0, p0);
      sts128(to1, p1);
      expand<DT>(b0.x, p2.x, p2.y);
      expand<DT>(b0.y, p2.z, p2.w);
      expand<DT>(b1.x, p3.x, p3.y);
      expand<DT>(b1.y, p3.z, p3.w);
      sts128(to0 + step, p2);
      sts128(to1 + step, p3);
      from += 4096;
      to0 += 2 * step;
      to1 += 2 * step;
    }
    warp_arrive(&bars[RAW_FREE + item % L::RAWS], lane);
    ++item;
  };
  // The open block, over what was converted there (by the same threads).  Keys behind its last token are masked in the scores,
  // whatever they are; values there count as zero: a weight of 0 times anything else might be NaN.
  auto open_keys = [&](uint32_t tile, size_t bh, int open) {
    const uint16_t* const tail = static_cast<const uint16_t*>(c.k_tail) + bh * NKV_BLOCK * D;
#pragma unroll 1
    for (int i = 0; i < LOADS; ++i) {
      const int at = ((i / 2) * 128 + tid) * 16 + (i % 2) * 8, row = at / D, col = at % D;
      sts128(tile + (col / 64) * SUB + sw128_offset(open * NKV_BLOCK + row, col % 64), *reinterpret_cast<const uint4*>(tail + at));
    }
  };
  const float2* const scales = reinterpret_cast<const float2*>(smem + M_SCALES);
  auto open_values = [&](uint32_t tile, size_t bh, int open, int held) {
    const int e = DT == NKV_BF16 ? static_cast<int>(scales[(seq % NMETA) * 2 + open].y) : 0;   // (written ahead of the tile's codes)
    const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    const uint16_t* const tail = static_cast<const uint16_t*>(c.v_tail) + bh * NKV_BLOCK * D;
#pragma unroll 1
    for (int i = 0; i < (2 - open) * LOADS; ++i) {     // the open block, and the one behind it where the tile has room
      const int at = ((i % LOADS / 2) * 128 + tid) * 16 + (i % 2) * 8, row = at / NKV_BLOCK, col = at % NKV_BLOCK;
      uint32_t w[4] = {0, 0, 0, 0};
      if (i < LOADS && col < held) {
        const uint4 v = *reinterpret_cast<const uint4*>(tail + at);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] &= col + 2 * j + 1 < held ? 0xFFFFFFFFu : col + 2 * j < held ? 0xFFFFu : 0u;
          const float2 f = unpack2<DT>(w[j]);
          if (DT == NKV_BF16) w[j] = pack2<DT>(f.x * down, f.y * down);
        }
      }
      sts128(tile + (open + i / LOADS) * L::V_SUB + sw128_offset(row, col), make_uint4(w[0], w[1], w[2], w[3]));
    }
  };
  while (ok && walk.next(plan, a, seqs, c.kv_heads, p)) {
    const size_t bh = static_cast<size_t>(p.b) * c.kv_heads + p.h;
    const int length = seqs.length[p.b], full = length / NKV_BLOCK, held = length - full * NKV_BLOCK;
    // ---- queries: the first rows are on their way while the piece before still reads its own
    const uint16_t* const q_head = a.q + p.b * a.q_batch + static_cast<long long>(p.h) * a.group * a.q_head + q_col;
    int r = p.unit * UNIT + q_row, token = r / a.group, head = r - token * a.group;
    const int token_step = ROWS / a.group, head_step = ROWS - token_step * a.group;
#pragma unroll 1
    for (int row0 = q_row; row0 < UNIT && ok; row0 += AHEAD * ROWS) {
      uint4 v[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const uint16_t* const src = q_head + token * a.q_token + head * a.q_head;
        v[k] = make_uint4(0, 0, 0, 0);
        if (a.q_vector && r < a.rows) v[k] = __ldg(reinterpret_cast<const uint4*>(src));
        r += ROWS;
        token += token_step;
        head += head_step;
        if (head >= a.group) { head -= a.group; ++token; }
      }
      if (row0 == q_row && pieces > 0) ok = wait(&bars[Q_FREE], (pieces - 1) & 1, ctx, 970);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int row = row0 + k * ROWS;
        sts128(q_to + (row / QT) * DCH * SUB + sw128_offset(row % QT, q_col % 64),
               make_uint4(v[k].x ^ flip, v[k].y ^ flip, v[k].z ^ flip, v[k].w ^ flip));
      }
    }
    if (!ok) break;
    ++pieces;
    if (!a.q_vector) {   // rows that start anywhere
#pragma unroll 1
      for (int row = q_row; row < UNIT; row += ROWS) {
        const int at = p.unit * UNIT + row, t = at / a.group;
        if (at >= a.rows) break;
        const uint4 v = gather16(q_head + t * a.q_token + (at - t * a.group) * a.q_head);
        sts128(q_to + (row / QT) * DCH * SUB + sw128_offset(row % QT, q_col % 64), make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip));
      }
    }
    fence_proxy_async();
    warp_arrive(&bars[Q_FULL], lane);
    // ---- tiles: K, then V
#pragma unroll 1
    for (int t = 0; t < 2 * p.nt && ok; ++t) {
      const int value = t & 1, stage = seq % STAGES, use = seq / STAGES;
      ok = wait(&bars[RAW_FULL + item % L::RAWS], (item / L::RAWS) & 1, ctx, 971);
      if (ok && use >= 1) ok = wait(&bars[(value ? V_FREE : K_FREE) + stage], (use - 1) & 1, ctx, 972 + value);
      if (!ok) break;
      const uint32_t at = stage * (value ? 2 * L::V_SUB : DCH * SUB);
      convert((value ? v0 : kf) + at, (value ? v1 : ks) + at, value ? V_STEP : K_STEP, value ? 0 : swap);
      const int open = full - 2 * (p.tile0 + t / 2);   // 0 or 1: that half of the tile is not a full block
      if (open <= 1) {
        if (value) open_values(v_to + at, bh, open, held); else open_keys(base + L::K_OFF + at, bh, open);
      }
      fence_proxy_async();
      warp_arrive(&bars[(value ? V_FULL : K_FULL) + stage], lane);
      seq += value;
    }
  }
}

// ---- warp 12: MMA issue -----------------------------------------------------------------------------------------
template <int DT, int D>
__device__ __forceinline__ void mma_role(uint8_t* smem, uint64_t* bars, uint32_t tmem, const Call& a, const Sequences& seqs,
                                         const Plan& plan, const Ctx& ctx, int kv_heads) {
  using L = Layout<D>;
  constexpr int DCH = L::DCH;
  const bool leader = elect_one();   // the whole warp runs the (uniform) control flow; one elected lane issues
  const uint32_t base = smem_u32(smem);
  // operand descriptors of the first tile and stage; the others lie a whole number of 16-byte units on
  const uint64_t q_desc = make_smem_desc_sw128(base + L::Q_OFF), k_desc = make_smem_desc_sw128(base + L::K_OFF);
  const uint64_t v_desc = make_smem_desc_sw128(base + L::V_OFF);
  auto issue_s = [&](int i, uint32_t stage) {
    const uint64_t qd = q_desc + static_cast<uint32_t>(i * (DCH * SUB / 16)), kd = k_desc + stage * static_cast<uint32_t>(DCH * SUB / 16);
    const uint32_t d = tmem + i * 128;
#pragma unroll
    for (int ch = 0; ch < DCH; ++ch)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (leader) mma_bf16(d, qd + ch * (SUB / 16) + 2 * k, kd + ch * (SUB / 16) + 2 * k, idesc<DT>(TOK), ch + k > 0);
    if (leader) mma_commit(&bars[S_FULL + i]);
  };
  // weights of 64 tokens (a block) times V of it: [128 rows x 64] [D x 64]^T, both with the tokens running along rows
  auto issue_pv = [&](int i, uint32_t stage, int half, bool accumulate) {
    const uint64_t vd = v_desc + (stage * 2 + half) * static_cast<uint32_t>(L::V_SUB / 16);
    const uint32_t d = tmem + 256 + i * 128, w = tmem + i * 128 + half * 32;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (leader) mma_bf16_ts(d, w + 8 * k, vd + 2 * k, idesc<DT>(D), accumulate || k > 0);
    if (half == 0 && leader) mma_commit(&bars[PV_HALF + i]);
  };
  Walk walk(plan, a, seqs, blockIdx.x, kv_heads);
  Piece p;
  bool ok = true;
  const uint32_t lane = threadIdx.x & 31;
  uint32_t seq = 0;
  int pieces = 0, done[NQ] = {0, 0}, used[NQ] = {0, 0};   // tiles and pieces of each query tile so far
  while (ok && walk.next(plan, a, seqs, kv_heads, p)) {
    const int n[NQ] = {tiles_for(a, seqs, p, 0), tiles_for(a, seqs, p, 1)};
    const int longest = max(n[0], n[1]);
    ok = wait(&bars[Q_FULL], pieces & 1, ctx, 980);
    ++pieces;
    // The first and the last query tile to use tile t: each K and V stage is waited for once and given back once.
    auto first_of = [&](int t) { return t < n[0] ? 0 : 1; };
    auto last_of = [&](int t) { return t < n[1] ? 1 : 0; };
#pragma unroll 1
    for (int t = 0; t <= longest && ok; ++t) {
      // PV of tile t - 1 and S of tile t, query tile by query tile.  Between the first and the last tiles that both take part in
      // there is nothing to decide, and V is waited for with the first weights.
#pragma unroll 1
      for (; t > 1 && t < min(n[0], n[1]); ++t) {
        const uint32_t now = (seq + t - 1) & 1, next = now ^ 1, now_phase = (seq + t - 1) >> 1 & 1, next_phase = (seq + t) >> 1 & 1;
        const uint32_t phase0 = (done[0] + t - 1) & 1, phase1 = (done[1] + t - 1) & 1;
        ok = wait_both(lane == 0 ? &bars[P_READY] : &bars[V_FULL + now], lane == 0 ? phase0 : now_phase, lane < 2, ctx, 981);
        if (!ok) break;
        tc_fence_after();
        issue_pv(0, now, 0, true);
        ok = wait(&bars[P_READY + 1], phase0, ctx, 984);
        if (!ok) break;
        tc_fence_after();
        issue_pv(0, now, 1, true);
        ok = wait(&bars[K_FULL + next], next_phase, ctx, 985);   // (converted just ahead of its use)
        if (!ok) break;
        tc_fence_after();
        issue_s(0, next);
        ok = wait(&bars[P_READY + 2], phase1, ctx, 981);
        if (!ok) break;
        tc_fence_after();
        issue_pv(1, now, 0, true);
        ok = wait(&bars[P_READY + 3], phase1, ctx, 984);
        if (!ok) break;
        tc_fence_after();
        issue_pv(1, now, 1, true);
        if (leader) mma_commit(&bars[V_FREE + now]);
        issue_s(1, next);
        if (leader) mma_commit(&bars[K_FREE + next]);
      }
      if (!ok) break;
      const uint32_t now = (seq + t - 1) % STAGES, next = (seq + t) % STAGES;
      const uint32_t now_phase = ((seq + t - 1) / STAGES) & 1, next_phase = ((seq + t) / STAGES) & 1;
#pragma unroll 1
      for (int i = 0; i < NQ; ++i) {
        const int tiles = i ? n[1] : n[0];
        if (t > 0 && t - 1 < tiles) {
          const uint32_t phase = ((i ? done[1] : done[0]) + t - 1) & 1;
          if (i == first_of(t - 1)) ok = wait(&bars[V_FULL + now], now_phase, ctx, 982);
          if (t == 1) {   // the first PV of a piece overwrites O: the rows of the piece before must have been read
            const int pieces_before = i ? used[1] : used[0];
            if (ok && pieces_before > 0) ok = wait(&bars[O_FREE + i], (pieces_before - 1) & 1, ctx, 983);
          }
          ok = ok && wait(&bars[P_READY + 2 * i], phase, ctx, 981);
          if (!ok) break;
          tc_fence_after();
          issue_pv(i, now, 0, t > 1);
          ok = wait(&bars[P_READY + 2 * i + 1], phase, ctx, 984);
          if (!ok) break;
          tc_fence_after();
          issue_pv(i, now, 1, true);
          if (t == tiles && leader) mma_commit(&bars[O_DONE + i]);
          if (i == last_of(t - 1) && leader) mma_commit(&bars[V_FREE + now]);
        }
        if (t < tiles) {
          // S of the next tile overwrites P of this one, right behind the PV that reads it: the tensor core executes one
          // thread's MMAs in order
          if (i == first_of(t)) {
            ok = wait(&bars[K_FULL + next], next_phase, ctx, 985);
            if (!ok) break;
            tc_fence_after();
          }
          issue_s(i, next);
          if (i == last_of(t) && leader) mma_commit(&bars[K_FREE + next]);
        }
      }
    }
    if (!ok) break;
    if (leader) mma_commit(&bars[Q_FREE]);
    // tiles of the list that no query tile of the piece uses do not exist: the longest of the two is the piece's length
    seq += p.nt;
    for (int i = 0; i < NQ; ++i) {
      done[i] += n[i];
      used[i] += n[i] > 0 ? 1 : 0;
    }
  }
  __syncwarp();
}

// ---- warps 0-7: softmax -------------------------------------------------------------------------------------------
template <int DT, int D>
__device__ __forceinline__ void softmax_role(uint8_t* smem, uint64_t* bars, uint32_t tmem, const Call& a, const Sequences& seqs,
                                             const Plan& plan, const Parts& parts, const Ctx& ctx, int kv_heads) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const int wg = warp / 4, row = tid & 127;
  const uint32_t lane_sel = static_cast<uint32_t>(32 * (warp & 3)) << 16;
  const uint32_t o_addr = tmem + lane_sel + 256 + wg * 128;
  const float2* const scales = reinterpret_cast<const float2*>(smem + M_SCALES);
  const float scale = fabsf(a.scale_log2);
  Walk walk(plan, a, seqs, blockIdx.x, kv_heads);
  Piece p;
  bool ok = true, more = true;
  int seq = 0, ci = 0, pieces = 0;   // tiles of the list, and tiles and pieces of this query tile
  auto place_of = [&](const Piece& pc) { return 2 * static_cast<size_t>(blockIdx.x) + (pc.tile0 == 0 ? 1 : 0); };
  while (ok && (more = walk.next(plan, a, seqs, kv_heads, p))) {
    const int r = p.unit * UNIT + wg * QT + row;
    const int length = seqs.length[p.b], count = seqs.count[p.b];
    const int seen = r < a.rows ? visible_to(a, length, count, r) : 0;
    const int seen_least = __reduce_min_sync(0xffffffffu, seen);
    const int tiles = tiles_for(a, seqs, p, wg);
    const size_t bh = static_cast<size_t>(p.b) * kv_heads + p.h;
    const int token = r / a.group;
    const size_t at = (static_cast<size_t>(p.b) * a.tokens + token) * a.heads + p.h * a.group + r - token * a.group;
    float m = NOTHING, l = 0.f, c = NOTHING;   // m' and the row sum relative to 2^c
    // half a tile, a block of the cache, at a time
#pragma unroll 1
    for (int n = 0; n < 2 * tiles && ok; ++n) {
      const int half = n & 1, block = 2 * p.tile0 + n, first = block * NKV_BLOCK;
      auto partial_at = [&]() { return a.partial + (bh * a.most_blocks + block) * a.rows + r; };
      const bool partial_wanted = a.partial && r < a.rows && block < a.most_blocks;
      const uint32_t s_addr = tmem + lane_sel + wg * 128 + half * 64, p_addr = tmem + lane_sel + wg * 128 + half * 32;
      if (half == 0) {
        ok = wait(&bars[S_FULL + wg], ci & 1, ctx, 990);
        if (!ok) break;
        tc_fence_after();
      }
      uint32_t raw[2][32];
      tmem_ld32_issue(s_addr, raw[0]);
      tmem_ld32_issue(s_addr + 32, raw[1]);
      const float2 sc = scales[(2 * seq + n) % (2 * NMETA)];   // (written ahead of the request for the codes that this S came from)
      tmem_ld32_wait(raw[0]);
      tmem_ld32_wait(raw[1]);
      float f = scale * sc.x;
      if (first + NKV_BLOCK > seen_least) {   // some row of the warp does not see all of the block
        // scaled before they are masked: -inf times a scale of 0 would be NaN
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            raw[k][j] = first + 32 * k + j < seen ? __float_as_uint(__uint_as_float(raw[k][j]) * f) : 0xFF800000u;
        f = 1.f;
      }
      const float top = fmaxf(max32(raw[0]), max32(raw[1])) * f;
      float off = sc.y - m, rise = m - sc.y - c;   // rise: log2 of what P' counts in the row sum
      if (__any_sync(0xffffffffu, top + off > RAISE<DT> + RESCALE_THRESHOLD || top - c > SUM_THRESHOLD || rise > MOST_APART)) {
        // Move the references: O and the sum are scaled by 2^(old - new).  S was issued behind PV of the tile before and its commit
        // covers both; PV of this tile's first half may still run.
        const float m_new = fmaxf(m, top + sc.y - RAISE<DT>), c_new = fmaxf(c, top);
        const float alpha = exp2f(0.5f * (m - m_new));   // twice: the whole may leave fp32 where O does not
        if (n > 0) {
          if (half) {
            ok = wait(&bars[PV_HALF + wg], ci & 1, ctx, 991);
            if (!ok) break;
            tc_fence_after();
          }
#pragma unroll 1
          for (int cc = 0; cc < D / 16; ++cc) {
            uint32_t v[16];
            tmem_ld16(o_addr + cc * 16, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha * alpha);
            tmem_st16(o_addr + cc * 16, v);
          }
          tmem_wait_st();
        }
        l *= exp2f(c - c_new);
        m = m_new;
        c = c_new;
        off = sc.y - m;
        rise = m - sc.y - c;
        if (__any_sync(0xffffffffu, rise > MOST_APART)) {   // the sum apart from P', from scores read again (a short loop)
          float own = 0.f;
#pragma unroll 1
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t v[16];
            tmem_ld16(s_addr + 16 * cc, v);
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (first + 16 * cc + j < seen) own += exp2_fast(fmaf(__uint_as_float(v[j]), scale * sc.x, -c));
          }
          if (rise > MOST_APART) {
            l += own;
            if (partial_wanted) *partial_at() = log2f(own) + c;
            rise = -INFINITY;
          }
        }
      }
      // P' (16-bit pairs) replaces S, the first half's of the first columns.  (The compiler interleaves the groups: spelling out
      // exponentials of one beside arguments and sums of its neighbours changes nothing.)
      const uint64_t scale2 = pair_f32(f, f), off2 = pair_f32(off, off);
      uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float lo, hi;
          split_f32(fma_f32x2(pair_bits(raw[k][2 * i], raw[k][2 * i + 1]), scale2, off2), lo, hi);
          lo = exp2_fast(lo);
          hi = exp2_fast(hi);
          sum2[i & 1] = add_f32x2(sum2[i & 1], pair_f32(lo, hi));
          packed[i] = pack2<DT>(lo, hi);
        }
        tmem_st16(p_addr + k * 16, packed);
      }
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&bars[P_READY + 2 * wg + half], lane);
      float lo, hi;
      split_f32(add_f32x2(sum2[0], sum2[1]), lo, hi);
      const float sum = lo + hi;
      l = fmaf(sum, exp2_fast(rise), l);
      if (partial_wanted && rise > -INFINITY) *partial_at() = log2f(sum) - off;
      ci += half;
    }
    seq += p.nt;
    if (!ok) break;
    // ---- the rows: results, or a part of them
    if (tiles > 0) {
      ok = wait(&bars[O_DONE + wg], pieces & 1, ctx, 992);
      ++pieces;
      if (!ok) break;
      tc_fence_after();
    }
    const float half = exp2f(0.5f * (m - c)), inv = half / l;   // in two factors: 2^(m' - c) alone may leave fp32
    const uint64_t half2 = pair_f32(half, half), inv2 = pair_f32(inv, inv), zero2 = pair_f32(-0.f, -0.f);
    const bool wide_out = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0, wide_part = (reinterpret_cast<uintptr_t>(parts.o) & 31) == 0;
    float* const part = parts.o + (place_of(p) * UNIT + wg * QT + row) * D;
#pragma unroll 1
    for (int cc = 0; cc < D / 32; ++cc) {
      uint32_t v[32];
      if (tiles > 0) {
        tmem_ld32_issue(o_addr + cc * 32, v);
        tmem_ld32_wait(v);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0u;
      }
      if (r >= a.rows) continue;
      if (p.whole) {
#pragma unroll
        for (int j = 0; j < 32; j += 16) {
          uint32_t o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float lo, hi;
            split_f32(fma_f32x2(fma_f32x2(pair_bits(v[j + 2 * e], v[j + 2 * e + 1]), half2, zero2), inv2, zero2), lo, hi);
            o[e] = seen > 0 ? pack2<DT>(lo, hi) : 0u;
          }
          store32(a.out + at * D + cc * 32 + j, o, wide_out);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          const uint32_t o[8] = {v[j], v[j + 1], v[j + 2], v[j + 3], v[j + 4], v[j + 5], v[j + 6], v[j + 7]};
          store32(part + cc * 32 + j, o, wide_part);
        }
      }
    }
    if (r < a.rows) {
      if (p.whole) a.lse[at] = seen > 0 ? (c + log2f(l)) * LN2 : -INFINITY;
      else parts.ml[place_of(p) * UNIT + wg * QT + row] = make_float4(m, l, c, 0.f);
    }
    if (tiles > 0) {
      tc_fence_before();
      warp_arrive(&bars[O_FREE + wg], lane);
    }
  }
  // a launch that gave up: NaN for the piece it stopped in and all later ones
  if (!ok) {
    while (more) {
      const int r = p.unit * UNIT + wg * QT + row, token = r / a.group;
      if (r < a.rows) {
        if (p.whole) a.lse[(static_cast<size_t>(p.b) * a.tokens + token) * a.heads + p.h * a.group + r - token * a.group] = CUDART_NAN_F;
        else parts.ml[place_of(p) * UNIT + wg * QT + row] = make_float4(0.f, CUDART_NAN_F, 0.f, 0.f);
      }
      more = walk.next(plan, a, seqs, kv_heads, p);
    }
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(THREADS, 1)
tile_kernel(BlockArrays c, Call a, const __grid_constant__ Sequences seqs, const __grid_constant__ Plan plan, Parts parts, int32_t* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + M_SLOT);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + M_ABORT);
  const int warp = threadIdx.x / 32;
  if (threadIdx.x == 0) {
    mbar_init(&bars[Q_FULL], OPERAND_WARPS);
    mbar_init(&bars[Q_FREE], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[K_FULL + i], OPERAND_WARPS);
      mbar_init(&bars[K_FREE + i], 1);
      mbar_init(&bars[V_FULL + i], OPERAND_WARPS);
      mbar_init(&bars[V_FREE + i], 1);
      mbar_init(&bars[S_FULL + i], 1);
      mbar_init(&bars[PV_HALF + i], 1);
      mbar_init(&bars[O_DONE + i], 1);
      mbar_init(&bars[O_FREE + i], QT / 32);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars[P_READY + i], QT / 32);
      mbar_init(&bars[RAW_FULL + i], 1);
      mbar_init(&bars[RAW_FREE + i], OPERAND_WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == MMA_WARP) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Ctx ctx{abort_flag};
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp < SOFTMAX_WARPS) softmax_role<DT, D>(smem, bars, tmem, a, seqs, plan, parts, ctx, c.kv_heads);
  else if (warp < SOFTMAX_WARPS + OPERAND_WARPS) operand_role<DT, D>(smem, bars, c, a, seqs, plan, ctx);
  else if (warp > MMA_WARP) codes_role<DT, D>(smem, bars, c, a, seqs, plan, ctx);
  else mma_role<DT, D>(smem, bars, tmem, a, seqs, plan, ctx, c.kv_heads);
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag) atomicCAS(status, 0, *abort_flag);
}

// Joins the parts of cut units and fills the rows of units that see nothing; a thread block per (unit, kv head,
// sequence) and 32 rows, a thread per row and 16 bytes of it.
template <int DT, int D>
__global__ void __launch_bounds__(256)
join_units_kernel(Call a, const __grid_constant__ Sequences seqs, const __grid_constant__ Plan plan, Parts parts, int kv_heads, int slices) {
  __shared__ uint32_t before;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int unit = blockIdx.x / slices, slice = blockIdx.x % slices, h = blockIdx.y, b = blockIdx.z;
  const int length = seqs.length[b], count = seqs.count[b];
  auto tiles_of = [&](int u) { return tiles_seen(length, count, a.group, a.rows, a.causal, u * UNIT, UNIT); };
  const int nt = tiles_of(unit);
  uint32_t r0 = 0, r1 = 0, begin = 0;
  if (nt > 0) {
    if (threadIdx.x == 0) before = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (int u = threadIdx.x; u < unit; u += 256) mine += cost_of(tiles_of(u));
    if (mine) atomicAdd(&before, mine);
    __syncthreads();
    begin = plan.start[b] + h * ((plan.start[b + 1] - plan.start[b]) / kv_heads) + before + PIECE_TILES;
    r0 = plan.run_of(begin);
    r1 = plan.run_of(begin + nt - 1);
    if (r0 == r1) return;   // one run had all of it and wrote the results
  }
  constexpr int PER_ROW = D / 8, ROWS = 256 / PER_ROW;
  const int row0 = slice * (UNIT / slices);
  for (int row = row0 + threadIdx.x / PER_ROW; row < row0 + UNIT / slices; row += ROWS) {
    const int r = unit * UNIT + row, col = (threadIdx.x % PER_ROW) * 8;
    if (r >= a.rows) break;
    const int token = r / a.group;
    const size_t at = (static_cast<size_t>(b) * a.tokens + token) * a.heads + h * a.group + r - token * a.group;
    const bool any = nt > 0 && visible_to(a, length, count, r) > 0;
    float top = -INFINITY, sum_top = -INFINITY, sum = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    if (any) {
      // the run the unit starts in has it as a piece that starts with the unit, the others as one that starts inside
      auto place = [&](uint32_t run) { return (2 * static_cast<size_t>(run) + (run == r0 ? 1 : 0)) * UNIT + row; };
      for (uint32_t run = r0; run <= r1; ++run) {
        const float4 ml = __ldcg(&parts.ml[place(run)]);
        top = fmaxf(top, ml.x);
        sum_top = fmaxf(sum_top, ml.z);
      }
      for (uint32_t run = r0; run <= r1; ++run) {
        const float4 ml = __ldcg(&parts.ml[place(run)]);
        const float4 lo = __ldcg(reinterpret_cast<const float4*>(parts.o + place(run) * D + col));
        const float4 hi = __ldcg(reinterpret_cast<const float4*>(parts.o + place(run) * D + col + 4));
        const float f = exp2f(0.5f * (ml.x - top));   // twice, as in the kernel above
        sum = fmaf(ml.y, exp2f(ml.z - sum_top), sum);
        const float part[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(part[e] * f, f, acc[e]);
      }
    }
    const float half = any ? exp2f(0.5f * (top - sum_top)) : 0.f, inv = any ? half / sum : 0.f;
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack2<DT>(acc[2 * e] * half * inv, acc[2 * e + 1] * half * inv);
    *reinterpret_cast<uint4*>(a.out + at * D + col) = make_uint4(o[0], o[1], o[2], o[3]);
    if (col == 0) a.lse[at] = any ? (sum_top + log2f(sum)) * LN2 : -INFINITY;
  }
}

Plan plan_of(const Sequences& seqs, int n, int kv_heads, int group, int rows, bool causal) {
  Plan p;
  p.sequences = n;
  p.units = ceil_div(rows, UNIT);
  uint64_t total = 0;
  for (int i = 0; i < n; ++i) {
    p.start[i] = static_cast<uint32_t>(total);
    uint64_t tiles = 0;
    for (int u = 0; u < p.units; ++u) tiles += cost_of(tiles_seen(seqs.length[i], seqs.count[i], group, rows, causal, u * UNIT, UNIT));
    total += tiles * kv_heads;
  }
  p.start[n] = static_cast<uint32_t>(total);
  p.fits = total <= UINT32_MAX;
  p.runs = static_cast<int>(min(total, static_cast<uint64_t>(sm_count())));
  p.run = p.runs ? static_cast<uint32_t>(total / p.runs) : 0;
  p.longer = p.runs ? static_cast<uint32_t>(total % p.runs) : 0;
  return p;
}


size_t part_bytes(int runs, int d) { return static_cast<size_t>(runs) * 2 * UNIT * (d + 4) * sizeof(float); }

}  // namespace

size_t block_tile_bytes(int d) { return part_bytes(sm_count(), d); }

int block_tile(const BlockArrays& c, const Call& a, const Sequences& seqs, int n, int dtype, int d, void* workspace, int32_t* status,
               cudaStream_t stream) {
  const Plan plan = plan_of(seqs, n, c.kv_heads, a.group, a.rows, a.causal);
  NKV_REQUIRE(plan.fits, NKV_ERR_TOO_LARGE, "block_attend: more tiles of %d x %d than 32 bits count", UNIT, TOK);
  Parts parts;
  parts.o = static_cast<float*>(workspace);
  parts.ml = reinterpret_cast<float4*>(parts.o + static_cast<size_t>(plan.runs) * 2 * UNIT * d);
  const bool bf16 = dtype == NKV_BF16, wide = d == 128;
  if (plan.runs > 0) {
    auto run = [&](auto kernel, int smem) {
      NKV_CUDA(allow_shared(reinterpret_cast<const void*>(kernel), smem));
      kernel<<<plan.runs, THREADS, smem, stream>>>(c, a, seqs, plan, parts, status);
      NKV_CUDA(cudaGetLastError());
      return NKV_OK;
    };
    const int rc = wide ? (bf16 ? run(tile_kernel<NKV_BF16, 128>, Layout<128>::DYNAMIC) : run(tile_kernel<NKV_F16, 128>, Layout<128>::DYNAMIC))
                        : (bf16 ? run(tile_kernel<NKV_BF16, 64>, Layout<64>::DYNAMIC) : run(tile_kernel<NKV_F16, 64>, Layout<64>::DYNAMIC));
    if (rc != NKV_OK) return rc;
  }
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  const int slices = 8;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(plan.units * slices, c.kv_heads, n);
  config.blockDim = dim3(256);
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = plan.runs > 0 ? 1 : 0;
  auto join = wide ? (bf16 ? join_units_kernel<NKV_BF16, 128> : join_units_kernel<NKV_F16, 128>)
                   : (bf16 ? join_units_kernel<NKV_BF16, 64> : join_units_kernel<NKV_F16, 64>);
  NKV_CUDA(cudaLaunchKernelEx(&config, join, a, seqs, plan, parts, c.kv_heads, slices));
  return NKV_OK;
}

}  // namespace nkv
