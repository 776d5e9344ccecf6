// Attention of few query rows over the 8-bit block cache: the read of a decoding step.
//
// The rows of a kv head are its group's heads of all query tokens, up to 16 (32 of heads of 64).  Every byte of the cache is used once per
// row, so memory is the bound, and the work is cut by bytes: the blocks of all sequences and kv heads form one list, and
// each warp takes an equal run of it, whatever heads and sequences that run cuts through.  A warp is on its own: its
// blocks arrive by bulk copies in a ring that only it uses, it keeps the running softmax of its rows in registers, and
// where its run leaves a head it stores what it has.  A second small launch joins the parts of a head.
//
// Scores are computed as S^T = K Q^T and the result as O^T = V^T P^T: the codes are the 16-row operand of the tensor
// cores, the rows the 8-wide one, so that one row costs half of what the other way round would.  Codes become fp16
// by two instructions per pair (a byte beside 0x64 is the number 1024 + byte; 1152 is subtracted, exactly), queries are
// scaled by a power of two per row into the middle of fp16's range.  Weights become 16-bit numbers relative to the largest of
// their own block and row, which is 2^7: 2^-21 of it keeps all its bits, 2^-32 is still a number, however small the block's weights are
// beside others'.  The block scales are applied in fp32: K's to the scores, V's, with the block's own weight, as its
// product is added to the running result.
//
// Measured, both launches, among other calls: 40 heads of 128 over 99,840 tokens, one row each: 1.02 GB in 166 us, 6.2 TB/s.  8 heads
// of 32 ragged sequences of up to 16,411 tokens, five rows each: 0.61 GB in 113 to 117 us, 5.3 TB/s.  8 heads of 64 of 8
// sequences of up to 8,191, twenty rows each: 38 MB in 25.6 us, about half of them the two launches' fixed cost and the rest the
// arithmetic of twenty rows a byte.
#include "nkv_block.cuh"
#include "nkv_internal.h"
#include "nkv_tc.cuh"

namespace nkv {
namespace {

using tc::smem_u32;

constexpr int WARPS = 4, CTAS_PER_SM = 2;
constexpr int RING_BYTES = 24576;                 // per warp: three K or V blocks of 128-wide heads, six of 64-wide ones
template <int D> constexpr int SLOT = NKV_BLOCK * D;
template <int D> constexpr int STAGES = RING_BYTES / SLOT<D>;
constexpr int STEP_SMEM = WARPS * RING_BYTES + 1024;
constexpr float RAISE = 7.f;                      // log2 of a block's largest weight as an fp16 number (as a bf16 one: 0)

// Where the blocks of a launch's sequences lie in the list, and how the list is cut.
struct Plan {
  uint32_t start[MAX_SEQUENCES + 1];   // first block of every sequence in the list (kv head by kv head)
  int sequences, workers;
  uint32_t run, longer;                // every worker takes `run` blocks, the first `longer` of them one more
  __host__ __device__ uint32_t first_of(uint32_t worker) const { return worker * run + min(worker, longer); }
  __host__ __device__ uint32_t worker_of(uint32_t g) const {
    const uint32_t edge = longer * (run + 1);
    return g < edge ? g / (run + 1) : longer + (g - edge) / run;
  }
};

__device__ __forceinline__ uint32_t blocks_of(int length, int count) {
  return count > 0 ? static_cast<uint32_t>(length + NKV_BLOCK - 1) / NKV_BLOCK : 0u;
}

struct Place { int b, h, block; };
__device__ __forceinline__ Place place_of(const Plan& p, const Sequences& seqs, uint32_t g) {
  int lo = 0, hi = p.sequences - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.start[mid] <= g) lo = mid; else hi = mid - 1;
  }
  Place r;
  r.b = lo;
  const uint32_t n = max(1u, blocks_of(seqs.length[lo], seqs.count[lo])), at = g - p.start[lo];
  r.h = static_cast<int>(at / n);
  r.block = static_cast<int>(at - r.h * n);
  return r;
}

// partial results: part (worker, head) lies at worker + head's number in the list of heads -- each next part raises one
// of the two, so no two share a place
struct Parts {
  float* o;        // [parts][rows][D], relative to 2^m
  float2* ml;      // [parts][rows] reference point, sum
};

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// four codes (plus 128) as two fp16 pairs, exactly
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const __half2 off = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), off), hb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
  lo = *reinterpret_cast<const uint32_t*>(&ha);
  hi = *reinterpret_cast<const uint32_t*>(&hb);
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// the tokens of an 8 x 8 piece of scores: with them a lane's four neighbouring bytes of a V row are its operand as they lie
__device__ __forceinline__ int token_of(int tile, int hi, int row) { return 16 * (row >> 1) + 4 * tile + 2 * hi + (row & 1); }

// NT: 8-wide groups of rows
template <int DT, int D, int NT>
__global__ void __launch_bounds__(32 * WARPS, CTAS_PER_SM)
step_kernel(BlockArrays c, Call a, const __grid_constant__ Sequences seqs, const __grid_constant__ Plan plan, Parts parts,
            int32_t* status) {
  constexpr int KSTEPS = D / 16, MTILES = D / 16, CHUNKS = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~static_cast<uintptr_t>(127));
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + WARPS * RING_BYTES);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + WARPS * RING_BYTES + 512);
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
  uint8_t* const ring = smem + warp * RING_BYTES;
  uint64_t* const full = bars + warp * STAGES<D>;
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0)
    for (int s = 0; s < STAGES<D>; ++s) tc::mbar_init(full + s, 1);
  tc::fence_barrier_init();
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int worker = blockIdx.x * WARPS + warp;
  if (worker >= plan.workers) return;
  const uint32_t first = plan.first_of(worker), last = plan.first_of(worker + 1);

  // ---- the ring: K and V of a block are two items; item i lies in slot i % STAGES.  An open block has none.
  // Lane l of a window knows block first + window + l.
  uint32_t ahead = first, ahead_window = first - 32;   // next block to request, blocks whose slots the lanes hold
  long long ahead_slot = 0;                            // -1: open
  uint32_t put = 0, got = 0;                           // items requested, items taken
  int put_half = 0;                                    // next item of block `ahead`: K or V
  auto request = [&]() {                               // fills the ring as far as there is room
    while (ahead < last && put - got < STAGES<D>) {
      if (ahead - ahead_window >= 32u) {
        ahead_window = ahead;
        ahead_slot = -1;
        if (ahead + lane < last) {
          const Place at = place_of(plan, seqs, ahead + lane);
          const size_t bh = static_cast<size_t>(at.b) * c.kv_heads + at.h;
          if ((at.block + 1) * NKV_BLOCK <= seqs.length[at.b]) ahead_slot = static_cast<long long>(slot_of(c, bh, at.block));
        }
      }
      const long long slot = __shfl_sync(0xffffffffu, ahead_slot, static_cast<int>(ahead - ahead_window));
      if (slot >= 0) {
        if (lane == 0) {
          const int s = put % STAGES<D>;
          tc::mbar_arrive_expect_tx(full + s, SLOT<D>);
          tc::bulk_load_1d(ring + s * SLOT<D>, (put_half ? c.v_codes : c.k_codes) + static_cast<size_t>(slot) * SLOT<D>, SLOT<D>, full + s);
        }
        ++put;
      } else {
        put_half = 1;
      }
      if (put_half) ++ahead;
      put_half ^= 1;
    }
  };
  request();

  // ---- per head: the rows as operand, their scale, what they see
  uint32_t qb[NT][KSTEPS][2];
  float factor[NT][2];               // of rows 8 nt + 2 t4 (+ 1): scale * log2 e * the row's power of two
  int seen[NT][2], seen_least = 0;   // tokens they see, and the least that any row of the head sees
  float m[NT][2], l[NT][2], o[NT][MTILES][4];
  int head_b = -1, head_h = -1;
  bool ok = true;

  auto load_rows = [&](int b, int h) {
    seen_least = seqs.length[b];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = 8 * nt + g8, token = r / a.group;
      const bool in = r < a.rows;
      const uint16_t* row = a.q + b * a.q_batch + (in ? token : 0) * a.q_token + (h * a.group + (in ? r - token * a.group : 0)) * a.q_head;
      float x[CHUNKS][16], top = 0.f;
#pragma unroll
      for (int ch = 0; ch < CHUNKS; ++ch)
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
          const uint16_t* const src = row + 64 * ch + 16 * t4 + e;
          uint32_t w[4] = {0, 0, 0, 0};
          if (in && a.q_vector) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
          } else if (in) {
#pragma unroll 1
            for (int k = 0; k < 4; ++k) {
              const uint32_t pair = __ldg(src + 2 * k) | (static_cast<uint32_t>(__ldg(src + 2 * k + 1)) << 16);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) w[kk] = kk == k ? pair : w[kk];
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = unpack2<DT>(w[k]);
            x[ch][e + 2 * k] = f.x;
            x[ch][e + 2 * k + 1] = f.y;
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the largest element goes to [2^14, 2^15): 16 bits hold what lies up to 2^-29 of it below exactly
      int shift = top > 0.f ? 14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127) : 0;
      shift = max(-126, min(126, shift));
      const float up = __uint_as_float(static_cast<uint32_t>(shift + 127) << 23);
      const float down = __uint_as_float(static_cast<uint32_t>(127 - shift) << 23) * fabsf(a.scale_log2);
      const float sign = a.scale_log2 < 0.f ? -up : up;
#pragma unroll
      for (int i = 0; i < KSTEPS; ++i) {
        const float* v = &x[i / 4][4 * (i & 3)];
        qb[nt][i][0] = pack2<NKV_F16>(v[0] * sign, v[1] * sign);
        qb[nt][i][1] = pack2<NKV_F16>(v[2] * sign, v[3] * sign);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rr = 8 * nt + 2 * t4 + e;
        factor[nt][e] = __shfl_sync(0xffffffffu, down, (2 * t4 + e) * 4);
        seen[nt][e] = rr < a.rows ? visible_to(a, seqs.length[b], seqs.count[b], rr) : 0;
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < MTILES; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][j][e] = 0.f;
    }
    // rows behind the last one and queries that see less: their blocks are masked
    seen_least = a.causal || seqs.count[b] < a.tokens ? visible_to(a, seqs.length[b], seqs.count[b], 0) : seqs.length[b];
    if (seqs.count[b] < a.tokens) seen_least = 0;
  };

  auto store_part = [&](int b, int h) {
    const size_t part = static_cast<size_t>(worker) + static_cast<size_t>(b) * c.kv_heads + h;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int r = 8 * nt + 2 * t4 + e;
        if (r >= a.rows) continue;
        if (g8 == 0) parts.ml[part * a.rows + r] = make_float2(m[nt][e], ok ? sum : CUDART_NAN_F);
        float* to = parts.o + (part * a.rows + r) * D;
#pragma unroll
        for (int j = 0; j < MTILES; ++j) {
          to[16 * j + g8] = o[nt][j][e];
          to[16 * j + 8 + g8] = o[nt][j][2 + e];
        }
      }
  };

  // softmax of one block: s -> P^T operand (fp16, or the cache's type for an open block), relative to the block's largest; alpha and
  // share: what the results so far and the block's product count from now on
  auto softmax = [&](float (&s)[NT][4][4], int t0, float k_scale, int b, int h, int block, uint32_t (&pb)[NT][4][2], float (&alpha)[NT][2],
                     float (&share)[NT][2], bool plain_type) {
    const bool masked = t0 + NKV_BLOCK > seen_least;
    const float raise = plain_type && DT == NKV_BF16 ? 0.f : RAISE;   // (bf16 values may leave no room for it)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = s[nt][i][e] * (factor[nt][e & 1] * k_scale);
          if (masked && t0 + token_of(i, e >> 1, g8) >= seen[nt][e & 1]) v = -INFINITY;
          s[nt][i][e] = v;
          top[e & 1] = fmaxf(top[e & 1], v);
        }
      float ref[2], sum[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], x));
        const float next = fmaxf(m[nt][e], top[e]), now = next == -INFINITY ? 0.f : next;
        alpha[nt][e] = exp2_fast(m[nt][e] - now);
        share[nt][e] = exp2_fast(top[e] - now - raise);
        ref[e] = (top[e] == -INFINITY ? 0.f : top[e]) - raise;
        m[nt][e] = next;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][i][e] = exp2_fast(s[nt][i][e] - ref[e & 1]);
          sum[e & 1] += s[nt][i][e];
        }
#pragma unroll
        for (int hi = 0; hi < 2; ++hi)
          pb[nt][i][hi] = transpose8x8(plain_type ? pack2<DT>(s[nt][i][2 * hi], s[nt][i][2 * hi + 1])
                                                  : pack2<NKV_F16>(s[nt][i][2 * hi], s[nt][i][2 * hi + 1]));
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[nt][e] = fmaf(sum[e], share[nt][e], l[nt][e] * alpha[nt][e]);
        if (a.partial) {
          float total = sum[e];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
          const int r = 8 * nt + 2 * t4 + e;
          if (g8 == 0 && r < a.rows)
            a.partial[((static_cast<size_t>(b) * c.kv_heads + h) * a.most_blocks + block) * a.rows + r] = log2f(total) + ref[e];
        }
      }
    }
  };

  // result += block product
  auto add = [&](int nt, int j, const float (&part)[4], const float (&alpha)[2], const float (&share)[2]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[nt][j][e] = fmaf(part[e], share[e & 1], o[nt][j][e] * alpha[e & 1]);
  };

  float2 scales = make_float2(0.f, 0.f);   // lane l: of block window + l
  Place place{0, 0, 0};
  uint32_t window = first - 32;
  for (uint32_t g = first; g < last && ok; ++g) {
    if (g - window >= 32u) {
      window = g;
      if (g + lane < last) {
        place = place_of(plan, seqs, g + lane);
        const size_t bh = static_cast<size_t>(place.b) * c.kv_heads + place.h;
        if ((place.block + 1) * NKV_BLOCK <= seqs.length[place.b])
          scales = __ldg(reinterpret_cast<const float2*>(c.scales) + slot_of(c, bh, place.block));
      }
    }
    const int at = static_cast<int>(g - window);
    const int b = __shfl_sync(0xffffffffu, place.b, at), h = __shfl_sync(0xffffffffu, place.h, at);
    const int block = __shfl_sync(0xffffffffu, place.block, at), t0 = block * NKV_BLOCK;
    if (b != head_b || h != head_h) {
      if (head_b >= 0) store_part(head_b, head_h);
      load_rows(b, h);
      head_b = b;
      head_h = h;
    }
    float s[NT][4][4];
    uint32_t pb[NT][4][2];
    float alpha[NT][2], share[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][i][e] = 0.f;
    if (t0 + NKV_BLOCK <= seqs.length[b]) {
      const float k_scale = __shfl_sync(0xffffffffu, scales.x, at), v_scale = __shfl_sync(0xffffffffu, scales.y, at);
      // ---- S^T = K Q^T: tokens x rows
      ok = tc::wait_all(full + got % STAGES<D>, (got / STAGES<D>) & 1, abort_flag, 960);
      if (!ok) break;
      const uint8_t* codes = ring + (got % STAGES<D>) * SLOT<D>;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* row_lo = codes + token_of(i, 0, g8) * D + 16 * t4;
        const uint8_t* row_hi = codes + token_of(i, 1, g8) * D + 16 * t4;
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ++ch) {
          const uint4 lo = *reinterpret_cast<const uint4*>(row_lo + 64 * ch), hi = *reinterpret_cast<const uint4*>(row_hi + 64 * ch);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a0, a1, a2, a3;
            codes_to_half(word_of(lo, w), a0, a2);
            codes_to_half(word_of(hi, w), a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<false>(s[nt][i], a0, a1, a2, a3, qb[nt][4 * ch + w][0], qb[nt][4 * ch + w][1]);
          }
        }
      }
      __syncwarp();
      ++got;
      request();
      softmax(s, t0, k_scale, b, h, block, pb, alpha, share, false);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) share[nt][e] *= v_scale;
      // ---- O^T = V^T P^T: columns x rows
      ok = tc::wait_all(full + got % STAGES<D>, (got / STAGES<D>) & 1, abort_flag, 961);
      if (!ok) break;
      codes = ring + (got % STAGES<D>) * SLOT<D>;
#pragma unroll
      for (int j = 0; j < MTILES; ++j) {
        const uint4 lo = *reinterpret_cast<const uint4*>(codes + (16 * j + g8) * NKV_BLOCK + 16 * t4);
        const uint4 hi = *reinterpret_cast<const uint4*>(codes + (16 * j + 8 + g8) * NKV_BLOCK + 16 * t4);
        float part[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[nt][e] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a0, a1, a2, a3;
          codes_to_half(word_of(lo, w), a0, a2);
          codes_to_half(word_of(hi, w), a1, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<false>(part[nt], a0, a1, a2, a3, pb[nt][w][0], pb[nt][w][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) add(nt, j, part[nt], alpha[nt], share[nt]);
      }
      __syncwarp();
      ++got;
      request();
    } else {
      // ---- the open block: 16-bit rows straight from memory, in their own type; tokens behind the last one count as zero
      const size_t tail = (static_cast<size_t>(b) * c.kv_heads + h) * NKV_BLOCK * D;
      const uint16_t* kt = static_cast<const uint16_t*>(c.k_tail) + tail;
      const uint16_t* vt = static_cast<const uint16_t*>(c.v_tail) + tail;
      const int held = seqs.length[b] - t0;
      // (64 columns at a time, all loads of them in flight: one warp has this block, and the others wait for it)
#pragma unroll 1
      for (int ch = 0; ch < CHUNKS; ++ch) {
        uint2 k_lo[4][4], k_hi[4][4], q2[NT][4];
        const int d0 = 64 * ch + 16 * t4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            k_lo[i][w] = *reinterpret_cast<const uint2*>(kt + token_of(i, 0, g8) * D + d0 + 4 * w);
            k_hi[i][w] = *reinterpret_cast<const uint2*>(kt + token_of(i, 1, g8) * D + d0 + 4 * w);
          }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int r = 8 * nt + g8, token = r / a.group;
          const uint16_t* const row = a.q + b * a.q_batch + token * a.q_token + (h * a.group + r - token * a.group) * a.q_head + d0;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            q2[nt][w] = make_uint2(0, 0);
            if (r < a.rows && a.q_vector) q2[nt][w] = __ldg(reinterpret_cast<const uint2*>(row + 4 * w));
            else if (r < a.rows)
              q2[nt][w] = make_uint2(__ldg(row + 4 * w) | (static_cast<uint32_t>(__ldg(row + 4 * w + 1)) << 16),
                                     __ldg(row + 4 * w + 2) | (static_cast<uint32_t>(__ldg(row + 4 * w + 3)) << 16));
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<DT == NKV_BF16>(s[nt][i], k_lo[i][w].x, k_hi[i][w].x, k_lo[i][w].y, k_hi[i][w].y, q2[nt][w].x, q2[nt][w].y);
      }
      // `factor` carries the rows' powers of two and the sign of the scale is in the operand: neither is here
      float kept[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          kept[nt][e] = factor[nt][e];
          factor[nt][e] = a.scale_log2;
        }
      const int least = seen_least;
      seen_least = min(seen_least, 0);   // tokens behind the last one are masked
      softmax(s, t0, 1.f, b, h, block, pb, alpha, share, true);
      seen_least = least;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) factor[nt][e] = kept[nt][e];
#pragma unroll
      for (int j = 0; j < MTILES; ++j) {
        float part[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[nt][e] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int t = 16 * t4 + 4 * w;
          uint2 lo = *reinterpret_cast<const uint2*>(vt + (16 * j + g8) * NKV_BLOCK + t);
          uint2 hi = *reinterpret_cast<const uint2*>(vt + (16 * j + 8 + g8) * NKV_BLOCK + t);
          const uint32_t keep0 = t + 1 < held ? 0xFFFFFFFFu : t < held ? 0xFFFFu : 0u;
          const uint32_t keep1 = t + 3 < held ? 0xFFFFFFFFu : t + 2 < held ? 0xFFFFu : 0u;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<DT == NKV_BF16>(part[nt], lo.x & keep0, hi.x & keep0, lo.y & keep1, hi.y & keep1, pb[nt][w][0], pb[nt][w][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) add(nt, j, part[nt], alpha[nt], share[nt]);
      }
    }
  }
  if (!ok) {   // a copy never came: the worker's heads get NaN, copies in flight land before the block goes away
    if (lane == 0) atomicCAS(status, 0, *abort_flag);
    for (uint32_t g = first; g < last; ++g) {
      const Place at = place_of(plan, seqs, g);
      if (at.b == head_b && at.h == head_h && g > first) continue;
      head_b = at.b;
      head_h = at.h;
      store_part(head_b, head_h);
    }
    const long long begin = clock64();
    while (clock64() - begin < (1ll << 21)) {}
    return;
  }
  if (head_b >= 0) store_part(head_b, head_h);
}

// Joins the parts of `slice` rows of a kv head.  A thread has four columns of a row; where the rows leave threads over, the parts
// are dealt out to several of them.  With weights, every block's share of the rows' attention as well,
// rows in a fixed order.
constexpr int JOIN_THREADS = 512;
template <int DT, int D>
__global__ void __launch_bounds__(JOIN_THREADS)
join_kernel(BlockArrays c, Call a, const __grid_constant__ Sequences seqs, const __grid_constant__ Plan plan, Parts parts, int slice) {
  __shared__ float lse2[32];
  __shared__ float4 accs[JOIN_THREADS];
  __shared__ float2 mls[JOIN_THREADS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int h = blockIdx.x, b = blockIdx.y;
  const int length = seqs.length[b], count = seqs.count[b];
  const uint32_t n = blocks_of(length, count);
  const size_t bh = static_cast<size_t>(b) * c.kv_heads + h;
  const uint32_t begin = plan.start[b] + h * n;
  const uint32_t w0 = n ? plan.worker_of(begin) : 0u, w1 = n ? plan.worker_of(begin + n - 1) : 0u;
  constexpr int COLS = D / 4;
  const int row0 = blockIdx.z * slice, wanted = min(slice, a.rows - row0) * COLS;
  const int groups = max(1, min(JOIN_THREADS / wanted, static_cast<int>(w1 - w0) + 1));   // threads that share the parts of four columns
  for (int base = 0; base < wanted; base += JOIN_THREADS) {
    const int i = groups > 1 ? threadIdx.x % wanted : base + threadIdx.x, group = groups > 1 ? threadIdx.x / wanted : 0;
    const bool in = i < wanted && group < groups;
    const int r = row0 + i / COLS, col = (i % COLS) * 4;
    const bool any = in && visible_to(a, length, count, r) > 0;
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float m, float l, const float4& o) {
      const float next = fmaxf(top, m), ref = next == -INFINITY ? 0.f : next, f = exp2f(top - ref), g = exp2f(m - ref);
      top = next;
      sum = fmaf(sum, f, l * g);
      acc.x = fmaf(acc.x, f, o.x * g);
      acc.y = fmaf(acc.y, f, o.y * g);
      acc.z = fmaf(acc.z, f, o.z * g);
      acc.w = fmaf(acc.w, f, o.w * g);
    };
    if (any) {
#pragma unroll 4
      for (uint32_t w = w0 + group; w <= w1; w += groups) {
        const float2 ml = __ldcg(&parts.ml[(w + bh) * a.rows + r]);
        add(ml.x, ml.y, __ldcg(reinterpret_cast<const float4*>(parts.o + ((w + bh) * a.rows + r) * D + col)));
      }
    }
    for (int left = groups; left > 1;) {
      const int half = (left + 1) / 2;
      accs[threadIdx.x] = acc;
      mls[threadIdx.x] = make_float2(top, sum);
      __syncthreads();
      const int other = threadIdx.x + half * wanted;
      if (any && group + half < left) add(mls[other].x, mls[other].y, accs[other]);
      __syncthreads();
      left = half;
    }
    if (in && group == 0) {
      const int token = r / a.group, head = h * a.group + r - token * a.group;
      const size_t at = (static_cast<size_t>(b) * a.tokens + token) * a.heads + head;
      const float inv = any ? 1.f / sum : 0.f;
      *reinterpret_cast<uint2*>(a.out + at * D + col) = make_uint2(pack2<DT>(acc.x * inv, acc.y * inv), pack2<DT>(acc.z * inv, acc.w * inv));
      if (col == 0) {
        const float v = any ? top + log2f(sum) : -INFINITY;
        a.lse[at] = v * LN2;
        lse2[r] = v;
      }
    }
  }
  if (a.weights == nullptr) return;
  __syncthreads();
  for (uint32_t block = threadIdx.x; block < n; block += JOIN_THREADS) {
    const float* partial = a.partial + (bh * a.most_blocks + block) * a.rows;
    float sum = 0.f;
    for (int r = 0; r < a.rows; ++r)
      if (visible_to(a, length, count, r) > static_cast<int>(block) * NKV_BLOCK) sum += exp2f(__ldcg(partial + r) - lse2[r]);
    a.weights[bh * c.blocks + block] += sum;
  }
}

// workers of a launch: a warp each, as many as are resident, and none without a block
Plan plan_of(const Sequences& seqs, int n, int kv_heads) {
  Plan p;
  uint32_t total = 0;
  for (int i = 0; i < n; ++i) {
    p.start[i] = total;
    total += (seqs.count[i] > 0 ? ceil_div(seqs.length[i], NKV_BLOCK) : 0) * kv_heads;
  }
  p.start[n] = total;
  p.sequences = n;
  const uint32_t resident = static_cast<uint32_t>(sm_count()) * CTAS_PER_SM * WARPS;
  p.workers = static_cast<int>(min(resident, total));
  p.run = p.workers ? total / p.workers : 0;
  p.longer = p.workers ? total % p.workers : 0;
  return p;
}

size_t parts_of(const Plan& p, int kv_heads) { return p.workers + static_cast<size_t>(p.sequences) * kv_heads; }

}  // namespace

// Up to as many rows as a warp's registers hold: four groups of eight rows of 64 columns, two of 128.  The tile kernel costs the
// same for one row as for 128 (single calls, 24,960 tokens x 24 heads of 128: 1 row 48 us and 16 rows 56 here, 17 to 128 rows 97 to
// 101 there; heads of 64: 1 row 32, 24 rows 48 and 32 rows 62 here, 33 rows 87 there).
bool block_step_supported(int rows, int d) { return rows <= (d == 64 ? 32 : 16); }

// bytes of the parts of one launch
size_t block_step_bytes(const Sequences& seqs, int n, int kv_heads, int rows, int d) {
  return parts_of(plan_of(seqs, n, kv_heads), kv_heads) * rows * (d + 2) * sizeof(float);
}

int block_step(const BlockArrays& c, const Call& a, const Sequences& seqs, int n, int dtype, int d, void* workspace, int32_t* status,
               cudaStream_t stream) {
  const Plan plan = plan_of(seqs, n, c.kv_heads);
  Parts parts;
  parts.o = static_cast<float*>(workspace);
  parts.ml = reinterpret_cast<float2*>(parts.o + parts_of(plan, c.kv_heads) * a.rows * d);
  if (plan.workers > 0) {
    auto run = [&](auto kernel) {
      NKV_CUDA(allow_shared(reinterpret_cast<const void*>(kernel), STEP_SMEM));
      kernel<<<ceil_div(plan.workers, WARPS), 32 * WARPS, STEP_SMEM, stream>>>(c, a, seqs, plan, parts, status);
      NKV_LAUNCH_CHECK("step_kernel");
      return NKV_OK;
    };
    const bool bf16 = dtype == NKV_BF16;
    const int groups = ceil_div(a.rows, 8);
    int rc;
    if (d == 128) rc = groups == 1 ? (bf16 ? run(step_kernel<NKV_BF16, 128, 1>) : run(step_kernel<NKV_F16, 128, 1>))
                                   : (bf16 ? run(step_kernel<NKV_BF16, 128, 2>) : run(step_kernel<NKV_F16, 128, 2>));
    else if (groups == 1) rc = bf16 ? run(step_kernel<NKV_BF16, 64, 1>) : run(step_kernel<NKV_F16, 64, 1>);
    else if (groups == 2) rc = bf16 ? run(step_kernel<NKV_BF16, 64, 2>) : run(step_kernel<NKV_F16, 64, 2>);
    else if (groups == 3) rc = bf16 ? run(step_kernel<NKV_BF16, 64, 3>) : run(step_kernel<NKV_F16, 64, 3>);
    else rc = bf16 ? run(step_kernel<NKV_BF16, 64, 4>) : run(step_kernel<NKV_F16, 64, 4>);
    if (rc != NKV_OK) return rc;
  }
  // the joining launch is set up under the first one's tail and waits for its results
  cudaLaunchConfig_t config = {};
  // few heads: their rows are cut too (not with weights, which take all rows of a head)
  const int slices = a.weights ? 1 : min(a.rows, max(1, 2 * sm_count() / (c.kv_heads * n)));
  const int slice = ceil_div(a.rows, slices);
  config.gridDim = dim3(c.kv_heads, n, ceil_div(a.rows, slice));
  config.blockDim = dim3(JOIN_THREADS);
  config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = plan.workers > 0 ? 1 : 0;
  auto join = d == 128 ? (dtype == NKV_BF16 ? join_kernel<NKV_BF16, 128> : join_kernel<NKV_F16, 128>)
                       : (dtype == NKV_BF16 ? join_kernel<NKV_BF16, 64> : join_kernel<NKV_F16, 64>);
  NKV_CUDA(cudaLaunchKernelEx(&config, join, c, a, seqs, plan, parts, slice));
  return NKV_OK;
}

}  // namespace nkv
