// The 8-bit block cache without its attention: tokens in (append), rows out (read), blocks freed (evict), and the rotary
// positions of queries and keys.  All four are bound by memory, the small calls by the latency of a launch.
#include "nkv_block.cuh"
#include "nkv_block_plan.h"
#include "nkv_internal.h"

namespace nkv {
static_assert(BLOCK_TOKENS == NKV_BLOCK, "one block size");
namespace {

// ---- rotary positions -----------------------------------------------------------------------------------------

struct Rotation {
  const float2* table;        // [rows][rotary_dim / 2] cosine, sine
  const int32_t* positions;   // [batch][tokens]
  int rows, dim, layout;      // dim 0: no rotation
};

// cosine and sine of one pair; a position outside the table gives NaN, never a wrong angle
__device__ __forceinline__ float2 turn_of(const Rotation& r, int position, int pair, bool transposed) {
  if (static_cast<unsigned>(position) >= static_cast<unsigned>(r.rows)) return make_float2(CUDART_NAN_F, CUDART_NAN_F);
  float2 cs = __ldg(r.table + static_cast<size_t>(position) * (r.dim / 2) + pair);
  if (transposed) cs.y = -cs.y;
  return cs;
}

// Products and sum are rounded one by one (no contraction to a fused multiply-add): the keys that enter the cache do not
// depend on which kernel rotated them, and elementwise fp32 arithmetic anywhere gives the same bits.
__device__ __forceinline__ float turn_first(float x0, float x1, float2 cs) {
  return __fsub_rn(__fmul_rn(x0, cs.x), __fmul_rn(x1, cs.y));
}
__device__ __forceinline__ float turn_second(float x0, float x1, float2 cs) {
  return __fadd_rn(__fmul_rn(x0, cs.y), __fmul_rn(x1, cs.x));
}

struct RotarySide {
  const void* x;
  void* out;
  long long stride_batch, stride_token, stride_head;
  int heads;
};

// 16 bytes of a row as floats and back
template <int DT>
struct Piece {
  static constexpr int N = DT == NKV_F32 ? 4 : 8;
  static __device__ __forceinline__ void unpack(const uint4& raw, float (&v)[N]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (DT == NKV_F32) {
        v[i] = __uint_as_float(w[i]);
      } else {
        const float2 f = unpack2<DT>(w[i]);
        v[(2 * i) % N] = f.x;
        v[(2 * i + 1) % N] = f.y;
      }
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = DT == NKV_F32 ? __float_as_uint(v[i]) : pack2<DT>(v[(2 * i) % N], v[(2 * i + 1) % N]);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// A thread takes two 16-byte pieces whose elements are each other's partners (or two that are only copied).
// HEADS heads per thread share the table entries; one where the call is short of threads.  Bound: memory (24,960 tokens x 24
// heads x 128, interleaved, half of each head turned: 307 MB in and out in 102 us, 6.0 TB/s).
template <int DT, int HEADS>
__global__ void __launch_bounds__(256)
rotary_kernel(RotarySide a, RotarySide b, int batch, int tokens, int d, Rotation rot, int transposed) {
  constexpr int N = Piece<DT>::N;
  const int units = d / (2 * N), groups = (a.heads + HEADS - 1) / HEADS + (b.heads + HEADS - 1) / HEADS;
  const long long index = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (index >= static_cast<long long>(batch) * tokens * groups * units) return;
  const int u = static_cast<int>(index % units);
  const long long rest = index / units;
  int group = static_cast<int>(rest % groups);
  const long long row = rest / groups;
  const int groups_a = (a.heads + HEADS - 1) / HEADS;
  const bool second = group >= groups_a;
  if (second) group -= groups_a;
  const RotarySide& side = second ? b : a;
  using E = typename Elem<DT>::type;
  const int half = rot.dim / 2, turned = rot.dim / (2 * N);
  const bool turns = u < turned;
  const int first = turns && rot.layout == NKV_ROTARY_HALF ? u * N : 2 * u * N;
  const int other = turns && rot.layout == NKV_ROTARY_HALF ? first + half : first + N;
  const int head0 = group * HEADS;
  const int bi = static_cast<int>(row / tokens), ti = static_cast<int>(row % tokens);
  const E* src = static_cast<const E*>(side.x) + bi * side.stride_batch + ti * side.stride_token + head0 * side.stride_head;
  E* dst = static_cast<E*>(side.out) + (row * side.heads + head0) * d;
  uint4 lo[HEADS], hi[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (HEADS > 1 && head0 + h >= side.heads) break;
    lo[h] = *reinterpret_cast<const uint4*>(src + h * side.stride_head + first);
    hi[h] = *reinterpret_cast<const uint4*>(src + h * side.stride_head + other);
  }
  float2 cs[N];
  if (turns) {
    const int position = __ldg(rot.positions + row);
#pragma unroll
    for (int e = 0; e < N; ++e) cs[e] = turn_of(rot, position, u * N + e, transposed);
  }
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (HEADS > 1 && head0 + h >= side.heads) break;
    if (turns) {
      float x[N], y[N];
      Piece<DT>::unpack(lo[h], x);
      Piece<DT>::unpack(hi[h], y);
      if (rot.layout == NKV_ROTARY_HALF) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float x0 = x[e], x1 = y[e];
          x[e] = turn_first(x0, x1, cs[e]);
          y[e] = turn_second(x0, x1, cs[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
          const float x0 = x[2 * e], x1 = x[2 * e + 1], y0 = y[2 * e], y1 = y[2 * e + 1];
          x[2 * e] = turn_first(x0, x1, cs[e]);
          x[2 * e + 1] = turn_second(x0, x1, cs[e]);
          y[2 * e] = turn_first(y0, y1, cs[N / 2 + e]);
          y[2 * e + 1] = turn_second(y0, y1, cs[N / 2 + e]);
        }
      }
      lo[h] = Piece<DT>::pack(x);
      hi[h] = Piece<DT>::pack(y);
    }
    *reinterpret_cast<uint4*>(dst + h * d + first) = lo[h];
    *reinterpret_cast<uint4*>(dst + h * d + other) = hi[h];
  }
}

// Rows that do not start on 16 bytes, or widths that do not divide into such pieces: one pair per thread.
template <int DT>
__global__ void __launch_bounds__(256)
rotary_pairs_kernel(RotarySide a, RotarySide b, int batch, int tokens, int d, Rotation rot, int transposed) {
  const int pairs = (d + 1) / 2, half = rot.dim / 2;
  const long long index = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (index >= static_cast<long long>(batch) * tokens * (a.heads + b.heads) * pairs) return;
  const int p = static_cast<int>(index % pairs);
  const long long rest = index / pairs;
  int head = static_cast<int>(rest % (a.heads + b.heads));
  const long long row = rest / (a.heads + b.heads);
  const bool second = head >= a.heads;
  if (second) head -= a.heads;
  const RotarySide& side = second ? b : a;
  const bool turns = p < half;
  const int first = turns && rot.layout == NKV_ROTARY_HALF ? p : 2 * p;
  const int other = turns && rot.layout == NKV_ROTARY_HALF ? p + half : first + 1;
  const int bi = static_cast<int>(row / tokens), ti = static_cast<int>(row % tokens);
  const size_t src = bi * side.stride_batch + ti * side.stride_token + head * side.stride_head;
  const size_t dst = (static_cast<size_t>(row) * side.heads + head) * d;
  float x0 = load_float(side.x, DT, src + first), x1 = other < d ? load_float(side.x, DT, src + other) : 0.f;
  if (turns) {
    const float2 cs = turn_of(rot, __ldg(rot.positions + row), p, transposed);
    const float y0 = turn_first(x0, x1, cs);
    x1 = turn_second(x0, x1, cs);
    x0 = y0;
  }
  store_float(side.out, DT, dst + first, x0);
  if (other < d) store_float(side.out, DT, dst + other, x1);
}

// ---- append ----------------------------------------------------------------------------------------------------

// the eight elements from d0 on of a token's row
template <int DT>
__device__ __forceinline__ uint4 load_piece(const uint16_t* row, int d0, bool vector) {
  if (vector) return __ldg(reinterpret_cast<const uint4*>(row + d0));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __ldg(row + d0 + 2 * i) | (static_cast<uint32_t>(__ldg(row + d0 + 2 * i + 1)) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// entries of eight neighbouring pairs from the one of element d0 on (half layout); rows of the table start on 16 bytes where its
// base does, as dim is a multiple of 16
__device__ __forceinline__ void turns_of(const Rotation& rot, int position, int d0, float2 (&cs)[8]) {
  const bool in = static_cast<unsigned>(position) < static_cast<unsigned>(rot.rows);
  const float2* const from = rot.table + static_cast<size_t>(in ? position : 0) * (rot.dim / 2) + d0;
  if ((reinterpret_cast<uintptr_t>(rot.table) & 15) == 0) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(from + e));
      cs[e] = make_float2(v.x, v.y);
      cs[e + 1] = make_float2(v.z, v.w);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = __ldg(from + e);
  }
  if (!in)
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = make_float2(CUDART_NAN_F, CUDART_NAN_F);
}

template <int DT>
__device__ __forceinline__ uint4 rotated_piece(const uint16_t* row, int d0, bool vector, const Rotation& rot, int position) {
  const uint4 raw = load_piece<DT>(row, d0, vector);
  if (d0 >= rot.dim) return raw;
  float x[8], y[8];
  Piece<DT>::unpack(raw, x);
  if (rot.layout == NKV_ROTARY_HALF) {
    const int half = rot.dim / 2;
    const bool low = d0 < half;
    Piece<DT>::unpack(load_piece<DT>(row, low ? d0 + half : d0 - half, vector), y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 cs = turn_of(rot, position, (low ? d0 : d0 - half) + e, false);
      x[e] = low ? turn_first(x[e], y[e], cs) : turn_second(y[e], x[e], cs);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 cs = turn_of(rot, position, (d0 + e) / 2, false);
      const float x0 = x[e], x1 = x[e + 1];
      x[e] = turn_first(x0, x1, cs);
      x[e + 1] = turn_second(x0, x1, cs);
    }
  }
  return Piece<DT>::pack(x);
}

template <int DT>
__device__ __forceinline__ bool not_finite(const uint4& v) {
  constexpr uint32_t E = DT == NKV_BF16 ? 0x7F80u : 0x7C00u;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & E) == E || ((w[i] >> 16) & E) == E;
  return bad;
}

// A block's scale as codes_of takes it.  Scales below 1e-20 are lifted by 2^64, and the elements with them, so that no residual
// falls below the normal numbers.
struct Quotient {
  float scale, inv, lift;   // inv: the reciprocal, rounded to nearest; lift: 1 or 2^64
  __device__ __forceinline__ explicit Quotient(float s) {
    lift = s < 1e-20f ? 18446744073709551616.f : 1.f;
    scale = s * lift;
    inv = __frcp_rn(scale);
  }
};

// Codes (plus 128) of eight elements: rint(x / scale), quotient rounded to fp32.  The quotient comes from the reciprocal y by one
// step of Markstein's division: q = x y, then q + (x - q scale) y with the residual exact.  It is x / scale correctly rounded for
// every 16-bit x and every scale that is a 16-bit number / 127 (the tests compare all of them).  Adding
// 1.5 * 2^23 + 128 rounds it to an integer, whose low byte is the code.  A subnormal scale is a coarse multiple of the
// maximum / 127: there the codes are clamped.
__device__ __forceinline__ uint2 codes_of(float (&x)[8], const Quotient& by) {
  constexpr float MAGIC = 12583040.0f;
  const uint64_t inv2 = pair_f32(by.inv, by.inv), neg2 = pair_f32(-by.scale, -by.scale), magic2 = pair_f32(MAGIC, MAGIC);
  if (by.lift != 1.f)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= by.lift;
  uint32_t t[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint64_t v = pair_f32(x[e], x[e + 1]), q = fma_f32x2(v, inv2, 0ull);
    float t0, t1;
    split_f32(add_f32x2(fma_f32x2(fma_f32x2(q, neg2, v), inv2, q), magic2), t0, t1);
    t[e] = __float_as_uint(t0);
    t[e + 1] = __float_as_uint(t1);
  }
  if (by.lift != 1.f)
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = __float_as_uint(fminf(fmaxf(__uint_as_float(t[e]), MAGIC - 127.f), MAGIC + 127.f));
  uint2 w;
  w.x = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
  w.y = __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410);
  return w;
}

// largest magnitudes of the two halves, as bits: those of 16-bit floating-point numbers are ordered as the numbers are, and what
// is not finite comes out as NOT_FINITE or more
__device__ __forceinline__ uint32_t magnitude(const uint4& v) {
  constexpr uint32_t M = 0x7FFF7FFFu;
  return __vmaxu2(__vmaxu2(v.x & M, v.y & M), __vmaxu2(v.z & M, v.w & M));
}
template <int DT> constexpr uint32_t NOT_FINITE = DT == NKV_BF16 ? 0x7F80u : 0x7C00u;

// 16 bytes from memory to shared memory; the thread that asked for them may read them once they have landed
__device__ __forceinline__ void copy16_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_landed() { asm volatile("cp.async.wait_all;" ::: "memory"); }

struct AppendSide {
  const uint16_t* x;
  long long stride_batch, stride_token, stride_head;
  int vector;   // rows and strides on 16 bytes
};

// One block of one sequence and head that the call touches.  K: a thread has the pieces p and p + D / 16 of a token's row, which
// are each other's partners where all of a head turns in the half layout, in two passes of 32 tokens.  V: it has eight
// columns of four neighbouring tokens, so that four codes of a column make a word of the transposed block.  A block that
// the call completes takes its old tokens from the tail; one that stays open only gets its new tokens stored there, in a
// second launch where the first one reads old tokens of the same tail.
// Rows come in past the registers, all at once; the table entries, fetched by position, are what the rotation waits for.
// Bound: the arithmetic, then memory (24,967 tokens x 40 heads x 128 rotated and written: 767 MB in and out in 177 us,
// 4.3 TB/s; 227 with a division where a quotient lay near a half, 238 with rows in registers, 503 before pairs were turned once).
// The second launch: 1,560 tokens x 40 heads behind 24 others take 22.2 us, 15.7 behind none; the same thread block going on
// with the new open block instead took 26.6.
template <int DT, int D>
__global__ void __launch_bounds__(2 * D, 640 / D)
append_kernel(BlockArrays c, AppendSide k, AppendSide v, Rotation rot, int tokens, Sequences seqs, bool second_launch) {
  constexpr int PIECES = D / 8, PAIRS = PIECES / 2, THREADS = 2 * D, WARPS = THREADS / 32;
  __shared__ __align__(16) uint4 k_rows[NKV_BLOCK * PIECES], v_rows[NKV_BLOCK * PIECES];   // a thread's own pieces, on their way in
  __shared__ uint32_t reduced[2][WARPS];
  uint32_t* const words = reinterpret_cast<uint32_t*>(k_rows);   // later: [column][16 words of 4 tokens], word index xor column / 8
  const int b = blockIdx.z, h = blockIdx.y;
  const int length = seqs.length[b], count = seqs.count[b];
  const int block = append_block(length, count, blockIdx.x, second_launch);
  if (block < 0) return;
  const int t0 = block * NKV_BLOCK;         // first token of the block
  const int held = max(0, length - t0), filled = min(NKV_BLOCK, length + count - t0);
  const bool whole = filled == NKV_BLOCK;
  const int lane = threadIdx.x & 31;
  const size_t bh = static_cast<size_t>(b) * c.kv_heads + h;
  uint16_t* const k_tail = static_cast<uint16_t*>(c.k_tail) + bh * NKV_BLOCK * D;
  uint16_t* const v_tail = static_cast<uint16_t*>(c.v_tail) + bh * NKV_BLOCK * D;
  const int pair = threadIdx.x % PAIRS, d_lo = pair * 8, d_hi = d_lo + D / 2;
  const int k_token = threadIdx.x / PAIRS;   // and 32 on
  const int piece = threadIdx.x % PIECES, group = threadIdx.x / PIECES, d0 = piece * 8;
  const bool partners = rot.dim == D && rot.layout == NKV_ROTARY_HALF && k.vector != 0;
  const bool k_ahead = k.vector != 0 && (partners || rot.dim == 0), v_ahead = v.vector != 0;
  const uint16_t* const k_row = k.x + b * k.stride_batch + h * k.stride_head;
  const uint16_t* const v_row = v.x + b * v.stride_batch + h * v.stride_head;
  // ---- all rows that start on 16 bytes, past the registers and at once
  if (k_ahead)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = k_token + 32 * i;
      if (t < held || t >= filled) continue;
      const uint16_t* const row = k_row + static_cast<long long>(t0 + t - length) * k.stride_token;
      copy16_async(&k_rows[t * PIECES + pair], row + d_lo);
      copy16_async(&k_rows[t * PIECES + pair + PAIRS], row + d_hi);
    }
  if (v_ahead)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * group + i;
      if (t < held || t >= filled) continue;
      copy16_async(&v_rows[t * PIECES + piece], v_row + static_cast<long long>(t0 + t - length) * v.stride_token + d0);
    }
  int position[2] = {0, 0};
  if (rot.dim > 0)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = k_token + 32 * i;
      if (t >= held && t < filled) position[i] = __ldg(rot.positions + static_cast<size_t>(b) * tokens + (t0 + t - length));
    }
  // ---- K
  uint4 kp[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = k_token + 32 * i;
    kp[i][0] = kp[i][1] = make_uint4(0, 0, 0, 0);
    if (t >= held && t < filled) {
      if (partners) {
        float2 cs[8];
        turns_of(rot, position[i], d_lo, cs);
        copies_landed();
        float x[8], y[8];
        Piece<DT>::unpack(k_rows[t * PIECES + pair], x);
        Piece<DT>::unpack(k_rows[t * PIECES + pair + PAIRS], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x0 = x[e], x1 = y[e];
          x[e] = turn_first(x0, x1, cs[e]);
          y[e] = turn_second(x0, x1, cs[e]);
        }
        kp[i][0] = Piece<DT>::pack(x);
        kp[i][1] = Piece<DT>::pack(y);
      } else if (k_ahead) {
        copies_landed();
        kp[i][0] = k_rows[t * PIECES + pair];
        kp[i][1] = k_rows[t * PIECES + pair + PAIRS];
      } else {
        const uint16_t* const row = k_row + static_cast<long long>(t0 + t - length) * k.stride_token;
        kp[i][0] = rot.dim > 0 ? rotated_piece<DT>(row, d_lo, k.vector != 0, rot, position[i]) : load_piece<DT>(row, d_lo, k.vector != 0);
        kp[i][1] = rot.dim > 0 ? rotated_piece<DT>(row, d_hi, k.vector != 0, rot, position[i]) : load_piece<DT>(row, d_hi, k.vector != 0);
      }
    } else if (whole && t < held) {
      kp[i][0] = *reinterpret_cast<const uint4*>(k_tail + t * D + d_lo);
      kp[i][1] = *reinterpret_cast<const uint4*>(k_tail + t * D + d_hi);
    }
  }
  // ---- V
  copies_landed();
  uint4 vp[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * group + i;
    vp[i] = make_uint4(0, 0, 0, 0);
    if (t >= held && t < filled) {
      vp[i] = v_ahead ? v_rows[t * PIECES + piece] : load_piece<DT>(v_row + static_cast<long long>(t0 + t - length) * v.stride_token, d0, false);
    } else if (whole && t < held) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = v_tail[(d0 + 2 * e) * NKV_BLOCK + t] | (static_cast<uint32_t>(v_tail[(d0 + 2 * e + 1) * NKV_BLOCK + t]) << 16);
      vp[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (!whole) {
    // a token with an element that is not finite: NaN keys, zero values
    __shared__ uint32_t bad_tokens[2];
    if (threadIdx.x < 2) bad_tokens[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (not_finite<DT>(kp[i][0]) || not_finite<DT>(kp[i][1])) atomicOr(&bad_tokens[i], 1u << k_token);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (not_finite<DT>(vp[i])) atomicOr(&bad_tokens[(4 * group + i) >> 5], 1u << ((4 * group + i) & 31));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (bad_tokens[i] >> k_token & 1) kp[i][0] = kp[i][1] = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (bad_tokens[(4 * group + i) >> 5] >> ((4 * group + i) & 31) & 1) vp[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = k_token + 32 * i;
      if (t < held || t >= filled) continue;
      *reinterpret_cast<uint4*>(k_tail + t * D + d_lo) = kp[i][0];
      *reinterpret_cast<uint4*>(k_tail + t * D + d_hi) = kp[i][1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * group + i;
      if (t < held || t >= filled) continue;
      const uint32_t w[4] = {vp[i].x, vp[i].y, vp[i].z, vp[i].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) v_tail[(d0 + e) * NKV_BLOCK + t] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
    }
    return;
  }
  // ---- the block's scales; one with an element that is not finite: NaN for K, zero for V
  uint32_t k_most = __vmaxu2(__vmaxu2(magnitude(kp[0][0]), magnitude(kp[0][1])), __vmaxu2(magnitude(kp[1][0]), magnitude(kp[1][1])));
  uint32_t v_most = __vmaxu2(__vmaxu2(magnitude(vp[0]), magnitude(vp[1])), __vmaxu2(magnitude(vp[2]), magnitude(vp[3])));
  k_most = __reduce_max_sync(0xffffffffu, max(k_most & 0xFFFFu, k_most >> 16));
  v_most = __reduce_max_sync(0xffffffffu, max(v_most & 0xFFFFu, v_most >> 16));
  if (lane == 0) {
    reduced[0][threadIdx.x / 32] = k_most;
    reduced[1][threadIdx.x / 32] = v_most;
  }
  __syncthreads();
  k_most = __reduce_max_sync(0xffffffffu, reduced[0][lane % WARPS]);
  v_most = __reduce_max_sync(0xffffffffu, reduced[1][lane % WARPS]);
  const bool bad = max(k_most, v_most) >= NOT_FINITE<DT>;
  const float k_scale = bad ? 0.f : __fdiv_rn(unpack2<DT>(k_most).x, 127.f), v_scale = bad ? 0.f : __fdiv_rn(unpack2<DT>(v_most).x, 127.f);
  const Quotient k_by(k_scale), v_by(v_scale);
  const size_t slot = slot_of(c, bh, block);
  if (threadIdx.x == 0) {
    c.scales[2 * slot] = bad ? CUDART_NAN_F : k_scale;
    c.scales[2 * slot + 1] = v_scale;
  }
  // ---- codes: K rows as they are, V through shared memory
  uint8_t* const k_codes = c.k_codes + slot * NKV_BLOCK * D;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x[8];
      uint2 w = make_uint2(0x80808080u, 0x80808080u);
      Piece<DT>::unpack(kp[i][half], x);
      if (k_scale > 0.f) w = codes_of(x, k_by);
      *reinterpret_cast<uint2*>(k_codes + (k_token + 32 * i) * D + (half ? d_hi : d_lo)) = w;
    }
  uint2 vw[4];   // codes of the thread's columns, token by token
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[8];
    Piece<DT>::unpack(vp[i], x);
    vw[i] = v_scale > 0.f ? codes_of(x, v_by) : make_uint2(0x80808080u, 0x80808080u);
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {   // four columns: a 4 x 4 transposition of bytes
    const uint32_t w0 = half ? vw[0].y : vw[0].x, w1 = half ? vw[1].y : vw[1].x, w2 = half ? vw[2].y : vw[2].x, w3 = half ? vw[3].y : vw[3].x;
    const uint32_t a = __byte_perm(w0, w1, 0x5140), e = __byte_perm(w0, w1, 0x7362);
    const uint32_t f = __byte_perm(w2, w3, 0x5140), g = __byte_perm(w2, w3, 0x7362);
    const int col = d0 + 4 * half, at = group ^ (piece & 15);
    words[(col + 0) * 16 + at] = __byte_perm(a, f, 0x5410);
    words[(col + 1) * 16 + at] = __byte_perm(a, f, 0x7632);
    words[(col + 2) * 16 + at] = __byte_perm(e, g, 0x5410);
    words[(col + 3) * 16 + at] = __byte_perm(e, g, 0x7632);
  }
  __syncthreads();
  uint32_t* const v_codes = reinterpret_cast<uint32_t*>(c.v_codes + slot * NKV_BLOCK * D);
#pragma unroll
  for (int i = 0; i < D * 16 / THREADS; ++i) {
    const int w = threadIdx.x + i * THREADS;
    v_codes[w] = words[(w & ~15) + ((w & 15) ^ ((w >> 7) & 15))];
  }
}

// ---- read ------------------------------------------------------------------------------------------------------

// One block of one sequence and head as rows; the same split as append, the other way round.  Bound: memory (24,960 tokens x 40
// heads x 128: 767 MB in and out in 124 us, 6.2 TB/s).
template <int DT, int D>
__global__ void __launch_bounds__(2 * D)
read_kernel(BlockArrays c, int start, int stop, uint16_t* k_out, uint16_t* v_out, Sequences seqs) {
  constexpr int PIECES = D / 8, THREADS = 2 * D;
  __shared__ uint32_t words[D * 16];
  const int b = blockIdx.z, h = blockIdx.y, length = seqs.length[b];
  const int block = start / NKV_BLOCK + blockIdx.x, t0 = block * NKV_BLOCK;
  const int piece = threadIdx.x % PIECES, group = threadIdx.x / PIECES, d0 = piece * 8;
  const size_t bh = static_cast<size_t>(b) * c.kv_heads + h;
  const bool whole = t0 + NKV_BLOCK <= length;
  uint4 kp[4], vp[4];
  if (whole) {
    const size_t slot = slot_of(c, bh, block);
    const float2 scale = *reinterpret_cast<const float2*>(c.scales + 2 * slot);
    const uint32_t* v_codes = reinterpret_cast<const uint32_t*>(c.v_codes + slot * NKV_BLOCK * D);
#pragma unroll
    for (int i = 0; i < D * 16 / THREADS; ++i) {
      const int w = threadIdx.x + i * THREADS;
      words[(w & ~15) + ((w & 15) ^ ((w >> 7) & 15))] = __ldg(v_codes + w);
    }
    __syncthreads();
    uint32_t column[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) column[e] = words[(d0 + e) * 16 + (group ^ (piece & 15))];
    const uint8_t* k_codes = c.k_codes + slot * NKV_BLOCK * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint2 raw = __ldg(reinterpret_cast<const uint2*>(k_codes + (4 * group + i) * D + d0));
      float x[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = code_value(((e < 4 ? raw.x : raw.y) >> (8 * (e & 3))) & 0xFFu) * scale.x;
        y[e] = code_value((column[e] >> (8 * i)) & 0xFFu) * scale.y;
      }
      kp[i] = Piece<DT>::pack(x);
      vp[i] = Piece<DT>::pack(y);
    }
  } else {
    const uint16_t* k_tail = static_cast<const uint16_t*>(c.k_tail) + bh * NKV_BLOCK * D;
    const uint16_t* v_tail = static_cast<const uint16_t*>(c.v_tail) + bh * NKV_BLOCK * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * group + i;
      kp[i] = vp[i] = make_uint4(0, 0, 0, 0);
      if (t0 + t >= length) continue;
      kp[i] = *reinterpret_cast<const uint4*>(k_tail + t * D + d0);
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = v_tail[(d0 + 2 * e) * NKV_BLOCK + t] | (static_cast<uint32_t>(v_tail[(d0 + 2 * e + 1) * NKV_BLOCK + t]) << 16);
      vp[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + 4 * group + i;
    if (t < start || t >= stop) continue;
    const size_t at = ((static_cast<size_t>(b) * (stop - start) + (t - start)) * c.kv_heads + h) * D + d0;
    *reinterpret_cast<uint4*>(k_out + at) = kp[i];
    *reinterpret_cast<uint4*>(v_out + at) = vp[i];
  }
}

// ---- evict -----------------------------------------------------------------------------------------------------

// larger weight = larger key; NaN above all numbers, -0 as 0
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t bits = __float_as_uint(w + 0.f);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

constexpr int EVICT_THREADS = 256;

// One table row per thread block.  The smallest kept key is found digit by digit (8 bits, most significant first) from
// counts of the candidates that agree with the digits found so far; then one pass in index order keeps what lies
// above it and the first of its equals, and writes every entry to its place.
__global__ void __launch_bounds__(EVICT_THREADS)
evict_kernel(const float* weights, const int32_t* table, int blocks, int keep, int sinks, int recent, float* weights_out,
             int32_t* table_out, Sequences seqs) {
  __shared__ int counts[256];
  __shared__ int warp_eq[EVICT_THREADS / 32], warp_kept[EVICT_THREADS / 32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int full = seqs.length[blockIdx.y], partial = seqs.count[blockIdx.y];
  const size_t base = (static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x) * blocks;
  weights += base; table += base; weights_out += base; table_out += base;
  const int lo = min(sinks, full), hi = max(lo, full - recent);   // candidates [lo, hi)
  const int forced = lo + (full - hi);
  const int live = full + partial;
  uint32_t threshold = 0;
  int equals = 0;                       // entries at the threshold that stay
  const bool all = keep >= full;
  if (!all) {
    int need = keep - forced;           // candidates that stay
    if (need > 0) {
      for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += EVICT_THREADS) counts[i] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (int i = lo + tid; i < hi; i += EVICT_THREADS) {
          const uint32_t key = weight_key(weights[i]);
          if ((key & mask) == threshold) atomicAdd(&counts[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (warp == 0) {
          // 8 digits per lane, from the largest down: lane l has digits 255 - 8 l ... 248 - 8 l
          int own = 0;
          for (int i = 0; i < 8; ++i) own += counts[255 - 8 * lane - i];
          int above = own;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, above, o);
            if (lane >= o) above += up;
          }
          above -= own;
          if (above < need && above + own >= need) {
            int left = need - above, digit = 255 - 8 * lane;
            while (left > counts[digit]) left -= counts[digit--];
            s_prefix = threshold | (static_cast<uint32_t>(digit) << shift);
            s_need = left;
          }
        }
        __syncthreads();
        threshold = s_prefix;
        need = s_need;
      }
      equals = need;
    } else {
      threshold = 0xFFFFFFFFu;          // nothing lies above it and none of its equals stays
    }
  }
  const int kept_total = (all ? full : keep) + partial;
  int eq_before = 0, kept_before = 0;
  for (int start = 0; start < blocks; start += EVICT_THREADS) {
    const int i = start + tid;
    const bool in = i < blocks;
    const float w = in && i < live ? weights[i] : 0.f;
    const uint32_t key = weight_key(w);
    const bool candidate = in && i >= lo && i < hi;
    const bool eq = !all && candidate && key == threshold;
    const uint32_t eq_mask = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) warp_eq[warp] = __popc(eq_mask);
    __syncthreads();
    int eq_rank = eq_before + __popc(eq_mask & ((1u << lane) - 1u)), eq_tile = 0;
#pragma unroll
    for (int k = 0; k < EVICT_THREADS / 32; ++k) {
      if (k < warp) eq_rank += warp_eq[k];
      eq_tile += warp_eq[k];
    }
    const bool kept = in && i < live && (all || !candidate || key > threshold || (eq && eq_rank < equals));
    const uint32_t kept_mask = __ballot_sync(0xffffffffu, kept);
    if (lane == 0) warp_kept[warp] = __popc(kept_mask);
    __syncthreads();
    int kept_rank = kept_before + __popc(kept_mask & ((1u << lane) - 1u)), kept_tile = 0;
#pragma unroll
    for (int k = 0; k < EVICT_THREADS / 32; ++k) {
      if (k < warp) kept_rank += warp_kept[k];
      kept_tile += warp_kept[k];
    }
    if (in) {
      const int to = i >= live ? i : (kept ? kept_rank : kept_total + i - kept_rank);
      table_out[to] = table[i];
      weights_out[to] = kept ? w : 0.f;
    }
    eq_before += eq_tile;
    kept_before += kept_tile;
  }
}

// The same for rows of 257 to 2,048 entries, whose keys stay in registers, sixteen neighbouring entries to a thread.  The
// digits begin at the highest bit in which keys differ (weights share most of their exponents, and counts of equal digits
// collide), and end as soon as all that is left of a digit stays.  Two prefix sums then place every entry.  32 x 40 rows
// of 1,564: 18.6 us, 25.6 with the kernel above, which has the longer rows (32 x 40 of 2,048 here 19.6 us, of 2,100 there 29.3, of
// 4,096 53).
constexpr int SMALL_THREADS = 128, EVICT_ITEMS = 16;
__global__ void __launch_bounds__(SMALL_THREADS)
evict_small_kernel(const float* weights, const int32_t* table, int blocks, int keep, int sinks, int recent, float* weights_out,
                   int32_t* table_out, Sequences seqs) {
  constexpr int WARPS = SMALL_THREADS / 32;
  __shared__ float staged[SMALL_THREADS * (EVICT_ITEMS + 1)];
  __shared__ int32_t slots[SMALL_THREADS * (EVICT_ITEMS + 1)];
  __shared__ uint16_t order[SMALL_THREADS * EVICT_ITEMS];
  __shared__ int counts[256];
  __shared__ uint32_t extremes[2][WARPS];
  __shared__ uint32_t s_threshold;
  __shared__ int s_need;
  __shared__ int sums[2][WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int full = seqs.length[blockIdx.y], partial = seqs.count[blockIdx.y];
  const size_t base = (static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x) * blocks;
  weights += base; table += base; weights_out += base; table_out += base;
  const int lo = min(sinks, full), hi = max(lo, full - recent);   // candidates [lo, hi)
  const int live = full + partial, kept_total = min(keep, full) + partial;
  // coalesced in, sixteen neighbours (one word of padding behind them) out
#pragma unroll 4
  for (int i = tid; i < blocks; i += SMALL_THREADS) {
    staged[i + i / EVICT_ITEMS] = weights[i];
    slots[i + i / EVICT_ITEMS] = table[i];
  }
  __syncthreads();
  uint32_t key[EVICT_ITEMS];
  uint32_t candidates = 0;
#pragma unroll
  for (int k = 0; k < EVICT_ITEMS; ++k) {
    const int i = tid * EVICT_ITEMS + k;
    key[k] = i < live ? weight_key(staged[tid * (EVICT_ITEMS + 1) + k]) : 0u;
    if (i >= lo && i < hi) candidates |= 1u << k;
  }
  int need = keep - (lo + full - hi);   // candidates that stay
  uint32_t threshold = 0xFFFFFFFFu;
  int equals = 0;                       // candidates at the threshold that stay; others stay above it
  const bool all = keep >= full;
  if (!all && need > 0) {
    uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
    for (int k = 0; k < EVICT_ITEMS; ++k)
      if (candidates >> k & 1) {
        most = max(most, key[k]);
        least = min(least, key[k]);
      }
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    if (lane == 0) {
      extremes[0][warp] = most;
      extremes[1][warp] = least;
    }
    counts[tid] = counts[tid + 128] = 0;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < WARPS; ++x) {
      most = max(most, extremes[0][x]);
      least = min(least, extremes[1][x]);
    }
    int top = 32 - __clz(most ^ least);            // bits that are still open
    threshold = top < 32 ? most >> top << top : 0u;
    equals = need;                                 // (all keys equal: the first of them)
#pragma unroll 1
    while (top > 0) {
      const int shift = max(0, top - 8);
      const uint32_t digits = (1u << (top - shift)) - 1u;
      const uint32_t prefix = top < 32 ? threshold >> top : 0u;
#pragma unroll
      for (int k = 0; k < EVICT_ITEMS; ++k)
        if ((candidates >> k & 1) && (top == 32 || key[k] >> top == prefix)) atomicAdd(&counts[(key[k] >> shift) & digits], 1);
      __syncthreads();
      if (warp == 0) {
        // 8 digits per lane, from the largest down: lane l has digits 255 - 8 l ... 248 - 8 l
        int own = 0, here[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          here[x] = counts[255 - 8 * lane - x];
          own += here[x];
        }
        int above = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, above, o);
          if (lane >= o) above += up;
        }
        above -= own;
        if (above < need && above + own >= need) {
          int left = need - above, digit = 255 - 8 * lane, inside = 0;
          bool found = false;
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (!found) {
              if (left <= here[x]) {
                found = true;
                inside = here[x];
                digit -= x;
              } else {
                left -= here[x];
              }
            }
          s_threshold = threshold | (static_cast<uint32_t>(digit) << shift);
          s_need = inside == left ? -1 : left;   // -1: everything of this digit stays
        }
      }
      __syncthreads();
      threshold = s_threshold;
      const int left = s_need;
      top = shift;
      if (left < 0) {                            // keys of the digit and above stay: none is compared further
        --threshold;                             // (a key of 0 would be -NaN's: there is none)
        equals = 0;
        break;
      }
      need = equals = left;
      counts[tid] = counts[tid + 128] = 0;
      __syncthreads();
    }
  }
  // exclusive prefix sum over the thread block
  auto before = [&](int own, int which) {
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) sums[which][warp] = sum;
    __syncthreads();
    int first = sum - own;
#pragma unroll
    for (int x = 0; x < WARPS; ++x)
      if (x < warp) first += sums[which][x];
    return first;
  };
  uint32_t eq = 0, kept = 0;
#pragma unroll
  for (int k = 0; k < EVICT_ITEMS; ++k)
    if ((candidates >> k & 1) && key[k] == threshold) eq |= 1u << k;
  int rank = before(__popc(eq), 0);
#pragma unroll
  for (int k = 0; k < EVICT_ITEMS; ++k) {
    const int i = tid * EVICT_ITEMS + k;
    const bool stays = all || !(candidates >> k & 1) || key[k] > threshold || ((eq >> k & 1) && rank < equals);
    if (i < live && stays) kept |= 1u << k;
    rank += eq >> k & 1;
  }
  int at = before(__popc(kept), 1);
#pragma unroll
  for (int k = 0; k < EVICT_ITEMS; ++k) {
    const int i = tid * EVICT_ITEMS + k;
    if (i < blocks) {
      const bool stays = kept >> k & 1;
      const int to = i >= live ? i : (stays ? at : kept_total + i - at);
      order[to] = tid * (EVICT_ITEMS + 1) + k;
      at += stays;
    }
  }
  __syncthreads();
#pragma unroll 4
  for (int i = tid; i < blocks; i += SMALL_THREADS) {   // and coalesced out
    table_out[i] = slots[order[i]];
    weights_out[i] = i < kept_total ? staged[order[i]] : 0.f;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// ---- host ------------------------------------------------------------------------------------------------------

Sequences sequences_of(const nkv_block_cache& c, int first, int count, const int32_t* counts, int tokens) {
  Sequences s;
  for (int i = 0; i < count; ++i) {
    s.length[i] = c.lengths[first + i];
    s.count[i] = counts ? counts[first + i] : tokens;
  }
  return s;
}

BlockArrays block_arrays(const nkv_block_cache& c, int first) {
  const size_t heads = static_cast<size_t>(first) * c.kv_heads, slots = heads * c.blocks;
  const size_t block = static_cast<size_t>(NKV_BLOCK) * c.head_dim;
  BlockArrays a;
  a.k_codes = c.k_codes + slots * block;
  a.v_codes = c.v_codes + slots * block;
  a.scales = c.scales + 2 * slots;
  a.table = c.table + slots;
  a.k_tail = static_cast<uint8_t*>(c.k_tail) + heads * block * 2;
  a.v_tail = static_cast<uint8_t*>(c.v_tail) + heads * block * 2;
  a.kv_heads = c.kv_heads;
  a.blocks = c.blocks;
  return a;
}

int rotary(const nkv_tokens& x, void* out_x, const nkv_tokens* y, void* out_y, int dtype, int batch, int tokens, int d,
           const nkv_rotation& rotation, bool transposed, cudaStream_t stream) {
  const RotarySide a{x.data, out_x, x.stride_batch, x.stride_token, x.stride_head, x.heads};
  const RotarySide b = y ? RotarySide{y->data, out_y, y->stride_batch, y->stride_token, y->stride_head, y->heads}
                         : RotarySide{nullptr, nullptr, 0, 0, 0, 0};
  const Rotation rot{reinterpret_cast<const float2*>(rotation.table), rotation.positions, rotation.rows, rotation.rotary_dim,
                     rotation.layout};
  const long long rows = static_cast<long long>(batch) * tokens;
  if (rows == 0 || a.heads + b.heads == 0) return NKV_OK;
  const int n = dtype == NKV_F32 ? 4 : 8;   // elements of 16 bytes
  auto fits = [&](const RotarySide& s) {
    return s.heads == 0 || (aligned16(s.x) && aligned16(s.out) && s.stride_batch % n == 0 && s.stride_token % n == 0 &&
                            s.stride_head % n == 0);
  };
  const bool vector = d % (2 * n) == 0 && rotation.rotary_dim % (2 * n) == 0 && fits(a) && fits(b);
  if (vector) {
    const int units = d / (2 * n);
    auto run = [&](auto kernel, int heads) {
      const long long total = rows * units * (ceil_div(a.heads, heads) + ceil_div(b.heads, heads));
      kernel<<<static_cast<unsigned>((total + 255) / 256), 256, 0, stream>>>(a, b, batch, tokens, d, rot, transposed);
    };
    // four heads per thread share the table entries once that still leaves every SM a block of threads (one / four heads per
    // thread, bf16: 32 tokens x 48 heads of 128 2.5 / 3.0 us, 1,024 x 32 10.2 / 8.2, 24,960 x 24 77.8 / 57.3)
    const bool many = rows * units * (a.heads + b.heads) >= 4ll * 256 * sm_count();
    if (dtype == NKV_F32) many ? run(rotary_kernel<NKV_F32, 4>, 4) : run(rotary_kernel<NKV_F32, 1>, 1);
    else if (dtype == NKV_BF16) many ? run(rotary_kernel<NKV_BF16, 4>, 4) : run(rotary_kernel<NKV_BF16, 1>, 1);
    else many ? run(rotary_kernel<NKV_F16, 4>, 4) : run(rotary_kernel<NKV_F16, 1>, 1);
    NKV_LAUNCH_CHECK("rotary_kernel");
    return NKV_OK;
  }
  const long long total = rows * (a.heads + b.heads) * ((d + 1) / 2);
  auto kernel = dtype == NKV_F32 ? rotary_pairs_kernel<NKV_F32>
                                 : (dtype == NKV_BF16 ? rotary_pairs_kernel<NKV_BF16> : rotary_pairs_kernel<NKV_F16>);
  kernel<<<static_cast<unsigned>((total + 255) / 256), 256, 0, stream>>>(a, b, batch, tokens, d, rot, transposed);
  NKV_LAUNCH_CHECK("rotary_pairs_kernel");
  return NKV_OK;
}

int block_append(const nkv_block_cache& c, const nkv_tokens& k, const nkv_tokens& v, int tokens, const int32_t* counts,
                 const nkv_rotation* rotation, cudaStream_t stream) {
  auto side = [](const nkv_tokens& x) {
    AppendSide s{static_cast<const uint16_t*>(x.data), x.stride_batch, x.stride_token, x.stride_head, 0};
    s.vector = aligned16(x.data) && x.stride_batch % 8 == 0 && x.stride_token % 8 == 0 && x.stride_head % 8 == 0;
    return s;
  };
  AppendSide ks = side(k), vs = side(v);
  Rotation rot{nullptr, nullptr, 0, 0, 0};
  if (rotation)
    rot = Rotation{reinterpret_cast<const float2*>(rotation->table), rotation->positions, rotation->rows, rotation->rotary_dim,
                   rotation->layout};
  for (int first = 0; first < c.batch; first += MAX_SEQUENCES) {
    const int n = min(MAX_SEQUENCES, c.batch - first);
    const Sequences seqs = sequences_of(c, first, n, counts, tokens);
    int touched = 0;
    bool twice = false;
    for (int i = 0; i < n; ++i) {
      touched = max(touched, append_blocks(seqs.length[i], seqs.count[i]));
      twice |= append_twice(seqs.length[i], seqs.count[i]);
    }
    if (touched == 0) continue;
    AppendSide kf = ks, vf = vs;
    kf.x += first * ks.stride_batch;
    vf.x += first * vs.stride_batch;
    Rotation rf = rot;
    if (rotation) rf.positions += static_cast<size_t>(first) * tokens;
    auto kernel = c.head_dim == 128 ? (c.dtype == NKV_BF16 ? append_kernel<NKV_BF16, 128> : append_kernel<NKV_F16, 128>)
                                    : (c.dtype == NKV_BF16 ? append_kernel<NKV_BF16, 64> : append_kernel<NKV_F16, 64>);
    for (int launch = 0; launch < (twice ? 2 : 1); ++launch) {
      const dim3 grid(launch ? 1 : touched, c.kv_heads, n);
      kernel<<<grid, 2 * c.head_dim, 0, stream>>>(block_arrays(c, first), kf, vf, rf, tokens, seqs, launch == 1);
      NKV_LAUNCH_CHECK("append_kernel");
    }
  }
  return NKV_OK;
}

int block_read(const nkv_block_cache& c, int start, int stop, void* k_out, void* v_out, cudaStream_t stream) {
  const int touched = (stop - 1) / NKV_BLOCK - start / NKV_BLOCK + 1;
  for (int first = 0; first < c.batch; first += MAX_SEQUENCES) {
    const int n = min(MAX_SEQUENCES, c.batch - first);
    const Sequences seqs = sequences_of(c, first, n, nullptr, 0);
    const size_t skip = static_cast<size_t>(first) * (stop - start) * c.kv_heads * c.head_dim;
    auto kernel = c.head_dim == 128 ? (c.dtype == NKV_BF16 ? read_kernel<NKV_BF16, 128> : read_kernel<NKV_F16, 128>)
                                    : (c.dtype == NKV_BF16 ? read_kernel<NKV_BF16, 64> : read_kernel<NKV_F16, 64>);
    kernel<<<dim3(touched, c.kv_heads, n), 2 * c.head_dim, 0, stream>>>(
        block_arrays(c, first), start, stop, static_cast<uint16_t*>(k_out) + skip, static_cast<uint16_t*>(v_out) + skip, seqs);
    NKV_LAUNCH_CHECK("read_kernel");
  }
  return NKV_OK;
}

int block_evict(const float* weights, const int32_t* table, const int32_t* full, const int32_t* partial, int batch, int kv_heads,
                int blocks, int keep, int sinks, int recent, float* weights_out, int32_t* table_out, cudaStream_t stream) {
  for (int first = 0; first < batch; first += MAX_SEQUENCES) {
    const int n = min(MAX_SEQUENCES, batch - first);
    Sequences seqs;
    for (int i = 0; i < n; ++i) {
      seqs.length[i] = full[first + i];
      seqs.count[i] = partial[first + i];
    }
    const size_t skip = static_cast<size_t>(first) * kv_heads * blocks;
    // one round of the plain kernel's threads: it is shorter there (8 rows of 132: 4.4 us, 5.9)
    const bool small = blocks > EVICT_THREADS && blocks <= EVICT_ITEMS * SMALL_THREADS;
    auto kernel = small ? evict_small_kernel : evict_kernel;
    kernel<<<dim3(kv_heads, n), small ? SMALL_THREADS : EVICT_THREADS, 0, stream>>>(weights + skip, table + skip, blocks, keep, sinks, recent,
                                                            weights_out + skip, table_out + skip, seqs);
    NKV_LAUNCH_CHECK("evict_kernel");
  }
  return NKV_OK;
}

}  // namespace nkv
