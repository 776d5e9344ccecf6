// The 8-bit block cache without its attention: tokens in (append), rows out (read), blocks freed (evict), and the rotary
// positions of queries and keys.  All four are bound by memory, the small calls by the latency of a launch.
#include "nkv_block.cuh"
#include "nkv_internal.h"

namespace nkv {
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
// HEADS heads per thread share the table entries; one where the call is short of threads.
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

// Code (plus 128) of x for a block scale: rint(x / scale).  x * inv is within 2 ulp of the IEEE quotient, less than 1e-4 at
// 127, so only products that near to a half take the division; rint is the addition of 1.5 * 2^23 + 128, whose low
// byte is the code.  A scale too small for its reciprocal divides always, and clamps: such a scale is a subnormal
// number, a coarse multiple of the maximum / 127.
__device__ __forceinline__ uint32_t code_of(float x, float scale, float inv) {
  constexpr float MAGIC = 12583040.0f;
  float q = x * inv;
  float t = __fadd_rn(q, MAGIC);
  if (fabsf(q - (t - MAGIC)) > 0.4999f || !(inv < 1e37f)) {
    q = fminf(fmaxf(__fdiv_rn(x, scale), -127.f), 127.f);
    t = __fadd_rn(q, MAGIC);
  }
  return __float_as_uint(t) & 0xFFu;
}

struct AppendSide {
  const uint16_t* x;
  long long stride_batch, stride_token, stride_head;
  int vector;   // rows and strides on 16 bytes
};

// One block of one sequence and head that the call touches.  A thread holds eight columns of four neighbouring tokens, so
// that four codes of a column make a word of the transposed V block.  A block that the call completes takes its old
// tokens from the tail; one that stays open only gets its new tokens stored there.
template <int DT, int D>
__global__ void __launch_bounds__(2 * D)
append_kernel(BlockArrays c, AppendSide k, AppendSide v, Rotation rot, int tokens, Sequences seqs) {
  constexpr int PIECES = D / 8, THREADS = 2 * D;
  __shared__ uint32_t words[D * 16];        // [column][16 words of 4 tokens], word index xor column / 8
  __shared__ float reduced[2][THREADS / 32];
  const int b = blockIdx.z, h = blockIdx.y;
  const int length = seqs.length[b], count = seqs.count[b];
  const int block = length / NKV_BLOCK + blockIdx.x;
  const int t0 = block * NKV_BLOCK;         // first token of the block
  if (t0 >= length + count || block >= c.blocks || count <= 0) return;
  const int held = max(0, length - t0), filled = min(NKV_BLOCK, length + count - t0);
  const bool whole = filled == NKV_BLOCK;
  const int piece = threadIdx.x % PIECES, group = threadIdx.x / PIECES, lane = threadIdx.x & 31;
  const int d0 = piece * 8;
  const size_t bh = static_cast<size_t>(b) * c.kv_heads + h;
  uint16_t* const k_tail = static_cast<uint16_t*>(c.k_tail) + bh * NKV_BLOCK * D;
  uint16_t* const v_tail = static_cast<uint16_t*>(c.v_tail) + bh * NKV_BLOCK * D;
  uint4 kp[4], vp[4];
  uint32_t bad_tokens = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * group + i;
    kp[i] = vp[i] = make_uint4(0, 0, 0, 0);
    if (t >= held && t < filled) {
      const long long n = t0 + t - length;   // token of the call
      const uint16_t* kr = k.x + b * k.stride_batch + n * k.stride_token + h * k.stride_head;
      const uint16_t* vr = v.x + b * v.stride_batch + n * v.stride_token + h * v.stride_head;
      const int position = rot.dim > 0 && d0 < rot.dim ? __ldg(rot.positions + static_cast<size_t>(b) * tokens + n) : 0;
      kp[i] = rot.dim > 0 ? rotated_piece<DT>(kr, d0, k.vector != 0, rot, position) : load_piece<DT>(kr, d0, k.vector != 0);
      vp[i] = load_piece<DT>(vr, d0, v.vector != 0);
    } else if (whole && t < held) {
      kp[i] = *reinterpret_cast<const uint4*>(k_tail + t * D + d0);
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = v_tail[(d0 + 2 * e) * NKV_BLOCK + t] | (static_cast<uint32_t>(v_tail[(d0 + 2 * e + 1) * NKV_BLOCK + t]) << 16);
      vp[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // a token with an element that is not finite: NaN keys, zero values (all pieces of a token lie in one warp)
    const uint32_t flags = __ballot_sync(0xffffffffu, not_finite<DT>(kp[i]) || not_finite<DT>(vp[i]));
    const uint32_t mine = (PIECES == 32 ? 0xffffffffu : ((1u << PIECES) - 1u) << (lane / PIECES * PIECES));
    if (flags & mine) {
      kp[i] = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
      vp[i] = make_uint4(0, 0, 0, 0);
      bad_tokens |= 1u << i;
    }
  }
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * group + i;
      if (t < held || t >= filled) continue;
      *reinterpret_cast<uint4*>(k_tail + t * D + d0) = kp[i];
      const uint32_t w[4] = {vp[i].x, vp[i].y, vp[i].z, vp[i].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) v_tail[(d0 + e) * NKV_BLOCK + t] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
    }
    return;
  }
  // ---- the block's scales
  float kmax = 0.f, vmax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[8];
    if (!(bad_tokens & (1u << i))) {
      Piece<DT>::unpack(kp[i], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) kmax = fmaxf(kmax, fabsf(x[e]));
    }
    Piece<DT>::unpack(vp[i], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) vmax = fmaxf(vmax, fabsf(x[e]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, o));
    vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
  }
  if (lane == 0) {
    reduced[0][threadIdx.x / 32] = kmax;
    reduced[1][threadIdx.x / 32] = vmax;
  }
  const bool bad = __syncthreads_or(bad_tokens != 0) != 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    kmax = fmaxf(kmax, reduced[0][w]);
    vmax = fmaxf(vmax, reduced[1][w]);
  }
  const float k_scale = bad ? 0.f : __fdiv_rn(kmax, 127.f), v_scale = bad ? 0.f : __fdiv_rn(vmax, 127.f);
  const float k_inv = __frcp_rn(k_scale), v_inv = __frcp_rn(v_scale);
  const size_t slot = slot_of(c, bh, block);
  if (threadIdx.x == 0) {
    c.scales[2 * slot] = bad ? CUDART_NAN_F : k_scale;
    c.scales[2 * slot + 1] = v_scale;
  }
  // ---- codes: K rows as they are, V through shared memory
  uint8_t* const k_codes = c.k_codes + slot * NKV_BLOCK * D;
  uint32_t column[8];   // four tokens of each of this thread's columns
#pragma unroll
  for (int e = 0; e < 8; ++e) column[e] = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[8];
    uint32_t word[2] = {0x80808080u, 0x80808080u};
    if (k_scale > 0.f) {
      Piece<DT>::unpack(kp[i], x);
      word[0] = word[1] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) word[e / 4] |= code_of(x[e], k_scale, k_inv) << (8 * (e & 3));
    }
    *reinterpret_cast<uint2*>(k_codes + (4 * group + i) * D + d0) = make_uint2(word[0], word[1]);
    Piece<DT>::unpack(vp[i], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) column[e] |= (v_scale > 0.f ? code_of(x[e], v_scale, v_inv) : 128u) << (8 * i);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) words[(d0 + e) * 16 + (group ^ (piece & 15))] = column[e];
  __syncthreads();
  uint32_t* const v_codes = reinterpret_cast<uint32_t*>(c.v_codes + slot * NKV_BLOCK * D);
#pragma unroll
  for (int i = 0; i < D * 16 / THREADS; ++i) {
    const int w = threadIdx.x + i * THREADS;
    v_codes[w] = words[(w & ~15) + ((w & 15) ^ ((w >> 7) & 15))];
  }
}

// ---- read ------------------------------------------------------------------------------------------------------

// One block of one sequence and head as rows; the same split as append, the other way round.
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

// Sequences of a launch, passed by value: no upload, no device state that a call would have to order against others.
Sequences sequences_of(const nkv_block_cache& c, int first, int count, const int32_t* counts, int tokens) {
  Sequences s;
  for (int i = 0; i < count; ++i) {
    s.length[i] = c.lengths[first + i];
    s.count[i] = counts ? counts[first + i] : tokens;
  }
  return s;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// ---- host ------------------------------------------------------------------------------------------------------

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
    // four heads per thread share the table entries once that still leaves every SM its 2,048 threads
    const bool many = rows * units * (a.heads + b.heads) >= 4ll * 2048 * sm_count();
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
    for (int i = 0; i < n; ++i)
      if (seqs.count[i] > 0)
        touched = max(touched, (seqs.length[i] + seqs.count[i] - 1) / NKV_BLOCK - seqs.length[i] / NKV_BLOCK + 1);
    if (touched == 0) continue;
    AppendSide kf = ks, vf = vs;
    kf.x += first * ks.stride_batch;
    vf.x += first * vs.stride_batch;
    Rotation rf = rot;
    if (rotation) rf.positions += static_cast<size_t>(first) * tokens;
    const dim3 grid(touched, c.kv_heads, n);
    auto kernel = c.head_dim == 128 ? (c.dtype == NKV_BF16 ? append_kernel<NKV_BF16, 128> : append_kernel<NKV_F16, 128>)
                                    : (c.dtype == NKV_BF16 ? append_kernel<NKV_BF16, 64> : append_kernel<NKV_F16, 64>);
    kernel<<<grid, 2 * c.head_dim, 0, stream>>>(block_arrays(c, first), kf, vf, rf, tokens, seqs);
    NKV_LAUNCH_CHECK("append_kernel");
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
    evict_kernel<<<dim3(kv_heads, n), EVICT_THREADS, 0, stream>>>(weights + skip, table + skip, blocks, keep, sinks, recent,
                                                                  weights_out + skip, table_out + skip, seqs);
    NKV_LAUNCH_CHECK("evict_kernel");
  }
  return NKV_OK;
}

}  // namespace nkv
