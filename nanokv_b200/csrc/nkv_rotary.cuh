// Rotary positions and rows in 16-byte pieces, as the kernels that turn queries or keys share them.
#pragma once

#include "nkv_block.cuh"

namespace nkv {

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

}  // namespace nkv
