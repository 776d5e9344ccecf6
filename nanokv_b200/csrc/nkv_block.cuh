// What the kernels of the 8-bit block cache share.
#pragma once

#include <math_constants.h>

#include "nkv_common.cuh"

namespace nkv {

constexpr int MAX_SEQUENCES = 128;   // sequences of one launch; longer batches are cut

// Lengths and token counts of a launch's sequences, passed by value: no upload, no device state that a call would have to order
// against others.
struct Sequences {
  int32_t length[MAX_SEQUENCES];
  int32_t count[MAX_SEQUENCES];
};
// of `count` sequences from `first` on; counts NULL: `tokens` each
Sequences sequences_of(const nkv_block_cache& c, int first, int count, const int32_t* counts, int tokens);

// device arrays of nkv_block_cache from one of its sequences on
struct BlockArrays {
  uint8_t* k_codes;
  uint8_t* v_codes;
  float* scales;
  const int32_t* table;
  void* k_tail;
  void* v_tail;
  int kv_heads, blocks;
};
BlockArrays block_arrays(const nkv_block_cache& c, int first);

// slot of a logical block among all slots; an entry outside the row's slots is taken to its end, never followed out of the arrays
__device__ __forceinline__ size_t slot_of(const BlockArrays& c, size_t bh, int block) {
  return bh * c.blocks + min(static_cast<unsigned>(__ldg(c.table + bh * c.blocks + block)), static_cast<unsigned>(c.blocks - 1));
}

template <int DT> struct Elem { using type = uint16_t; };
template <> struct Elem<NKV_F32> { using type = float; };

// two 16-bit elements of a word, the even one in the low half
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (DT == NKV_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (DT == NKV_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// (a NaN among them is passed over, as by fmaxf)
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// value of a stored byte: 2^23 + byte is an fp32 number whose low mantissa bits are the byte
__device__ __forceinline__ float code_value(uint32_t byte) { return __uint_as_float(0x4B000000u | byte) - 8388736.0f; }

// ---- attention ----
// Shared memory by its own addresses: a dynamic buffer aligned by hand has a generic pointer, and 16-byte accesses through
// one are slower.
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// One call, from one of its sequences on.  The queries of a kv head are rows r = token * group + (head within the group).
struct Call {
  const uint16_t* q;
  long long q_batch, q_token, q_head;
  uint16_t* out;
  float* lse;
  float* partial;      // log2 of every (row, block)'s weight sum, or NULL: [sequence][kv head][most blocks][rows]
  float* weights;      // block weights to add to
  int tokens, heads, group, rows, causal, most_blocks;
  float scale_log2;    // scale * log2(e)
  int q_vector;        // the queries' rows start on 16 bytes
};

// tokens that row r of a sequence sees
__device__ __forceinline__ int visible_to(const Call& a, int length, int count, int r) {
  const int t = r / a.group;
  if (t >= count) return 0;
  return a.causal ? max(0, min(length, length - count + t + 1)) : length;
}

// dynamic shared memory allowed to a kernel: asked for once per kernel and device, not with every call (nkv_block_attn.cu)
cudaError_t allow_shared(const void* kernel, int bytes);

// few rows per kv head (nkv_block_step.cu)
bool block_step_supported(int rows, int d);
size_t block_step_bytes(const Sequences& seqs, int n, int kv_heads, int rows, int d);
int block_step(const BlockArrays& c, const Call& a, const Sequences& seqs, int n, int dtype, int d, void* workspace, int32_t* status,
               cudaStream_t stream);

// many rows per kv head (nkv_block_tile.cu)
size_t block_tile_bytes(int d);
int block_tile(const BlockArrays& c, const Call& a, const Sequences& seqs, int n, int dtype, int d, void* workspace, int32_t* status,
               cudaStream_t stream);

}  // namespace nkv
