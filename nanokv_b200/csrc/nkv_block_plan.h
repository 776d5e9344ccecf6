// How an append to the 8-bit block cache is dealt out to launches and thread blocks.  Plain C++, so that it can be checked
// without a GPU.
#pragma once

#ifdef __CUDACC__
#define NKV_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define NKV_HOST_DEVICE inline
#endif

namespace nkv {

constexpr int BLOCK_TOKENS = 64;

// Blocks that an append of `count` tokens behind `length` touches, of one sequence and kv head.
NKV_HOST_DEVICE int append_blocks(int length, int count) {
  return count > 0 ? (length + count - 1) / BLOCK_TOKENS - length / BLOCK_TOKENS + 1 : 0;
}

// Whether the call completes an open block and leaves another one open.  The two share one store of 16-bit rows: the block
// that is completed reads its old rows there, the new one puts its rows in their place.  The new one is left to a second launch.
NKV_HOST_DEVICE bool append_twice(int length, int count) {
  const int before = length / BLOCK_TOKENS, open = (length + count) / BLOCK_TOKENS;
  return length % BLOCK_TOKENS != 0 && (length + count) % BLOCK_TOKENS != 0 && open > before;
}

// The block that thread block x of a launch takes; -1: none.
NKV_HOST_DEVICE int append_block(int length, int count, int x, bool second_launch) {
  const int block = length / BLOCK_TOKENS + x, open = (length + count) / BLOCK_TOKENS;
  const bool twice = append_twice(length, count);
  if (second_launch) return twice && x == 0 ? open : -1;
  return x < append_blocks(length, count) && !(twice && block == open) ? block : -1;
}

}  // namespace nkv
