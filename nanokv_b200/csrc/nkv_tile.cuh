// What the attention kernels on tcgen05 share beside nkv_tc.cuh: bounded waits of whole warps, the instruction descriptor of
// both 16-bit types, small loads of tensor memory, stores of result rows.
#pragma once

#include "nkv_block.cuh"
#include "nkv_tc.cuh"

namespace nkv {
namespace tc {

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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 columns of this thread's TMEM lane; the load apart from the wait, so that several can be in flight
__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  tmem_ld16_issue(taddr, r);
  tmem_ld16_wait(r);
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

}  // namespace tc
}  // namespace nkv
