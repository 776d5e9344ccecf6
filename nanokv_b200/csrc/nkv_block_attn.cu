// Attention over the 8-bit block cache.
#include <atomic>

#include "nkv_block.cuh"
#include "nkv_internal.h"

namespace nkv {
namespace {

// ---- CUDA cores ------------------------------------------------------------------------------------------------

// The formula as it stands, in fp32: a warp per row, the rows of a block share its dequantised K and V.  Runs where the
// tensor-core kernels are switched off, to check them.
constexpr int ROWS = 8;
template <int DT, int D>
__global__ void __launch_bounds__(32 * ROWS)
attend_plain_kernel(BlockArrays c, Call a, Sequences seqs) {
  extern __shared__ float smem[];
  float* const ks = smem;                            // [64][D + 1]
  float* const vs = ks + NKV_BLOCK * (D + 1);        // [D][65]
  float* const qs = vs + D * (NKV_BLOCK + 1);        // [ROWS][D]
  float* const ps = qs + ROWS * D;                   // [ROWS][64]
  const int b = blockIdx.z, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int length = seqs.length[b], count = seqs.count[b];
  const int r = blockIdx.x * ROWS + warp;
  const size_t bh = static_cast<size_t>(b) * c.kv_heads + h;
  const bool row = r < a.rows;
  const int token = r / a.group, head = h * a.group + r % a.group;
  const int seen = row ? visible_to(a, length, count, r) : 0;
  const int last = min(a.rows, (static_cast<int>(blockIdx.x) + 1) * ROWS) - 1;
  const int seen_most = a.causal ? visible_to(a, length, count, min(last, count * a.group - 1)) : (count > 0 ? length : 0);
  if (row)
    for (int d = lane; d < D; d += 32)
      qs[warp * D + d] = load_float(a.q, DT, b * a.q_batch + token * a.q_token + head * a.q_head + d);
  float m = -INFINITY, l = 0.f, o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
  for (int t0 = 0; t0 < seen_most; t0 += NKV_BLOCK) {
    const int block = t0 / NKV_BLOCK;
    __syncthreads();
    if (t0 + NKV_BLOCK <= length) {
      const size_t slot = slot_of(c, bh, block);
      const float k_scale = c.scales[2 * slot], v_scale = c.scales[2 * slot + 1];
      for (int i = threadIdx.x; i < NKV_BLOCK * D; i += 32 * ROWS) {
        ks[i / D * (D + 1) + i % D] = code_value(c.k_codes[slot * NKV_BLOCK * D + i]) * k_scale;
        vs[i / NKV_BLOCK * (NKV_BLOCK + 1) + i % NKV_BLOCK] = code_value(c.v_codes[slot * NKV_BLOCK * D + i]) * v_scale;
      }
    } else {
      const size_t tail = bh * NKV_BLOCK * D;
      for (int i = threadIdx.x; i < NKV_BLOCK * D; i += 32 * ROWS) {
        ks[i / D * (D + 1) + i % D] = t0 + i / D < length ? load_float(c.k_tail, DT, tail + i) : 0.f;
        vs[i / NKV_BLOCK * (NKV_BLOCK + 1) + i % NKV_BLOCK] = t0 + i % NKV_BLOCK < length ? load_float(c.v_tail, DT, tail + i) : 0.f;
      }
    }
    __syncthreads();
    if (t0 >= seen) continue;
    float s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = lane + 32 * j;
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = fmaf(qs[warp * D + d], ks[t * (D + 1) + d], dot);
      s[j] = t0 + t < seen ? dot * a.scale_log2 : -INFINITY;
    }
    // NaN has to reach the row: the maximum of a NaN and a number is the number
    float top = fmaxf(s[0], s[1]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float next = fmaxf(m, top), ref = next == -INFINITY ? 0.f : next;
    const float alpha = exp2f(m - ref), p0 = exp2f(s[0] - ref), p1 = exp2f(s[1] - ref);
    float sum = p0 + p1;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (a.partial && lane == 0) a.partial[(bh * a.most_blocks + block) * a.rows + r] = log2f(sum) + ref;
    l = l * alpha + sum;
    m = next;
    ps[warp * NKV_BLOCK + lane] = p0;
    ps[warp * NKV_BLOCK + lane + 32] = p1;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      float acc = o[i] * alpha;
      for (int t = 0; t < NKV_BLOCK; ++t) acc = fmaf(ps[warp * NKV_BLOCK + t], vs[(lane + 32 * i) * (NKV_BLOCK + 1) + t], acc);
      o[i] = acc;
    }
    __syncwarp();
  }
  if (!row) return;
  const size_t at = (static_cast<size_t>(b) * a.tokens + token) * a.heads + head;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) store_float(a.out, DT, at * D + lane + 32 * i, seen > 0 ? o[i] / l : 0.f);
  if (lane == 0) a.lse[at] = seen > 0 ? (m + log2f(l)) * LN2 : -INFINITY;
}

// weights[block] += sum over rows of 2^(partial - lse), rows in a fixed order: a thread block per WEIGHT_BLOCKS blocks of a kv
// head, so that a row's lse, scattered over the query heads, is fetched once for all of them.  Bound: memory, four bytes a row and
// block (16 heads of 16,380 rows x 64 blocks: 67 MB, part of it still in L2, in 29 us).
constexpr int WEIGHT_BLOCKS = 2, WEIGHT_THREADS = 512;
__global__ void __launch_bounds__(WEIGHT_THREADS)
block_weights_kernel(BlockArrays c, Call a, Sequences seqs) {
  __shared__ float sums[WEIGHT_BLOCKS][WEIGHT_THREADS / 32];
  const int block0 = blockIdx.x * WEIGHT_BLOCKS, h = blockIdx.y, b = blockIdx.z;
  const int length = seqs.length[b], count = seqs.count[b];
  const int blocks = min(WEIGHT_BLOCKS, (length + NKV_BLOCK - 1) / NKV_BLOCK - block0);
  if (blocks <= 0 || count <= 0) return;
  const size_t bh = static_cast<size_t>(b) * c.kv_heads + h;
  const float* const partial = a.partial + (bh * a.most_blocks + block0) * a.rows;
  const float* const lse = a.lse + static_cast<size_t>(b) * a.tokens * a.heads + h * a.group;
  // the first token that sees anything of these blocks
  const int first = a.causal ? max(0, block0 * NKV_BLOCK - (length - count)) : 0;
  float sum[WEIGHT_BLOCKS] = {};
#pragma unroll 4
  for (int r = first * a.group + threadIdx.x; r < count * a.group; r += WEIGHT_THREADS) {
    const int token = r / a.group;
    const float ref = lse[static_cast<size_t>(token) * a.heads + r - token * a.group] * LOG2E;
    const int seen = visible_to(a, length, count, r) - block0 * NKV_BLOCK;
#pragma unroll
    for (int k = 0; k < WEIGHT_BLOCKS; ++k)
      if (k < blocks && seen > k * NKV_BLOCK) sum[k] += exp2f(partial[static_cast<size_t>(k) * a.rows + r] - ref);
  }
#pragma unroll
  for (int k = 0; k < WEIGHT_BLOCKS; ++k) {
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], x);
    if ((threadIdx.x & 31) == 0) sums[k][threadIdx.x / 32] = sum[k];
  }
  __syncthreads();
  if (threadIdx.x < blocks) {
    float total = 0.f;
    for (int w = 0; w < WEIGHT_THREADS / 32; ++w) total += sums[threadIdx.x][w];
    a.weights[bh * c.blocks + block0 + threadIdx.x] += total;
  }
}

int most_blocks_of(const nkv_block_cache& c) {
  int most = 0;
  for (int i = 0; i < c.batch; ++i) most = max(most, ceil_div(c.lengths[i], NKV_BLOCK));
  return most;
}

// scratch of one launch over n sequences: the rows' weight sums per block, then the kernel's own
struct Scratch { size_t partial, own; };
Scratch scratch_of(const nkv_block_cache& c, const Sequences& seqs, int n, int group, int tokens, int most_blocks, bool with_weights) {
  const int rows = group * tokens;
  Scratch s{0, 0};
  if (with_weights) s.partial = (static_cast<size_t>(n) * c.kv_heads * most_blocks * rows * 4 + 255) & ~static_cast<size_t>(255);
  if (!simt_forced())
    s.own = block_step_supported(rows, c.head_dim) ? block_step_bytes(seqs, n, c.kv_heads, rows, c.head_dim)
                                       : block_tile_bytes(c.head_dim);
  return s;
}

}  // namespace

cudaError_t allow_shared(const void* kernel, int bytes) {
  constexpr int DEVICES = 64, KERNELS = 32;
  static std::atomic<const void*> known[DEVICES][KERNELS];
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) return err;
  std::atomic<const void*>* const row = device < DEVICES ? known[device] : nullptr;
  for (int i = 0; row && i < KERNELS; ++i) {
    const void* const k = row[i].load(std::memory_order_acquire);
    if (k == kernel) return cudaSuccess;
    if (k == nullptr) break;
  }
  err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  for (int i = 0; row && err == cudaSuccess && i < KERNELS; ++i) {
    const void* none = nullptr;
    if (row[i].compare_exchange_strong(none, kernel) || none == kernel) break;
  }
  return err;
}

size_t block_attend_workspace_bytes(const nkv_block_cache& c, int heads, int tokens, const int32_t* counts, bool causal,
                                    bool with_weights) {
  size_t most = 0;   // launches follow one another on the stream and share it
  for (int first = 0; first < c.batch; first += MAX_SEQUENCES) {
    const int n = min(MAX_SEQUENCES, c.batch - first);
    const Scratch s = scratch_of(c, sequences_of(c, first, n, counts, tokens), n, heads / c.kv_heads, tokens, most_blocks_of(c), with_weights);
    if (s.partial + s.own > most) most = s.partial + s.own;
  }
  return most;
}

int block_attend(const nkv_block_cache& c, const nkv_tokens& q, int tokens, const int32_t* counts, bool causal, float scale,
                 void* out, float* lse, float* weights, int32_t* status, void* workspace, cudaStream_t stream) {
  for (int first = 0; first < c.batch; first += MAX_SEQUENCES) {
    const int n = min(MAX_SEQUENCES, c.batch - first);
    const Sequences seqs = sequences_of(c, first, n, counts, tokens);
    Call a;
    a.q = static_cast<const uint16_t*>(q.data) + first * q.stride_batch;
    a.q_batch = q.stride_batch;
    a.q_token = q.stride_token;
    a.q_head = q.stride_head;
    a.out = static_cast<uint16_t*>(out) + static_cast<size_t>(first) * tokens * q.heads * c.head_dim;
    a.lse = lse + static_cast<size_t>(first) * tokens * q.heads;
    a.partial = weights ? static_cast<float*>(workspace) : nullptr;
    a.weights = weights ? weights + static_cast<size_t>(first) * c.kv_heads * c.blocks : nullptr;
    a.tokens = tokens;
    a.heads = q.heads;
    a.group = q.heads / c.kv_heads;
    a.rows = tokens * a.group;
    a.causal = causal;
    a.most_blocks = most_blocks_of(c);
    a.scale_log2 = scale * LOG2E;
    a.q_vector = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.q_batch % 8 == 0 && a.q_token % 8 == 0 && a.q_head % 8 == 0;
    const BlockArrays arrays = block_arrays(c, first);
    void* const own = static_cast<uint8_t*>(workspace) + scratch_of(c, seqs, n, a.group, tokens, a.most_blocks, weights != nullptr).partial;
    if (!simt_forced() && block_step_supported(a.rows, c.head_dim)) {
      const int rc = block_step(arrays, a, seqs, n, c.dtype, c.head_dim, own, status, stream);
      if (rc != NKV_OK) return rc;
      continue;
    }
    if (!simt_forced()) {
      const int rc = block_tile(arrays, a, seqs, n, c.dtype, c.head_dim, own, status, stream);
      if (rc != NKV_OK) return rc;
    } else {
      auto kernel = c.head_dim == 128
                        ? (c.dtype == NKV_BF16 ? attend_plain_kernel<NKV_BF16, 128> : attend_plain_kernel<NKV_F16, 128>)
                        : (c.dtype == NKV_BF16 ? attend_plain_kernel<NKV_BF16, 64> : attend_plain_kernel<NKV_F16, 64>);
      const size_t smem = sizeof(float) * (NKV_BLOCK * (c.head_dim + 1) + c.head_dim * (NKV_BLOCK + 1) +
                                           ROWS * (c.head_dim + NKV_BLOCK));
      NKV_CUDA(allow_shared(reinterpret_cast<const void*>(kernel), static_cast<int>(smem)));
      kernel<<<dim3(ceil_div(a.rows, ROWS), c.kv_heads, n), 32 * ROWS, smem, stream>>>(arrays, a, seqs);
      NKV_LAUNCH_CHECK("attend_plain_kernel");
    }
    if (weights && a.most_blocks > 0) {
      block_weights_kernel<<<dim3(ceil_div(a.most_blocks, WEIGHT_BLOCKS), c.kv_heads, n), WEIGHT_THREADS, 0, stream>>>(arrays, a, seqs);
      NKV_LAUNCH_CHECK("block_weights_kernel");
    }
  }
  return NKV_OK;
}

}  // namespace nkv
