// Attention over the paged 16-bit cache.
#include "nkv_internal.h"
#include "nkv_page.cuh"

namespace nkv {
namespace {

// The formula as it stands, in fp32: a warp per row, the rows of a thread block share 64 tokens of K and V at a time.  Runs where the
// tensor-core kernel is switched off, to check it.
constexpr int ROWS = 8, STEP = 64;
template <int DT, int D>
__global__ void __launch_bounds__(32 * ROWS)
page_plain_kernel(PageArrays c, PageCall a, int32_t* status) {
  extern __shared__ float smem[];
  float* const ks = smem;                      // [STEP][D + 1]
  float* const vs = ks + STEP * (D + 1);       // [STEP][D]
  float* const qs = vs + STEP * D;             // [ROWS][D]
  float* const ps = qs + ROWS * D;             // [ROWS][STEP]
  const int b = blockIdx.z, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  bool bad;
  const Extent e = extent_of(c, a.counts, a.tokens, b, bad);
  const int r = blockIdx.x * ROWS + warp;
  const bool row = r < a.rows;
  const int token = r / a.group, head = h * a.group + r % a.group;
  const bool asked = row && token < e.count;
  const int last = min(e.count, (min(a.rows, (static_cast<int>(blockIdx.x) + 1) * ROWS) - 1) / a.group + 1);   // queries up to here
  const int most = static_cast<int>(blockIdx.x) * ROWS / a.group >= e.count ? 0 : e.length + (a.sight == page::SEES_CAUSAL ? min(last, e.there) : e.there);
  if (row)
    for (int d = lane; d < D; d += 32)
      qs[warp * D + d] = load_float(a.q, DT, b * a.q_batch + token * a.q_token + head * a.q_head + d);
  // weights are taken so far below 1 that their sum stays below it: sums of the largest bf16 values are numbers then
  const float below = 32 - __clz(e.length + e.there);
  float m = -INFINITY, l = 0.f, o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
  for (int t0 = 0; t0 < most; t0 += STEP) {
    __syncthreads();
    for (int i = threadIdx.x; i < STEP * D; i += 32 * ROWS) {
      const int t = t0 + i / D, page = t < e.length + e.there ? page_of(c, b, t) : -1;
      bad |= t < e.length + e.there && page < 0;
      const size_t at = page < 0 ? 0 : row_at(c, page, h, t, D) + i % D;
      ks[i / D * (D + 1) + i % D] = page < 0 ? 0.f : load_float(c.k, DT, at);
      vs[i] = page < 0 ? 0.f : load_float(c.v, DT, at);
    }
    __syncthreads();
    if (!asked) continue;
    uint32_t sees[2];
    float s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sees[j] = sight_of(a, e, b, token, t0 + 32 * j);
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = fmaf(qs[warp * D + d], ks[(lane + 32 * j) * (D + 1) + d], dot);
      s[j] = sees[j] >> lane & 1 ? dot * a.scale_log2 : -INFINITY;
    }
    float top = fmaxf(s[0], s[1]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float next = fmaxf(m, top), ref = next == -INFINITY ? 0.f : next;
    const float alpha = exp2f(m - ref), p0 = exp2f(s[0] - ref - below), p1 = exp2f(s[1] - ref - below);
    float sum = p0 + p1;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * alpha + sum;
    m = next;
    ps[warp * STEP + lane] = p0;
    ps[warp * STEP + lane + 32] = p1;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      float acc = o[i] * alpha;
      // what a row does not see has no part in it, whatever it is
      for (int t = 0; t < STEP; ++t)
        if (sees[t / 32] >> (t & 31) & 1) acc = fmaf(ps[warp * STEP + t], vs[t * D + lane + 32 * i], acc);
      o[i] = acc;
    }
    __syncwarp();
  }
  if (bad) report(status, STATUS_PAGE);
  if (!row) return;
  const size_t at = (static_cast<size_t>(b) * a.tokens + token) * a.heads + head;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) store_float(a.out, DT, at * D + lane + 32 * i, l == 0.f ? 0.f : o[i] / l);
  if (lane == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + below + log2f(l)) * LN2;
}

}  // namespace

size_t page_attend_workspace_bytes(const nkv_page_cache& c, int heads, int tokens) {
  const int n = min(page::MOST_SEQUENCES, c.batch);
  return page_tile_bytes(page_arrays(c, 0), n, heads / c.kv_heads * tokens, c.head_dim);   // launches follow one another on the stream and share it
}

int page_attend(const nkv_page_cache& c, const nkv_tokens& q, int tokens, const int32_t* counts, const uint32_t* mask,
                int64_t mask_stride, bool causal, float scale, void* out, float* lse, int32_t* status, void* workspace,
                cudaStream_t stream) {
  for (int first = 0; first < c.batch; first += page::MOST_SEQUENCES) {
    const int n = min(page::MOST_SEQUENCES, c.batch - first);
    PageCall a;
    a.q = static_cast<const uint16_t*>(q.data) + first * q.stride_batch;
    a.q_batch = q.stride_batch;
    a.q_token = q.stride_token;
    a.q_head = q.stride_head;
    a.out = static_cast<uint16_t*>(out) + static_cast<size_t>(first) * tokens * q.heads * c.head_dim;
    a.lse = lse + static_cast<size_t>(first) * tokens * q.heads;
    a.counts = counts ? counts + first : nullptr;
    a.mask = mask ? mask + first * mask_stride : nullptr;
    a.mask_batch = mask_stride;
    a.words = ceil_div(tokens, 32);
    a.sight = mask ? page::SEES_TREE : causal ? page::SEES_CAUSAL : page::SEES_ALL;
    a.tokens = tokens;
    a.heads = q.heads;
    a.group = q.heads / c.kv_heads;
    a.rows = tokens * a.group;
    a.scale_log2 = scale * LOG2E;
    a.q_vector = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.q_batch % 8 == 0 && a.q_token % 8 == 0 && a.q_head % 8 == 0;
    const PageArrays arrays = page_arrays(c, first);
    if (!simt_forced()) {
      const int rc = page_tile(arrays, a, n, c.dtype, c.head_dim, workspace, status, stream);
      if (rc != NKV_OK) return rc;
      continue;
    }
    auto kernel = c.head_dim == 128 ? (c.dtype == NKV_BF16 ? page_plain_kernel<NKV_BF16, 128> : page_plain_kernel<NKV_F16, 128>)
                                    : (c.dtype == NKV_BF16 ? page_plain_kernel<NKV_BF16, 64> : page_plain_kernel<NKV_F16, 64>);
    const int smem = static_cast<int>(sizeof(float)) * (STEP * (2 * c.head_dim + 1) + ROWS * (c.head_dim + STEP));
    NKV_CUDA(allow_shared(reinterpret_cast<const void*>(kernel), smem));
    kernel<<<dim3(ceil_div(a.rows, ROWS), c.kv_heads, n), 32 * ROWS, smem, stream>>>(arrays, a, status);
    NKV_LAUNCH_CHECK("page_plain_kernel");
  }
  return NKV_OK;
}

}  // namespace nkv
