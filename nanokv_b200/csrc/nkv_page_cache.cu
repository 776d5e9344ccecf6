// The paged 16-bit cache without its attention: pending tokens in (append), accepted rows to their places (keep), and what drafted
// tokens see of one another (tree mask).
#include "nkv_internal.h"
#include "nkv_page.cuh"
#include "nkv_rotary.cuh"

namespace nkv {
namespace {

// ---- append ----------------------------------------------------------------------------------------------------

struct Side {
  const uint16_t* x;
  long long stride_batch, stride_token, stride_head;
  int heads, vector;   // vector: rows start on 16 bytes
};

// A thread takes two 16-byte pieces of a head row whose elements are each other's partners (or two that are only copied), of HEADS
// heads, which share the table's entries and the page; one where the call is short of threads.  Bound: memory (24,967 tokens x 40 heads of
// keys, values and queries: 1.55 GB in and out in 270 us, 5.7 TB/s); the smallest calls the chain of loads, length, page, store (32 tokens x 56 heads
// 2.7 us).  Rows of the call are counted from row0 on; a launch has fewer than 2^31 threads.
template <int DT, int HEADS>
__global__ void __launch_bounds__(256)
page_append_kernel(PageArrays c, Side k, Side v, Side q, uint16_t* q_out, const int32_t* counts, long long row0, unsigned rows, unsigned tokens,
                   int d, Rotation rot, int32_t* status) {
  const unsigned units = d / 16, groups_kv = (k.heads + HEADS - 1) / HEADS, groups_q = (q.heads + HEADS - 1) / HEADS, groups = 2 * groups_kv + groups_q;
  const unsigned index = blockIdx.x * 256 + threadIdx.x;
  if (index >= rows * groups * units) return;
  const unsigned u = index & (units - 1), rest = index / units, group = rest % groups;   // (units: 4 or 8)
  const long long row = row0 + rest / groups;
  const int b = static_cast<int>(row / tokens), t = static_cast<int>(row - static_cast<long long>(b) * tokens);
  const int kind = group < groups_kv ? 0 : group < groups_kv + groups_q ? 1 : 2;   // keys, queries, values
  const int head0 = (group - (kind == 0 ? 0 : kind == 1 ? groups_kv : groups_kv + groups_q)) * HEADS;
  const Side& side = kind == 0 ? k : kind == 1 ? q : v;
  const bool turns = kind != 2 && static_cast<int>(u) < rot.dim / 16;
  const int first = turns && rot.layout == NKV_ROTARY_HALF ? u * 8 : 16 * u;
  const int other = turns && rot.layout == NKV_ROTARY_HALF ? first + rot.dim / 2 : first + 8;
  // all that comes from memory first
  const uint16_t* const from = side.x + b * side.stride_batch + t * side.stride_token + head0 * side.stride_head;
  uint4 lo[HEADS], hi[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (HEADS > 1 && head0 + h >= side.heads) break;
    lo[h] = load_piece<DT>(from + h * side.stride_head, first, side.vector);
    hi[h] = load_piece<DT>(from + h * side.stride_head, other, side.vector);
  }
  bool bad;
  const Extent e = extent_of(c, counts, tokens, b, bad);
  if (bad && t == 0 && u == 0) report(status, STATUS_PAGE);
  uint16_t* to;
  size_t apart;
  if (kind == 1) {
    to = q_out + (row * q.heads + head0) * d;
    apart = d;
  } else {
    if (t >= e.there) return;
    const int page = page_of(c, b, e.length + t);
    if (page < 0) {
      report(status, STATUS_PAGE);
      return;
    }
    to = (kind == 0 ? c.k : c.v) + row_at(c, page, head0, e.length + t, d);
    apart = static_cast<size_t>(d) << c.shift;
  }
  float2 cs[8];
  if (turns) turns_of(rot, rot.positions ? __ldg(rot.positions + row) : e.length + t, u * 8, cs);
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (HEADS > 1 && head0 + h >= side.heads) break;
    if (turns) {
      float x[8], y[8];
      Piece<DT>::unpack(lo[h], x);
      Piece<DT>::unpack(hi[h], y);
      if (rot.layout == NKV_ROTARY_HALF) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x0 = x[i], x1 = y[i];
          x[i] = turn_first(x0, x1, cs[i]);
          y[i] = turn_second(x0, x1, cs[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x0 = x[2 * i], x1 = x[2 * i + 1], y0 = y[2 * i], y1 = y[2 * i + 1];
          x[2 * i] = turn_first(x0, x1, cs[i]);
          x[2 * i + 1] = turn_second(x0, x1, cs[i]);
          y[2 * i] = turn_first(y0, y1, cs[4 + i]);
          y[2 * i + 1] = turn_second(y0, y1, cs[4 + i]);
        }
      }
      lo[h] = Piece<DT>::pack(x);
      hi[h] = Piece<DT>::pack(y);
    }
    *reinterpret_cast<uint4*>(to + h * apart + first) = lo[h];
    *reinterpret_cast<uint4*>(to + h * apart + other) = hi[h];
  }
}

// ---- keep ------------------------------------------------------------------------------------------------------

struct Kept {
  uint16_t* pools[2 * MOST_KEPT];   // keys and values of every cache
};

// A thread moves one 16-byte column of a kv head: the rows of the path lie at or behind the places they move to, in order, so
// that none is written before it is read; a node ahead of its place, as those behind a refused one may be, is refused as well.  Bound:
// the chain length, node, page, row (one sequence 2.0 us); 32 sequences x 40 layers x 9 rows of 8 heads 9.2 us over four states in turn
// (47 MB, 5.1 TB/s), 8.2 over one, whose rows stay in L2.
constexpr int AT_ONCE = 8;   // rows in flight
__global__ void __launch_bounds__(256)
page_keep_kernel(const __grid_constant__ Kept kept, PageArrays c, const int32_t* path, int accepted, const int32_t* counts, int d,
                 int32_t* status) {
  const int b = blockIdx.y, per_row = d / 8;
  const int index = blockIdx.z * 256 + threadIdx.x;
  if (index >= c.kv_heads * per_row) return;
  const int head = index / per_row, col = index % per_row * 8;
  uint16_t* const pool = kept.pools[blockIdx.x];
  const int32_t* const nodes = path + static_cast<size_t>(b) * accepted;
  bool bad;
  const Extent e = extent_of(c, counts, accepted, b, bad);
  const int room = c.row_pages << c.shift;
  int before = -1;
  for (int j0 = 0; j0 < e.there; j0 += AT_ONCE) {
    uint4 rows[AT_ONCE];
    bool moves[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      moves[i] = false;
      if (j0 + i >= e.there) continue;
      const int node = __ldg(nodes + j0 + i);
      const bool in = node > before && node >= j0 + i && node < room - e.length;
      bad |= !in;
      if (!in) continue;
      before = node;
      if (node == j0 + i) continue;
      const int page = page_of(c, b, e.length + node);
      bad |= page < 0;
      if (page < 0) continue;
      rows[i] = *reinterpret_cast<const uint4*>(pool + row_at(c, page, head, e.length + node, d) + col);
      moves[i] = true;
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      if (!moves[i]) continue;
      const int token = e.length + j0 + i, page = page_of(c, b, token);
      bad |= page < 0;
      if (page >= 0) *reinterpret_cast<uint4*>(pool + row_at(c, page, head, token, d) + col) = rows[i];
    }
  }
  if (bad && index == 0 && blockIdx.x == 0) report(status, STATUS_PAGE);
}

// ---- tree mask --------------------------------------------------------------------------------------------------

// A thread per node and word walks the node's ancestors as far as the word's first node: parents are in shared memory, and a draft is a few
// levels deep (a chain of n nodes takes n steps).  16 nodes 1.7 us, 32 drafts of 511 nodes 3.3 us, both a launch's latency.
__global__ void __launch_bounds__(256)
tree_mask_kernel(const int32_t* parents, int tokens, int words, uint32_t* mask, int32_t* depth, int32_t* status) {
  extern __shared__ int32_t up[];
  const int32_t* const from = parents + static_cast<size_t>(blockIdx.y) * tokens;
  bool bad = false;
  for (int i = threadIdx.x; i < tokens; i += 256) {
    const int p = __ldg(from + i);
    const bool in = p >= -1 && p < i;
    bad |= !in;
    up[i] = in ? p : -1;
  }
  if (bad && status) report(status, STATUS_TREE);
  __syncthreads();
  const int index = blockIdx.x * 256 + threadIdx.x;
  if (index >= tokens * words) return;
  const int node = index / words, w = index % words;
  uint32_t bits = 0;
  int steps = 0;
  for (int p = node; p >= 32 * w; p = up[p]) {
    if (p < 32 * w + 32) bits |= 1u << (p - 32 * w);
    ++steps;
  }
  mask[static_cast<size_t>(blockIdx.y) * tokens * words + index] = bits;
  if (w == 0) depth[static_cast<size_t>(blockIdx.y) * tokens + node] = steps - 1;
}

bool starts_on_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

// ---- host ------------------------------------------------------------------------------------------------------

PageArrays page_arrays(const nkv_page_cache& c, int first) {
  PageArrays a;
  a.k = static_cast<uint16_t*>(c.k_pages);
  a.v = static_cast<uint16_t*>(c.v_pages);
  a.table = c.table + static_cast<size_t>(first) * c.row_pages;
  a.lengths = c.lengths + first;
  a.kv_heads = c.kv_heads;
  a.pages = c.pages;
  a.shift = 0;
  while (1 << a.shift < c.page) ++a.shift;
  a.row_pages = c.row_pages;
  return a;
}

int page_append(const nkv_page_cache& c, const nkv_tokens& k, const nkv_tokens& v, const nkv_tokens* q, void* q_out, int tokens,
                const int32_t* counts, const nkv_rotation* rotation, int32_t* status, cudaStream_t stream) {
  auto side = [](const nkv_tokens& x) {
    Side s{static_cast<const uint16_t*>(x.data), x.stride_batch, x.stride_token, x.stride_head, x.heads, 0};
    s.vector = starts_on_16(x.data) && x.stride_batch % 8 == 0 && x.stride_token % 8 == 0 && x.stride_head % 8 == 0;
    return s;
  };
  const Side ks = side(k), vs = side(v), qs = q ? side(*q) : Side{nullptr, 0, 0, 0, 0, 0};
  Rotation rot{nullptr, nullptr, 0, 0, 0};
  if (rotation)
    rot = Rotation{reinterpret_cast<const float2*>(rotation->table), rotation->positions, rotation->rows, rotation->rotary_dim,
                   rotation->layout};
  const long long rows = static_cast<long long>(c.batch) * tokens;
  const int units = c.head_dim / 16;
  auto run = [&](auto kernel, int heads) {
    const long long per_row = static_cast<long long>(units) * (2 * ceil_div(ks.heads, heads) + ceil_div(qs.heads, heads)), most = ((1ll << 31) - 1) / per_row;
    for (long long row0 = 0; row0 < rows; row0 += most) {
      const long long n = min(most, rows - row0);
      kernel<<<static_cast<unsigned>((n * per_row + 255) / 256), 256, 0, stream>>>(page_arrays(c, 0), ks, vs, qs, static_cast<uint16_t*>(q_out), counts,
                                                                                  row0, static_cast<unsigned>(n), tokens, c.head_dim, rot, status);
      NKV_LAUNCH_CHECK("page_append_kernel");
    }
    return NKV_OK;
  };
  // four heads per thread share the table entries and the page once that still leaves every SM half a block of threads (one / four heads per
  // thread, 32 sequences x 56 heads of 128: 1 token 3.2 / 4.1 us, 4 tokens 3.6 / 4.2, 8 tokens 4.6 / 4.2, 64 tokens 15.9 / 12.0; 24,967 tokens x 120
  // heads 362 / 257)
  const bool many = rows * units * (2 * ks.heads + qs.heads) >= 2ll * 256 * sm_count();
  if (c.dtype == NKV_BF16) return many ? run(page_append_kernel<NKV_BF16, 4>, 4) : run(page_append_kernel<NKV_BF16, 1>, 1);
  return many ? run(page_append_kernel<NKV_F16, 4>, 4) : run(page_append_kernel<NKV_F16, 1>, 1);
}

int page_keep(const nkv_page_cache* caches, int count, const int32_t* path, int accepted, const int32_t* counts, int32_t* status,
              cudaStream_t stream) {
  const nkv_page_cache& c = caches[0];
  for (int first = 0; first < count; first += MOST_KEPT) {
    const int n = min(MOST_KEPT, count - first);
    Kept kept;
    for (int i = 0; i < n; ++i) {
      kept.pools[2 * i] = static_cast<uint16_t*>(caches[first + i].k_pages);
      kept.pools[2 * i + 1] = static_cast<uint16_t*>(caches[first + i].v_pages);
    }
    page_keep_kernel<<<dim3(2 * n, c.batch, ceil_div(c.kv_heads * (c.head_dim / 8), 256)), 256, 0, stream>>>(
        kept, page_arrays(c, 0), path, accepted, counts, c.head_dim, status);
    NKV_LAUNCH_CHECK("page_keep_kernel");
  }
  return NKV_OK;
}

int tree_mask(const int32_t* parents, int batch, int tokens, uint32_t* mask, int32_t* depth, int32_t* status, cudaStream_t stream) {
  const int words = ceil_div(tokens, 32);
  tree_mask_kernel<<<dim3(ceil_div(tokens * words, 256), batch), 256, tokens * sizeof(int32_t), stream>>>(parents, tokens, words, mask, depth,
                                                                                                          status);
  NKV_LAUNCH_CHECK("tree_mask_kernel");
  return NKV_OK;
}

}  // namespace nkv
