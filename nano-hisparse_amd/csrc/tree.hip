// Verifying a tree of drafted tokens: ancestor masks and positions from the
// nodes' parents (nhs_tree_plan), and attention of every node over its
// request's selected pool rows and its own ancestors (nhs_tree_attention).
#include <math.h>

#include <algorithm>

#include "nhs_common.h"

namespace nhs {

constexpr int kTreeNodes = NHS_MAX_TREE_NODES;  // one bit of a mask word each

// ---- masks and positions ------------------------------------------------------------

// One wave per tree, one lane per node: mask[t] = mask[parent[t]] | 1 << t by
// pointer doubling (every lane takes over the mask and the parent of the node
// it points at; six rounds reach the root of any chain of 64), and the node's
// position is its request's length plus its depth. A parent outside [-1, t)
// marks the node absent, and whatever hangs below an absent node is absent
// too: mask 0, position 0. Bound by its launch (a few KB at most).
__global__ __launch_bounds__(kWave) void tree_plan_kernel(const int32_t* parents, int64_t parents_stride, int nodes,
                                                          const int64_t* lengths, int64_t* mask, int64_t* positions) {
  const int b = blockIdx.x, t = threadIdx.x;
  int p = t < nodes ? parents[(int64_t)b * parents_stride + t] : -2;
  if (p < -1 || p >= t) p = -2;
  uint64_t m = 1ull << t;
#pragma unroll
  for (int round = 0; round < 6; ++round) {
    const int at = max(p, 0);
    const uint32_t lo = __shfl((uint32_t)m, at), hi = __shfl((uint32_t)(m >> 32), at);
    const int up = __shfl(p, at);
    if (p >= 0) {
      m |= (uint64_t)hi << 32 | lo;
      p = up;
    }
  }
  if (t >= nodes) return;
  const bool present = p == -1;
  const int64_t i = (int64_t)b * nodes + t;
  mask[i] = present ? (int64_t)m : 0;
  positions[i] = present ? lengths[b] + __popcll(m) - 1 : 0;
}

// ---- attention ----------------------------------------------------------------------

// For request b, node t and query head h (KV head h / group), over the keys
// x of the request's rows (0 <= row < pool rows) and the drafted nodes j whose
// bit the node's mask word holds:
//   out[b, t, h] = sum_x softmax_x(q . K[x] * D^-1/2) V[x]
// and zeros where the mask word is 0. The group's heads of every node share
// the KV head's keys, so the query rows of a (request, KV head) are the
// nodes x group (row r = node * group + head of the group).
struct TreeArgs {
  const char* q;
  const char* k;
  const char* v;
  const int64_t* mask;
  int64_t q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, mask_b;  // element strides
  const char* pool;
  int64_t pool_rows, row_bytes, plane_bytes, block_stride;  // bytes, but pool_rows
  const int64_t* rows;
  int64_t r_b, r_c;
  int n_rows, rows_per_split, n_splits;
  int nodes, q_heads, kv_heads, group, head_dim, page_size;
  int query_rows, row_blocks;  // nodes * group, and blocks of them
  FastDiv group_div, page_div;
  float scale_log2;  // D^-1/2 * log2(e)
  char* out;
  int64_t o_b, o_n, o_h;
  float* stats;    // n_splits > 1: [n_splits, batch * nodes * q_heads, 2] (max in base 2, sum)
  float* partial;  // and [n_splits, batch * nodes * q_heads, head_dim], not divided by the sum
  int64_t out_rows;  // batch * nodes * q_heads
};

constexpr int kTgThreads = 256, kTgRows = 16, kTgMaxDim = NHS_MAX_TREE_HEAD_DIM;

// Every element type and head_dim up to 256. A workgroup takes 16 query rows
// of one (request, KV head) and one split of its rows; the last split takes
// the drafted keys too. Tiles of KEYS keys and values go to LDS in fp32; the
// 16 lanes of a query row score KEYS / 16 keys each, keep the row's online
// softmax in base 2 and hold its output dims (lane, lane + 16, ...). KEYS is
// 32, and 16 where 32 keys of head_dim above 128 would not leave two
// workgroups' LDS on a CU.
template <typename T, int KEYS, int DIMS>
__global__ __launch_bounds__(kTgThreads) void tree_general_kernel(TreeArgs a) {
  constexpr int pitch = DIMS + 1;
  __shared__ float qs[kTgRows * pitch], ks[KEYS * pitch], vs[KEYS * pitch], ps[kTgRows * (KEYS + 1)];
  __shared__ int valid[KEYS];  // of the tile's keys: a row, or a present drafted node
  const int D = a.head_dim;
  const int tid = threadIdx.x, row = tid >> 4, sub = tid & 15;
  const int split = blockIdx.x % a.n_splits, item = blockIdx.x / a.n_splits;
  const int block = item % a.row_blocks, bk = item / a.row_blocks;
  const int b = bk / a.kv_heads, kv = bk - b * a.kv_heads;

  const int r = block * kTgRows + row;
  const bool live = r < a.query_rows;
  const int node = live ? (int)a.group_div.div((uint32_t)r) : 0;
  const int head = kv * a.group + (live ? r - node * a.group : 0);
  const uint64_t word = live ? (uint64_t)a.mask[(int64_t)b * a.mask_b + node] : 0;
  for (int d = sub; d < D; d += 16)
    qs[row * pitch + d] =
        live ? load_elem(a.q, T::dtype, (int64_t)b * a.q_b + (int64_t)node * a.q_n + (int64_t)head * a.q_h + d) : 0.f;

  float m = -INFINITY, l = 0.f, acc[DIMS / 16];
#pragma unroll
  for (int i = 0; i < DIMS / 16; ++i) acc[i] = 0.f;

  const int begin = split * a.rows_per_split, end = min(a.n_rows, begin + a.rows_per_split);
  const int tiles = (max(end - begin, 0) + KEYS - 1) / KEYS;
  const int drafted = split == a.n_splits - 1 ? (a.nodes + KEYS - 1) / KEYS : 0;
  for (int t = 0; t < tiles + drafted; ++t) {
    const bool own = t >= tiles;
    const int first = own ? (t - tiles) * KEYS : begin + t * KEYS;
    const int count = min(KEYS, (own ? a.nodes : end) - first);
    __syncthreads();
    for (int j = row; j < KEYS; j += kTgThreads / 16) {  // 16 lanes a key
      const char *kp = nullptr, *vp = nullptr;
      if (j < count) {
        if (own) {
          if (a.mask[(int64_t)b * a.mask_b + first + j] != 0) {  // absent nodes hold anything
            kp = a.k + ((int64_t)b * a.k_b + (int64_t)(first + j) * a.k_n + (int64_t)kv * a.k_h) * T::bytes;
            vp = a.v + ((int64_t)b * a.v_b + (int64_t)(first + j) * a.v_n + (int64_t)kv * a.v_h) * T::bytes;
          }
        } else {
          const int64_t at = a.rows[(int64_t)b * a.r_b + (int64_t)(first + j) * a.r_c];
          if (at >= 0 && at < a.pool_rows) {
            const uint32_t page = a.page_div.div((uint32_t)at);
            kp = a.pool + page * a.block_stride + (int64_t)((uint32_t)at - page * a.page_size) * a.row_bytes +
                 (int64_t)kv * D * T::bytes;
            vp = kp + a.plane_bytes;
          }
        }
      }
      if (sub == 0) valid[j] = kp != nullptr;
      for (int d = sub; d < D; d += 16) {
        ks[j * pitch + d] = kp ? load_elem(kp, T::dtype, d) : 0.f;
        vs[j * pitch + d] = kp ? load_elem(vp, T::dtype, d) : 0.f;
      }
    }
    __syncthreads();
    // scores of keys sub and sub + 16, in base 2
    float s[KEYS / 16];
#pragma unroll
    for (int x = 0; x < KEYS / 16; ++x) {
      const int j = sub + 16 * x;
      float dot = 0.f;
      for (int d = 0; d < D; ++d) dot = __builtin_fmaf(qs[row * pitch + d], ks[j * pitch + d], dot);
      const bool seen = valid[j] && (!own || (word >> (first + j) & 1));
      s[x] = seen ? dot * a.scale_log2 : -INFINITY;
      // a key that is not seen adds nothing, whatever its value holds: -1 tells its weight from one that underflowed
      ps[row * (KEYS + 1) + j] = seen ? 0.f : -1.f;
    }
    float mx = s[0];
#pragma unroll
    for (int x = 1; x < KEYS / 16; ++x) mx = fmaxf(mx, s[x]);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    const float moved = fmaxf(m, mx), ref = moved == -INFINITY ? 0.f : moved;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = moved;
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < KEYS / 16; ++x) {
      float& p = ps[row * (KEYS + 1) + sub + 16 * x];
      if (p == 0.f) {
        p = __builtin_amdgcn_exp2f(s[x] - ref);
        sum += p;
      }
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d);
    l = l * alpha + sum;
    // a row's weights are written and read by its own 16 lanes of one wave, in order
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < DIMS / 16; ++i) {
      const int d = sub + 16 * i;
      if (d >= D) break;
      float o = acc[i] * alpha;
      for (int j = 0; j < count; ++j) {
        const float p = ps[row * (KEYS + 1) + j];
        if (!(p < 0.f)) o = __builtin_fmaf(p, vs[j * pitch + d], o);
      }
      acc[i] = o;
    }
  }
  if (!live) return;
  const int64_t out_row = ((int64_t)b * a.nodes + node) * a.q_heads + head;
  if (a.n_splits > 1) {
    const int64_t at = (int64_t)split * a.out_rows + out_row;
    if (sub == 0) {
      a.stats[2 * at] = m;
      a.stats[2 * at + 1] = l;
    }
    for (int i = 0, d = sub; i < DIMS / 16 && d < D; ++i, d += 16) a.partial[at * D + d] = acc[i];
    return;
  }
  const int64_t at = (int64_t)b * a.o_b + (int64_t)node * a.o_n + (int64_t)head * a.o_h;
  const bool some = word != 0 && m != -INFINITY;
#pragma unroll
  for (int i = 0; i < DIMS / 16; ++i)
    if (sub + 16 * i < D) store_elem(a.out, T::dtype, at + sub + 16 * i, some ? acc[i] / l : 0.f);
}

// Joins the splits of every output row, one wave per row: the sums are scaled
// to the largest of the splits' maxima, added and divided.
template <typename T>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a) {
  const int64_t out_row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (out_row >= a.out_rows) return;
  const int lane = threadIdx.x & 63, D = a.head_dim;
  const int64_t bn = out_row / a.q_heads;
  const int head = (int)(out_row - bn * a.q_heads);
  const int b = (int)(bn / a.nodes), node = (int)(bn - (int64_t)b * a.nodes);
  float top = -INFINITY;
  for (int s = 0; s < a.n_splits; ++s) top = fmaxf(top, a.stats[2 * ((int64_t)s * a.out_rows + out_row)]);
  const float ref = top == -INFINITY ? 0.f : top;
  const bool some = a.mask[(int64_t)b * a.mask_b + node] != 0 && top != -INFINITY;
  const int64_t at = (int64_t)b * a.o_b + (int64_t)node * a.o_n + (int64_t)head * a.o_h;
  for (int d = lane; d < D; d += kWave) {
    float total = 0.f, o = 0.f;
    for (int s = 0; s < a.n_splits; ++s) {
      const int64_t p = (int64_t)s * a.out_rows + out_row;
      const float f = __builtin_amdgcn_exp2f(a.stats[2 * p] - ref);
      total = __builtin_fmaf(f, a.stats[2 * p + 1], total);
      o = __builtin_fmaf(f, a.partial[p * D + d], o);
    }
    store_elem(a.out, T::dtype, at + d, some ? o / total : 0.f);
  }
}

struct TreeShape {
  int row_blocks, n_splits, rows_per_split;
};

// How the rows of a (request, KV head) are split: about 512 workgroups in
// all, none of less than 64 rows.
static TreeShape tree_shape(int batch, int nodes, int n_rows, int q_heads, int kv_heads) {
  TreeShape s;
  s.row_blocks = (nodes * (q_heads / kv_heads) + kTgRows - 1) / kTgRows;
  const int64_t items = (int64_t)batch * kv_heads * s.row_blocks;
  const int64_t wanted = std::max<int64_t>(1, 512 / items), most = std::max(1, n_rows / 64);
  s.n_splits = (int)std::min(wanted, most);
  s.rows_per_split = ((n_rows + s.n_splits - 1) / s.n_splits + 31) / 32 * 32;
  s.n_splits = std::max(1, (n_rows + std::max(s.rows_per_split, 1) - 1) / std::max(s.rows_per_split, 1));
  return s;
}

static bool tree_valid(int batch, int nodes, int n_rows, int q_heads, int kv_heads, int head_dim) {
  return batch >= 0 && nodes >= 1 && nodes <= kTreeNodes && n_rows >= 0 && q_heads >= 1 && kv_heads >= 1 &&
         q_heads % kv_heads == 0 && head_dim >= 1 && q_heads <= 65536 && batch <= (1 << 20);
}

}  // namespace nhs

using namespace nhs;

extern "C" int nhs_tree_plan(int32_t batch, int32_t nodes, const int32_t* parents, int64_t parents_stride,
                             const int64_t* lengths, int64_t* mask, int64_t* positions, void* stream) {
  const LaunchEvents ev = take_launch_events();
  if (!parents || !lengths || !mask || !positions) return fail(NHS_ERR_INVALID, "nhs_tree_plan: null pointer");
  if (batch < 0 || nodes < 1) return fail(NHS_ERR_INVALID, "nhs_tree_plan: invalid shape");
  if (nodes > kTreeNodes) return fail(NHS_ERR_UNSUPPORTED, "nhs_tree_plan: at most %d nodes", kTreeNodes);
  if (batch == 0) return NHS_OK;
  launch(tree_plan_kernel, dim3((unsigned)batch), dim3(kWave), 0, (hipStream_t)stream, ev.start, ev.stop, parents,
         parents_stride, nodes, lengths, mask, positions);
  return launch_status("nhs_tree_plan");
}

extern "C" int64_t nhs_tree_attention_workspace_bytes(int32_t batch, int32_t nodes, int32_t n_rows, int32_t q_heads,
                                                      int32_t kv_heads, int32_t head_dim) {
  if (!tree_valid(batch, nodes, n_rows, q_heads, kv_heads, head_dim)) return 0;
  const TreeShape s = tree_shape(std::max(batch, 1), nodes, n_rows, q_heads, kv_heads);
  if (s.n_splits == 1) return 0;
  return (int64_t)s.n_splits * batch * nodes * q_heads * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int nhs_tree_attention(const void* q, int64_t q_batch_stride, int64_t q_node_stride, int64_t q_head_stride,
                                  const void* k, int64_t k_batch_stride, int64_t k_node_stride, int64_t k_head_stride,
                                  const void* v, int64_t v_batch_stride, int64_t v_node_stride, int64_t v_head_stride,
                                  const int64_t* mask, int64_t mask_batch_stride, int32_t dtype, const void* pool,
                                  int64_t pool_rows, int64_t pool_block_stride, const int64_t* rows,
                                  int64_t rows_batch_stride, int64_t rows_col_stride, int32_t batch, int32_t nodes,
                                  int32_t n_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                  int32_t page_size, void* out, int64_t out_batch_stride, int64_t out_node_stride,
                                  int64_t out_head_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  const LaunchEvents ev = take_launch_events();
  const char* who = "nhs_tree_attention";
  if (!tree_valid(batch, nodes, n_rows, q_heads, kv_heads, head_dim) || page_size < 1 || pool_rows < 0 ||
      !valid_dtype(dtype))
    return fail(NHS_ERR_INVALID, "%s: invalid shape or dtype", who);
  if (batch == 0) return NHS_OK;
  if (!q || !k || !v || !mask || !out || (n_rows > 0 && (!pool || !rows)))
    return fail(NHS_ERR_INVALID, "%s: null pointer", who);
  if (head_dim > kTgMaxDim) return fail(NHS_ERR_UNSUPPORTED, "%s: head_dim up to %d", who, kTgMaxDim);
  if (pool_rows >= (1ll << 31)) return fail(NHS_ERR_UNSUPPORTED, "%s: pool rows must be < 2^31", who);
  const int esize = elem_size(dtype);
  const int64_t row_bytes = (int64_t)kv_heads * head_dim * esize, block = 2 * page_size * row_bytes;
  if (pool_block_stride == 0) pool_block_stride = block;
  if (pool_block_stride < block || pool_block_stride % esize)
    return fail(NHS_ERR_INVALID, "%s: pool_block_stride is 0 or at least one block of whole elements", who);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)pool) % esize ||
      ((uintptr_t)mask | (uintptr_t)rows) % 8)
    return fail(NHS_ERR_INVALID, "%s: misaligned pointer", who);
  const TreeShape shape = tree_shape(batch, nodes, n_rows, q_heads, kv_heads);
  const int64_t need = nhs_tree_attention_workspace_bytes(batch, nodes, n_rows, q_heads, kv_heads, head_dim);
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(NHS_ERR_WORKSPACE, "%s: needs %lld bytes of 16-byte aligned workspace", who, (long long)need);
  const int64_t blocks = (int64_t)batch * kv_heads * shape.row_blocks * shape.n_splits;
  if (blocks > 0x7fffffff || (int64_t)batch * nodes * q_heads > 0x7fffffff)
    return fail(NHS_ERR_UNSUPPORTED, "%s: too many workgroups", who);
  TreeArgs a;
  a.q = static_cast<const char*>(q), a.k = static_cast<const char*>(k), a.v = static_cast<const char*>(v);
  a.mask = mask;
  a.q_b = q_batch_stride, a.q_n = q_node_stride, a.q_h = q_head_stride;
  a.k_b = k_batch_stride, a.k_n = k_node_stride, a.k_h = k_head_stride;
  a.v_b = v_batch_stride, a.v_n = v_node_stride, a.v_h = v_head_stride;
  a.mask_b = mask_batch_stride;
  a.pool = static_cast<const char*>(pool);
  a.pool_rows = pool_rows, a.row_bytes = row_bytes, a.plane_bytes = page_size * row_bytes;
  a.block_stride = pool_block_stride;
  a.rows = rows, a.r_b = rows_batch_stride, a.r_c = rows_col_stride;
  a.n_rows = n_rows, a.rows_per_split = shape.rows_per_split, a.n_splits = shape.n_splits;
  a.nodes = nodes, a.q_heads = q_heads, a.kv_heads = kv_heads, a.group = q_heads / kv_heads;
  a.head_dim = head_dim, a.page_size = page_size;
  a.query_rows = nodes * a.group, a.row_blocks = shape.row_blocks;
  a.group_div = FastDiv((uint32_t)a.group), a.page_div = FastDiv((uint32_t)page_size);
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  a.out = static_cast<char*>(out);
  a.o_b = out_batch_stride, a.o_n = out_node_stride, a.o_h = out_head_stride;
  a.out_rows = (int64_t)batch * nodes * q_heads;
  a.stats = static_cast<float*>(workspace);
  a.partial = a.stats + 2 * a.out_rows * shape.n_splits;
  hipStream_t s = (hipStream_t)stream;
  const hipEvent_t none = nullptr;
  auto run = [&](auto kernel, auto join) {
    const bool joined = shape.n_splits > 1;
    launch(kernel, dim3((unsigned)blocks), dim3(kTgThreads), 0, s, ev.start, joined ? none : ev.stop, a);
    if (joined) launch(join, dim3((unsigned)((a.out_rows + 3) / 4)), dim3(256), 0, s, none, ev.stop, a);
  };
  const auto general = [&](auto tag) {
    using T = decltype(tag);
    if (head_dim <= 128)
      run(tree_general_kernel<T, 32, 128>, tree_join_kernel<T>);
    else
      run(tree_general_kernel<T, 16, kTgMaxDim>, tree_join_kernel<T>);
  };
  if (dtype == NHS_BF16)
    general(BF16{});
  else if (dtype == NHS_F16)
    general(F16{});
  else
    general(F32{});
  return launch_status(who);
}
