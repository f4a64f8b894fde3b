// Decode attention over pool rows held in 8 bits (rows8.h): nhs_attend_rows8.
//
// For request b and query head h (KV head h / group), over the rows r of the
// list with 0 <= r < pool rows:
//   out[b, h] = sum_r softmax_r(q[b, h] . K[r] D^-1/2) V[r]
// and zeros where the list holds none. The scale of a row's keys multiplies
// its score, that of its values its weight, so the products run on the codes.
#include <math.h>

#include <algorithm>
#include <mutex>
#include <type_traits>
#include <vector>

#include "rows8.h"

namespace nhs {

struct Attend8Args {
  const void* q;
  int q_dtype;
  int64_t q_bs, q_hs;
  const char* pool;
  int64_t pool_rows, block_stride, row_bytes, scales_at, plane_bytes;
  const int64_t* rows;
  int64_t r_bs, r_hs, r_cs;
  int batch, n_rows, q_heads, kv_heads, group, head_dim, page_size;
  int rows_per_split, n_splits;
  FastDiv page_div;
  float scale_log2;  // D^-1/2 * log2(e)
  void* out;
  int64_t o_bs, o_hs;
  float* partial;  // n_splits > 1: [n_splits, batch * q_heads, head_dim], not divided by the sum
  float* stats;    // and [n_splits, batch * q_heads, 2] (max in base 2, sum)
};

// ---- any head_dim up to NHS_MAX_HEAD_DIM8 -----------------------------------------------

constexpr int kG8Threads = 256, kG8Waves = kG8Threads / kWave, kG8Rows = 4;

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// A workgroup takes one query head of one request and one split of its rows;
// a wave takes four rows at a time (lane l dims l, l + 64, ...; N of them at
// most) and keeps its own online softmax in base 2.
template <typename C, int N>
__global__ __launch_bounds__(kG8Threads) void attend8_general_kernel(Attend8Args a) {
  __shared__ float merged[kG8Waves][N * kWave + 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, D = a.head_dim;
  const int heads = a.batch * a.q_heads;
  const int item = blockIdx.x % heads, split = blockIdx.x / heads;
  const int b = item / a.q_heads, h = item - b * a.q_heads, kv = h / a.group;
  float q[N], acc[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane + i * kWave;
    q[i] = d < D ? load_elem(a.q, a.q_dtype, (int64_t)b * a.q_bs + (int64_t)h * a.q_hs + d) : 0.f;
    acc[i] = 0.f;
  }
  const int64_t* list = a.rows + (int64_t)b * a.r_bs + (int64_t)h * a.r_hs;
  const int begin = split * a.rows_per_split, end = min(a.n_rows, begin + a.rows_per_split);
  for (int r0 = begin + wave * kG8Rows; r0 < end; r0 += kG8Waves * kG8Rows) {
    float s[kG8Rows], vs[kG8Rows], v[kG8Rows][N];
    bool seen[kG8Rows];
    float top = m;
#pragma unroll
    for (int j = 0; j < kG8Rows; ++j) {
      const int64_t row = r0 + j < end ? list[(int64_t)(r0 + j) * a.r_cs] : -1;
      seen[j] = row >= 0 && row < a.pool_rows;
      const uint32_t at = seen[j] ? (uint32_t)row : 0u, page = a.page_div.div(at);
      const char* kp = a.pool + page * a.block_stride + (int64_t)(at - page * a.page_size) * a.row_bytes;
      const char* vp = kp + a.plane_bytes;
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int d = lane + i * kWave;
        const bool here = seen[j] && d < D;
        dot = here ? __builtin_fmaf(q[i], decode8<C>((uint8_t)kp[kv * D + d]), dot) : dot;
        v[j][i] = here ? decode8<C>((uint8_t)vp[kv * D + d]) : 0.f;
      }
      const float ks = seen[j] ? reinterpret_cast<const float*>(kp + a.scales_at)[kv] : 0.f;
      vs[j] = seen[j] ? reinterpret_cast<const float*>(vp + a.scales_at)[kv] : 0.f;
      s[j] = seen[j] ? wave_sum(dot) * (ks * a.scale_log2) : -INFINITY;
      top = fmaxf(top, s[j]);
    }
    const float ref = top == -INFINITY ? 0.f : top, alpha = __builtin_amdgcn_exp2f(m - ref);
    m = top;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= alpha;
#pragma unroll
    for (int j = 0; j < kG8Rows; ++j) {
      if (!seen[j]) continue;
      const float p = __builtin_amdgcn_exp2f(s[j] - ref), w = p * vs[j];
      l += p;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = __builtin_fmaf(w, v[j][i], acc[i]);
    }
  }
  if (lane == 0) {
    merged[wave][0] = m;
    merged[wave][1] = l;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) merged[wave][2 + lane + i * kWave] = acc[i];
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kG8Waves; ++w) top = fmaxf(top, merged[w][0]);
  const float ref = top == -INFINITY ? 0.f : top;
  float f[kG8Waves], total = 0.f;
#pragma unroll
  for (int w = 0; w < kG8Waves; ++w) {
    f[w] = __builtin_amdgcn_exp2f(merged[w][0] - ref);
    total = __builtin_fmaf(merged[w][1], f[w], total);
  }
  for (int d = threadIdx.x; d < D; d += kG8Threads) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < kG8Waves; ++w) o = __builtin_fmaf(merged[w][2 + d], f[w], o);
    if (a.n_splits > 1)
      a.partial[((int64_t)split * heads + item) * D + d] = o;
    else
      store_elem(a.out, a.q_dtype, (int64_t)b * a.o_bs + (int64_t)h * a.o_hs + d, total != 0.f ? o / total : 0.f);
  }
  if (a.n_splits > 1 && threadIdx.x == 0) {
    a.stats[2 * ((int64_t)split * heads + item)] = top;
    a.stats[2 * ((int64_t)split * heads + item) + 1] = total;
  }
}

// ---- joining the splits ------------------------------------------------------------------

// A wave per (request, query head).
__global__ __launch_bounds__(kWave) void attend8_join_kernel(Attend8Args a) {
  const int heads = a.batch * a.q_heads, item = blockIdx.x, lane = threadIdx.x, D = a.head_dim;
  float top = -INFINITY;
  for (int s = 0; s < a.n_splits; ++s) top = fmaxf(top, a.stats[2 * ((int64_t)s * heads + item)]);
  const float ref = top == -INFINITY ? 0.f : top;
  const int b = item / a.q_heads, h = item - b * a.q_heads;
  float total = 0.f;
  for (int s = 0; s < a.n_splits; ++s) {
    const float* st = a.stats + 2 * ((int64_t)s * heads + item);
    total = __builtin_fmaf(st[1], __builtin_amdgcn_exp2f(st[0] - ref), total);
  }
  for (int d = lane; d < D; d += kWave) {
    float o = 0.f;
    for (int s = 0; s < a.n_splits; ++s) {
      const int64_t at = (int64_t)s * heads + item;
      o = __builtin_fmaf(a.partial[at * D + d], __builtin_amdgcn_exp2f(a.stats[2 * at] - ref), o);
    }
    store_elem(a.out, a.q_dtype, (int64_t)b * a.o_bs + (int64_t)h * a.o_hs + d, total != 0.f ? o / total : 0.f);
  }
}

// ---- host --------------------------------------------------------------------------------

constexpr int kA8MaxSplits = 64;

// About two workgroups per CU, splits of at least 64 rows.
static int splits8(int64_t items, int n_rows) {
  const int64_t most = std::min<int64_t>(kA8MaxSplits, (n_rows + 63) / 64);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, 512 / items));
}

}  // namespace nhs

extern "C" int64_t nhs_attend_rows8_workspace_bytes(int32_t batch, int32_t n_rows, int32_t q_heads, int32_t kv_heads,
                                                    int32_t head_dim) {
  using namespace nhs;
  if (batch < 1 || n_rows < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1) return 0;
  const int64_t heads = (int64_t)batch * q_heads;
  const int splits = splits8(heads, n_rows);
  return splits == 1 ? 0 : splits * heads * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int nhs_attend_rows8(const void* query, int32_t q_dtype, int64_t q_batch_stride, int64_t q_head_stride,
                                const void* pool, int64_t pool_rows, int64_t pool_block_stride, int32_t code,
                                const int64_t* rows, int64_t rows_batch_stride, int64_t rows_head_stride,
                                int64_t rows_col_stride, int32_t batch, int32_t n_rows, int32_t q_heads,
                                int32_t kv_heads, int32_t head_dim, int32_t page_size, void* out,
                                int64_t out_batch_stride, int64_t out_head_stride, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  using namespace nhs;
  const LaunchEvents ev = take_launch_events();
  if (!query || !pool || !rows || !out) return fail(NHS_ERR_INVALID, "nhs_attend_rows8: null pointer");
  if (!valid_dtype(q_dtype) || !valid_code(code)) return fail(NHS_ERR_INVALID, "nhs_attend_rows8: bad dtype or code");
  if (batch < 1 || n_rows < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1 || page_size < 1 || q_heads % kv_heads ||
      n_rows > (1 << 30) || pool_rows < 0 || pool_rows >= (1ll << 31))
    return fail(NHS_ERR_INVALID, "nhs_attend_rows8: invalid shape");
  if (head_dim > NHS_MAX_HEAD_DIM8 || (int64_t)kv_heads * head_dim > (1 << 24))
    return fail(NHS_ERR_UNSUPPORTED, "nhs_attend_rows8: head_dim must be <= %d and rows of at most 2^24 elements",
                NHS_MAX_HEAD_DIM8);
  const Row8 form = row8(kv_heads, head_dim);
  const int64_t block = 2 * (int64_t)page_size * form.bytes;
  if (pool_block_stride == 0) pool_block_stride = block;
  if (pool_block_stride < block || pool_block_stride % 16 || (uintptr_t)pool % 16)
    return fail(NHS_ERR_INVALID, "nhs_attend_rows8: the pool and its block stride must be multiples of 16 bytes, the "
                "stride at least a block");
  const int64_t heads = (int64_t)batch * q_heads;
  const int64_t need = nhs_attend_rows8_workspace_bytes(batch, n_rows, q_heads, kv_heads, head_dim);
  if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
    return fail(NHS_ERR_WORKSPACE, "nhs_attend_rows8: needs a 16-byte aligned workspace of %lld bytes",
                (long long)need);
  Attend8Args a;
  a.q = query;
  a.q_dtype = q_dtype;
  a.q_bs = q_batch_stride;
  a.q_hs = q_head_stride;
  a.pool = static_cast<const char*>(pool);
  a.pool_rows = pool_rows;
  a.block_stride = pool_block_stride;
  a.row_bytes = form.bytes;
  a.scales_at = form.scales_at;
  a.plane_bytes = page_size * form.bytes;
  a.rows = rows;
  a.r_bs = rows_batch_stride;
  a.r_hs = rows_head_stride;
  a.r_cs = rows_col_stride;
  a.batch = batch;
  a.n_rows = n_rows;
  a.q_heads = q_heads;
  a.kv_heads = kv_heads;
  a.group = q_heads / kv_heads;
  a.head_dim = head_dim;
  a.page_size = page_size;
  a.page_div = FastDiv((uint32_t)page_size);
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  a.out = out;
  a.o_bs = out_batch_stride;
  a.o_hs = out_head_stride;
  a.n_splits = splits8(heads, n_rows);
  a.rows_per_split = (n_rows + a.n_splits - 1) / a.n_splits;
  a.partial = static_cast<float*>(workspace);
  a.stats = a.partial ? a.partial + a.n_splits * heads * head_dim : nullptr;
  if (heads * a.n_splits > 0x7fffffff) return fail(NHS_ERR_UNSUPPORTED, "nhs_attend_rows8: grid too large");
  const bool join = a.n_splits > 1;
  const auto run = [&](auto c, auto n) {
    launch(attend8_general_kernel<decltype(c), decltype(n)::value>, dim3((unsigned)(heads * a.n_splits)),
           dim3(kG8Threads), 0, (hipStream_t)stream, ev.start, join ? nullptr : ev.stop, a);
  };
  const auto wide = [&](auto c) {
    if (head_dim <= 2 * kWave)
      run(c, std::integral_constant<int, 2>());
    else if (head_dim <= 4 * kWave)
      run(c, std::integral_constant<int, 4>());
    else
      run(c, std::integral_constant<int, NHS_MAX_HEAD_DIM8 / kWave>());
  };
  if (code == NHS_CODE_I8)
    wide(I8());
  else
    wide(E4M3());
  if (join)
    launch(attend8_join_kernel, dim3((unsigned)heads), dim3(kWave), 0, (hipStream_t)stream, nullptr, ev.stop, a);
  return launch_status("nhs_attend_rows8");
}
