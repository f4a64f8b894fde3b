// A KV cache held in 8 bits (rows8.h): K and V rows quantised as they are
// appended to a pool page and its host mirror, with the page's key bounds and
// mean (nhs_append_page8, nhs_append_items8), and pool rows read back in a
// model's type (nhs_read_rows8).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "rows8.h"

namespace nhs {

constexpr int kA8Threads = 256;
constexpr int kA8Waves = kA8Threads / kWave;
constexpr int kA8Held = 16;     // new rows whose codes are in LDS at a time
constexpr int kA8Batch = 16;    // earlier rows loaded together for the page's mean
constexpr int kA8MaxDim = NHS_MAX_HEAD_DIM8;

struct Append8Args {
  const char* k;
  const char* v;
  int64_t token_stride;  // elements between consecutive tokens of k and v
  Row8 form;
  int page_size;
  char* pool_block;  // the page's pool block [2, page_size, form.bytes]
  char* host_block;  // its host block, or null
  int within, count;
  float* summary;
  void* minimum;
  void* maximum;
};

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) x = max(x, (uint32_t)__shfl_xor((int)x, d));
  return x;
}

// torch.minimum and torch.maximum: a NaN stays
__device__ __forceinline__ float least(float a, float b) { return (a != a || b != b) ? a + b : fminf(a, b); }
__device__ __forceinline__ float most(float a, float b) { return (a != a || b != b) ? a + b : fmaxf(a, b); }

// One plane of one KV head of a page: a wave quantises a row at a time (lane
// l its elements l, l + 64, ...; N of them at most), and for the keys a thread
// per element folds the bounds of the keys as they were given and sums what
// the page holds of them, in 64 bits and in row order, for the mean.
template <typename T, typename C, int N>
__device__ __forceinline__ void append8_head(const Append8Args& a, int plane, int head) {
  constexpr int kCols = (N * kWave + kA8Threads - 1) / kA8Threads;  // elements per folding thread
  __shared__ uint8_t held[kA8Held][N * kWave];
  __shared__ float scales[kA8Held];
  const int D = a.form.head_dim, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t slice = (int64_t)head * D;                       // of a row: elements and codes
  const int64_t at_scale = a.form.scales_at + 4 * (int64_t)head;
  const int64_t plane_at = (int64_t)plane * a.page_size * a.form.bytes;
  const char* src = plane ? a.v : a.k;
  double sum[kCols];
  float lo[kCols], hi[kCols];
  if (plane == 0) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int e = min(tid + c * kA8Threads, D - 1);
      lo[c] = load_elem(a.minimum, T::dtype, slice + e);
      hi[c] = load_elem(a.maximum, T::dtype, slice + e);
      sum[c] = 0.0;
      // unconditional loads (rows past the earlier ones re-read the last of them), masked sums
      for (int r0 = 0; r0 < a.within; r0 += kA8Batch) {
        float code[kA8Batch], scale[kA8Batch];
#pragma unroll
        for (int j = 0; j < kA8Batch; ++j) {
          const char* row = a.pool_block + (int64_t)min(r0 + j, a.within - 1) * a.form.bytes;
          code[j] = decode8<C>(static_cast<uint8_t>(row[slice + e]));
          scale[j] = *reinterpret_cast<const float*>(row + at_scale);
        }
#pragma unroll
        for (int j = 0; j < kA8Batch; ++j)
          if (r0 + j < a.within) sum[c] += (double)code[j] * (double)scale[j];
      }
    }
  }
  for (int t0 = 0; t0 < a.count; t0 += kA8Held) {
    const int n = min(kA8Held, a.count - t0);
    for (int t = wave; t < n; t += kA8Waves) {
      float x[N];
      uint32_t largest = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = lane + i * kWave;
        x[i] = e < D ? load_elem(src, T::dtype, (int64_t)(t0 + t) * a.token_stride + slice + e) : 0.f;
        largest = max(largest, __float_as_uint(x[i]) & 0x7fffffffu);
      }
      const float scale = scale8<C>(wave_max(largest)), inv = __fdiv_rn(1.f, scale);
      const int64_t row = plane_at + (int64_t)(a.within + t0 + t) * a.form.bytes;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = lane + i * kWave;
        if (e >= D) break;
        const float four[4] = {x[i], 0.f, 0.f, 0.f};
        const uint8_t code = (uint8_t)codes8<C>(four, scale, inv);
        a.pool_block[row + slice + e] = (char)code;
        if (a.host_block) a.host_block[row + slice + e] = (char)code;
        held[t][e] = code;
      }
      if (lane == 0) {
        *reinterpret_cast<float*>(a.pool_block + row + at_scale) = scale;
        if (a.host_block) *reinterpret_cast<float*>(a.host_block + row + at_scale) = scale;
        scales[t] = scale;
      }
    }
    if (plane) continue;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int e = min(tid + c * kA8Threads, D - 1);
      for (int t = 0; t < n; ++t) {
        const float key = load_elem(a.k, T::dtype, (int64_t)(t0 + t) * a.token_stride + slice + e);
        lo[c] = least(lo[c], key);
        hi[c] = most(hi[c], key);
        sum[c] += (double)decode8<C>(held[t][e]) * (double)scales[t];
      }
    }
    __syncthreads();  // the next rows overwrite the held ones
  }
  if (plane) return;
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int e = tid + c * kA8Threads;
    if (e >= D) break;
    store_elem(a.minimum, T::dtype, slice + e, lo[c]);
    store_elem(a.maximum, T::dtype, slice + e, hi[c]);
    a.summary[slice + e] = (float)(sum[c] / (double)(a.within + a.count));
  }
}

template <typename T, typename C, int N>
__global__ __launch_bounds__(kA8Threads) void append8_page_kernel(Append8Args a) {
  const int plane = (int)blockIdx.x >= a.form.kv_heads;
  append8_head<T, C, N>(a, plane, (int)blockIdx.x - plane * a.form.kv_heads);
}

struct Append8ItemsArgs {
  Append8Args a;  // k, v, token_stride, form and page_size; pool_block and host_block are the whole pool and host
  int64_t pool_block_bytes;
  const nhs_layer_item* items;
  const int64_t* lengths;
};

// The page and row that an item's one token goes to follow from its length and
// its page tables; false for one whose page is not bound, which is left alone.
template <typename T>
__device__ __forceinline__ bool item8(const Append8ItemsArgs& g, int b, Append8Args* a) {
  const nhs_layer_item& item = g.items[b];
  *a = g.a;
  const int64_t length = g.lengths[b], page = length / a->page_size;
  if (length < 0 || page >= item.n_pages) return false;
  const int block = item.resident[page], host_page = item.source[page];
  if (block < 0) return false;
  const int64_t row_elems = (int64_t)a->form.kv_heads * a->form.head_dim;
  a->k += (int64_t)b * a->token_stride * T::bytes;
  a->v += (int64_t)b * a->token_stride * T::bytes;
  a->pool_block += block * g.pool_block_bytes;
  a->host_block =
      a->host_block && host_page >= 0 ? a->host_block + host_page * 2 * (a->page_size * a->form.bytes) : nullptr;
  a->within = (int)(length - page * a->page_size);
  a->count = 1;
  a->summary = item.summaries + page * row_elems;
  a->minimum = static_cast<char*>(item.minimum) + page * row_elems * T::bytes;
  a->maximum = static_cast<char*>(item.maximum) + page * row_elems * T::bytes;
  return true;
}

template <typename T, typename C, int N>
__global__ __launch_bounds__(kA8Threads) void append8_items_kernel(Append8ItemsArgs g) {
  Append8Args a;
  if (!item8<T>(g, blockIdx.y, &a)) return;
  const int plane = (int)blockIdx.x >= a.form.kv_heads;
  append8_head<T, C, N>(a, plane, (int)blockIdx.x - plane * a.form.kv_heads);
}

// ---- heads of a multiple of 16 dims up to 256: rows of whole chunks ------------------------

// Some workgroups copy: a wave takes 64 chunks of 16 elements of a row's plane
// (so whole heads), quantises them and writes 1 KB of codes to the pool and
// past the caches to the host block, whose rows are consecutive. Others fold
// the keys of one head each: they quantise them too (the copies' codes are not
// written yet), hold 64 rows of codes and keys in LDS and walk them, a thread
// per element and share of the rows. A head is N chunks, a power of two, the
// last of them beyond its dims where its own number is none.
constexpr int kFold8Rows = 64;
constexpr int kR8Threads = 512, kR8Waves = kR8Threads / kWave;

template <typename T, int N>
struct Fold8 {
  uint32_t codes[kFold8Rows * N * 4];
  std::conditional_t<T::bytes == 4, float, uint16_t> keys[kFold8Rows * N * 16];
  float scales[kFold8Rows];
  double sums[kR8Threads];
  float low[kR8Threads], high[kR8Threads];
};

// 16 elements of one lane as they lie, and as fp32
template <typename T>
struct Chunk8 {
  u32x4 raw[T::bytes];
  float x[16];
  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int i = 0; i < T::bytes; ++i) raw[i] = reinterpret_cast<const NHS_GLOBAL u32x4*>(to_global(p))[i];
  }
  __device__ __forceinline__ void widen() {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if constexpr (T::dtype == NHS_F32) {
        x[e] = __uint_as_float(raw[e / 4][e % 4]);
      } else {
        const uint32_t half = raw[e / 8][e / 2 % 4] >> (e % 2 * 16) & 0xffffu;
        x[e] = T::dtype == NHS_BF16 ? bf16_bits_to_f32(half) : f16_bits_to_f32(half);
      }
    }
  }
};

// The codes and the scale of a slice that N neighbouring lanes hold (those that are not `live` hold none of it).
template <typename T, typename C, int N>
__device__ __forceinline__ u32x4 quantise8(Chunk8<T>& c, bool live, float* scale) {
  c.widen();
  uint32_t largest = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) largest = max(largest, __float_as_uint(c.x[e]) & 0x7fffffffu);
  largest = live ? largest : 0;
#pragma unroll
  for (int d = 1; d < N; d <<= 1) largest = max(largest, (uint32_t)__shfl_xor((int)largest, d));
  *scale = scale8<C>(largest);
  const float inv = __fdiv_rn(1.f, *scale);
  u32x4 codes;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float four[4] = {c.x[4 * i], c.x[4 * i + 1], c.x[4 * i + 2], c.x[4 * i + 3]};
    codes[i] = codes8<C>(four, *scale, inv);
  }
  return codes;
}

template <typename T, typename C, int N>
__device__ __forceinline__ void copy8(const Append8Args& a, int unit, int groups) {
  constexpr int kHeads = kWave / N;  // of a wave
  const int lane = threadIdx.x & 63, row = unit / groups, group = unit - row * groups;
  if (row >= 2 * a.count) return;
  const int plane = row >= a.count, t = row - plane * a.count;
  const int head = group * kHeads + lane / N, from = lane % N * 16;  // the lane's elements of its head
  const bool live = head < a.form.kv_heads && from < a.form.head_dim;
  const int at_elem = live ? head * a.form.head_dim + from : 0;
  Chunk8<T> c;
  c.load((plane ? a.v : a.k) + ((int64_t)t * a.token_stride + at_elem) * T::bytes);
  float scale;
  const u32x4 codes = quantise8<T, C, N>(c, live, &scale);
  const int64_t at = ((int64_t)plane * a.page_size + a.within + t) * a.form.bytes;
  const float head_scale = __shfl(scale, lane * N % kWave);
  const bool scales = lane < kHeads && group * kHeads + lane < a.form.kv_heads;
  const int64_t to_scale = at + a.form.scales_at + 4 * (group * kHeads + lane);
  if (live) {
    *(NHS_GLOBAL u32x4*)to_global(a.pool_block + at + at_elem) = codes;
    if (a.host_block) store_through(to_global(a.host_block + at + at_elem), codes);
  }
  if (scales) {
    *(NHS_GLOBAL float*)to_global(a.pool_block + to_scale) = head_scale;
    if (a.host_block) *(NHS_GLOBAL float*)to_global(a.host_block + to_scale) = head_scale;
  }
}

template <typename T, typename C, int N>
__device__ __forceinline__ void fold8(const Append8Args& a, int head) {
  constexpr int D = N * 16, kParts = kR8Threads / D, kRowsPerPass = kR8Threads / N;
  constexpr int kPasses = (kFold8Rows + kRowsPerPass - 1) / kRowsPerPass;
  __shared__ __attribute__((aligned(16))) Fold8<T, N> s;
  const int tid = threadIdx.x, chunk = tid % N, slot = tid / N;
  const int dims = a.form.head_dim, from = chunk * 16 < dims ? chunk * 16 : 0;
  const int col = min(tid % D, dims - 1), part = tid / D;
  const int64_t slice = (int64_t)head * dims, at_scale = a.form.scales_at + 4 * (int64_t)head;
  const int total = a.within + a.count;
  double sum = 0.0;
  float low = INFINITY, high = -INFINITY, low0 = 0.f, high0 = 0.f;
  if (part == 0) {
    low0 = load_elem(a.minimum, T::dtype, slice + col);
    high0 = load_elem(a.maximum, T::dtype, slice + col);
  }
  for (int r0 = 0; r0 < total; r0 += kFold8Rows) {
    const int rows = min(kFold8Rows, total - r0);
    // every load of the rows before the first wait: earlier ones from the pool, new ones as they were given (both in
    // bounds for every thread)
    u32x4 held[kPasses];
    float scale[kPasses];
    Chunk8<T> fresh[kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = min(r0 + slot + i * kRowsPerPass, total - 1);
      if (r < a.within) {
        const char* row = a.pool_block + (int64_t)r * a.form.bytes;
        held[i] = *(const NHS_GLOBAL u32x4*)to_global(row + slice + from);
        scale[i] = *(const NHS_GLOBAL float*)to_global(row + at_scale);
      }
      fresh[i].load(a.k + ((int64_t)max(r - a.within, 0) * a.token_stride + slice + from) * T::bytes);
    }
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int j = slot + i * kRowsPerPass, r = r0 + j;
      float own;
      const u32x4 codes = quantise8<T, C, N>(fresh[i], chunk * 16 < dims, &own);
      if (j >= rows) continue;
      const bool earlier = r < a.within;
      *reinterpret_cast<u32x4*>(&s.codes[(j * N + chunk) * 4]) = earlier ? held[i] : codes;
      if (!earlier)
#pragma unroll
        for (int x = 0; x < T::bytes; ++x)
          reinterpret_cast<u32x4*>(&s.keys[(j * N + chunk) * 16])[x] = fresh[i].raw[x];
      if (chunk == 0) s.scales[j] = earlier ? scale[i] : own;
    }
    __syncthreads();
    const uint8_t* codes = reinterpret_cast<const uint8_t*>(s.codes) + col;
#pragma unroll 8
    for (int j = part; j < rows; j += kParts) sum += (double)decode8<C>(codes[j * D]) * (double)s.scales[j];
#pragma unroll 8
    for (int j = max(a.within - r0, 0) + part; j < rows; j += kParts) {
      const float key = load_elem(s.keys, T::dtype, j * D + col);
      low = least(low, key);
      high = most(high, key);
    }
    __syncthreads();
  }
  s.sums[tid] = sum;
  s.low[tid] = low;
  s.high[tid] = high;
  __syncthreads();
  if (part || tid % D >= dims) return;
#pragma unroll
  for (int p = 1; p < kParts; ++p) {
    sum += s.sums[p * D + col];
    low = least(low, s.low[p * D + col]);
    high = most(high, s.high[p * D + col]);
  }
  store_elem(a.minimum, T::dtype, slice + col, least(low0, low));
  store_elem(a.maximum, T::dtype, slice + col, most(high0, high));
  a.summary[slice + col] = (float)(sum / (double)total);
}

template <typename T, typename C, int N>
__device__ __forceinline__ void append8_rows(const Append8Args& a) {
  const int group = blockIdx.x;
  if (group < a.form.kv_heads) return fold8<T, C, N>(a, group);
  const int groups = (a.form.kv_heads * N + kWave - 1) / kWave;
  copy8<T, C, N>(a, (group - a.form.kv_heads) * kR8Waves + ((int)threadIdx.x >> 6), groups);
}

// Workgroups of a launch for `count` rows of heads of N chunks.
static unsigned rows8_grid(const Row8& form, int count, int N) {
  const int64_t groups = ((int64_t)form.kv_heads * N + kWave - 1) / kWave;
  return (unsigned)(form.kv_heads + (2 * count * groups + kR8Waves - 1) / kR8Waves);
}

template <typename T, typename C, int N>
__global__ __launch_bounds__(kR8Threads) void append8_rows_kernel(Append8Args a) {
  append8_rows<T, C, N>(a);
}

template <typename T, typename C, int N>
__global__ __launch_bounds__(kR8Threads) void append8_item_rows_kernel(Append8ItemsArgs g) {
  Append8Args a;
  if (item8<T>(g, blockIdx.y, &a)) append8_rows<T, C, N>(a);
}

// ---- read back ----------------------------------------------------------------------

struct Read8Args {
  const char* pool;
  int64_t pool_rows, block_stride;
  Row8 form;
  int page_size;
  FastDiv page_div, dim_div;
  const int64_t* rows;
  int64_t rows_stride;
  int64_t n;
  char* out[2];
  int64_t out_stride[2];  // elements between rows
};

__device__ __forceinline__ const char* row8_at(const char* pool, int64_t row, int64_t pool_rows, int64_t block_stride,
                                               int64_t row_bytes, int page_size, FastDiv page_div) {
  if (row < 0 || row >= pool_rows) return nullptr;
  const uint32_t page = page_div.div((uint32_t)row);
  return pool + page * block_stride + (int64_t)((uint32_t)row - page * page_size) * row_bytes;
}

// A wave per row and plane.
template <typename T, typename C>
__global__ __launch_bounds__(256) void read8_kernel(Read8Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= 2 * a.n) return;
  const int plane = (int)(unit & 1);
  const int64_t i = unit >> 1;
  const char* row = row8_at(a.pool, a.rows[i * a.rows_stride], a.pool_rows, a.block_stride, a.form.bytes, a.page_size,
                            a.page_div);
  if (row) row += (int64_t)plane * a.page_size * a.form.bytes;
  char* out = a.out[plane] + i * a.out_stride[plane] * T::bytes;
  const int width = a.form.kv_heads * a.form.head_dim;
  for (int e = lane; e < width; e += kWave) {
    float value = 0.f;
    if (row) {
      const int head = (int)a.dim_div.div((uint32_t)e);
      value = value8(decode8<C>((uint8_t)row[e]), *reinterpret_cast<const float*>(row + a.form.scales_at + 4 * head));
    }
    store_elem(out, T::dtype, e, value);
  }
}

// Heads of a multiple of 8 dims: a thread turns V codes into 16 bytes, kRead8
// of them in flight (heads and units of a row by exact division).
constexpr int kRead8 = 4;

// STREAM: past the caches. Whoever reads the outputs finds them there only if
// they fit beside its own traffic; then the plain stores are better, else
// these. us of a read, its rows not in a cache, and a copy of its outputs,
// plain and streamed: 8 MB 13.9, 15.7; 32 MB 34.5, 37.5; 64 MB 55.9, 63.4; 128
// MB 113.5, 108.9; 256 MB 201, 196.
constexpr int64_t kRead8Stream = 96 << 20;  // bytes of both outputs

template <typename T, typename C, bool STREAM>
__global__ __launch_bounds__(256) void read8_chunks_kernel(Read8Args a, FastDiv per_row, FastDiv per_head,
                                                           int rows_per_group) {
  constexpr int V = 16 / T::bytes;
  const int64_t first = (int64_t)blockIdx.x * rows_per_group;
  const uint32_t units = (uint32_t)min((int64_t)rows_per_group, a.n - first) * per_row.d, half = per_row.d / 2;
  for (uint32_t x0 = threadIdx.x; x0 < units; x0 += 256 * kRead8) {
    uint32_t code[kRead8][V / 4];
    float scale[kRead8];
    bool there[kRead8];
    char* out[kRead8];
#pragma unroll
    for (int u = 0; u < kRead8; ++u) {
      const uint32_t x = min(x0 + u * 256, units - 1), i = per_row.div(x), in_row = x - i * per_row.d;
      const uint32_t plane = in_row >= half, unit = in_row - plane * half;
      const int64_t at = first + i;
      const char* row = row8_at(a.pool, a.rows[at * a.rows_stride], a.pool_rows, a.block_stride, a.form.bytes,
                                a.page_size, a.page_div);
      out[u] = (plane ? a.out[1] : a.out[0]) + (at * (plane ? a.out_stride[1] : a.out_stride[0]) + unit * V) * T::bytes;
      // unconditional loads (row 0 in place of one outside the pool), so that no branch separates them
      const char* from = (row ? row : a.pool) + (int64_t)plane * a.page_size * a.form.bytes;
#pragma unroll
      for (int w = 0; w < V / 4; ++w)
        code[u][w] = reinterpret_cast<const NHS_GLOBAL uint32_t*>(to_global(from) + unit * V)[w];
      scale[u] = *(const NHS_GLOBAL float*)(to_global(from) + a.form.scales_at + 4 * per_head.div(unit));
      there[u] = row != nullptr;
    }
#pragma unroll
    for (int u = 0; u < kRead8; ++u) {
      if (x0 + u * 256 >= units) break;
      float v[V];
#pragma unroll
      for (int w = 0; w < V / 4; ++w) {
        float four[4];
        decode8<C>(code[u][w], four);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * w + e] = there[u] ? value8(four[e], scale[u]) : 0.f;
      }
      u32x4 words;
      if constexpr (T::dtype == NHS_F32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) words[e] = __float_as_uint(v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          words[e] = T::dtype == NHS_BF16
                         ? f32_to_bf16_bits(v[2 * e]) | (uint32_t)f32_to_bf16_bits(v[2 * e + 1]) << 16
                         : f32_to_f16_bits(v[2 * e]) | (uint32_t)f32_to_f16_bits(v[2 * e + 1]) << 16;
      }
      NHS_GLOBAL u32x4* to = (NHS_GLOBAL u32x4*)to_global(out[u]);
      if constexpr (STREAM)
        __builtin_nontemporal_store(words, to);
      else
        *to = words;
    }
  }
}

// Calls f with the tags of a storage type and a code.
template <typename F>
static void with_types(int dtype, int code, F f) {
  const auto second = [&](auto t) {
    if (code == NHS_CODE_I8)
      f(t, I8());
    else
      f(t, E4M3());
  };
  if (dtype == NHS_BF16)
    second(BF16());
  else if (dtype == NHS_F16)
    second(F16());
  else
    second(F32());
}

// Common checks of a pool of rows in 8 bits; sets a zero block stride to that of contiguous blocks.
static int check_pool8(const char* who, const void* pool, int code, int kv_heads, int head_dim, int page_size,
                       int64_t* block_stride) {
  if (!pool) return fail(NHS_ERR_INVALID, "%s: null pointer", who);
  if (!valid_code(code)) return fail(NHS_ERR_INVALID, "%s: bad code", who);
  if (kv_heads < 1 || head_dim < 1 || page_size < 1) return fail(NHS_ERR_INVALID, "%s: invalid shape", who);
  if (head_dim > NHS_MAX_HEAD_DIM8 || (int64_t)kv_heads * head_dim > (1 << 24))
    return fail(NHS_ERR_UNSUPPORTED, "%s: head_dim must be <= %d and rows of at most 2^24 elements", who,
                NHS_MAX_HEAD_DIM8);
  const int64_t block = 2 * (int64_t)page_size * row8(kv_heads, head_dim).bytes;
  if (*block_stride == 0) *block_stride = block;
  if (*block_stride < block || *block_stride % 16 || (uintptr_t)pool % 16)
    return fail(NHS_ERR_INVALID, "%s: the pool and its block stride must be multiples of 16 bytes, the stride at least "
                "a block", who);
  return NHS_OK;
}

// Whether rows are whole chunks of 16 elements wherever append8_rows touches them.
static bool whole_chunks8(const Append8Args& a, int dtype) {
  const int d = a.form.head_dim;
  return d % 16 == 0 && d <= 256 && a.token_stride * elem_size(dtype) % 16 == 0 &&
         ((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0;
}

// Calls f with the chunks of 16 elements of a head, rounded up to a power of two.
template <typename F>
static void with_chunks(int head_dim, F f) {
  if (head_dim <= 32)
    f(std::integral_constant<int, 2>());
  else if (head_dim <= 64)
    f(std::integral_constant<int, 4>());
  else if (head_dim <= 128)
    f(std::integral_constant<int, 8>());
  else
    f(std::integral_constant<int, 16>());
}

template <typename T, typename C, typename F>
static void with_width(int head_dim, F f) {
  if (head_dim <= 2 * kWave)
    f(std::integral_constant<int, 2>());
  else if (head_dim <= 4 * kWave)
    f(std::integral_constant<int, 4>());
  else
    f(std::integral_constant<int, kA8MaxDim / kWave>());
}

}  // namespace nhs

extern "C" int64_t nhs_row8_bytes(int32_t kv_heads, int32_t head_dim) {
  return kv_heads < 1 || head_dim < 1 ? 0 : nhs::row8(kv_heads, head_dim).bytes;
}

extern "C" int nhs_append_page8(const void* k, const void* v, int64_t token_stride, int32_t kv_dtype, int32_t code,
                                int32_t kv_heads, int32_t head_dim, int32_t page_size, void* pool,
                                int64_t pool_block_stride, int64_t block, int32_t within, int32_t count,
                                void* host_alias, int64_t host_page, float* summary, void* minimum, void* maximum,
                                void* stream) {
  using namespace nhs;
  const LaunchEvents ev = take_launch_events();
  if (!k || !v || !summary || !minimum || !maximum) return fail(NHS_ERR_INVALID, "nhs_append_page8: null pointer");
  if (!valid_dtype(kv_dtype)) return fail(NHS_ERR_INVALID, "nhs_append_page8: bad dtype");
  if (const int st = check_pool8("nhs_append_page8", pool, code, kv_heads, head_dim, page_size, &pool_block_stride))
    return st;
  if (block < 0 || within < 0 || count < 1 || count > page_size || within > page_size - count ||
      token_stride < (int64_t)kv_heads * head_dim || (host_alias && host_page < 0) || (uintptr_t)host_alias % 16)
    return fail(NHS_ERR_INVALID, "nhs_append_page8: invalid page, rows, strides or host alignment");
  Append8Args a;
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.token_stride = token_stride;
  a.form = row8(kv_heads, head_dim);
  a.page_size = page_size;
  a.pool_block = static_cast<char*>(pool) + block * pool_block_stride;
  a.host_block = host_alias ? static_cast<char*>(host_alias) + host_page * 2 * (page_size * a.form.bytes) : nullptr;
  a.within = within;
  a.count = count;
  a.summary = summary;
  a.minimum = minimum;
  a.maximum = maximum;
  if (whole_chunks8(a, kv_dtype)) {
    with_types(kv_dtype, code, [&](auto t, auto c) {
      with_chunks(head_dim, [&](auto n) {
        launch(append8_rows_kernel<decltype(t), decltype(c), decltype(n)::value>,
               dim3(rows8_grid(a.form, count, decltype(n)::value)), dim3(kR8Threads), 0, (hipStream_t)stream, ev.start,
               ev.stop, a);
      });
    });
    return launch_status("nhs_append_page8");
  }
  with_types(kv_dtype, code, [&](auto t, auto c) {
    using T = decltype(t);
    using C = decltype(c);
    with_width<T, C>(head_dim, [&](auto n) {
      launch(append8_page_kernel<T, C, decltype(n)::value>, dim3((unsigned)(2 * kv_heads)), dim3(kA8Threads), 0,
             (hipStream_t)stream, ev.start, ev.stop, a);
    });
  });
  return launch_status("nhs_append_page8");
}

extern "C" int nhs_append_items8(int32_t batch, const void* k, const void* v, int64_t token_stride, int32_t kv_dtype,
                                 int32_t code, int32_t kv_heads, int32_t head_dim, int32_t page_size, void* pool,
                                 int64_t pool_block_stride, void* host_alias, const nhs_layer_item* items,
                                 const int64_t* lengths, void* stream) {
  using namespace nhs;
  const LaunchEvents ev = take_launch_events();
  if (!k || !v || !items || !lengths) return fail(NHS_ERR_INVALID, "nhs_append_items8: null pointer");
  if (!valid_dtype(kv_dtype)) return fail(NHS_ERR_INVALID, "nhs_append_items8: bad dtype");
  if (const int st = check_pool8("nhs_append_items8", pool, code, kv_heads, head_dim, page_size, &pool_block_stride))
    return st;
  if (batch < 0 || batch > 65535 || token_stride < (int64_t)kv_heads * head_dim || (uintptr_t)host_alias % 16)
    return fail(NHS_ERR_INVALID, "nhs_append_items8: invalid batch, strides or host alignment");
  if (batch == 0) return NHS_OK;
  Append8ItemsArgs g;
  g.a = Append8Args();
  g.a.k = static_cast<const char*>(k);
  g.a.v = static_cast<const char*>(v);
  g.a.token_stride = token_stride;
  g.a.form = row8(kv_heads, head_dim);
  g.a.page_size = page_size;
  g.a.pool_block = static_cast<char*>(pool);
  g.a.host_block = static_cast<char*>(host_alias);
  g.pool_block_bytes = pool_block_stride;
  g.items = items;
  g.lengths = lengths;
  if (whole_chunks8(g.a, kv_dtype)) {
    with_types(kv_dtype, code, [&](auto t, auto c) {
      with_chunks(head_dim, [&](auto n) {
        launch(append8_item_rows_kernel<decltype(t), decltype(c), decltype(n)::value>,
               dim3(rows8_grid(g.a.form, 1, decltype(n)::value), (unsigned)batch), dim3(kR8Threads), 0,
               (hipStream_t)stream, ev.start, ev.stop, g);
      });
    });
    return launch_status("nhs_append_items8");
  }
  with_types(kv_dtype, code, [&](auto t, auto c) {
    using T = decltype(t);
    using C = decltype(c);
    with_width<T, C>(head_dim, [&](auto n) {
      launch(append8_items_kernel<T, C, decltype(n)::value>, dim3((unsigned)(2 * kv_heads), (unsigned)batch),
             dim3(kA8Threads), 0, (hipStream_t)stream, ev.start, ev.stop, g);
    });
  });
  return launch_status("nhs_append_items8");
}

extern "C" int nhs_read_rows8(const void* pool, int64_t pool_rows, int64_t pool_block_stride, int32_t code,
                              int32_t kv_heads, int32_t head_dim, int32_t page_size, const int64_t* rows,
                              int64_t rows_stride, int64_t n, int32_t out_dtype, void* k_out, int64_t k_stride,
                              void* v_out, int64_t v_stride, void* stream) {
  using namespace nhs;
  const LaunchEvents ev = take_launch_events();
  if (!rows || !k_out || !v_out) return fail(NHS_ERR_INVALID, "nhs_read_rows8: null pointer");
  if (!valid_dtype(out_dtype)) return fail(NHS_ERR_INVALID, "nhs_read_rows8: bad dtype");
  if (const int st = check_pool8("nhs_read_rows8", pool, code, kv_heads, head_dim, page_size, &pool_block_stride))
    return st;
  const int64_t width = (int64_t)kv_heads * head_dim;
  if (n < 0 || pool_rows < 0 || pool_rows >= (1ll << 31) || k_stride < width || v_stride < width)
    return fail(NHS_ERR_INVALID, "nhs_read_rows8: invalid rows or strides");
  if (n == 0) return NHS_OK;
  const int64_t groups = (2 * n + 3) / 4;
  if (groups > 0x7fffffff) return fail(NHS_ERR_UNSUPPORTED, "nhs_read_rows8: too many rows");
  Read8Args a;
  a.pool = static_cast<const char*>(pool);
  a.pool_rows = pool_rows;
  a.block_stride = pool_block_stride;
  a.form = row8(kv_heads, head_dim);
  a.page_size = page_size;
  a.page_div = FastDiv((uint32_t)page_size);
  a.dim_div = FastDiv((uint32_t)head_dim);
  a.rows = rows;
  a.rows_stride = rows_stride;
  a.n = n;
  a.out[0] = static_cast<char*>(k_out);
  a.out[1] = static_cast<char*>(v_out);
  a.out_stride[0] = k_stride;
  a.out_stride[1] = v_stride;
  const int esize = elem_size(out_dtype), vec = 16 / esize;
  if (pool_rows > 0 && head_dim % 8 == 0 && ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0 &&
      k_stride * esize % 16 == 0 && v_stride * esize % 16 == 0) {
    const uint32_t per_row = (uint32_t)(2 * width / vec);
    const int rows_per_group = (int)std::max<int64_t>(1, 256 * kRead8 / per_row);
    const int64_t grid = (n + rows_per_group - 1) / rows_per_group;
    if (grid > 0x7fffffff) return fail(NHS_ERR_UNSUPPORTED, "nhs_read_rows8: too many rows");
    with_types(out_dtype, code, [&](auto t, auto c) {
      using T = decltype(t);
      using C = decltype(c);
      launch(2 * n * width * esize >= kRead8Stream ? read8_chunks_kernel<T, C, true> : read8_chunks_kernel<T, C, false>,
             dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, ev.start, ev.stop, a, FastDiv(per_row),
             FastDiv((uint32_t)(head_dim / vec)), rows_per_group);
    });
    return launch_status("nhs_read_rows8");
  }
  with_types(out_dtype, code, [&](auto t, auto c) {
    launch(read8_kernel<decltype(t), decltype(c)>, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, ev.start,
           ev.stop, a);
  });
  return launch_status("nhs_read_rows8");
}
