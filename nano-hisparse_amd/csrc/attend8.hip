// Decode attention over pool rows held in 8 bits (rows8.h): nhs_attend_rows8.
//
// For request b and query head h (KV head h / group), over the rows r of the
// list with 0 <= r < pool rows:
//   out[b, h] = sum_r softmax_r(q[b, h] . K[r] D^-1/2) V[r]
// and zeros where the list holds none. The scale of a row's keys multiplies
// its score, that of its values its weight, so the products run on the codes.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "rows8.h"

namespace nhs {

// An element of a query, NaN in place of an infinity. With an infinity every
// score is one too, or NaN, so the softmax is NaN; but where all of them are
// minus infinity the sums below would read as those of a list without a row.
__device__ __forceinline__ float query8(float x) { return x + (x - x); }

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
  // the kernel on the matrix cores: items of a (request, split) = kv_heads x chunks of heads_per_item query heads
  int heads_per_item, chunks, subs, groups;
  bool near, q_aligned;  // near: the items of a (request, split) on one XCD
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
    q[i] = d < D ? query8(load_elem(a.q, a.q_dtype, (int64_t)b * a.q_bs + (int64_t)h * a.q_hs + d)) : 0.f;
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

// ---- heads of a multiple of 16 dims up to 256, on the matrix cores -------------------------

// A workgroup of 8 waves takes up to 16 query heads of one (request, KV head)
// and one split of the rows; wave w takes tiles w, w + 8, ... of 32 rows.
// Codes are exact in bf16, so the products run on v_mfma_f32_16x16x32_bf16:
// S^T = K Q^T and O^T = V^T P^T. Lane l supplies A[l % 16][8 (l / 16) + j] and
// B[8 (l / 16) + j][l % 16], j = 0..7, and holds D[4 (l / 16) + i][l % 16],
// i = 0..3: so lane l has the scores of head l % 16 against rows 4 (l / 16) + i
// of the tile's halves, which are the rows it has to supply to P^T (the order
// of rows within a product is free), its softmax is a lane's own work, and V
// comes transposed from LDS (ds_read_b64_tr_b8: of each 16 lanes, lanes 2r and
// 2r + 1 name 16 bytes of row r, and lane i receives column i of the 8 rows).
//
// A bf16 query is one operand, an fp16 query the sum of two bf16 numbers and
// an fp32 query of three, exactly; a weight (times the scale of the row's
// values) goes as two bf16 numbers, 2^-17 of it lost, or for fp32 queries as
// three.
//
// Measured (MI355X, rows from HBM, graphs; us with the join of the splits): 16
// requests x 2048 rows of 32/8 heads of 128, bf16 and e4m3, 21.8 (69 MB; the
// general kernel 887); 64 x 1024 rows of 28/4 heads, int8, 21.1 in one launch;
// one request x 32768 rows 22.6; 32 x 2048 rows 33.3. The rows stream at 5.6
// TB/s once they flow (1.03 times their bytes are read), but 3.5 us pass
// before the first are in; the scales, a line for each row and head, take 2.4,
// what follows the last row 2, the join 3 to 4.
//
// The heads of a (request, split) are workgroups on one XCD (`near`): a head's
// slice of a row begins at any multiple of 32 bytes, so neighbours share cache
// lines, and all share those of the scales (spread over the XCDs: 16 x 2048 rows
// 33.9 us where they take 21.9, 8 x 2048 21.0 where 15.2). With fewer than 8
// such groups the heads are spread instead, over more of the XCDs.
//
// Heads that are no power of two run in the next larger D (PAD): chunks past
// their dims are zeros, which add nothing to a score and to no one's output.
constexpr int kF8Threads = 512, kF8Waves = kF8Threads / kWave, kF8Tile = 32, kF8Heads = 16;

typedef __bf16 f8_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 f8_bf16x2 __attribute__((ext_vector_type(2)));
typedef float f8_f32x2 __attribute__((ext_vector_type(2)));
typedef float f8_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t f8_u32x4 __attribute__((ext_vector_type(4)));
typedef int f8_i32x2 __attribute__((ext_vector_type(2)));

__device__ __attribute__((aligned(256))) char attend8_zeros[256];  // read in place of a masked row

__device__ __forceinline__ f8_f32x4 f8_mfma(f8_u32x4 a, f8_u32x4 b, f8_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(f8_bf16x8, a), __builtin_bit_cast(f8_bf16x8, b), c,
                                                 0, 0, 0);
}

// two codes (the lower or the upper half of a word) as a pair of bf16 numbers, exactly
template <typename C, bool UPPER>
__device__ __forceinline__ uint32_t f8_pair(uint32_t word) {
  if constexpr (C::code == NHS_CODE_E4M3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)word, 1.f, UPPER));
  } else {
    const float a = (float)(int8_t)(word >> (UPPER ? 16 : 0)), b = (float)(int8_t)(word >> (UPPER ? 24 : 8));
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
}

// eight codes as an operand
template <typename C>
__device__ __forceinline__ f8_u32x4 f8_operand(uint32_t lo, uint32_t hi) {
  return (f8_u32x4){f8_pair<C, false>(lo), f8_pair<C, true>(lo), f8_pair<C, false>(hi), f8_pair<C, true>(hi)};
}

__device__ __forceinline__ uint32_t f8_round(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f8_f32x2){lo, hi}, f8_bf16x2));
}

// eight fp32 numbers as P bf16 operands: their sum with one part for bf16 numbers, two for fp16, three for fp32, else
// near it (two parts of an fp32 weight lose up to 2^-17 of it; the denominator takes the weight as it was)
template <int P>
__device__ __forceinline__ void f8_split(float (&x)[8], f8_u32x4 (&out)[P]) {
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = f8_round(x[2 * j], x[2 * j + 1]);
      out[p][j] = pair;
      if (p + 1 < P) {
        x[2 * j] -= __uint_as_float(pair << 16);
        x[2 * j + 1] -= __uint_as_float(pair & 0xffff0000u);
      }
    }
}

// LDS slot of 16-byte chunk c of K row r (N chunks a row): eight consecutive rows at one chunk fall on distinct banks
template <int N>
__device__ __forceinline__ int f8_k_slot(int r, int c) {
  return N >= 8 ? c ^ (r & 7) : N == 4 ? c ^ ((r >> 1) & 3) : c ^ ((r >> 2) & 1);
}
// and of V row r: the eight rows of a transposing read, 4g .. 4g + 3 of both halves of a tile
template <int N>
__device__ __forceinline__ int f8_v_slot(int r, int c) {
  return N >= 8   ? c ^ ((r & 3) | (r >> 2 & 4))
         : N == 4 ? c ^ ((r >> 1 & 1) | (r >> 3 & 2))
                  : c ^ (r >> 4 & 1);
}

// The tiles in LDS are written and read by the lanes of one wave, whose LDS instructions the hardware runs in order:
// only the compiler has to keep them so.
__device__ __forceinline__ void f8_order() { asm volatile("" ::: "memory"); }

template <typename C, int QP, int D, int DEPTH, bool LOOP, bool PAD>
__global__ __launch_bounds__(kF8Threads) void attend8_flash_kernel(Attend8Args a) {
  constexpr int PP = QP == 3 ? 3 : 2;     // operands of the weights
  constexpr int N = D / 16;               // 16-byte chunks of a head's row
  constexpr int RI = kWave / N;           // rows of a load instruction
  constexpr int KI = kF8Tile / RI;        // load instructions of a tile, for K and for V each
  constexpr int KS = D / 32;              // products of a score
  constexpr int kRows = DEPTH * kF8Tile;  // of a wave's round
  constexpr bool kAhead = D != 256 || QP == 1;  // (the others have no registers left for it)
  struct Wave {
    f8_u32x4 k[kF8Tile * N], v[kF8Tile * N];
    const char* at[kRows][2];  // the rows' K and V
    float ks[kRows], vs[kRows];
  };
  constexpr int kMerged = kF8Waves * kF8Heads * (D + 4) * 4;
  constexpr int kBytes = kF8Waves * (int)sizeof(Wave) > kMerged ? kF8Waves * (int)sizeof(Wave) : kMerged;
  __shared__ __attribute__((aligned(16))) char lds[kBytes];

  const int dims = PAD ? a.head_dim : D;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  __builtin_amdgcn_s_setprio(3);  // (see the loads)
  int sub, group;
  if (a.near) {
    const int rest = blockIdx.x >> 3;
    sub = rest % a.subs;
    group = rest / a.subs * 8 + (blockIdx.x & 7);
    if (group >= a.groups) return;
  } else {
    sub = blockIdx.x % a.subs;
    group = blockIdx.x / a.subs;
  }
  const int b = group / a.n_splits, split = group - b * a.n_splits;
  const int kv = sub / a.chunks, h0 = kv * a.group + (sub - kv * a.chunks) * a.heads_per_item;
  const int heads = min(a.heads_per_item, (kv + 1) * a.group - h0);
  Wave& w = reinterpret_cast<Wave*>(lds)[wave];

  const int64_t* list = a.rows + (int64_t)b * a.r_bs + (int64_t)h0 * a.r_hs;
  const int begin = split * a.rows_per_split, end = min(a.n_rows, begin + a.rows_per_split);
  // row of the wave's round that entry e of its addresses is for
  const auto row_of = [&](int round, int e) {
    return begin + ((round * DEPTH + e / kF8Tile) * kF8Waves + wave) * kF8Tile + e % kF8Tile;
  };
  constexpr int kMine = (kRows + kWave - 1) / kWave;  // addresses of a lane
  int64_t index[kMine];
  const auto fetch = [&](int round) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int r = row_of(round, (lane + i * kWave) % kRows);
      index[i] = r < end ? list[(int64_t)r * a.r_cs] : -1;
    }
  };
  fetch(0);

  // the query as operand B: head n, dims in the order in which K's chunks give them
  f8_u32x4 q[QP][KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int d0 = N >= 4 ? 16 * (4 * (s / 2) + g) + 8 * (s % 2) : 8 * g;
    float x[8];
    const int64_t at = (int64_t)b * a.q_bs + (int64_t)(h0 + min(n, heads - 1)) * a.q_hs + d0;
    if (PAD && d0 >= dims) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
    } else if (a.q_aligned) {
      if constexpr (QP == 1)
        load_vec<BF16, 8>(a.q, at, x);
      else if constexpr (QP == 2)
        load_vec<F16, 8>(a.q, at, x);
      else
        load_vec<F32, 8>(a.q, at, x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = load_elem(a.q, QP == 1 ? NHS_BF16 : QP == 2 ? NHS_F16 : NHS_F32, at + j);
    }
    if constexpr (QP == 1)  // (in parts an infinity leaves NaN)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = query8(x[j]);
    f8_u32x4 parts[QP];
    f8_split<QP>(x, parts);
#pragma unroll
    for (int p = 0; p < QP; ++p) q[p][s] = parts[p];
  }

  f8_f32x4 acc[N];
#pragma unroll
  for (int t = 0; t < N; ++t) acc[t] = (f8_f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  const int rounds = (end - begin + kF8Waves * kRows - 1) / (kF8Waves * kRows);
  uint64_t seen[kMine];
  float ks[kMine], vs[kMine];
  // addresses of a round's rows to LDS, their scales asked for
  const auto stage = [&] {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const bool in = index[i] >= 0 && index[i] < a.pool_rows;
      const uint32_t at = in ? (uint32_t)index[i] : 0u, page = a.page_div.div(at);
      const char* row = a.pool + page * a.block_stride + (int64_t)(at - page * a.page_size) * a.row_bytes;
      const char* kp = in ? row + kv * dims : attend8_zeros;
      const char* vp = in ? row + a.plane_bytes + kv * dims : attend8_zeros;
      const int64_t to_scale = in ? a.scales_at + 4 * (int64_t)kv - kv * dims : 0;
      seen[i] = __ballot(in);
      if (kMine * kWave == kRows || lane < kRows) {
        w.at[lane + i * kWave][0] = kp;
        w.at[lane + i * kWave][1] = vp;
      }
      ks[i] = *(const NHS_GLOBAL float*)(kp + to_scale);
      vs[i] = *(const NHS_GLOBAL float*)(vp + to_scale);
    }
    f8_order();
  };
  // The loads of a round's keys or values. Non-temporal, since no one reads a row's codes again (their lines are shared
  // with the neighbouring heads of the same moment), and ahead of the arithmetic of the wave's neighbours. us of 16 x
  // 2048 rows of 32/8 heads, 64 x 1024 of 28/4: 23.8, 22.3 plain, 22.3, 21.2 non-temporal, 21.8, 20.9 with the
  // priority; with non-temporal scales too (whose lines all heads read) 23.3, 23.2.
  f8_u32x4 k[DEPTH][KI], v[DEPTH][KI];
  const auto load = [&](int plane, f8_u32x4(&to)[DEPTH][KI]) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const char* at = w.at[d * kF8Tile + i * RI + lane / N][plane] + lane % N * 16;
        if (PAD && lane % N * 16 >= dims) at = attend8_zeros;
        to[d][i] = __builtin_nontemporal_load((const NHS_GLOBAL f8_u32x4*)at);
      }
  };
  if (rounds > 0) {
    stage();
    if (LOOP && rounds > 1) fetch(1);
    load(0, k);
  }
  // Keys first: scores and weights are there when the last values come. Where there are several rounds, the next one's
  // keys are asked for as soon as this one's have been multiplied (32 requests x 2048 rows of 32/8 heads 33.4 us, 36.2
  // without).
  for (int round = 0; round < (LOOP ? rounds : min(rounds, 1)); ++round) {  // (without LOOP there is one, see plan8)
    load(1, v);
    __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (kMine * kWave == kRows || lane < kRows) {
        w.ks[lane + i * kWave] = ks[i] * a.scale_log2;
        w.vs[lane + i * kWave] = vs[i];
      }
    // scores of rows 4g + i and 16 + 4g + i of every tile
    float p[DEPTH][8], top = m;
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      f8_order();
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int r = i * RI + lane / N;
        w.k[r * N + f8_k_slot<N>(r, lane % N)] = k[d][i];
      }
      f8_order();
      const uint32_t word = (uint32_t)(seen[d * kF8Tile / kWave] >> (d * kF8Tile % kWave));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f8_f32x4 s = (f8_f32x4){0.f, 0.f, 0.f, 0.f};
        const int r = 16 * u + n;
        if constexpr (N >= 4) {
#pragma unroll
          for (int c = 0; c < N / 4; ++c) {
            const f8_u32x4 x = w.k[r * N + f8_k_slot<N>(r, 4 * c + g)];
            const f8_u32x4 lo = f8_operand<C>(x[0], x[1]), hi = f8_operand<C>(x[2], x[3]);
#pragma unroll
            for (int part = 0; part < QP; ++part) {
              s = f8_mfma(lo, q[part][2 * c], s);
              s = f8_mfma(hi, q[part][2 * c + 1], s);
            }
          }
        } else {
          const char* at = reinterpret_cast<const char*>(&w.k[r * N + f8_k_slot<N>(r, g >> 1)]) + 8 * (g & 1);
          const uint2 x = *reinterpret_cast<const uint2*>(at);
#pragma unroll
          for (int part = 0; part < QP; ++part) s = f8_mfma(f8_operand<C>(x.x, x.y), q[part][0], s);
        }
        const f8_f32x4 scale = *reinterpret_cast<const f8_f32x4*>(&w.ks[d * kF8Tile + 16 * u + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float score = word >> (16 * u + 4 * g + i) & 1 ? s[i] * scale[i] : -INFINITY;
          p[d][4 * u + i] = score;
          top = fmaxf(top, score);
        }
      }
    }
    const auto next = [&] {
      if (!LOOP || round + 1 >= rounds) return;
      f8_order();
      stage();
      if (round + 2 < rounds) fetch(round + 2);
      load(0, k);
    };
    if constexpr (kAhead) next();
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float ref = top == -INFINITY ? 0.f : top, alpha = __builtin_amdgcn_exp2f(m - ref);
    m = top;
    l *= alpha;
    if (round > 0 && __ballot(alpha != 1.f) != 0) {
#pragma unroll
      for (int t = 0; t < N; ++t) acc[t] *= alpha;
    }
    f8_u32x4 weights[DEPTH][PP];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f8_f32x4 scale = *reinterpret_cast<const f8_f32x4*>(&w.vs[d * kF8Tile + 16 * u + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(p[d][4 * u + i] - ref);
          l += e;
          p[d][4 * u + i] = e * scale[i];
        }
      }
      f8_split<PP>(p[d], weights[d]);
    }
    const int vr = (n >> 1 & 3) + 4 * g + (n >> 3) * 16;  // the row that this lane names for a transposing read
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      f8_order();
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int r = i * RI + lane / N;
        w.v[r * N + f8_v_slot<N>(r, lane % N)] = v[d][i];
      }
      f8_order();
#pragma unroll
      for (int t = 0; t < N; ++t) {
        const char* at = reinterpret_cast<const char*>(&w.v[vr * N + f8_v_slot<N>(vr, t)]) + 8 * (n & 1);
        const f8_i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) f8_i32x2*)const_cast<char*>(at));
        const f8_u32x4 values = f8_operand<C>((uint32_t)x.x, (uint32_t)x.y);
#pragma unroll
        for (int part = 0; part < PP; ++part) acc[t] = f8_mfma(values, weights[d][part], acc[t]);
      }
    }
    if constexpr (!kAhead) next();
    f8_order();
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // the waves' sums are joined through LDS: [wave][head][D, max, sum]
  __syncthreads();
  constexpr int kPitch = D + 4;
  float* merged = reinterpret_cast<float*>(lds);
  if (n < heads) {
    float* mine = merged + (wave * heads + n) * kPitch;
#pragma unroll
    for (int t = 0; t < N; ++t) *reinterpret_cast<f8_f32x4*>(mine + 16 * t + 4 * g) = acc[t];
    if (g == 0) {
      mine[D] = m;
      mine[D + 1] = l;
    }
  }
  __syncthreads();
  const int64_t all = (int64_t)a.batch * a.q_heads;
  for (int i = threadIdx.x; i < heads * dims; i += kF8Threads) {
    const int h = i / dims, d = i - h * dims;
    const float* from = merged + h * kPitch;
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < kF8Waves; ++x) top = fmaxf(top, from[x * heads * kPitch + D]);
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f, o = 0.f;
#pragma unroll
    for (int x = 0; x < kF8Waves; ++x) {
      const float* one = from + x * heads * kPitch;
      const float f = __builtin_amdgcn_exp2f(one[D] - ref);
      total = __builtin_fmaf(one[D + 1], f, total);
      o = __builtin_fmaf(one[d], f, o);
    }
    if (a.n_splits > 1) {
      const int64_t at = split * all + (int64_t)b * a.q_heads + h0 + h;
      a.partial[at * dims + d] = o;
      if (d == 0) {
        a.stats[2 * at] = top;
        a.stats[2 * at + 1] = total;
      }
    } else {
      const int64_t at = (int64_t)b * a.o_bs + (int64_t)(h0 + h) * a.o_hs + d;
      store_elem(a.out, a.q_dtype, at, total != 0.f ? o / total : 0.f);
    }
  }
}

constexpr int kA8MaxSplits = 64;  // (one lane of the joining waves each)

// ---- joining the splits ------------------------------------------------------------------

// Heads of a multiple of four dims: a thread takes four dims of every parts-th
// split, up to 8 of them and all their loads in flight at once; the parts of a
// sum are lanes of one wave. (One wave per head that walked its 32 splits took
// 29.8 us for 32 heads of 128.)
constexpr int kJ8Threads = 256, kJ8Each = 8;

template <int EACH>
__global__ __launch_bounds__(kJ8Threads) void attend8_join_kernel(Attend8Args a, FastDiv quads, int parts) {
  const uint32_t heads = (uint32_t)(a.batch * a.q_heads), lane = threadIdx.x & 63, span = kWave / parts;
  const uint32_t part = lane / span, wave = blockIdx.x * (kJ8Threads / kWave) + (threadIdx.x >> 6);
  const uint32_t x = min(wave * span + lane % span, heads * quads.d - 1), item = quads.div(x);
  const uint32_t d = 4 * (x - item * quads.d);
  float m[EACH], l[EACH], top = -INFINITY, total = 0.f;
  f8_f32x4 v[EACH], o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < EACH; ++i) {  // (past the last split that one again, without a weight)
    const int s = (int)part + i * parts;
    const int64_t at = (int64_t)min(s, a.n_splits - 1) * heads + item;
    const f8_f32x2 st = *(const NHS_GLOBAL f8_f32x2*)to_global(a.stats + 2 * at);
    m[i] = s < a.n_splits ? st[0] : -INFINITY;
    l[i] = st[1];
    v[i] = *(const NHS_GLOBAL f8_f32x4*)to_global(a.partial + at * a.head_dim + d);
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) top = fmaxf(top, m[i]);
  for (uint32_t step = span; step < kWave; step *= 2) top = fmaxf(top, __shfl_xor(top, step));
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const bool there = (int)part + i * parts < a.n_splits;
    const float f = there ? __builtin_amdgcn_exp2f(m[i] - ref) : 0.f;
    total = there ? __builtin_fmaf(l[i], f, total) : total;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = there ? __builtin_fmaf(v[i][e], f, o[e]) : o[e];
  }
  for (uint32_t step = span; step < kWave; step *= 2) {
    total += __shfl_xor(total, step);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], step);
  }
  if (part || wave * span + lane >= heads * quads.d) return;
  const uint32_t b = item / a.q_heads, h = item - b * a.q_heads;
  const int64_t at = (int64_t)b * a.o_bs + (int64_t)h * a.o_hs + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) store_elem(a.out, a.q_dtype, at + e, total != 0.f ? o[e] / total : 0.f);
}

// Other heads: a wave per (request, query head).
__global__ __launch_bounds__(kWave) void attend8_join_any_kernel(Attend8Args a) {
  const int64_t heads = (int64_t)a.batch * a.q_heads;
  const int item = blockIdx.x, lane = threadIdx.x, D = a.head_dim;
  const float* st = a.stats + 2 * ((int64_t)min(lane, a.n_splits - 1) * heads + item);
  const float m = lane < a.n_splits ? st[0] : -INFINITY, l = lane < a.n_splits ? st[1] : 0.f;
  float top = m;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float f = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
  const float total = wave_sum(l * f);
  const int b = item / a.q_heads, h = item - b * a.q_heads;
  for (int d0 = 0; d0 < D; d0 += kWave) {
    const int d = min(d0 + lane, D - 1);
    float o = 0.f;
    for (int s = 0; s < a.n_splits; ++s) o = __builtin_fmaf(a.partial[(s * heads + item) * D + d], __shfl(f, s), o);
    if (d0 + lane < D)
      store_elem(a.out, a.q_dtype, (int64_t)b * a.o_bs + (int64_t)h * a.o_hs + d, total != 0.f ? o / total : 0.f);
  }
}

// ---- host --------------------------------------------------------------------------------

struct Plan8 {
  bool flash;
  int heads_per_item, chunks, subs, splits, rows_per_split, depth;
};

// own_lists: every query head has a row list of its own.
static Plan8 plan8(int batch, int n_rows, int q_heads, int kv_heads, int head_dim, bool own_lists) {
  Plan8 p;
  p.flash = head_dim % 16 == 0 && head_dim <= 256;
  p.heads_per_item = p.flash && !own_lists ? kF8Heads : 1;
  const int group = q_heads / kv_heads;
  p.chunks = (group + p.heads_per_item - 1) / p.heads_per_item;
  p.subs = kv_heads * p.chunks;
  const int64_t items = (int64_t)batch * p.subs;
  if (!p.flash) {
    // the general kernel: about two workgroups per CU, splits of at least 64 rows
    const int64_t most = std::min<int64_t>(kA8MaxSplits, (n_rows + 63) / 64);
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(most, 512 / items));
    p.rows_per_split = (n_rows + p.splits - 1) / p.splits;
    p.depth = 1;
    return p;
  }
  // About one workgroup per CU, in splits of whole tiles for its eight waves. Twice as many, of half the rows: 16 x 2048
  // rows 26.6 us against 21.8, 8 x 2048 15.9 against 15.6, 64 x 1024 of 28/4 heads 27.9 against 21.0, one request x
  // 32768 27.3 against 22.6, x 2048 the same. A wave asks for all its rows at once (one tile, or four), or for two tiles
  // in a round.
  constexpr int kStep = kF8Waves * kF8Tile;
  const int64_t most = std::min<int64_t>(kA8MaxSplits, (n_rows + kStep - 1) / kStep);
  int splits = (int)std::max<int64_t>(1, std::min<int64_t>(most, (256 + items / 2) / items));
  int per = (n_rows + splits - 1) / splits;
  per = (per + kStep - 1) / kStep * kStep;
  p.splits = (n_rows + per - 1) / per;
  p.rows_per_split = per;
  p.depth = per <= kStep ? 1 : per > 2 * kStep && per <= 4 * kStep ? 4 : 0;
  return p;
}

static int64_t workspace8(const Plan8& p, int64_t heads, int head_dim) {
  return p.splits == 1 ? 0 : p.splits * heads * (head_dim + 2) * (int64_t)sizeof(float);
}

// depth: tiles of a wave's only round, or 0 for the loop over rounds. (A kernel of its own for a single round of two
// tiles: 8 requests x 2048 rows of 32/8 heads 15.3 us against 15.7 in the loop, int8 15.9 against 15.4, fp32 16.0
// against 15.3.) Padded heads have no four tiles: 16 requests x 2048 rows of 32/8 heads of 96 21.5 us with them and 20.7
// in the loop, of 112 in int8 23.7 and 22.8, of 48 16.8 and 16.4.
template <typename C, int QP, int D, bool PAD>
static void (*flash8_deep(int depth))(Attend8Args) {
  constexpr int kRound = D == 256 ? 1 : 2;
  if constexpr (D != 256) {
    if (depth == 1) return attend8_flash_kernel<C, QP, D, 1, false, PAD>;
    if constexpr (!PAD && (QP != 3 || D != 128))  // (four tiles of fp32 queries and heads of 128: registers)
      if (depth == 4) return attend8_flash_kernel<C, QP, D, 4, false, PAD>;
  }
  return attend8_flash_kernel<C, QP, D, kRound, true, PAD>;
}

template <typename C, int QP>
static void (*flash8(int head_dim, int depth))(Attend8Args) {
  switch (head_dim) {
    case 32: return flash8_deep<C, QP, 32, false>(depth);
    case 64: return flash8_deep<C, QP, 64, false>(depth);
    case 128: return flash8_deep<C, QP, 128, false>(depth);
    case 256: return flash8_deep<C, QP, 256, false>(depth);
  }
  return head_dim < 64    ? flash8_deep<C, QP, 64, true>(depth)
         : head_dim < 128 ? flash8_deep<C, QP, 128, true>(depth)
                          : flash8_deep<C, QP, 256, true>(depth);
}

}  // namespace nhs

extern "C" int64_t nhs_attend_rows8_workspace_bytes(int32_t batch, int32_t n_rows, int32_t q_heads, int32_t kv_heads,
                                                    int32_t head_dim) {
  using namespace nhs;
  if (batch < 1 || n_rows < 1 || q_heads < 1 || kv_heads < 1 || head_dim < 1) return 0;
  const int64_t heads = (int64_t)batch * q_heads;
  if (q_heads % kv_heads || n_rows > (1 << 30)) return 0;
  return std::max(workspace8(plan8(batch, n_rows, q_heads, kv_heads, head_dim, false), heads, head_dim),
                  workspace8(plan8(batch, n_rows, q_heads, kv_heads, head_dim, true), heads, head_dim));
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
  const Plan8 plan = plan8(batch, n_rows, q_heads, kv_heads, head_dim, rows_head_stride != 0);
  const int64_t need = workspace8(plan, heads, head_dim);
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
  a.n_splits = plan.splits;
  a.rows_per_split = plan.rows_per_split;
  a.partial = static_cast<float*>(workspace);
  a.stats = a.partial ? a.partial + a.n_splits * heads * head_dim : nullptr;
  const bool join = a.n_splits > 1;
  hipStream_t s = (hipStream_t)stream;
  hipEvent_t stop = join ? nullptr : ev.stop;
  if (plan.flash) {
    a.heads_per_item = plan.heads_per_item;
    a.chunks = plan.chunks;
    a.subs = plan.subs;
    if ((int64_t)batch * plan.splits * plan.subs > (1 << 30))
      return fail(NHS_ERR_UNSUPPORTED, "nhs_attend_rows8: grid too large");
    a.groups = batch * plan.splits;
    a.near = a.groups >= 8;
    const int vec = q_dtype == NHS_F32 ? 4 : 8;  // elements of 16 bytes
    a.q_aligned = (uintptr_t)query % 16 == 0 && q_batch_stride % vec == 0 && q_head_stride % vec == 0;
    const int64_t grid = (int64_t)plan.subs * (a.near ? (a.groups + 7) / 8 * 8 : a.groups);
    const auto pick = [&](auto c) {
      using C = decltype(c);
      return q_dtype == NHS_BF16  ? flash8<C, 1>(head_dim, plan.depth)
             : q_dtype == NHS_F16 ? flash8<C, 2>(head_dim, plan.depth)
                                  : flash8<C, 3>(head_dim, plan.depth);
    };
    launch(code == NHS_CODE_I8 ? pick(I8()) : pick(E4M3()), dim3((unsigned)grid), dim3(kF8Threads), 0, s, ev.start,
           stop, a);
  } else {
    if (heads * a.n_splits > 0x7fffffff) return fail(NHS_ERR_UNSUPPORTED, "nhs_attend_rows8: grid too large");
    const auto run = [&](auto c, auto n) {
      launch(attend8_general_kernel<decltype(c), decltype(n)::value>, dim3((unsigned)(heads * a.n_splits)),
             dim3(kG8Threads), 0, s, ev.start, stop, a);
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
  }
  if (join && head_dim % 4 == 0 && heads * head_dim < (1ll << 31)) {
    int parts = 1;
    while (parts * kJ8Each < plan.splits) parts *= 2;
    const int64_t per_group = kJ8Threads / parts, threads = heads * (head_dim / 4);
    launch(plan.splits <= 2   ? attend8_join_kernel<2>
           : plan.splits <= 4 ? attend8_join_kernel<4>
                              : attend8_join_kernel<kJ8Each>,
           dim3((unsigned)((threads + per_group - 1) / per_group)), dim3(kJ8Threads), 0, s, nullptr, ev.stop, a,
           FastDiv((uint32_t)(head_dim / 4)), parts);
  } else if (join) {
    launch(attend8_join_any_kernel, dim3((unsigned)heads), dim3(kWave), 0, s, nullptr, ev.stop, a);
  }
  return launch_status("nhs_attend_rows8");
}
