// Verifying a tree of drafted tokens: ancestor masks and positions from the
// nodes' parents (nhs_tree_plan), and attention of every node over its
// request's selected pool rows and its own ancestors (nhs_tree_attention).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "flash_common.h"

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
  int batch, nodes, q_heads, kv_heads, group, head_dim, page_size;
  int query_rows, row_blocks;  // nodes * group, and blocks of them
  FastDiv group_div, page_div;
  float scale_log2;  // D^-1/2 * log2(e)
  char* out;
  int64_t o_b, o_n, o_h;
  float* partial;  // n_splits > 1: [n_splits, batch * nodes * q_heads, head_dim], not divided by the sum
  float* stats;    // and [n_splits, batch * nodes * q_heads, 2] (max in base 2, sum)
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
  const bool some = word != 0 && l != 0.f;  // (a NaN among the scores makes l one)
#pragma unroll
  for (int i = 0; i < DIMS / 16; ++i)
    if (sub + 16 * i < D) store_elem(a.out, T::dtype, at + sub + 16 * i, some ? acc[i] / l : 0.f);
}

// ---- heads whose rows are 64 to 512 bytes, on the matrix cores ----

constexpr int kTfStage = 2048;  // rows whose addresses are in LDS at a time
constexpr int kTfRowBytes = 512;  // the longest row of a head
__device__ __attribute__((aligned(kTfRowBytes))) char tree_zeros[kTfRowBytes];  // read in place of a masked row

// LDS slot of 16-byte chunk c of K row r (C chunks a row): any 16 consecutive rows at one chunk fall on distinct banks
template <int C>
__device__ __forceinline__ int tf_k_slot(int r, int c) {
  return C >= 16 ? c ^ (r & 15) : C == 8 ? c ^ ((r >> 1) & 7) : c ^ ((r >> 2) & 3);
}
// and of V row (key) r. 16 bits: the 4 rows of a transposing read fall on distinct banks; fp32: rows r and r + 4, of
// which the halves of a wave read the same dims (two to a bank with 8 chunks a row).
template <typename T, int C>
__device__ __forceinline__ int tf_v_slot(int r, int c) {
  if constexpr (T::dtype == NHS_F32) return C >= 16 ? c ^ (8 * ((r >> 2) & 1)) : c;
  return C >= 16 ? c ^ (4 * (r & 3)) : C == 8 ? c ^ (4 * ((r >> 1) & 1)) : c;
}

// a packed pair as fp32
template <typename T>
__device__ __forceinline__ float2 tf_unpack(uint32_t pair) {
  if constexpr (T::dtype == NHS_BF16)
    return make_float2(__uint_as_float(pair << 16), __uint_as_float(pair & 0xffff0000u));
  else
    return make_float2(f16_bits_to_f32(pair & 0xffffu), f16_bits_to_f32(pair >> 16));
}

// 16 bytes of K and Q each: one 32x32x16 product of 16-bit elements, or four 32x32x2 of fp32
template <typename T>
__device__ __forceinline__ pf_f32x16 tf_qk(uint4 k, uint4 q, pf_f32x16 c) {
  if constexpr (T::dtype != NHS_F32) {
    return mfma32x32x16<T>(k, q, c);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.x), __uint_as_float(q.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.y), __uint_as_float(q.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.z), __uint_as_float(q.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k.w), __uint_as_float(q.w), c, 0, 0, 0);
  }
}

// QW waves hold 32 query rows each; KW such sets share the keys (KW tiles of
// BN keys a round). The layouts are those of prefill_attention_kernel:
// S^T = K Q^T and O^T = V^T P^T, tiles straight from global memory to LDS. A
// row of K and V is read once per block of 32 QW query rows, where a pass per
// node would read it once per node.
//
// Every row of a tile has an address of its own, so a stage of up to 2048 rows
// is turned into addresses in LDS first (a masked row's is that of zeros, and
// its bit of the tile's word is clear); the loads of a round then need one LDS
// read each. The drafted keys are the first round of the last split, asked
// for before the row indices are read. A masked weight is 0, which a matrix
// core would multiply with whatever V holds, so what a mask hides must be
// finite: masked rows read zeros, absent nodes' values are cleared in the tile,
// and NaN and infinities of drafted values are taken out of it, then added to
// the outputs of the nodes that see them.
//
// 16-bit weights go to the matrix cores as the nearest value of the type and,
// in a second product against the same V, the rest of that rounding; the
// denominator sums them as they are. The output is the exact one rounded once
// (error against float64 0.0017 in bf16; with the rounded weights alone, which
// the prompt attention takes, 0.0022). us without / with the rests: one request
// x 16 nodes x 2048 rows 15.5 / 15.8, eight of them 28.8 / 30.0, the long
// history and the widest trees below 44.0 / 48.7 and 89.7 / 108.5.
//
// With QW = 1 a wave loads and reads its own tiles only and no barrier stands
// in the loop (the four shares are joined in two steps: one share after the
// other took 8.0 us where two steps take 7.5, one request of 128 rows).
//
// Measured (MI355X, bf16, rows read from HBM, graphs replayed for a second, us
// with the join of the splits): 8 requests x 16 nodes x 32/8 heads of 128 x
// 2048 rows 30.0 (the rows stream at 5.5 TB/s once they flow, but 6 us pass
// before the first are in, and 2.5 at the end; the join is 5); one request x
// 32 nodes x 32768 rows 48.7 (join 6.7); 16 requests x 64 nodes x 28/4 heads x
// 4096 rows 108.5 (559 TFLOP/s, 838 with the rests' products): bound by the
// matrix cores, LDS reads and softmax together, which follow each other in a
// wave. With the general kernel 932, 3685 and 10818. Other figures of this file
// compare variants without the rests, in short runs after an idle card, which
// take 5 to 14% longer (the widest trees 102, 85 of them without the loads, 65
// with the loads alone).
//
// fp32 runs on v_mfma_f32_32x32x2_f32 (lane l: row l%32 of A at k = l/32). The
// dims of a dot product may come in any order, so four of them take the
// 16-byte chunks as they lie; for O^T a score register is the B operand as it
// stands, its two keys (4 rows apart) against one V element per lane.
template <typename T, int D, int QW, int KW, int BN>
__global__ __launch_bounds__(QW * KW * kWave) void tree_flash_kernel(TreeArgs a) {
  constexpr int W = QW * KW, THREADS = W * kWave;
  constexpr bool F = T::dtype == NHS_F32;
  constexpr int RB = D * T::bytes;             // bytes of a head's row
  constexpr int KS = RB / 32, DB = D / 32, C = RB / 16, NB = BN / 32;
  constexpr int kRows = 1024 / RB;             // of a load instruction
  constexpr int kMine = BN / kRows / QW;       // instructions of a wave per tile, for K and for V each
  constexpr int kTile = BN * RB;               // bytes
  constexpr int kRound = BN * KW;              // keys
  // fp16 weights, denominators and sums are all 2^15 times too large: what both products leave of a weight is then
  // 2^-40 of the largest at most (which itself is below 2^15.2 and fp16's numbers end at 2^16, see `large`)
  constexpr float kLift = T::dtype == NHS_F16 ? 15.f : 0.f;
  // exponent bits of NaN and infinities
  constexpr uint32_t kOdd = F ? 0x7f800000u : T::dtype == NHS_BF16 ? 0x7f80u : 0x7c00u;
  static_assert(kRound >= kTreeNodes && kTfStage % kRound == 0 && kMine >= 1 && RB <= kTfRowBytes, "tile shape");
  // Tiles under names of their own, used by rounds in turn: the compiler then knows that reads of one need not wait for
  // loads into the others.
  __shared__ __attribute__((aligned(16))) char k0[KW * kTile], k1[KW * kTile];
  __shared__ __attribute__((aligned(16))) char v0[KW * kTile], v1[KW * kTile];
  __shared__ __attribute__((aligned(16))) int64_t stage[kTfStage];
  __shared__ uint32_t words[kTfStage / 32];
  __shared__ int odd;  // the draft's values hold a NaN or an infinity

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave_id = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = wave_id % QW, share = wave_id / QW;
  const int half = lane >> 5, n = lane & 31;
  // The items of one (request, KV head) and split are a multiple of the items apart: on one XCD where they are a
  // multiple of 8, so that the blocks of query rows read the keys from one L2.
  const int items = a.batch * a.kv_heads;
  const int bk = blockIdx.x % items, rest = blockIdx.x / items;
  const int block = rest % a.row_blocks, split = rest / a.row_blocks;
  const int b = bk / a.kv_heads, kv = bk - b * a.kv_heads;

  const int r = (block * QW + wave) * 32 + n;  // this lane's query row (column of S^T)
  const bool live = r < a.query_rows;
  const int rr = min(r, a.query_rows - 1);
  const int node = (int)a.group_div.div((uint32_t)rr), head = kv * a.group + rr - node * a.group;
  const int64_t* mask = a.mask + (int64_t)b * a.mask_b;
  const uint64_t word = live ? (uint64_t)mask[node] : 0;
  uint4 qf[KS];
  {
    const char* qp = a.q + ((int64_t)b * a.q_b + (int64_t)node * a.q_n + (int64_t)head * a.q_h) * T::bytes + half * 16;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const uint4*>(qp + s * 32);
  }
  // a wave past the last query row only loads (448 rows in blocks of 128: 105.5 -> 102 us, widest trees)
  const bool alive = (block * QW + wave) * 32 < a.query_rows;
  float m = -INFINITY, l = 0.f;  // running max (of the unscaled scores) and this lane's share of the denominator
  pf_f32x16 o[DB];
#pragma unroll
  for (int x = 0; x < DB; ++x)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[x][i] = 0.f;

  const int lrow = lane / C, lchunk = lane % C;
  const int k_row = n * RB;
  const int j4 = (lane & 15) >> 2;
  int v_at[DB];
#pragma unroll
  for (int x = 0; x < DB; ++x)
    v_at[x] = F ? 4 * half * RB + tf_v_slot<T, C>(4 * half, x * 8 + n / 4) * 16 + n % 4 * 4
                : (4 * half + j4) * RB +
                      tf_v_slot<T, C>(j4, x * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;

  const int64_t head_bytes = (int64_t)kv * RB, plane = a.plane_bytes;
  const int64_t zeros = (int64_t)tree_zeros;
  auto load_tile = [&](int t, char* kb, char* vb) {  // this share's tile of the stage's round t
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int row = (i * QW + wave) * kRows + lrow;
      const int64_t at = stage[t * kRound + share * BN + row];
      const int dst = share * kTile + (i * QW + wave) * 1024;
      const char* ks = (const char*)at + tf_k_slot<C>(row, lchunk) * 16;
      const char* vs = (const char*)(at == zeros ? at : at + plane) + tf_v_slot<T, C>(row, lchunk) * 16;
      pf_load_lds(ks, kb + dst);
      pf_load_lds(vs, vb + dst);
    }
  };
  // the tile in (kb, vb), of which the lane's query sees the keys of `seen` (bit = key of the tile)
  auto tile = [&](const char* kb, const char* vb, const uint32_t (&seen)[NB]) {
    const char* kl = kb + share * kTile + k_row;
    const char* vl = vb + share * kTile;
    pf_f32x16 s[NB];
#pragma unroll
    for (int x = 0; x < NB; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[x][i] = 0.f;
#pragma unroll
    for (int st = 0; st < KS; ++st)
#pragma unroll
      for (int x = 0; x < NB; ++x) {
        const uint4 kf = *reinterpret_cast<const uint4*>(kl + x * 32 * RB + tf_k_slot<C>(n, 2 * st + half) * 16);
        s[x] = tf_qk<T>(kf, qf[st], s[x]);
      }
    if constexpr (!F && D == 128 && NB == 2) {  // as in the prompt attention: eight K reads ahead of the MFMAs
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, 8, 0);
    }
#pragma unroll
    for (int x = 0; x < NB; ++x)
      if (__any(seen[x] != 0xffffffffu)) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(seen[x] >> ((i >> 2) * 8 + half * 4 + (i & 3)) & 1)) s[x][i] = -INFINITY;
      }
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < NB; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[x][i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__any(mx > m)) {
      const float moved = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f((m - (moved == -INFINITY ? 0.f : moved)) * a.scale_log2);
      m = moved;
      l *= alpha;
#pragma unroll
      for (int x = 0; x < DB; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[x][i] *= alpha;
    }
    float ref = m == -INFINITY ? 0.f : m * a.scale_log2;
    // Scores are scaled and made relative to the maximum in one step, which is off by the rounding of ref. Where that
    // could exceed a thirtieth of a power of 2 (and overflow the weights in the end), they are made relative first.
    const bool large = fabsf(ref) > 0x1p20f;
    if (__any(large)) {
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[x][i] -= large ? m : 0.f;
      ref = large ? 0.f : ref;
    }
    ref -= kLift;
    float tile_sum = 0.f;
    if constexpr (F) {
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[x][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][i], a.scale_log2, -ref));
          tile_sum += s[x][i];
        }
      l += tile_sum;
#pragma unroll
      for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int y = 0; y < DB; ++y) {
            const float vf = *reinterpret_cast<const float*>(vl + v_at[y] + (x * 32 + (i >> 2) * 8 + (i & 3)) * RB);
            o[y] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, s[x][i], o[y], 0, 0, 0);
          }
    } else {
#pragma unroll
      for (int j = 0; j < 2 * NB; ++j) {  // 16 keys
        uint32_t w[4], r[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float e0 = s[j >> 1][(j & 1) * 8 + 2 * x], e1 = s[j >> 1][(j & 1) * 8 + 2 * x + 1];
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(e0, a.scale_log2, -ref));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(e1, a.scale_log2, -ref));
          w[x] = pf_pack<T>(p0, p1);
          const float2 rounded = tf_unpack<T>(w[x]);
          r[x] = pf_pack<T>(p0 - rounded.x, p1 - rounded.y);
          tile_sum += p0 + p1;
        }
        const uint4 pb = make_uint4(w[0], w[1], w[2], w[3]), rest = make_uint4(r[0], r[1], r[2], r[3]);
        uint4 vf[DB];
#pragma unroll
        for (int x = 0; x < DB; ++x) {
          const uint2 lo = pf_read_tr(vl + v_at[x] + (16 * j) * RB);
          const uint2 hi = pf_read_tr(vl + v_at[x] + (16 * j + 8) * RB);
          vf[x] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
#pragma unroll
        for (int x = 0; x < DB; ++x) o[x] = mfma32x32x16<T>(vf[x], pb, o[x]);
#pragma unroll
        for (int x = 0; x < DB; ++x) o[x] = mfma32x32x16<T>(vf[x], rest, o[x]);
      }
      l += tile_sum;
    }
  };

  const int begin = split * a.rows_per_split, end = min(a.n_rows, begin + a.rows_per_split);
  const int64_t* rows = a.rows + (int64_t)b * a.r_b;
  const bool draft = split == a.n_splits - 1;
  uint64_t present = 0;  // drafted nodes
  if (draft) {  // the drafted keys as they lie (node j is key j of a round), asked for before the rows' indices are read
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int row = (i * QW + wave) * kRows + lrow, j = min(share * BN + row, a.nodes - 1);
      const int dst = share * kTile + (i * QW + wave) * 1024;
      const char* ks = a.k + ((int64_t)b * a.k_b + (int64_t)j * a.k_n + (int64_t)kv * a.k_h) * T::bytes;
      const char* vs = a.v + ((int64_t)b * a.v_b + (int64_t)j * a.v_n + (int64_t)kv * a.v_h) * T::bytes;
      pf_load_lds(ks + tf_k_slot<C>(row, lchunk) * 16, k0 + dst);
      pf_load_lds(vs + tf_v_slot<T, C>(row, lchunk) * 16, v0 + dst);
    }
    present = __ballot(lane < a.nodes && mask[min(lane, a.nodes - 1)] != 0);
    if (tid == 0) odd = 0;
  }
  for (int s0 = begin; s0 < end || s0 == begin; s0 += kTfStage) {
    const int count = min(kTfStage, max(end - s0, 0)), rounds = (count + kRound - 1) / kRound;
    if (s0 != begin) __syncthreads();  // the last stage's addresses and tiles are read
    for (int i = tid; i < rounds * kRound; i += THREADS) {
      const int64_t at = i < count ? rows[(int64_t)(s0 + i) * a.r_c] : -1;
      const bool ok = at >= 0 && at < a.pool_rows;
      const uint32_t page = a.page_div.div((uint32_t)at);
      const int64_t in_page = (uint32_t)at - page * (uint32_t)a.page_size;
      stage[i] = ok ? (int64_t)a.pool + page * a.block_stride + in_page * a.row_bytes + head_bytes : zeros;
      const uint64_t live_rows = __ballot(ok);  // of this wave's 64 consecutive rows
      if (lane == 0) {
        words[i / 32] = (uint32_t)live_rows;
        words[i / 32 + 1] = (uint32_t)(live_rows >> 32);
      }
    }
    if (draft && s0 == begin) __builtin_amdgcn_s_waitcnt(kPfVmcnt0);
    __syncthreads();
    if (rounds > 0) load_tile(0, k1, v1);
    const bool with_draft = draft && s0 == begin;
    if (with_draft) {  // zeros for the values of absent nodes (those past the last are copies of it), NaN and infinities
      for (int c = tid; c < kTreeNodes * C; c += THREADS) {  // rows lie one after another, shares too
        uint4* p = reinterpret_cast<uint4*>(v0) + c;
        const bool here = present >> (c / C) & 1;
        uint32_t w[4] = {p->x, p->y, p->z, p->w};
        bool found = false;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const bool lo = (w[x] & kOdd) == kOdd, hi = !F && (w[x] >> 16 & kOdd) == kOdd;
          found |= lo || hi;
          const uint32_t keep = F ? (lo ? 0u : ~0u) : (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
          w[x] = here ? w[x] & keep : 0u;
        }
        if (found || !here) *p = make_uint4(w[0], w[1], w[2], w[3]);
        if (found && here) odd = 1;
      }
      __syncthreads();
    }
    // round t of the stage's rows; t = -1: the draft, whose tile is in place
    auto round = [&](int t, char* kb, char* vb, char* kb_next, char* vb_next) {
      uint32_t seen[NB];
      bool some;
      if (t >= 0) {
        // this wave's loads of round t are in; after the barrier every wave's are, and every wave is done with the
        // other buffers, which take round t + 1
        if constexpr (QW > 1) {
          __builtin_amdgcn_s_waitcnt(kPfVmcnt0);
          __syncthreads();
        } else {  // the wave's reads of the other buffers are back too
          __builtin_amdgcn_s_waitcnt(kPfVmcnt0 & kPfLgkmcnt0);
          asm volatile("" ::: "memory");
        }
#pragma unroll
        for (int x = 0; x < NB; ++x) seen[x] = words[(t * kRound + share * BN) / 32 + x];
        if (t + 1 < rounds) load_tile(t + 1, kb_next, vb_next);
        some = false;
#pragma unroll
        for (int x = 0; x < NB; ++x) {
          seen[x] = __builtin_amdgcn_readfirstlane(seen[x]);
          some |= seen[x] != 0;
        }
      } else {
        some = share * BN < a.nodes;
#pragma unroll
        for (int x = 0; x < NB; ++x)
          seen[x] = some ? (uint32_t)((word & present) >> (share * BN + 32 * x)) : 0u;
      }
      if (some && alive) tile(kb, vb, seen);
    };
    for (int t = -1; t < rounds; t += 2) {
      if (t >= 0 || with_draft) round(t, k0, v0, k1, v1);
      if (t + 1 < rounds) round(t + 1, k1, v1, k0, v0);
    }
  }

  l += __shfl_xor(l, 32);
  if constexpr (KW > 1) {
    // the upper half of the shares hands its sums over to the lower half through the tile buffers, until one is left
    // (registers by lane: the partners hold the same query rows and dims)
    static_assert(W <= 8 && DB * 16 * kWave * 4 <= KW * kTile && W * kWave * 4 <= kTfStage * 8, "merge space");
    for (int step = KW / 2; step > 0; step /= 2) {
      const int area = wave * (KW / 2) + share % step;  // below W / 2
      float* part = reinterpret_cast<float*>(area == 0 ? k0 : area == 1 ? v0 : area == 2 ? k1 : v1) + lane;
      float* stat = reinterpret_cast<float*>(stage) + area * 2 * kWave + lane;
      __syncthreads();
      if (share / step == 1) {
#pragma unroll
        for (int x = 0; x < DB; ++x)
#pragma unroll
          for (int i = 0; i < 16; ++i) part[(x * 16 + i) * kWave] = o[x][i];
        stat[0] = m;
        stat[kWave] = l;
      }
      __syncthreads();
      if (share < step) {
        const float m2 = stat[0], l2 = stat[kWave];
        const float both = fmaxf(m, m2), ref = both == -INFINITY ? 0.f : both;
        const float f1 = __builtin_amdgcn_exp2f((m - ref) * a.scale_log2);
        const float f2 = __builtin_amdgcn_exp2f((m2 - ref) * a.scale_log2);
        m = both;
        l = l * f1 + l2 * f2;
#pragma unroll
        for (int x = 0; x < DB; ++x)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[x][i] = o[x][i] * f1 + part[(x * 16 + i) * kWave] * f2;
      }
    }
    if (share) return;
  }
  if (!live) return;
  if (draft && odd) {
    for (int j = 0; j < a.nodes; ++j) {
      if (!((word & present) >> j & 1)) continue;
      const char* vs = a.v + ((int64_t)b * a.v_b + (int64_t)j * a.v_n + (int64_t)kv * a.v_h) * T::bytes;
#pragma unroll
      for (int x = 0; x < DB; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float value = load_elem(vs, T::dtype, x * 32 + (i >> 2) * 8 + half * 4 + (i & 3));
          if (!(fabsf(value) < INFINITY)) o[x][i] += value;
        }
    }
  }
  if (a.n_splits > 1) {
    const int64_t at = (int64_t)split * a.out_rows + ((int64_t)b * a.nodes + node) * a.q_heads + head;
    if (half == 0) *reinterpret_cast<float2*>(a.stats + 2 * at) = make_float2(m * a.scale_log2, l);
    float* p = a.partial + at * D + half * 4;
#pragma unroll
    for (int x = 0; x < DB; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y)  // dims x*32 + y*8 + half*4 .. +3 of the lane's query row
        *reinterpret_cast<float4*>(p + x * 32 + y * 8) =
            make_float4(o[x][4 * y], o[x][4 * y + 1], o[x][4 * y + 2], o[x][4 * y + 3]);
    return;
  }
  const bool some = word != 0 && l != 0.f;  // (a NaN among the scores makes l one)
  const float inv = some ? 1.f / l : 0.f;
  char* op = a.out + ((int64_t)b * a.o_b + (int64_t)node * a.o_n + (int64_t)head * a.o_h) * T::bytes;
#pragma unroll
  for (int x = 0; x < DB; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) {  // dims x*32 + y*8 + half*4 .. +3
      float r4[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r4[e] = some ? o[x][4 * y + e] * inv : 0.f;
      char* to = op + (x * 32 + y * 8 + half * 4) * T::bytes;
      if constexpr (F)
        *reinterpret_cast<float4*>(to) = make_float4(r4[0], r4[1], r4[2], r4[3]);
      else
        *reinterpret_cast<uint2*>(to) = make_uint2(pf_pack<T>(r4[0], r4[1]), pf_pack<T>(r4[2], r4[3]));
    }
}

// Joins the splits of every output row: the sums are scaled to the largest of
// the splits' maxima, added and divided. WAVES waves of a workgroup share a row
// (four from 17 splits on, where the rows are few and the chains of loads long;
// us of both launches with one / four: 32 splits 30.3 / 29.6, 8 splits 41.6 / 44.1);
// LANES lanes of four dims read one split while the others read the next ones,
// all the splits of a wave in flight at once.
template <typename T, int D, int WAVES>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a) {
  constexpr int LANES = D / 4, SIDE = kWave / LANES, U = 16 / SIDE;
  __shared__ __attribute__((aligned(16))) float part[WAVES > 1 ? 4 : 1][WAVES > 1 ? D : 4];
  __shared__ float stat[WAVES > 1 ? 4 : 1][2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t out_row = WAVES > 1 ? blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  if (out_row >= a.out_rows) return;  // (a whole workgroup or a wave without barriers)
  const int64_t bn = out_row / a.q_heads;
  const int head = (int)(out_row - bn * a.q_heads);
  const int b = (int)(bn / a.nodes), node = (int)(bn - (int64_t)b * a.nodes);
  const bool present = a.mask[(int64_t)b * a.mask_b + node] != 0;
  const int side = lane / LANES, d = lane % LANES * 4;
  const int each = (a.n_splits + WAVES - 1) / WAVES, begin = WAVES > 1 ? wave * each : 0;
  const int end = min(begin + each, a.n_splits);
  float top = -INFINITY, total = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = begin; s0 < end; s0 += SIDE * U) {
    float4 p[U];
    float2 st[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (int64_t)min(s0 + u * SIDE + side, end - 1) * a.out_rows + out_row;
      p[u] = *reinterpret_cast<const float4*>(a.partial + at * D + d);
      st[u] = *reinterpret_cast<const float2*>(a.stats + 2 * at);
    }
    float moved = top;
#pragma unroll
    for (int u = 0; u < U; ++u) moved = fmaxf(moved, st[u].x);
    const float ref = moved == -INFINITY ? 0.f : moved, alpha = __builtin_amdgcn_exp2f(top - ref);
    top = moved;
    total *= alpha;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= alpha;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * SIDE + side >= end) continue;
      const float f = __builtin_amdgcn_exp2f(st[u].x - ref);
      total = __builtin_fmaf(f, st[u].y, total);
      o[0] = __builtin_fmaf(f, p[u].x, o[0]), o[1] = __builtin_fmaf(f, p[u].y, o[1]);
      o[2] = __builtin_fmaf(f, p[u].z, o[2]), o[3] = __builtin_fmaf(f, p[u].w, o[3]);
    }
  }
  // the sides, then the waves
#pragma unroll
  for (int x = LANES; x < kWave; x <<= 1) {
    const float m2 = __shfl_xor(top, x), both = fmaxf(top, m2), ref = both == -INFINITY ? 0.f : both;
    const float f1 = __builtin_amdgcn_exp2f(top - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
    total = total * f1 + __shfl_xor(total, x) * f2;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f1 + __shfl_xor(o[e], x) * f2;
    top = both;
  }
  if constexpr (WAVES > 1) {
    if (side == 0) *reinterpret_cast<float4*>(&part[wave][d]) = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) stat[wave][0] = top, stat[wave][1] = total;
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < WAVES; ++w) {
      const float m2 = stat[w][0], both = fmaxf(top, m2), ref = both == -INFINITY ? 0.f : both;
      const float f1 = __builtin_amdgcn_exp2f(top - ref), f2 = __builtin_amdgcn_exp2f(m2 - ref);
      const float4 q = *reinterpret_cast<const float4*>(&part[w][d]);
      total = total * f1 + stat[w][1] * f2;
      o[0] = o[0] * f1 + q.x * f2, o[1] = o[1] * f1 + q.y * f2;
      o[2] = o[2] * f1 + q.z * f2, o[3] = o[3] * f1 + q.w * f2;
      top = both;
    }
  }
  if (side) return;
  const bool some = present && total != 0.f;
  const int64_t at = (int64_t)b * a.o_b + (int64_t)node * a.o_n + (int64_t)head * a.o_h + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) store_elem(a.out, T::dtype, at + e, some ? o[e] / total : 0.f);
}

// The same for every head_dim, one wave per row and a dim per lane.
template <typename T>
__global__ __launch_bounds__(256) void tree_join_general_kernel(TreeArgs a) {
  const int64_t out_row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (out_row >= a.out_rows) return;
  const int lane = threadIdx.x & 63, D = a.head_dim;
  const int64_t bn = out_row / a.q_heads;
  const int head = (int)(out_row - bn * a.q_heads);
  const int b = (int)(bn / a.nodes), node = (int)(bn - (int64_t)b * a.nodes);
  float top = -INFINITY, total = 0.f;
  for (int s = lane; s < a.n_splits; s += kWave) top = fmaxf(top, a.stats[2 * ((int64_t)s * a.out_rows + out_row)]);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float ref = top == -INFINITY ? 0.f : top;
  for (int s = lane; s < a.n_splits; s += kWave) {
    const float* st = a.stats + 2 * ((int64_t)s * a.out_rows + out_row);
    total = __builtin_fmaf(__builtin_amdgcn_exp2f(st[0] - ref), st[1], total);
  }
  total = group_sum(total, kWave);
  const bool some = a.mask[(int64_t)b * a.mask_b + node] != 0 && total != 0.f;
  const int64_t at = (int64_t)b * a.o_b + (int64_t)node * a.o_n + (int64_t)head * a.o_h;
  for (int d = lane; d < D; d += kWave) {
    float o = 0.f;
    for (int s = 0; s < a.n_splits; ++s) {
      const int64_t p = (int64_t)s * a.out_rows + out_row;
      o = __builtin_fmaf(__builtin_amdgcn_exp2f(a.stats[2 * p] - ref), a.partial[p * D + d], o);
    }
    store_elem(a.out, T::dtype, at + d, some ? o / total : 0.f);
  }
}

struct TreeShape {
  int waves, shares;  // of the matrix-core kernel (QW, KW); 0: the general one
  int row_blocks, n_splits, rows_per_split;
};

// How a (request, KV head)'s query rows and keys are divided. `row_bytes`: of a
// head's row where the matrix-core kernel takes the call, else 0.
static TreeShape tree_shape(int batch, int nodes, int n_rows, int q_heads, int kv_heads, int head_dim,
                            int row_bytes) {
  const bool flash = row_bytes > 0;
  TreeShape s;
  const int query_rows = nodes * (q_heads / kv_heads);
  int block_rows = kTgRows, per_cu = 2, least = 64;
  s.waves = s.shares = 0;
  if (flash) {
    // One set of waves per 32 query rows. us at up to 32 rows with one / two sets: rows of 128 bytes, 16 requests x
    // 16384 keys 38.3 / 41.3, fp32 heads of 32 x 528 keys 11.8 / 13.6; rows of 256 bytes, one request x 128 keys 11.9
    // / 10.4, x 2048 15.7 / 14.5, x 32768 37.5 / 37.0, 16 requests x 8192 equal. At 64 rows x 2048 keys two / four sets
    // 30.0 / 30.8. (Heads of 256: four would spill.)
    s.waves = query_rows <= 32 && row_bytes <= 128 ? 1 : query_rows <= 64 || head_dim == 256 ? 2 : 4;
    s.shares = s.waves == 1 ? 4 : 2;
    // Blocks of 256 rows where they fill the chip without splits (half the reads of the keys from L2; with splits their
    // joining costs more than that). us with blocks of 128 / 256: 32 requests x 448 rows x 4 KV heads (256 of 256) x
    // 2048 keys 118.5 / 98.5 (long runs with the rests 130 / 110), 16 of them (128) x 4096 keys 105 / 116.
    if (query_rows > 128 && head_dim == 128 && row_bytes == 256 &&
        (int64_t)batch * kv_heads * ((query_rows + 255) / 256) >= 256)
      s.waves = 8, s.shares = 1;
    block_rows = 32 * s.waves;
    // One workgroup per CU, of rounds of 128 keys. us with one / two per CU: one request of 8 nodes x 16384 keys
    // 27.4 / 36.8, rows of 64 bytes x 32768 keys 15.5 / 18.9. In rounds of 64 / 128 / 256: 8 nodes x 2048 keys
    // 19.0 / 16.7 / 18.0, 32 nodes 26.7 / 17.9 / 19.5, x 512 keys 15.0 / 14.9 / 16.5.
    per_cu = 1;
    least = 128;
  }
  s.row_blocks = (query_rows + block_rows - 1) / block_rows;
  const int64_t items = (int64_t)batch * kv_heads * s.row_blocks;
  const int64_t wanted = std::max<int64_t>(1, 256 * per_cu / items), most = std::max(1, n_rows / least);
  if (flash) {
    // The draft is a round too, of the last split, so the longest split has `longest` rounds, it among them, and the
    // last one may have nothing else. us with splits of equal numbers of keys, the draft on top / so: 16 nodes x 512
    // keys 14.3 / 12.5, 4 requests of them 16.6 / 14.4, x 960 keys 19.2 / 16.6, fp32 heads of 32 x 448 keys 13.2 / 9.9.
    // Splitting pays where it saves more than the join costs, which is about 2.3 us and the partial sums at 5.5 TB/s; a
    // round takes 1.6 us (16-bit heads of up to 128 and fp32 heads of 32; the products of a round of fp32 heads of 128
    // alone take about 6.8 us, and rounds of 512-byte rows are half as long, so for those the rule is only a guess). us
    // whole / split: 256 keys, 8 requests of 16 nodes 14.5 / 17.8, one request 13.3 / 12.3.
    const int rounds = (n_rows + least - 1) / least, total = rounds + 1;
    const int longest = (int)((total + wanted - 1) / wanted), splits = (total + longest - 1) / longest;
    const double joined = longest * 1.6 + 2.3 + (double)splits * batch * nodes * q_heads * head_dim * 8 / 5.5e6;
    s.n_splits = 1, s.rows_per_split = std::max(n_rows, 1);
    if (splits > 1 && joined < total * 1.6) {
      s.n_splits = splits;
      s.rows_per_split =
          std::max((rounds - longest + splits - 1) / (splits - 1), (rounds + splits - 1) / splits) * least;
    }
    return s;
  }
  s.n_splits = (int)std::min(wanted, most);
  s.rows_per_split = std::max(((n_rows + s.n_splits - 1) / s.n_splits + least - 1) / least * least, 1);
  s.n_splits = std::max(1, (n_rows + s.rows_per_split - 1) / s.rows_per_split);
  return s;
}

// Bytes of a head's row if the matrix-core kernel has it, else 0.
static int tree_flash_row(int dtype, int head_dim) {
  const int bytes = head_dim * elem_size(dtype);
  return (head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256) && bytes <= kTfRowBytes ? bytes : 0;
}

static bool tree_valid(int batch, int nodes, int n_rows, int q_heads, int kv_heads, int head_dim) {
  return batch >= 0 && nodes >= 1 && nodes <= kTreeNodes && n_rows >= 0 && n_rows <= (1 << 30) && q_heads >= 1 && kv_heads >= 1 &&
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
  if (batch > 0x3ffffff) return fail(NHS_ERR_UNSUPPORTED, "nhs_tree_plan: too many trees");
  launch(tree_plan_kernel, dim3((unsigned)batch), dim3(kWave), 0, (hipStream_t)stream, ev.start, ev.stop, parents,
         parents_stride, nodes, lengths, mask, positions);
  return launch_status("nhs_tree_plan");
}

extern "C" int64_t nhs_tree_attention_workspace_bytes(int32_t batch, int32_t nodes, int32_t n_rows, int32_t q_heads,
                                                      int32_t kv_heads, int32_t head_dim) {
  if (!tree_valid(batch, nodes, n_rows, q_heads, kv_heads, head_dim)) return 0;
  int splits = 0;  // the most that any kernel makes of the shape: which one runs depends on dtype and alignment too
  for (const int row : {0, tree_flash_row(NHS_BF16, head_dim), tree_flash_row(NHS_F32, head_dim)})
    splits = std::max(splits, tree_shape(std::max(batch, 1), nodes, n_rows, q_heads, kv_heads, head_dim, row).n_splits);
  if (splits == 1) return 0;
  return (int64_t)splits * batch * nodes * q_heads * (head_dim + 2) * (int64_t)sizeof(float);
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
  const int64_t row_bytes = (int64_t)kv_heads * head_dim * esize, block = 2ll * page_size * row_bytes;
  if (pool_block_stride == 0) pool_block_stride = block;
  if (pool_block_stride < block || pool_block_stride % esize)
    return fail(NHS_ERR_INVALID, "%s: pool_block_stride is 0 or at least one block of whole elements", who);
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)pool) % esize ||
      ((uintptr_t)mask | (uintptr_t)rows) % 8)
    return fail(NHS_ERR_INVALID, "%s: misaligned pointer", who);
  bool flash = tree_flash_row(dtype, head_dim) > 0 && pool_block_stride % 16 == 0 &&
               ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)pool) % 16 == 0;
  for (const int64_t stride : {q_batch_stride, q_node_stride, q_head_stride, k_batch_stride, k_node_stride,
                               k_head_stride, v_batch_stride, v_node_stride, v_head_stride, out_batch_stride,
                               out_node_stride, out_head_stride})
    flash = flash && stride * esize % 16 == 0;
  const TreeShape shape =
      tree_shape(batch, nodes, n_rows, q_heads, kv_heads, head_dim, flash ? tree_flash_row(dtype, head_dim) : 0);
  const int64_t need = nhs_tree_attention_workspace_bytes(batch, nodes, n_rows, q_heads, kv_heads, head_dim);
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(NHS_ERR_WORKSPACE, "%s: needs %lld bytes of 16-byte aligned workspace", who, (long long)need);
  const int64_t blocks = (int64_t)batch * kv_heads * shape.row_blocks * shape.n_splits;
  const int threads = flash ? shape.waves * shape.shares * kWave : kTgThreads;
  if (blocks * threads > 0xffffffffll || (int64_t)batch * nodes * q_heads > 0x7fffffff)  // (a launch has 32 bits of threads)
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
  a.batch = batch, a.nodes = nodes, a.q_heads = q_heads, a.kv_heads = kv_heads, a.group = q_heads / kv_heads;
  a.head_dim = head_dim, a.page_size = page_size;
  a.query_rows = nodes * a.group, a.row_blocks = shape.row_blocks;
  a.group_div = FastDiv((uint32_t)a.group), a.page_div = FastDiv((uint32_t)page_size);
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  a.out = static_cast<char*>(out);
  a.o_b = out_batch_stride, a.o_n = out_node_stride, a.o_h = out_head_stride;
  a.out_rows = (int64_t)batch * nodes * q_heads;
  a.partial = static_cast<float*>(workspace);
  a.stats = a.partial + a.out_rows * shape.n_splits * head_dim;
  hipStream_t s = (hipStream_t)stream;
  const hipEvent_t none = nullptr;
  const auto run = [&](auto kernel, auto join, int rows_each) {
    const bool joined = shape.n_splits > 1;
    launch(kernel, dim3((unsigned)blocks), dim3((unsigned)threads), 0, s, ev.start, joined ? none : ev.stop, a);
    if (joined)
      launch(join, dim3((unsigned)((a.out_rows + rows_each - 1) / rows_each)), dim3(256), 0, s, none, ev.stop, a);
  };
  const auto general = [&](auto tag) {
    using T = decltype(tag);
    if (head_dim <= 128)
      run(tree_general_kernel<T, 32, 128>, tree_join_general_kernel<T>, 4);
    else
      run(tree_general_kernel<T, 16, kTgMaxDim>, tree_join_general_kernel<T>, 4);
  };
  const auto on_mfma = [&](auto tag, auto dim) {
    using T = decltype(tag);
    constexpr int D = decltype(dim)::value;
    const auto go = [&](auto kernel) {
      if (shape.n_splits > 16)
        run(kernel, tree_join_kernel<T, D, 4>, 1);
      else
        run(kernel, tree_join_kernel<T, D, 1>, 4);
    };
    constexpr int RB = D * T::bytes, BN = RB < 512 ? 64 : 32;  // (tiles of at most 64 KB in two buffers)
    if (shape.waves == 2) return go(tree_flash_kernel<T, D, 2, 2, BN>);
    if constexpr (RB <= 128)
      if (shape.waves == 1) return go(tree_flash_kernel<T, D, 1, 4, 32>);
    if constexpr (D < 256)
      if (shape.waves == 4) return go(tree_flash_kernel<T, D, 4, 2, BN>);
    if constexpr (D == 128 && RB == 256)
      if (shape.waves == 8) return go(tree_flash_kernel<T, D, 8, 1, BN>);
  };
  const auto by_dim = [&](auto tag) {
    using T = decltype(tag);
    if (!flash) return general(tag);
    switch (head_dim) {
      case 32: return on_mfma(tag, std::integral_constant<int, 32>());
      case 64: return on_mfma(tag, std::integral_constant<int, 64>());
      case 128: return on_mfma(tag, std::integral_constant<int, 128>());
      default:
        if constexpr (T::bytes == 2) on_mfma(tag, std::integral_constant<int, 256>());
    }
  };
  if (dtype == NHS_BF16)
    by_dim(BF16{});
  else if (dtype == NHS_F16)
    by_dim(F16{});
  else
    by_dim(F32{});
  return launch_status(who);
}
