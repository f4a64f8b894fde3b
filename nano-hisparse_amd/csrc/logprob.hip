// Log probabilities of given tokens, the entropy and the most likely
// alternatives of every row of logits (nhs_token_logprobs).
//
// For a row x[0..V) with m = max x and S = sum exp(x - m):
//   log p(i) = (x[i] - m) - ln S
//   entropy  = ln S - sum exp(x - m) (x - m) / S
// both terms of the entropy are >= 0, so nothing cancels. The alternatives
// are the `top` largest logits, equal ones by ascending index, a NaN above
// every number. A token outside [0, V) has log probability -inf; a row that
// holds a NaN or +inf, or nothing above -inf, has no distribution: NaN.
#include <math.h>

#include <algorithm>

#include "nhs_common.h"

namespace nhs {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / kWave, kLpMaxTop = NHS_MAX_TOP_LOGPROBS;
constexpr int kLpCandidates = 1024;  // keys held in LDS
constexpr int kLpMaxSplits = 64;
// The most alternatives for which the bound comes from the maxima of four threads each: a quarter of the comparisons, but
// a lower bound, which more threads reach. us with one thread / four: one bf16 row of 32001, top 5 9.0 / 8.1, 128 of
// them, top 10 10.7 / 9.8, top 20 11.9 / 11.3, top 32 12.8 / 13.1.
constexpr int kLpQuadTop = 24;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.693147180559945309417;

struct LogprobArgs {
  const char* logits;
  int64_t row_stride;  // elements
  int vocab, top, per_row;
  const int64_t* tokens;
  int64_t tokens_stride;
  float* logprobs;   // [rows, per_row]
  float* entropy;    // [rows]
  int64_t* top_ids;  // [rows, top]
  float* top_logprobs;
  int splits, split_chunks;
  float4* sums;    // splits > 1: [rows, splits] (reference, S, W, unused)
  uint64_t* keys;  // and [rows, splits, top], 0 where a split has fewer elements
};

// The order of the alternatives as unsigned keys: larger logit, larger key (-0 equals +0, a NaN is above +inf); the
// low word is the complement of the index, so equal logits go by ascending index. 0 is below every key.
__device__ __forceinline__ uint32_t lp_order(float x) {
  uint32_t u = __float_as_uint(x);
  if (u == 0x80000000u) u = 0u;
  const uint32_t ordered = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (u & 0x7fffffffu) > 0x7f800000u ? 0xfffffffeu : ordered;
}
__device__ __forceinline__ uint64_t lp_key(float x, int index) {
  return (uint64_t)lp_order(x) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ int lp_index(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float lp_value(uint64_t key) {  // the logit (+0 for -0, a NaN for a NaN)
  const uint32_t o = key >> 32;
  return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

__device__ __forceinline__ uint64_t lp_wave_max(uint64_t key) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint64_t other = (uint64_t)__shfl_xor((uint32_t)(key >> 32), d) << 32 | __shfl_xor((uint32_t)key, d);
    key = key > other ? key : other;
  }
  return key;
}

struct LogprobShared {
  float m[kLpWaves], s[kLpWaves], w[kLpWaves];
  uint64_t best[2][kLpWaves];
  __attribute__((aligned(16))) uint32_t lane_max[kLpThreads];  // order of the largest logit of each thread, 0 without one
  int hot[kLpThreads];               // threads whose elements may be among the alternatives
  int n_hot, n_found, scan[kLpWaves + 1];
  uint32_t threshold;
  __attribute__((aligned(16))) uint64_t found[kLpCandidates];
  uint64_t sorted[kLpMaxTop];
};

// Sums of a row or of a part: S = sum 2^(x log2 e - ref), W = sum 2^(...) (x log2 e - ref).
struct LpSums {
  float ref, s, w;
};
__device__ __forceinline__ LpSums lp_join(LpSums a, LpSums b) {
  const float ref = fmaxf(a.ref, b.ref), da = a.ref - ref, db = b.ref - ref;
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  // (below -1e9 the factor is 0: the product must only be finite)
  return {ref, a.s * fa + b.s * fb,
          fa * __builtin_fmaf(fmaxf(da, -1e9f), a.s, a.w) + fb * __builtin_fmaf(fmaxf(db, -1e9f), b.s, b.w)};
}

// over the wave: every lane moves to the largest reference, then plain sums
__device__ __forceinline__ LpSums lp_wave_join(LpSums t) {
  float ref = t.ref;
  ref = fmaxf(ref, dpp_f32<0xB1>(ref));   // lane ^ 1, ^ 2, then the mirrored 8 and 16 lanes, as group_sum goes
  ref = fmaxf(ref, dpp_f32<0x4E>(ref));
  ref = fmaxf(ref, dpp_f32<0x141>(ref));
  ref = fmaxf(ref, dpp_f32<0x140>(ref));
  ref = fmaxf(ref, __shfl_xor(ref, 16));
  ref = fmaxf(ref, __shfl_xor(ref, 32));
  const float d = t.ref - ref, f = __builtin_amdgcn_exp2f(d);
  return {ref, group_sum(t.s * f, kWave), group_sum(f * __builtin_fmaf(fmaxf(d, -1e9f), t.s, t.w), kWave)};
}

// The chunks of 16 bytes of a row that lie wholly inside it, and the elements before and after them.
template <typename T>
struct LpRow {
  static constexpr int E = 16 / T::bytes;
  const char* base;  // the first whole chunk
  int lead, chunks, vocab;
  __device__ LpRow(const LogprobArgs& a, int64_t row) : vocab(a.vocab) {
    const char* p = a.logits + row * a.row_stride * T::bytes;
    lead = min(vocab, (int)(-(intptr_t)p & 15) / T::bytes);
    chunks = (vocab - lead) / E;
    base = p + lead * T::bytes;
  }
  __device__ int index(int chunk, int e) const { return lead + chunk * E + e; }
  __device__ uint4 load(int chunk) const { return *reinterpret_cast<const uint4*>(base + (int64_t)chunk * 16); }
  __device__ float at(int64_t i) const { return load_elem(base, T::dtype, i - lead); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[E]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (T::dtype == NHS_F32)
        x[e] = __uint_as_float(w[e]);
      else if constexpr (T::dtype == NHS_BF16)
        x[e] = __uint_as_float((e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
      else
        x[e] = f16_bits_to_f32((e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xffffu);
    }
  }
};

// Chunks [first, last) of a row and, with `lead` / `tail`, the elements around all chunks.
struct LpPart {
  int first, last;
  bool lead, tail;
};

// The keys of the part's `top` largest elements to sh.sorted, one pass over the part per key.
template <typename T>
__device__ void lp_top_by_rounds(const LpRow<T>& row, const LpPart& part, int top, LogprobShared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int begin = part.lead ? 0 : row.index(part.first, 0), end = part.tail ? row.vocab : row.index(part.last, 0);
  uint64_t last = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t key = 0;
    for (int i = begin + tid; i < end; i += kLpThreads) {
      const uint64_t x = lp_key(row.at(i), i);
      if (x < last && x > key) key = x;
    }
    key = lp_wave_max(key);
    if (lane == 0) sh.best[k & 1][wave] = key;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kLpWaves; ++i) key = key > sh.best[k & 1][i] ? key : sh.best[k & 1][i];
    last = key;
    if (tid == 0) sh.sorted[k] = key;
  }
  __syncthreads();
}

// The `top` largest of sh.found[0 .. n) in descending order to sh.sorted (0 beyond n): every key's place is the number
// of larger ones. Eight keys are read at a time, so that the wait for LDS is paid once for them.
__device__ __forceinline__ void lp_sort_found(int n, int top, LogprobShared& sh) {
  constexpr int kStep = 8;
  const int tid = threadIdx.x, padded = (n + kStep - 1) / kStep * kStep;
  if (tid < top) sh.sorted[tid] = 0;
  if (tid < padded - n) sh.found[n + tid] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kLpThreads) {
    const uint64_t key = sh.found[i];
    int place[2] = {0, 0};
    for (int x = 0; x < padded; x += kStep) {
      uint64_t other[kStep];
#pragma unroll
      for (int e = 0; e < kStep; ++e) other[e] = sh.found[x + e];
#pragma unroll
      for (int e = 0; e < kStep; ++e) place[e & 1] += other[e] > key;
    }
    if (key && place[0] + place[1] < top) sh.sorted[place[0] + place[1]] = key;
  }
  __syncthreads();
}

// The `top` largest elements of the part, given each thread's largest (of chunks first + thread, + kLpThreads, ...):
// the top-th largest of these (or of those of four threads each) is a lower bound, and only the few threads that reach
// it hold elements that count; their chunks are read again and compared by the whole workgroup. Where many threads
// reach it (masked vocabularies) or more elements than LDS holds, those above it are kept and the equal ones counted
// off in index order.
template <typename T>
__device__ void lp_top(const LpRow<T>& row, const LpPart& part, int top, bool any, float thread_max,
                       LogprobShared& sh) {
  constexpr int E = LpRow<T>::E;
  const int tid = threadIdx.x, lane = tid & 63;
  const uint32_t mine = any ? lp_order(thread_max) : 0u;
  const bool quads = top <= kLpQuadTop;
  uint32_t best = mine;
  if (quads) {  // the four threads of a quad stand for one
    best = max(best, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)best, 0xB1, 0xF, 0xF, false));
    best = max(best, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)best, 0x4E, 0xF, 0xF, false));
    if (tid % 4 == 0) sh.lane_max[tid / 4] = best;
  } else {
    sh.lane_max[tid] = mine;
  }
  if (tid == 0) sh.n_hot = sh.n_found = 0, sh.threshold = 0xffffffffu;
  __syncthreads();
  // the threads (or quads) with fewer than `top` larger ones; the least of them is the top-th largest
  int larger[2] = {0, 0};
  const uint4* all = reinterpret_cast<const uint4*>(sh.lane_max);
#pragma unroll 8
  for (int i = 0; i < (quads ? kLpThreads / 16 : kLpThreads / 4); ++i) {
    const uint4 v = all[i];
    larger[0] += (v.x > best) + (v.z > best);
    larger[1] += (v.y > best) + (v.w > best);
  }
  if (larger[0] + larger[1] < top) atomicMin(&sh.threshold, best);
  __syncthreads();
  const uint32_t threshold = sh.threshold;
  if (mine && mine >= threshold) sh.hot[atomicAdd(&sh.n_hot, 1)] = tid;
  __syncthreads();
  const int per_thread = (part.last - part.first + kLpThreads - 1) / kLpThreads;
  // pushes the elements whose order is at least `least`
  const auto collect = [&](uint32_t least) {
    const int log = 32 - __clz(max(per_thread, 1) - 1), pairs = sh.n_hot << log;  // (chunks of a thread, to a power of two)
    const auto push = [&](float x, int i) {
      if (lp_order(x) >= least) {
        const int at = atomicAdd(&sh.n_found, 1);
        if (at < kLpCandidates) sh.found[at] = lp_key(x, i);
      }
    };
    for (int p = tid; p < pairs; p += kLpThreads) {
      const int chunk = part.first + sh.hot[p >> log] + (p & ((1 << log) - 1)) * kLpThreads;
      if (chunk >= part.last) continue;
      float x[E];
      LpRow<T>::unpack(row.load(chunk), x);
#pragma unroll
      for (int e = 0; e < E; ++e) push(x[e], row.index(chunk, e));
    }
    const int behind = row.index(row.chunks, 0);
    const int lead = part.lead ? row.lead : 0, around = lead + (part.tail ? row.vocab - behind : 0);
    if (tid < around) {
      const int i = tid < lead ? tid : behind + tid - lead;
      push(row.at(i), i);
    }
  };
  // (a row of 128256 with half of it masked: 15 us, where looking through all that reach the bound first took 20)
  bool ties = sh.n_hot > 2 * top + 32;
  if (!ties) {
    collect(threshold);
    __syncthreads();
    ties = sh.n_found > kLpCandidates;
  }
  if (ties) {
    __syncthreads();
    if (tid == 0) sh.n_hot = sh.n_found = 0;
    __syncthreads();
    if (mine > threshold) sh.hot[atomicAdd(&sh.n_hot, 1)] = tid;
    __syncthreads();
    collect(threshold + 1);
    __syncthreads();
    const int above = sh.n_found;
    if (above > kLpCandidates - kLpMaxTop) {
      lp_top_by_rounds(row, part, top, sh);
      return;
    }
    // the first elements equal to the threshold, in index order: those before the chunks, chunk by chunk, those behind
    int left = max(top - above, 0), taken = above;
    const auto equal = [&](uint32_t bits, int first) {  // bit e: element first + e
      const int count = __popc(bits);
      int incl = count;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
      }
      if (lane == kWave - 1) sh.scan[tid >> 6] = incl;
      __syncthreads();
      int before = incl - count, total = 0;
#pragma unroll
      for (int w = 0; w < kLpWaves; ++w) {
        if (w < (tid >> 6)) before += sh.scan[w];
        total += sh.scan[w];
      }
      for (uint32_t b = bits; b && before < left; b &= b - 1, ++before)
        sh.found[taken + before] = (uint64_t)threshold << 32 | (uint32_t)~(first + __ffs(b) - 1);
      const int used = min(total, left);
      taken += used, left -= used;
      __syncthreads();
    };
    if (part.lead) equal(tid < row.lead && lp_order(row.at(tid)) == threshold, tid);
    for (int c = part.first; c < part.last && left > 0; c += kLpThreads) {
      uint32_t bits = 0;
      if (c + tid < part.last) {
        float x[E];
        LpRow<T>::unpack(row.load(c + tid), x);
#pragma unroll
        for (int e = 0; e < E; ++e) bits |= (uint32_t)(lp_order(x[e]) == threshold) << e;
      }
      equal(bits, row.index(c + tid, 0));
    }
    if (part.tail && left > 0) {  // fewer elements than threads
      const int i = row.index(row.chunks, 0) + tid;
      equal(i < row.vocab && lp_order(row.at(i)) == threshold, i);
    }
    lp_sort_found(taken, top, sh);
    return;
  }
  lp_sort_found(sh.n_found, top, sh);
}

// The logit of a given token.
struct LpToken {
  float x;
  bool known;
};
template <typename T>
__device__ __forceinline__ LpToken lp_token(const LogprobArgs& a, int64_t r, const LpRow<T>& row, int g) {
  const int64_t token = a.tokens[r * a.tokens_stride + g];
  const bool known = token >= 0 && token < a.vocab;
  return {row.at(known ? token : 0), known};
}

// The outputs of a row from its sums and sh.sorted. The sums are those of x * (1 + beta), where kLog2e rounds to
// log2 e * (1 + beta): to first order lse(x) = lse(x (1 + beta)) - beta * sum p x. (No rounding makes a probability more
// than 1 or an entropy less than 0.)
template <typename F>
__device__ __forceinline__ void lp_finish(const LogprobArgs& a, int64_t r, const LpSums& t, const LpToken& first,
                                          F logit, LogprobShared& sh) {
  constexpr double beta = (double)kLog2e * kLn2 - 1.0;
  const double bits = (double)log2f(t.s), mean = (double)t.w / (double)t.s;
  const double lse = ((double)t.ref + bits - beta * (mean + (double)t.ref)) * kLn2;
  const int tid = threadIdx.x;
  if (tid == 0) a.entropy[r] = (float)fmax((bits - mean) * kLn2, 0.0);
  for (int g = tid; g < a.per_row; g += kLpThreads) {
    const LpToken token = g == tid ? first : logit(g);
    a.logprobs[r * a.per_row + g] = token.known ? (float)fmin((double)token.x - lse, 0.0) : -INFINITY;
  }
  if (tid < a.top) {
    a.top_ids[r * a.top + tid] = lp_index(sh.sorted[tid]);
    a.top_logprobs[r * a.top + tid] = (float)fmin((double)lp_value(sh.sorted[tid]) - lse, 0.0);
  }
}

// A row whose sums overflow or vanish in the form above (a NaN, +inf, nothing above -inf, logits beyond 1e38): the
// formulas as they stand, one pass per step.
template <typename T>
__device__ void lp_unusual_row(const LogprobArgs& a, int64_t r, const LpRow<T>& row, LogprobShared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  float m = -INFINITY;
  bool nan = false;
  for (int i = tid; i < a.vocab; i += kLpThreads) {
    const float x = row.at(i);
    nan |= x != x;
    m = fmaxf(m, x);
  }
  if (nan) m = NAN;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const float other = __shfl_xor(m, d);
    m = m != m || other != other ? NAN : fmaxf(m, other);
  }
  __syncthreads();
  if (lane == 0) sh.m[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) m = m != m || sh.m[w] != sh.m[w] ? NAN : fmaxf(m, sh.m[w]);
  float s = 0.f, w = 0.f;
  for (int i = tid; i < a.vocab; i += kLpThreads) {
    const float y = (row.at(i) - m) * kLog2e, e = __builtin_amdgcn_exp2f(y);
    s += e;
    if (e != 0.f) w = __builtin_fmaf(e, y, w);
  }
  s = group_sum(s, kWave), w = group_sum(w, kWave);
  if (lane == 0) sh.s[wave] = s, sh.w[wave] = w;
  __syncthreads();
  s = w = 0.f;
#pragma unroll
  for (int i = 0; i < kLpWaves; ++i) s += sh.s[i], w += sh.w[i];
  const float log_s = logf(s), entropy = log_s - w / s * (float)kLn2;
  const auto at_most_0 = [](float x) { return x > 0.f ? 0.f : x; };  // a NaN stays
  if (tid == 0) a.entropy[r] = -at_most_0(-entropy);
  for (int g = tid; g < a.per_row; g += kLpThreads) {
    const LpToken token = lp_token(a, r, row, g);
    a.logprobs[r * a.per_row + g] = token.known ? at_most_0(token.x - m - log_s) : s == s ? -INFINITY : NAN;
  }
  lp_top_by_rounds(row, LpPart{0, row.chunks, true, true}, a.top, sh);
  if (tid < a.top) {
    a.top_ids[r * a.top + tid] = lp_index(sh.sorted[tid]);
    a.top_logprobs[r * a.top + tid] = at_most_0(lp_value(sh.sorted[tid]) - m - log_s);
  }
}

__device__ __forceinline__ bool lp_usual(const LpSums& t) { return t.s > 0.f && t.s < INFINITY; }

// One pass over a row or a part of it. Every thread keeps a reference of its
// own (its running maximum times log2 e, rounded: the exponents are exact
// relative to it, and references only ever meet as these numbers), S and W
// over blocks of four chunks, and its largest logit, which the search for the
// alternatives starts from. Long prompts are bound by memory: 4000 bf16 rows
// of 128256, read once, 185 us (5.5 TB/s; with a maximum, a sum and a search
// in passes of their own 1626). Short ones by the chain of steps, each waiting
// for the last: one row of 128256 takes 5.5 us without alternatives and 9.5 with
// five, 128 rows of 32001 6.7 and 9.5 (a launch that does nothing, 2).
template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_kernel(LogprobArgs a) {
  constexpr int E = LpRow<T>::E, U = 4;
  __shared__ LogprobShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x / (unsigned)a.splits;
  const int split = blockIdx.x - (int)r * a.splits;
  const LpRow<T> row(a, r);
  LpPart part;
  part.first = min(split * a.split_chunks, row.chunks);
  part.last = split == a.splits - 1 ? row.chunks : min(part.first + a.split_chunks, row.chunks);
  part.lead = split == 0, part.tail = split == a.splits - 1;

  // the given tokens' logits are asked for first
  const LpToken token = a.splits == 1 && tid < a.per_row ? lp_token(a, r, row, tid) : LpToken{0.f, false};
  float m = -1e38f, top = -INFINITY;  // (a finite start: nothing above it leaves S at 0)
  LpSums t{m * kLog2e, 0.f, 0.f};
  const auto raise = [&](float block_max) {
#pragma clang fp contract(off)  // d is the difference of the rounded references
    top = fmaxf(top, block_max);
    const float ref = fmaxf(m, block_max) * kLog2e, d = t.s > 0.f ? t.ref - ref : 0.f;
    const float f = __builtin_amdgcn_exp2f(d);
    m = fmaxf(m, block_max);
    t.w = f * __builtin_fmaf(fmaxf(d, -1e9f), t.s, t.w);
    t.s *= f;
    t.ref = ref;
  };
  const auto add = [&](float x, float& s, float& w) {
    const float y = __builtin_fmaf(x, kLog2e, -t.ref), e = __builtin_amdgcn_exp2f(y);
    s += e;
    w = __builtin_fmaf(e, fmaxf(y, -1e9f), w);  // 0 and not NaN where x is -inf
  };
  // (one copy of the loop's body, also for the last block: a row is often shorter than the code that it runs is long)
  for (int c = part.first + tid; c < part.last; c += U * kLpThreads) {
    constexpr uint32_t none = T::dtype == NHS_F32 ? 0xff800000u : T::dtype == NHS_BF16 ? 0xff80ff80u : 0xfc00fc00u;
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // chunks past the end count as -inf
      v[u] = make_uint4(none, none, none, none);
      if (c + u * kLpThreads < part.last) v[u] = row.load(c + u * kLpThreads);
    }
    float x[U][E], block_max = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      LpRow<T>::unpack(v[u], x[u]);
#pragma unroll
      for (int e = 0; e < E; ++e) block_max = fmaxf(block_max, x[u][e]);
    }
    raise(block_max);
    float s = 0.f, w = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) add(x[u][e], s, w);
    t.s += s, t.w += w;
  }
  const bool any = part.first + tid < part.last;
  const float thread_max = top;
  // the elements before and after the chunks, which the search looks at in any case
  const int behind = row.index(row.chunks, 0);
  const int lead = part.lead ? row.lead : 0, around = lead + (part.tail ? row.vocab - behind : 0);
  if (tid < around) {
    const float x = row.at(tid < lead ? tid : behind + tid - lead);
    raise(x);
    add(x, t.s, t.w);
  }
  t = lp_wave_join(t);
  if (lane == 0) sh.m[wave] = t.ref, sh.s[wave] = t.s, sh.w[wave] = t.w;
  __syncthreads();
  t = {sh.m[0], sh.s[0], sh.w[0]};
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) t = lp_join(t, LpSums{sh.m[w], sh.s[w], sh.w[w]});
  if (a.splits == 1 && !lp_usual(t)) {
    lp_unusual_row(a, r, row, sh);
    return;
  }
  if (a.top) lp_top(row, part, a.top, any, thread_max, sh);
  if (a.splits == 1) {
    lp_finish(a, r, t, token, [&](int g) { return lp_token(a, r, row, g); }, sh);
    return;
  }
  if (tid == 0) a.sums[blockIdx.x] = make_float4(t.ref, t.s, t.w, 0.f);
  if (tid < a.top) a.keys[(int64_t)blockIdx.x * a.top + tid] = sh.sorted[tid];
}

// Joins the parts of a row, one workgroup per row.
template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_join_kernel(LogprobArgs a) {
  __shared__ LogprobShared sh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t r = blockIdx.x;
  const LpRow<T> row(a, r);
  const int n = a.splits * a.top;  // at most kLpThreads
  const LpToken token = tid < a.per_row ? lp_token(a, r, row, tid) : LpToken{0.f, false};
  for (int i = tid; i < n; i += kLpThreads) sh.found[i] = a.keys[r * n + i];
  const float4 part = a.sums[r * a.splits + min(lane, a.splits - 1)];
  LpSums t{part.x, lane < a.splits ? part.y : 0.f, lane < a.splits ? part.z : 0.f};
  t = lp_wave_join(t);
  __syncthreads();
  if (!lp_usual(t)) {
    lp_unusual_row(a, r, row, sh);
    return;
  }
  if (a.top) lp_sort_found(n, a.top, sh);
  lp_finish(a, r, t, token, [&](int g) { return lp_token(a, r, row, g); }, sh);
}

struct LogprobShape {
  int splits, split_chunks;
};

// About 512 workgroups in all (two on a CU), none of less than 2048 chunks (eight loads of every thread): every part
// searches for alternatives, and parts have to be joined. us with at least 1024 / 2048 / 4096 chunks: one bf16 row of
// 32001 (top 5) 10.2 / 9.2 / 9.2, 128 of them (top 20) 14.1 / 11.8 / 11.9, one fp32 row of 128256 11.3 / 10.7 / 11.1,
// 16 bf16 rows of 128256 11.4 / 11.5 / 13.1. With 256 / 512 / 1024 workgroups: 100 rows of 128256 17.8 / 16.6 / 17.7,
// 250 fp32 rows (top 20) 47.8 / 38.1 / 38.1, 400 rows of 50257 16.7 / 16.7 / 20.9.
static LogprobShape logprob_shape(int rows, int vocab, int dtype, int top) {
  const int chunks = vocab / (16 / elem_size(dtype));
  int64_t splits = std::min<int64_t>(512 / std::max(rows, 1), chunks / 2048);
  // (the join sorts a key per thread)
  splits = std::min<int64_t>(splits, std::min(kLpMaxSplits, kLpThreads / std::max(top, 1)));
  LogprobShape s;
  s.splits = (int)std::max<int64_t>(splits, 1);
  s.split_chunks = (chunks + s.splits - 1) / s.splits;
  return s;
}

}  // namespace nhs

using namespace nhs;

extern "C" int64_t nhs_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t dtype, int32_t top) {
  if (rows < 1 || vocab < 1 || top < 0 || top > kLpMaxTop || !valid_dtype(dtype)) return 0;
  const LogprobShape s = logprob_shape(rows, vocab, dtype, top);
  return s.splits == 1 ? 0 : (int64_t)rows * s.splits * (int64_t)(sizeof(float4) + top * sizeof(uint64_t));
}

extern "C" int nhs_token_logprobs(const void* logits, int64_t row_stride, int32_t dtype, int32_t rows, int32_t vocab,
                                  const int64_t* tokens, int64_t tokens_stride, int32_t tokens_per_row, int32_t top,
                                  float* logprobs, float* entropy, int64_t* top_ids, float* top_logprobs,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  const LaunchEvents ev = take_launch_events();
  const char* who = "nhs_token_logprobs";
  if (!valid_dtype(dtype) || rows < 0 || vocab < 1 || tokens_per_row < 0 || top < 0 || top > vocab)
    return fail(NHS_ERR_INVALID, "%s: invalid shape or dtype", who);
  if (top > kLpMaxTop) return fail(NHS_ERR_UNSUPPORTED, "%s: at most %d alternatives", who, kLpMaxTop);
  if (vocab > (1 << 30)) return fail(NHS_ERR_UNSUPPORTED, "%s: vocab up to 2^30", who);
  if (rows == 0) return NHS_OK;
  if (!logits || !entropy || (tokens_per_row > 0 && (!tokens || !logprobs)) || (top > 0 && (!top_ids || !top_logprobs)))
    return fail(NHS_ERR_INVALID, "%s: null pointer", who);
  if ((uintptr_t)logits % elem_size(dtype) || ((uintptr_t)tokens | (uintptr_t)top_ids) % 8 ||
      ((uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)top_logprobs) % 4)
    return fail(NHS_ERR_INVALID, "%s: misaligned pointer", who);
  const LogprobShape shape = logprob_shape(rows, vocab, dtype, top);
  const int64_t need = nhs_token_logprobs_workspace_bytes(rows, vocab, dtype, top), parts = (int64_t)rows * shape.splits;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(NHS_ERR_WORKSPACE, "%s: needs %lld bytes of 16-byte aligned workspace", who, (long long)need);
  if (parts * kLpThreads > 0xffffffffll) return fail(NHS_ERR_UNSUPPORTED, "%s: too many rows", who);
  LogprobArgs a{static_cast<const char*>(logits), row_stride, vocab, top, tokens_per_row, tokens, tokens_stride,
                logprobs, entropy, top_ids, top_logprobs, shape.splits, shape.split_chunks,
                static_cast<float4*>(workspace), nullptr};
  a.keys = reinterpret_cast<uint64_t*>(a.sums + parts);
  hipStream_t s = (hipStream_t)stream;
  const hipEvent_t none = nullptr;
  const auto run = [&](auto kernel, auto join) {
    const bool joined = shape.splits > 1;
    launch(kernel, dim3((unsigned)parts), dim3(kLpThreads), 0, s, ev.start, joined ? none : ev.stop, a);
    if (joined) launch(join, dim3((unsigned)rows), dim3(kLpThreads), 0, s, none, ev.stop, a);
  };
  if (dtype == NHS_BF16)
    run(logprob_kernel<BF16>, logprob_join_kernel<BF16>);
  else if (dtype == NHS_F16)
    run(logprob_kernel<F16>, logprob_join_kernel<F16>);
  else
    run(logprob_kernel<F32>, logprob_join_kernel<F32>);
  return launch_status(who);
}
