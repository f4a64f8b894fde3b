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

constexpr int kLpThreads = 256, kLpMaxTop = NHS_MAX_TOP_LOGPROBS;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogprobArgs {
  const char* logits;
  int64_t row_stride;  // elements
  int vocab, top, per_row;
  const int64_t* tokens;
  int64_t tokens_stride;
  float* logprobs;  // [rows, per_row]
  float* entropy;   // [rows]
  int64_t* top_ids;  // [rows, top]
  float* top_logprobs;
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

__device__ __forceinline__ uint64_t lp_wave_max(uint64_t key) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint64_t other = (uint64_t)__shfl_xor((uint32_t)(key >> 32), d) << 32 | __shfl_xor((uint32_t)key, d);
    key = key > other ? key : other;
  }
  return key;
}

// One workgroup per row: a pass for the maximum and the sums, then a pass per alternative for the largest key below the
// last one.
template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_rows_kernel(LogprobArgs a) {
  __shared__ float sm[kLpThreads / kWave], ss[kLpThreads / kWave], sw[kLpThreads / kWave];
  __shared__ uint64_t best[2][kLpThreads / kWave];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t base = row * a.row_stride;
  float m = -INFINITY;
  bool nan = false;
  for (int i = tid; i < a.vocab; i += kLpThreads) {
    const float x = load_elem(a.logits, T::dtype, base + i);
    nan |= x != x;
    m = fmaxf(m, x);
  }
  if (nan) m = NAN;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const float other = __shfl_xor(m, d);
    m = m != m || other != other ? NAN : fmaxf(m, other);
  }
  if (lane == 0) sm[wave] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kLpThreads / kWave; ++w) m = m != m || sm[w] != sm[w] ? NAN : fmaxf(m, sm[w]);
  float s = 0.f, w = 0.f;
  for (int i = tid; i < a.vocab; i += kLpThreads) {
    const float y = (load_elem(a.logits, T::dtype, base + i) - m) * kLog2e, e = __builtin_amdgcn_exp2f(y);
    s += e;
    if (e != 0.f) w = __builtin_fmaf(e, y, w);
  }
  s = group_sum(s, kWave), w = group_sum(w, kWave);
  if (lane == 0) ss[wave] = s, sw[wave] = w;
  __syncthreads();
  s = w = 0.f;
#pragma unroll
  for (int i = 0; i < kLpThreads / kWave; ++i) s += ss[i], w += sw[i];
  const float log_s = logf(s);
  if (tid == 0) a.entropy[row] = log_s - w / s * kLn2;
  for (int g = tid; g < a.per_row; g += kLpThreads) {
    const int64_t token = a.tokens[row * a.tokens_stride + g];
    const bool known = token >= 0 && token < a.vocab;
    a.logprobs[row * a.per_row + g] =
        known ? load_elem(a.logits, T::dtype, base + token) - m - log_s : s == s ? -INFINITY : NAN;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t key = 0;
    for (int i = tid; i < a.vocab; i += kLpThreads) {
      const uint64_t x = lp_key(load_elem(a.logits, T::dtype, base + i), i);
      if (x < last && x > key) key = x;
    }
    key = lp_wave_max(key);
    if (lane == 0) best[k & 1][wave] = key;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kLpThreads / kWave; ++i) key = key > best[k & 1][i] ? key : best[k & 1][i];
    last = key;
    if (tid == 0) {
      const int index = (int)~(uint32_t)key;
      a.top_ids[row * a.top + k] = index;
      a.top_logprobs[row * a.top + k] = load_elem(a.logits, T::dtype, base + index) - m - log_s;
    }
  }
}

}  // namespace nhs

using namespace nhs;

extern "C" int64_t nhs_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t dtype, int32_t top) {
  return 0;
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
  if (rows == 0) return NHS_OK;
  if (!logits || !entropy || (tokens_per_row > 0 && (!tokens || !logprobs)) || (top > 0 && (!top_ids || !top_logprobs)))
    return fail(NHS_ERR_INVALID, "%s: null pointer", who);
  if ((uintptr_t)logits % elem_size(dtype) || ((uintptr_t)tokens | (uintptr_t)top_ids) % 8 ||
      ((uintptr_t)logprobs | (uintptr_t)entropy | (uintptr_t)top_logprobs) % 4)
    return fail(NHS_ERR_INVALID, "%s: misaligned pointer", who);
  LogprobArgs a{static_cast<const char*>(logits), row_stride, vocab, top, tokens_per_row, tokens, tokens_stride,
                logprobs, entropy, top_ids, top_logprobs};
  const dim3 grid((unsigned)rows), block(kLpThreads);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == NHS_BF16)
    launch(logprob_rows_kernel<BF16>, grid, block, 0, s, ev.start, ev.stop, a);
  else if (dtype == NHS_F16)
    launch(logprob_rows_kernel<F16>, grid, block, 0, s, ev.start, ev.stop, a);
  else
    launch(logprob_rows_kernel<F32>, grid, block, 0, s, ev.start, ev.stop, a);
  return launch_status(who);
}
