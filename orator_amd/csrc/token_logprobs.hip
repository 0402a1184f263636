// Log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
// With m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m):
//   lse = m + log S,  logprob = x_tok - lse,  entropy = log S - T / S.
// Entries of -infinity have weight 0 and add 0 to T.
//
// One workgroup per row, three kinds of passes over it: the maximum, the sums, and one per
// alternative for the largest entry that comes after the previous one in the order (value
// descending, id ascending).
#include <string>

#include "common.hpp"
#include "internal.hpp"

namespace orator_hip {
namespace {

constexpr int kTopMax = 32;
constexpr int kThreads = 1024;

struct LogprobArgs {
  const float* x;
  long row_stride;
  const int* tokens;
  int vocab, top_k;
  float* logprob;
  float* entropy;
  int* top_ids;
  float* top_logprobs;
};

// Order of the alternatives as one unsigned key: larger values above smaller ones, -0 as +0, every
// NaN below -infinity; equal values with the lower id first.
__device__ __forceinline__ uint64_t order_key(float x, int id) {
  uint32_t u = __float_as_uint(x + 0.0f);
  u = (u & 0x7fffffffu) > 0x7f800000u ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return static_cast<uint64_t>(u) << 32 | static_cast<uint32_t>(~id);
}

template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T* lds, Op op) {
  for (int s = 1; s < 64; s <<= 1) v = op(v, __shfl_xor(v, s));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  T r = lds[0];
  for (int w = 1; w < kThreads / 64; ++w) r = op(r, lds[w]);
  return r;
}

__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(LogprobArgs a) {
  __shared__ float red[kThreads / 64];
  __shared__ unsigned long long red64[kThreads / 64];
  const int row = blockIdx.x;
  const float* x = a.x + row * a.row_stride;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) m = fmaxf(m, x[i]);
  m = block_reduce(m, red, [](float p, float q) { return fmaxf(p, q); });
  const float ref = m == -INFINITY ? 0.0f : m;
  float S = 0.0f, T = 0.0f;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const float d = x[i] - ref;
    const float e = expf(d);
    S += e;
    T += d == -INFINITY ? 0.0f : e * d;
  }
  S = block_reduce(S, red, [](float p, float q) { return p + q; });
  T = block_reduce(T, red, [](float p, float q) { return p + q; });
  const float logS = logf(S), lse = ref + logS;  // -infinity for a row of -infinity only
  auto logp = [&](float v) { return v == -INFINITY && S == S ? -INFINITY : (v - ref) - logS; };
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const int t = a.tokens[row];
      a.logprob[row] = t >= 0 && t < a.vocab ? logp(x[t]) : __uint_as_float(0x7fc00000u);
    }
    if (a.entropy) a.entropy[row] = S == 0.0f ? 0.0f : logS - T / S;
  }
  (void)lse;
  unsigned long long prev = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const unsigned long long key = order_key(x[i], i);
      if (key < prev && key > best) best = key;
    }
    best = block_reduce(best, red64,
                        [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
    prev = best;
    if (threadIdx.x == 0) {
      const int id = static_cast<int>(~static_cast<uint32_t>(best));
      a.top_ids[static_cast<long>(row) * a.top_k + k] = id;
      a.top_logprobs[static_cast<long>(row) * a.top_k + k] = logp(x[id]);
    }
  }
}

}  // namespace
}  // namespace orator_hip

using namespace orator_hip;

extern "C" int orator_token_logprobs(const float* logits, long row_stride, const int* tokens,
                                     int rows, int vocab, int top_k, float* logprob,
                                     float* entropy, int* top_ids, float* top_logprobs,
                                     void* stream) {
  return guarded([&] {
    if (rows <= 0 || vocab <= 0) return ORATOR_OK;
    if (!logits || (logprob && !tokens))
      return fail(ORATOR_ERR_INVALID, "token_logprobs: null pointer");
    if (row_stride < vocab)
      return fail(ORATOR_ERR_INVALID, "token_logprobs: row_stride below vocab");
    if (top_k < 0 || top_k > kTopMax || top_k > vocab)
      return fail(ORATOR_ERR_UNSUPPORTED, "token_logprobs: top_k in [0, 32], at most vocab");
    if (!top_ids != !top_logprobs)
      return fail(ORATOR_ERR_INVALID, "token_logprobs: top_ids and top_logprobs go together");
    if (!top_ids) top_k = 0;
    if (!logprob && !entropy && top_k == 0) return ORATOR_OK;
    LogprobArgs a{logits, row_stride, tokens, vocab, top_k, logprob, entropy, top_ids, top_logprobs};
    hipLaunchKernelGGL(token_logprobs_kernel, dim3(rows), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    return check_launch("token_logprobs_kernel");
  });
}
