// Log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
// With m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m):
//   lse = m + log S,  logprob = x_tok - lse,  entropy = log S - T / S.
// Entries of -infinity have weight 0 and add 0 to T.
//
// Memory-bound: the logits are read once.  A row is cut into parts of up to 8192 entries, one
// workgroup each, which holds its part in registers (32 entries a thread): the maximum, the sums
// against it, and the part's best entries, all from the one read.  The last workgroup of a row to
// finish joins its parts.
//
// Best entries of a part: the k-th largest of the 64 lanes' maxima of a wave is a bound that k
// entries reach; entries at or above the largest of the waves' bounds (k to a few hundred) go to
// LDS, and each finds its rank by counting those before it.  Parts where that leaves too many (ties
// in masses) or too few (NaN) extract their best one after the other instead.
#include <algorithm>
#include <string>

#include "common.hpp"
#include "internal.hpp"

namespace orator_hip {
namespace {

typedef unsigned long long u64;

constexpr int kTopMax = 32;
constexpr int kThreads = 256;
constexpr int kWavesN = kThreads / 64;
constexpr int kVec = 8;                           // float4 per thread
constexpr int kPart = kThreads * kVec * 4;        // entries of a part, at most
constexpr int kCand = 768;                        // candidates kept in LDS
constexpr int kFirst = 256;                       // entries whose -infinity may be a candidate

struct LogprobArgs {
  const float* x;
  long row_stride;
  const int* tokens;
  int vocab, top_k;
  float* logprob;
  float* entropy;
  int* top_ids;
  float* top_logprobs;
  int parts, part_len;
  float* stats;      // [rows][parts][4]: m, S, T
  u64* best;         // [rows][parts][top_k], descending; 0: none
  unsigned* arrive;  // [rows], kCounterStride apart; null: one part
};

// Order of the values as an unsigned number: larger above smaller, -0 as +0, NaN at 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x7fffffffu) > 0x7f800000u ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return o == 0u ? __uint_as_float(0x7fc00000u)
                 : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
// Order of the entries: the larger value, then the lower id.
__device__ __forceinline__ u64 key_of(float x, int id) {
  return static_cast<u64>(order_of(x)) << 32 | static_cast<uint32_t>(~id);
}
__device__ __forceinline__ int id_of(u64 key) { return static_cast<int>(~static_cast<uint32_t>(key)); }

__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 wave_max64(u64 v) {
  for (int s = 1; s < 64; s <<= 1) v = max64(v, static_cast<u64>(__shfl_xor(static_cast<long long>(v), s)));
  return v;
}

template <typename T>
__device__ __forceinline__ void store_dev(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T load_dev(const T* p) {
  return __hip_atomic_load(const_cast<T*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct Vec4 {
  float v[4];
};
// 16 bytes at any 4-byte address.
__device__ __forceinline__ Vec4 load4(const float* p) {
  typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
  const f4 r = __builtin_nontemporal_load(reinterpret_cast<const f4*>(p));
  return {{r[0], r[1], r[2], r[3]}};
}

// The row's sums over its parts; every thread of a wave gets them.
struct RowSums {
  float ref, logS;  // lse = ref + logS
  float S, T;
  __device__ __forceinline__ float logp(float v) const {
    return v == -INFINITY && S == S ? -INFINITY : (v - ref) - logS;
  }
};

__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(LogprobArgs a) {
  __shared__ float s_red[kWavesN][3];
  __shared__ uint32_t s_bound[kWavesN];
  __shared__ u64 s_cand[kCand];
  __shared__ u64 s_best[kTopMax];
  __shared__ int s_n, s_inf, s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = blockIdx.x % a.parts;
  const int row = blockIdx.x / a.parts;
  const float* x = a.x + row * a.row_stride;
  const int base = part * a.part_len;
  const int n = min(a.part_len, a.vocab - base);  // >= 1
  const int k = a.top_k;

  // ---- the part, 4 consecutive entries at (i * kThreads + tid) * 4; behind its end -infinity ----
  float v[kVec][4];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int at = (i * kThreads + tid) * 4;
    if (at + 4 <= n) {
      const Vec4 r = load4(x + base + at);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = r.v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = at + j < n ? x[base + at + j] : -INFINITY;
    }
  }
  if (tid == 0) s_n = s_inf = 0;

  // ---- maximum, bound of the k-th best, sums ----
  float mine = -INFINITY;
#pragma unroll
  for (int i = 0; i < kVec; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) mine = fmaxf(mine, v[i][j]);
  const float wm = wave_max(mine);
  uint32_t bound = 0;
  if (k > 0) {
    // the upper 16 bits of the largest number that k lanes' maxima reach
    const uint32_t o = order_of(mine);
    for (int bit = 31; bit >= 16; --bit) {
      const uint32_t t = bound | 1u << bit;
      if (__popcll(__ballot(o >= t)) >= k) bound = t;
    }
  }
  if (lane == 0) {
    s_red[wave][0] = wm;
    s_bound[wave] = bound;
  }
  __syncthreads();
  float m = s_red[0][0];
  uint32_t limit = s_bound[0];
#pragma unroll
  for (int w = 1; w < kWavesN; ++w) {
    m = fmaxf(m, s_red[w][0]);
    limit = max(limit, s_bound[w]);
  }
  const float ref = m == -INFINITY ? 0.0f : m;
  float S = 0.0f, T = 0.0f;
#pragma unroll
  for (int i = 0; i < kVec; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = v[i][j] - ref;
      const float e = fast_exp2(d * 1.4426950408889634f);
      S += e;
      T += d == -INFINITY ? 0.0f : e * d;
    }
  S = wave_sum(S);
  T = wave_sum(T);
  __syncthreads();  // s_red is read
  if (lane == 0) {
    s_red[wave][1] = S;
    s_red[wave][2] = T;
  }

  // ---- the part's best entries ----
  if (k > 0) {
    // Entries that may be among the best: at or above the limit.  A limit that -infinity reaches
    // says nothing: then every number, and the -infinity entries among the first kFirst, which are
    // enough of them if they are k (ids count upwards).
    const bool low = limit <= order_of(-INFINITY);
    const float lim = low ? -INFINITY : value_of(limit);
#pragma unroll
    for (int i = 0; i < kVec; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = (i * kThreads + tid) * 4 + j;
        const bool inf = low && at < min(n, kFirst) && v[i][j] == -INFINITY;
        if (low ? inf || v[i][j] > lim : v[i][j] >= lim) {
          const int slot = atomicAdd(&s_n, 1);
          if (slot < kCand) s_cand[slot] = key_of(v[i][j], base + at);
          if (inf) atomicAdd(&s_inf, 1);
        }
      }
    __syncthreads();
    const int want = min(k, n);
    const int found = s_n;
    if (found >= want && found <= kCand && (!low || s_inf >= k || n <= kFirst)) {
      for (int c = tid; c < found; c += kThreads) {
        const u64 key = s_cand[c];
        int rank = 0;
        for (int o = 0; o < found; ++o) rank += s_cand[o] > key ? 1 : 0;
        if (rank < k) s_best[rank] = key;
      }
      if (tid < k && tid >= found) s_best[tid] = 0;
    } else {
      // one after the other: each wave takes its own largest entry below its last one
      __syncthreads();
      u64 last = ~0ull;
      for (int r = 0; r < k; ++r) {
        u64 top = 0;
#pragma unroll
        for (int i = 0; i < kVec; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = (i * kThreads + tid) * 4 + j;
            const u64 key = at < n ? key_of(v[i][j], base + at) : 0;
            if (key < last) top = max64(top, key);
          }
        last = wave_max64(top);
        if (lane == 0) s_cand[wave * kTopMax + r] = last;
      }
      if (tid < kTopMax) s_best[tid] = 0;
      __syncthreads();
      if (lane < k) {
        const u64 key = s_cand[wave * kTopMax + lane];
        int rank = 0;
        for (int w = 0; w < kWavesN; ++w)
          for (int r = 0; r < k; ++r) rank += s_cand[w * kTopMax + r] > key ? 1 : 0;
        if (key != 0 && rank < k) s_best[rank] = key;
      }
    }
  }
  __syncthreads();
  const long slot = static_cast<long>(row) * a.parts + part;
  if (tid < k) store_dev(a.best + slot * k + tid, s_best[tid]);
  if (tid == 0) {
    S = T = 0.0f;
    for (int w = 0; w < kWavesN; ++w) {
      S += s_red[w][1];
      T += s_red[w][2];
    }
    store_dev(a.stats + 4 * slot, m);
    store_dev(a.stats + 4 * slot + 1, S);
    store_dev(a.stats + 4 * slot + 2, T);
  }

  // ---- the last workgroup of the row joins the parts ----
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    s_last = 1;
    if (a.parts > 1) {
      unsigned* ctr = a.arrive + static_cast<long>(row) * kCounterStride;
      s_last = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 ==
               static_cast<unsigned>(a.parts);
      if (s_last) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    s_n = 0;
  }
  __syncthreads();
  if (!s_last) return;
  const float* stats = a.stats + static_cast<long>(row) * a.parts * 4;
  RowSums sum;
  float M = -INFINITY;
  for (int p = lane; p < a.parts; p += 64) M = fmaxf(M, load_dev(stats + 4 * p));
  M = wave_max(M);
  sum.ref = M == -INFINITY ? 0.0f : M;
  sum.S = sum.T = 0.0f;
  for (int p = lane; p < a.parts; p += 64) {
    const float mp = load_dev(stats + 4 * p);
    const float Sp = load_dev(stats + 4 * p + 1), Tp = load_dev(stats + 4 * p + 2);
    const float d = mp == -INFINITY ? 0.0f : mp - sum.ref;  // a part of -infinity: S = T = 0
    const float c = fast_exp2(d * 1.4426950408889634f);
    sum.S = fmaf(c, Sp, sum.S);
    // weight 0: d may be as large as the type's lowest value makes it, and 0 * inf is NaN
    sum.T += c == 0.0f ? 0.0f : c * fmaf(d, Sp, Tp);
  }
  sum.S = wave_sum(sum.S);
  sum.T = wave_sum(sum.T);
  sum.logS = logf(sum.S);
  if (tid == 0) {
    if (a.logprob) {
      const int t = a.tokens[row];
      a.logprob[row] = t >= 0 && t < a.vocab ? sum.logp(x[t]) : __uint_as_float(0x7fc00000u);
    }
    if (a.entropy) a.entropy[row] = sum.S == 0.0f ? 0.0f : sum.logS - sum.T / sum.S;
  }
  if (k == 0) return;
  // the best of the parts' k best: those at or above the largest k-th of a part, by rank
  const u64* best = a.best + static_cast<long>(row) * a.parts * k;
  u64 floor_key = 0;
  for (int p = lane; p < a.parts; p += 64) floor_key = max64(floor_key, load_dev(best + p * k + k - 1));
  floor_key = wave_max64(floor_key);
  if (floor_key == 0) floor_key = 1;  // parts of fewer than k entries
  for (int c = tid; c < a.parts * k; c += kThreads) {
    const u64 key = load_dev(best + c);
    if (key >= floor_key) {
      const int at = atomicAdd(&s_n, 1);
      if (at < kCand) s_cand[at] = key;
    }
  }
  __syncthreads();
  const int found = s_n;
  int* ids = a.top_ids + static_cast<long>(row) * k;
  float* top = a.top_logprobs + static_cast<long>(row) * k;
  if (found <= kCand) {
    for (int c = tid; c < found; c += kThreads) {
      const u64 key = s_cand[c];
      int rank = 0;
      for (int o = 0; o < found; ++o) rank += s_cand[o] > key ? 1 : 0;
      if (rank < k) {
        ids[rank] = id_of(key);
        top[rank] = sum.logp(value_of(static_cast<uint32_t>(key >> 32)));
      }
    }
  } else if (wave == 0) {  // many parts whose best lie close together
    u64 last = ~0ull;
    for (int r = 0; r < k; ++r) {
      u64 t = 0;
      for (int c = lane; c < a.parts * k; c += 64) {
        const u64 key = load_dev(best + c);
        if (key < last) t = max64(t, key);
      }
      last = wave_max64(t);
      if (lane == 0) {
        ids[r] = id_of(last);
        top[r] = sum.logp(value_of(static_cast<uint32_t>(last >> 32)));
      }
    }
  }
}

// Rows per launch: counters and a workspace of some 32 MB.
constexpr size_t kSlabBytes = size_t{32} << 20;

int token_logprobs(LogprobArgs a, int rows, hipStream_t stream) {
  const long parts = (static_cast<long>(a.vocab) + kPart - 1) / kPart;
  a.parts = static_cast<int>(parts);
  a.part_len = static_cast<int>(((a.vocab + parts - 1) / parts + 3) / 4 * 4);
  a.parts = static_cast<int>((static_cast<long>(a.vocab) + a.part_len - 1) / a.part_len);
  const size_t per_row = static_cast<size_t>(a.parts) * (4 * sizeof(float) + a.top_k * sizeof(u64));
  const int slab = static_cast<int>(
      std::clamp<size_t>(kSlabBytes / per_row, 1, static_cast<size_t>(std::min(rows, kArriveCounters))));
  char* ws = static_cast<char*>(workspace_graph(stream, per_row * slab, kWsLogprobs));
  if (!ws) return ORATOR_ERR_HIP;
  a.stats = reinterpret_cast<float*>(ws);
  a.best = reinterpret_cast<u64*>(ws + static_cast<size_t>(slab) * a.parts * 4 * sizeof(float));
  if (a.parts > 1)
    if (int rc = zeroed_counters(stream, kWsLogprobsArrive, &a.arrive, true)) return rc;
  for (long r0 = 0; r0 < rows; r0 += slab) {
    const int n = static_cast<int>(std::min<long>(slab, rows - r0));
    LogprobArgs s = a;
    s.x += r0 * a.row_stride;
    if (s.tokens) s.tokens += r0;
    if (s.logprob) s.logprob += r0;
    if (s.entropy) s.entropy += r0;
    if (s.top_ids) {
      s.top_ids += r0 * a.top_k;
      s.top_logprobs += r0 * a.top_k;
    }
    hipLaunchKernelGGL(token_logprobs_kernel, dim3(static_cast<unsigned>(a.parts) * n),
                       dim3(kThreads), 0, stream, s);
    if (int rc = check_launch("token_logprobs_kernel")) return rc;
  }
  return ORATOR_OK;
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
    LogprobArgs a{};
    a.x = logits;
    a.row_stride = row_stride;
    a.tokens = tokens;
    a.vocab = vocab;
    a.top_k = top_k;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_k ? top_ids : nullptr;
    a.top_logprobs = top_logprobs;
    return token_logprobs(a, rows, static_cast<hipStream_t>(stream));
  });
}
