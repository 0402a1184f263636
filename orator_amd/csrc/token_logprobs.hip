// Log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
// With m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m):
//   lse = m + log S,  logprob = x_tok - lse,  entropy = log S - T / S.
// Entries of -infinity have weight 0 and add 0 to T.
//
// Memory-bound: the logits are read once.  A row is cut into parts, one workgroup each, and a part
// into chunks of up to 4096 entries that a workgroup holds in registers (16 a thread) while the next
// one is loaded.  Every thread keeps its own maximum and sums; nothing is exchanged between chunks.
// The last workgroup of a row to finish joins its parts.
//
// Best entries: a wave keeps a list in LDS of entries that may be among the k best of its own.  The
// k-th largest of the 64 lanes' running maxima is a bound that k entries reach, so entries below it
// are left out (1024 entries of a wave add some 24 at first, then ever fewer).  A chunk with too many
// (ties in masses) gives its k best one after the other instead; a full list is cut to its k best.  What
// the waves listed is ranked by counting, per part and then per row.  Entries of -infinity and NaN
// are never listed: a row with fewer than k others is searched for them at the end.
//
// Measured, 151936 entries: 257 rows with 20 alternatives 42 us (3.7 TB/s, vector instructions half of
// the time; 5 alternatives 37, none 33), one row with 5 9.8 us.
#include <float.h>

#include <algorithm>
#include <string>

#include "common.hpp"
#include "internal.hpp"

namespace orator_hip {
namespace {

typedef unsigned long long u64;

constexpr int kTopMax = 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256;
constexpr int kWavesN = kThreads / 64;
constexpr int kVec = 4;                           // float4 per thread and chunk
constexpr int kChunk = kThreads * kVec * 4;       // entries of a chunk, at most
constexpr int kList = 192;                        // a wave's list
constexpr int kFew = 6;                           // lanes with entries to list that need no new bound
constexpr int kMost = 96;                         // entries that one chunk may add to it
constexpr int kCand = 768;                        // candidates ranked at once
static_assert(kTopMax + kMost <= kList && kWavesN * kList <= kCand && kTopMax <= 64);

struct LogprobArgs {
  const float* x;
  long row_stride;
  const int* tokens;
  int vocab, top_k;
  float* logprob;
  float* entropy;
  int* top_ids;
  float* top_logprobs;
  int parts, chunks;  // chunks of a part (the row's last part may have fewer)
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

// v >= above(t) says v > t.
__device__ __forceinline__ float above(float t) { return value_of(order_of(t) + 1u); }

// Writes the keys of list[0, n) that are among its k largest (all of them, if fewer) to best[0, k),
// in order, 0 behind them; `threads` threads take part, this one is number t.  List and best apart.
__device__ __forceinline__ void rank_into(u64* best, const u64* list, int n, int k, int t, int threads) {
  for (int c = t; c < n; c += threads) {
    const u64 key = list[c];
    int rank = 0, o = 0;
    for (; o + 8 <= n; o += 8) {  // eight reads on the way at a time
      u64 other[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) other[i] = list[o + i];
#pragma unroll
      for (int i = 0; i < 8; ++i) rank += other[i] > key ? 1 : 0;
    }
    for (; o < n; ++o) rank += list[o] > key ? 1 : 0;
    if (rank < k) best[rank] = key;
  }
  if (t < k && t >= n) best[t] = 0;
}

typedef float Chunk[kVec][4];

// Entries c0 + (i * kThreads + tid) * 4 + j of a part's n, as loaded: a group of four that does not
// lie in the part holds its last four entries (parts of fewer than 4: none), which finish_chunk puts
// right once they are there.  No branch stands between the loads, and a chunk behind the part's end
// reads that one line.
__device__ __forceinline__ void load_chunk(Chunk& v, const float* x, int c0, int n, int tid) {
  if (n < 4) return;  // uniform
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const Vec4 r = load4(x + min(c0 + (i * kThreads + tid) * 4, n - 4));
#pragma unroll
    for (int j = 0; j < 4; ++j) v[i][j] = r.v[j];
  }
}
// Entries behind the part's end become -infinity.
__device__ __forceinline__ void finish_chunk(Chunk& v, const float* x, int c0, int n, int tid) {
  if (n - c0 >= kChunk) return;  // uniform
  if (n < 4) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = i == 0 && tid == 0 && j < n ? x[j] : -INFINITY;
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    if (c0 + (i + 1) * kThreads * 4 <= n) continue;  // uniform
    const int past = c0 + (i * kThreads + tid) * 4 - (n - 4);  // entries that the load came too early
    if (past > 0) {
      v[i][0] = past == 1 ? v[i][1] : past == 2 ? v[i][2] : past == 3 ? v[i][3] : -INFINITY;
      v[i][1] = past == 1 ? v[i][2] : past == 2 ? v[i][3] : -INFINITY;
      v[i][2] = past == 1 ? v[i][3] : -INFINITY;
      v[i][3] = -INFINITY;
    }
  }
}

// A thread's sums over its entries so far; T in units of log 2, as the exponents are.
struct Sums {
  float m = -INFINITY, S = 0.0f, T = 0.0f;

  // To a maximum of m2 >= m.  d may be as large as the type's lowest value makes it: a weight of 0
  // leaves nothing (0 * inf is NaN); S keeps a NaN.
  __device__ __forceinline__ void move(float m2) {
    if (m2 == -INFINITY) return;
    const float t = m == -INFINITY ? 0.0f : (m - m2) * kLog2e;
    const float c = fast_exp2(t);
    T = c == 0.0f ? 0.0f : c * fmaf(t, S, T);
    S *= c;
    m = m2;
  }
  __device__ __forceinline__ void take(float x, float ref) {
    const float t = (x - ref) * kLog2e;
    const float e = fast_exp2(t);
    S += e;
    T = fmaf(e, fmaxf(t, -FLT_MAX), T);  // a weight of 0 leaves 0; S keeps a NaN
  }
};

// A wave's list of entries that may be among its k best.
struct List {
  u64* at;              // kList in LDS
  float* bounds;        // the waves' `reach`, in LDS: each writes its own, all read the largest
  int wave = 0;
  int n = 0;            // uniform
  float thr = -FLT_MAX; // entries below are not listed (NaN: none is)
  float reach = -INFINITY;  // k listed entries reach this
  float lane_max = -INFINITY;

  __device__ __forceinline__ void add(bool in, u64 key) {
    const u64 mask = __ballot(in);
    if (mask == 0) return;
    const int slot = n + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
    if (in) at[slot] = key;
    n += __popcll(mask);
  }

  __device__ __forceinline__ void publish(float r) {
    reach = fmaxf(reach, r);
    __hip_atomic_store(bounds + wave, reach, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }

  // The list cut to its k best (it has at least k); later entries have to be above the last.
  __device__ __forceinline__ void cut(int k, int lane) {
    wave_lds_sync();
    constexpr int N = kList / 64;
    u64 mine[N];
    int rank[N] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) mine[i] = 64 * i + lane < n ? at[64 * i + lane] : 0;
    for (int o = 0; o < n; ++o) {
      const u64 key = at[o];
#pragma unroll
      for (int i = 0; i < N; ++i) rank[i] += key > mine[i] ? 1 : 0;
    }
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (64 * i + lane < n && rank[i] < k) at[rank[i]] = mine[i];
    wave_lds_sync();
    n = k;
    publish(value_of(static_cast<uint32_t>(at[k - 1] >> 32)));
    thr = fmaxf(thr, above(reach));
  }

  // The chunk's entries, their ids from id0 on, all higher than those listed.
  // m4: the maxima of the lane's groups of four; chunk_max: of all.
  __device__ __forceinline__ void take(const Chunk& v, const float (&m4)[kVec], float chunk_max,
                                       int id0, int k, int tid, int lane) {
    lane_max = fmaxf(lane_max, chunk_max);
    // k entries of the part reach any wave's bound: what is below is not among the part's best
    // (bounds only grow, so one that is read late costs entries, never loses one)
    float part = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWavesN; ++w)
      part = fmaxf(part, __hip_atomic_load(bounds + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
    thr = fmaxf(thr, part);
    const int lanes = __popcll(__ballot(chunk_max >= thr));
    if (lanes == 0) return;
    if (lanes > kFew) {
      // the upper 16 bits of the largest number that k lanes' maxima reach
      const uint32_t o = order_of(lane_max);
      uint32_t bound = 0;
#pragma unroll
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = bound | 1u << bit;
        if (__popcll(__ballot(o >= t)) >= k) bound = t;
      }
      if (bound > order_of(-INFINITY)) {
        const float b = value_of(bound);
        // k of the wave's entries so far reach b, and those that do are listed or in this chunk
        if (b > reach) publish(b);
        if (b > thr) thr = b;
      }
    }
    int count = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) count += 4 * __popcll(__ballot(m4[i] >= thr));
    if (count > kMost) {  // at most that many: count them
      count = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) count += __popcll(__ballot(v[i][j] >= thr));
      if (count > kMost) {
        best_of(v, id0, k, tid, lane);
        return;
      }
    }
    if (n + count > kList) cut(k, lane);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (__ballot(m4[i] >= thr) == 0) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        add(v[i][j] >= thr, key_of(v[i][j], id0 + (i * kThreads + tid) * 4 + j));
    }
  }

  // The k best of a chunk that has more than kMost to list, one after the other.
  __device__ __forceinline__ void best_of(const Chunk& v, int id0, int k, int tid, int lane) {
    if (n + k > kList) cut(k, lane);
    u64 last = ~0ull;
    for (int r = 0; r < k; ++r) {
      u64 top = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y = v[i][j];
          asm volatile("" : "+v"(y));  // keys formed in the loop: 32 held across it are 64 registers
          const u64 key = key_of(y, id0 + (i * kThreads + tid) * 4 + j);
          if (y >= thr && key < last) top = max64(top, key);
        }
      last = wave_max64(top);
      if (lane == 0) at[n + r] = last;
    }
    n += k;
    cut(k, lane);
  }
};

__global__ __launch_bounds__(kThreads, 5) void token_logprobs_kernel(LogprobArgs a) {
  __shared__ float s_sums[kWavesN][3];
  __shared__ float s_reach[kWavesN];
  __shared__ u64 s_list[kWavesN][kList];
  __shared__ u64 s_cand[kCand];
  __shared__ u64 s_best[kTopMax];
  __shared__ int s_len[kWavesN], s_n, s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = blockIdx.x % a.parts;
  const int row = blockIdx.x / a.parts;
  const float* x = a.x + row * a.row_stride;
  const int k = a.top_k;
  const long base = static_cast<long>(part) * a.chunks * kChunk;
  x += base;
  const int entries = static_cast<int>(min(static_cast<long>(a.chunks) * kChunk, a.vocab - base));
  Sums sum;
  List list;
  list.at = s_list[wave];
  list.bounds = s_reach;
  list.wave = wave;
  if (tid < kWavesN) s_reach[tid] = -INFINITY;
  Chunk nxt = {};
  load_chunk(nxt, x, 0, entries, tid);
  lds_barrier();
  for (long c = 0; c < entries; c += kChunk) {
    const int c0 = static_cast<int>(c);
    Chunk v;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = nxt[i][j];
    load_chunk(nxt, x, min(c0, 0x7fffffff - 2 * kChunk) + kChunk, entries, tid);
    finish_chunk(v, x, c0, entries, tid);
    float m4[kVec], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      m4[i] = fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3]));
      mx = fmaxf(mx, m4[i]);
    }
    if (mx > sum.m) sum.move(mx);
    const float ref = sum.m == -INFINITY ? 0.0f : sum.m;
#pragma unroll
    for (int i = 0; i < kVec; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum.take(v[i][j], ref);
    if (k > 0) list.take(v, m4, mx, static_cast<int>(base) + c0, k, tid, lane);
  }

  x -= base;

  // ---- the part's sums and best entries ----
  sum.move(wave_max(sum.m));
  sum.S = wave_sum(sum.S);
  sum.T = wave_sum(sum.T);
  if (lane == 0) {
    s_sums[wave][0] = sum.m, s_sums[wave][1] = sum.S, s_sums[wave][2] = sum.T;
    s_len[wave] = list.n;
  }
  if (tid == 0) s_n = 0;
  __syncthreads();
  if (k > 0) {
    float reach = s_reach[0];
#pragma unroll
    for (int w = 1; w < kWavesN; ++w) reach = fmaxf(reach, s_reach[w]);
    const uint32_t lim = order_of(reach);
    for (int w = 0; w < kWavesN; ++w)
      for (int c = tid; c < s_len[w]; c += kThreads) {
        const u64 key = s_list[w][c];
        if (static_cast<uint32_t>(key >> 32) >= lim) s_cand[atomicAdd(&s_n, 1)] = key;
      }
    __syncthreads();
    rank_into(s_best, s_cand, s_n, k, tid, kThreads);
  }
  __syncthreads();
  const long slot = static_cast<long>(row) * a.parts + part;
  if (tid < k) store_dev(a.best + slot * k + tid, s_best[tid]);
  if (tid == 0) {
    Sums p;
    for (int w = 0; w < kWavesN; ++w) {
      Sums q{s_sums[w][0], s_sums[w][1], s_sums[w][2]};
      const float M = fmaxf(p.m, q.m);
      p.move(M);
      q.move(M);
      p.S += q.S;
      p.T += q.T;
    }
    store_dev(a.stats + 4 * slot, p.m);
    store_dev(a.stats + 4 * slot + 1, p.S);
    store_dev(a.stats + 4 * slot + 2, p.T);
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
  const u64* best = a.best + static_cast<long>(row) * a.parts * k;
  const long keys = static_cast<long>(a.parts) * k;
  // everything that is read is on its way before any of it is waited for (parts up to 64, and
  // kHeld keys a thread; what there is beyond is read in the loops)
  constexpr int kHeld = 4;
  u64 held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    held[i] = tid + i * kThreads < keys ? load_dev(best + tid + i * kThreads) : 0;
  Sums mine;
  if (lane < a.parts) {
    mine.m = load_dev(stats + 4 * lane);
    mine.S = load_dev(stats + 4 * lane + 1);
    mine.T = load_dev(stats + 4 * lane + 2);
  }
  const int token = a.logprob ? a.tokens[row] : -1;
  const bool known = token >= 0 && token < a.vocab;
  const float picked = known ? x[token] : 0.0f;
  float M = mine.m;
  for (int p = 64 + lane; p < a.parts; p += 64) M = fmaxf(M, load_dev(stats + 4 * p));
  M = wave_max(M);
  mine.move(M);
  Sums all = mine;
  for (int p = 64 + lane; p < a.parts; p += 64) {
    Sums q;
    q.m = load_dev(stats + 4 * p);
    q.S = load_dev(stats + 4 * p + 1);
    q.T = load_dev(stats + 4 * p + 2);
    q.move(M);
    all.S += q.S;
    all.T += q.T;
  }
  RowSums sums;
  sums.ref = M == -INFINITY ? 0.0f : M;
  sums.S = wave_sum(all.S);
  sums.T = wave_sum(all.T);
  sums.logS = logf(sums.S);
  if (tid == 0) {
    if (a.logprob) a.logprob[row] = known ? sums.logp(picked) : __uint_as_float(0x7fc00000u);
    if (a.entropy)
      a.entropy[row] = sums.S == 0.0f ? 0.0f : sums.logS - sums.T * 0.69314718055994531f / sums.S;
  }
  if (k == 0) return;
  int* ids = a.top_ids + static_cast<long>(row) * k;
  float* top = a.top_logprobs + static_cast<long>(row) * k;
  // the best of the parts' k best: those at or above the largest k-th of a part, by rank
  u64 lowest = 1;  // 0 stands behind the entries of a part that has fewer than k
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if ((tid + i * kThreads) % k == k - 1) lowest = max64(lowest, held[i]);
  for (long c = tid + kHeld * kThreads; c < keys; c += kThreads)
    if (c % k == k - 1) lowest = max64(lowest, load_dev(best + c));
  lowest = wave_max64(lowest);
  if (lane == 0) s_list[0][wave] = lowest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWavesN; ++w) lowest = max64(lowest, s_list[0][w]);
  auto keep = [&](u64 key) {
    if (key < lowest) return;
    const int at = atomicAdd(&s_n, 1);
    if (at < kCand) s_cand[at] = key;
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i) keep(held[i]);
  for (long c = tid + kHeld * kThreads; c < keys; c += kThreads) keep(load_dev(best + c));
  __syncthreads();
  const int found = s_n;
  if (found <= kCand) {
    rank_into(s_best, s_cand, found, k, tid, kThreads);
    __syncthreads();
    if (tid < min(k, found)) {
      const u64 key = s_best[tid];
      ids[tid] = id_of(key);
      top[tid] = sums.logp(value_of(static_cast<uint32_t>(key >> 32)));
    }
  } else if (wave == 0) {  // many parts whose best lie close together
    u64 last = ~0ull;
    for (int r = 0; r < k; ++r) {
      u64 t = 0;
      for (long c = lane; c < static_cast<long>(a.parts) * k; c += 64) {
        const u64 key = load_dev(best + c);
        if (key < last) t = max64(t, key);
      }
      last = wave_max64(t);
      if (lane == 0) {
        ids[r] = id_of(last);
        top[r] = sums.logp(value_of(static_cast<uint32_t>(last >> 32)));
      }
    }
  }
  if (found >= k || wave != 0) return;
  // fewer than k numbers above -infinity: the first entries of -infinity, then the first NaN
  int r = found;
  for (int nan = 0; nan < 2 && r < k; ++nan)
    for (long c = 0; c < a.vocab && r < k; c += 64) {
      const float y = c + lane < a.vocab ? x[c + lane] : 0.0f;
      const bool in = nan ? y != y : y == -INFINITY;
      const u64 mask = __ballot(in);
      const int at = r + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
      if (in && at < k) {
        ids[at] = static_cast<int>(c + lane);
        top[at] = sums.logp(y);
      }
      r += __popcll(mask);
    }
}

// Rows per launch: counters and a workspace of some 32 MB.
constexpr size_t kSlabBytes = size_t{32} << 20;

int token_logprobs(LogprobArgs a, int rows, hipStream_t stream) {
  // Parts of a row: the fewest rounds of workgroups (five to a CU) times chunks each, where a
  // workgroup's start and end cost about as much as two chunks.
  const long slots = 5L * (device_cu_count() > 0 ? device_cu_count() : 256);
  const long chunks = (static_cast<long>(a.vocab) + kChunk - 1) / kChunk;
  long parts = 1, least = 0;
  for (long p = 1; p <= std::min(chunks, slots); ++p) {
    const long cost = (rows * p + slots - 1) / slots * ((chunks + p - 1) / p + 2);
    if (p == 1 || cost < least) least = cost, parts = p;
  }
  a.chunks = static_cast<int>((chunks + parts - 1) / parts);
  a.parts = static_cast<int>((chunks + a.chunks - 1) / a.chunks);
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
