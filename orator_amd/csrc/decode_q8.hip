// Decode attention over the 8-bit KV cache on int8 matrix instructions, gfx950.
//
// One query row per q head attends S keys; HBM-bound (2 (Dh + 4) bytes per key and kv head).  The
// codes go from memory into the matrix cores as they are: no conversion, no transpose, no LDS.
//
//  * q as four int8 digits.  Per head, X = q * 2^(30 - e) with |q| < 2^e: an integer of 31 bits,
//    exact for q within 2^-7 of the largest, to 2^-31 of the largest below.  X = sum_k a_k 256^k
//    with digits a_k in [-128, 127] (the bytes of (X + 0x808080) ^ 0x808080), so q . codes =
//    2^(e - 30) sum_k 256^k (a_k . codes), each product an exact int32 (|a . codes| <= 2^21).
//  * QK: mfma_i32_16x16x64_i8, A = 16 keys' codes, B = 16 columns (head r, digit t): 4 heads at a
//    time.  Lane (r, t) of a quad gets 4 keys' digit sums; the four digits lie in the quad's lanes,
//    which add them while each keeps one key of four (reduce-scatter by DPP).
//  * softmax on 4 keys per lane and 64-key step: running maximum and sum, fp32.
//  * PV: the weights w_j = p_j vs_j (the value's scale) become digits in the same way, relative to
//    the step's largest; a quad exchanges them so that lane (r, t) holds digit t of 16 keys, the A
//    operand.  B = the V codes, [dim][16 keys] per block: the lane's 16 bytes as they lie in
//    memory.  The four digit rows of a head come out in one lane, which adds them to its fp32 sums.
//    Key (t, i) of a step's tile t is 16 g + 4 t + i for lane group g, so that A and B agree.
//  So one 64-key step of one wave is 8 + 8 MFMAs of 16 cycles per 4 heads (Dh 128) and some 490 VALU
//  instructions (counted over whole calls, with each wave's start and end), against 16.5 KB from HBM.
//  * one workgroup = (a range of one stream's keys, kv head), 4 waves that take 64-key steps in
//    turn; the next step's codes are loaded while the current one is worked on.  The streams share
//    the workgroups of a kv head by their lengths, which every workgroup reads at entry (two
//    workgroups per CU; streams of 2049 to 4097 keys each cut by the capacity instead left a quarter
//    of them idle).  A stream's ranges are joined by the last of its workgroups to finish.  Batches
//    of more streams than that take a workgroup per (stream, kv head).
//  Measured, 16 q / 8 kv heads of 128: 16 streams of 2049 to 4097 keys 24.4 us a call (106 MB, 4.35
//  TB/s; B = 64 of 4096 keys 98 us, 5.65 TB/s, where a chain of ~6 us weighs less), one stream of
//  1301 keys 8.0 us, of 16384 keys 16.8 us.
#include <algorithm>
#include <string>

#include "kv_q8.hpp"

namespace orator_hip {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kStep = 64;  // keys per wave step

struct DecodeQ8Args {
  KeysProblem p;
  Q8Map map;
  int groups;        // workgroups of a kv head and chunk, shared by the streams; 0: one per stream
  int chunks;        // chunks of 4 NG q heads per kv head
  float scale_log2e;
  float* part_o;     // [Hkv * chunks][groups][4 NG][Dh]
  float* part_ml;    // [Hkv * chunks][groups][4 NG][2]
  unsigned* arrive;  // [B * Hkv * chunks], kCounterStride apart
};
constexpr int kMaxGroups = 256;

// The four digits of x (|x| <= 2^30), the top one in byte 3.
__device__ __forceinline__ int digits_of(int x) { return (x + 0x808080) ^ 0x808080; }

// Byte (3 - digit) of four words as one word: sel = 0x0004 * 0x0100.. built by byte_sel.
__device__ __forceinline__ uint32_t byte_sel(int byte) { return byte | (4 + byte) << 8; }
__device__ __forceinline__ uint32_t gather_bytes(uint32_t z0, uint32_t z1, uint32_t z2, uint32_t z3,
                                                 uint32_t sel) {
  const uint32_t lo = __builtin_amdgcn_perm(z1, z0, sel);
  const uint32_t hi = __builtin_amdgcn_perm(z3, z2, sel);
  return (lo & 0xffffu) | hi << 16;
}

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xf, 0xf, false));
}

// Over the lanes of one (l & 15) >> 2: the quad, then the four lane groups.
__device__ __forceinline__ float row_max(float v) {
  v = quad_max(v);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float v) {
  v = quad_sum(v);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ i32x4_t mfma_i8(uint4 a, uint4 b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a),
                                               __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}

// Partials are read by another workgroup of the same launch: agent-scope accesses, which the
// XCDs' separate L2s agree on.
__device__ __forceinline__ void store_dev(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_dev(const float* p) {
  return __hip_atomic_load(const_cast<float*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int DH>
struct Q8Step {
  uint4 k[4][DH / 64];
  uint4 v[DH / 16];
  float ks[4], vs[4];
  bool mapped;  // this lane group's block
};

// Block numbers of step `s` (of 64 keys): for the K rows this lane loads and for its V and scales;
// blocks past the stream's last key take that key's (their keys are masked).
struct StepBlocks {
  long k, v;
};
__device__ __forceinline__ StepBlocks step_blocks(const Q8Map& m, int b, int h, int s, int last_blk,
                                                  int lane) {
  StepBlocks r;
  r.k = m.block(b, min(4 * s + ((lane & 15) >> 2), last_blk), h);
  r.v = m.block(b, min(4 * s + (lane >> 4), last_blk), h);
  return r;
}

template <int DH>
__device__ __forceinline__ void load_step(Q8Step<DH>& st, const KeysProblem& p, StepBlocks blk,
                                          int lane) {
  st.mapped = blk.v >= 0;
  // an unmapped block reads block 0 (a pool has one); its keys are masked
  const int8_t* k = p.kq + (max(blk.k, 0L) * kQ8Block + (lane & 3)) * DH + 16 * (lane >> 4);
  const long bv = max(blk.v, 0L);
  const int8_t* v = p.vq + (bv * DH + (lane & 15)) * kQ8Block;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int c = 0; c < DH / 64; ++c) st.k[t][c] = *reinterpret_cast<const uint4*>(k + 4 * t * DH + 64 * c);
#pragma unroll
  for (int n = 0; n < DH / 16; ++n) st.v[n] = load_nt(v + 256 * n);
  const float* ks = p.ks + bv * kQ8Block + (lane & 3);
  const float* vs = p.vs + bv * kQ8Block + (lane & 3);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    st.ks[t] = ks[4 * t];
    st.vs[t] = vs[4 * t];
  }
}

template <int DH, int NG>
struct RowState {
  uint4 q[NG][DH / 64];  // digits: column (head (l & 15) >> 2, digit l & 3), dims 16 (l >> 4) ..
  float f[NG];           // 256^(3 - digit) 2^(e - 30) scale log2(e): a digit sum's part of a score
  float m[NG], l[NG];    // of head (l & 15) >> 2; l is this lane's share
  float acc[NG][DH / 16];  // head l >> 4, dims 16 n + (l & 15)
};

template <int DH, int NG>
__device__ __forceinline__ void load_q(RowState<DH, NG>& st, const float* q, int heads, float scale,
                                       int lane) {
  const int digit = lane & 3;
  const uint32_t sel = byte_sel(3 - digit);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const int r = 4 * g + ((lane & 15) >> 2);
    const float* row = q + static_cast<long>(min(r, heads - 1)) * DH + 16 * (lane >> 4);
    float x[DH / 4];
    uint32_t amax = 0;
#pragma unroll
    for (int c = 0; c < DH / 64; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[16 * c + i] = row[64 * c + i];
        amax = max(amax, __float_as_uint(x[16 * c + i]) & 0x7fffffffu);
      }
    amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 16)));
    amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 32)));
    const int e = __builtin_amdgcn_frexp_expf(__uint_as_float(amax));  // |x| < 2^e
#pragma unroll
    for (int c = 0; c < DH / 64; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          z[j] = digits_of(static_cast<int>(__builtin_rintf(ldexpf(x[16 * c + 4 * i + j], 30 - e))));
        w[i] = gather_bytes(z[0], z[1], z[2], z[3], sel);
      }
      st.q[g][c] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // a head that is not finite has NaN scores
    st.f[g] = amax >= 0x7f800000u ? __uint_as_float(0x7fc00000u)
                                  : ldexpf(scale, e - 30 + 8 * (3 - digit));
    st.m[g] = -INFINITY;
    st.l[g] = 0.0f;
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) st.acc[g][n] = 0.0f;
  }
}

// One step: keys 64 s + 16 (l >> 4) + 4 t + (l & 3) of this lane, those before S attended.
template <int DH, int NG>
__device__ __forceinline__ void step(RowState<DH, NG>& st, const Q8Step<DH>& kv, int s, int S,
                                     int lane) {
  const bool odd = lane & 1, high = lane & 2;
  const uint32_t sel = byte_sel(3 - (lane & 3));
  const int key0 = kStep * s + 16 * (lane >> 4) + (lane & 3);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float sc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      i32x4_t d = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < DH / 64; ++c) d = mfma_i8(kv.k[t][c], st.q[g][c], d);
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(d[i]) * st.f[g];
      // the quad's four digit sums of each key, key i left in lane i of the quad
      const float y0 = (odd ? x[1] : x[0]) + dpp<0xB1>(odd ? x[0] : x[1]);
      const float y1 = (odd ? x[3] : x[2]) + dpp<0xB1>(odd ? x[2] : x[3]);
      const float z = (high ? y1 : y0) + dpp<0x4E>(high ? y0 : y1);
      const int key = key0 + 4 * t;
      const bool in = kv.mapped && key < S;
      sc[t] = in ? z * kv.ks[t] : -INFINITY;
    }
    const float mn = fmaxf(
        st.m[g], row_max(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]))));
    const float ref = mn == -INFINITY ? 0.0f : mn;  // no key yet
    const float corr = fast_exp2(st.m[g] - ref);
    st.m[g] = mn;
    float w[4], l = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int key = key0 + 4 * t;
      const bool in = kv.mapped && key < S;
      const float p = fast_exp2(sc[t] - ref);
      w[t] = in ? p * kv.vs[t] : 0.0f;
      // 0 w: a value's scale that is not finite has to show, and digits cannot hold it
      l += fmaf(w[t], 0.0f, p);
    }
    st.l[g] = fmaf(st.l[g], corr, l);
    const float wm = row_max(fmaxf(fmaxf(fabsf(w[0]), fabsf(w[1])), fmaxf(fabsf(w[2]), fabsf(w[3]))));
    const int e = __builtin_amdgcn_frexp_expf(wm);
    uint32_t a[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t z = digits_of(static_cast<int>(__builtin_rintf(ldexpf(w[t], 30 - e))));
      a[t] = gather_bytes(dpp_u<0x00>(z), dpp_u<0x55>(z), dpp_u<0xAA>(z), dpp_u<0xFF>(z), sel);
    }
    const uint4 wd = make_uint4(a[0], a[1], a[2], a[3]);
    // the sums are held by lanes of head l >> 4
    const int from = 4 * (lane >> 4);
    const float c = __shfl(corr, from);
    const float top = __shfl(ldexpf(1.0f, e - 30 + 24), from);
#pragma unroll
    for (int n = 0; n < DH / 16; ++n) {
      i32x4_t d = {0, 0, 0, 0};
      d = mfma_i8(wd, kv.v[n], d);
      float o = static_cast<float>(d[3]);
      o = fmaf(o, 1.0f / 256.0f, static_cast<float>(d[2]));
      o = fmaf(o, 1.0f / 256.0f, static_cast<float>(d[1]));
      o = fmaf(o, 1.0f / 256.0f, static_cast<float>(d[0]));
      st.acc[g][n] = fmaf(o, top, st.acc[g][n] * c);
    }
  }
}

// Keys that stream b attends.
__device__ __forceinline__ int keys_of(const DecodeQ8Args& a, int b) {
  const int pos = a.p.pos[b];
  return pos < 0 ? 0 : min(pos, a.map.capacity - 1) + 1;
}

// Inclusive sum over the lanes.
__device__ __forceinline__ int scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// What a workgroup does: range `part` of `parts` of stream b's S keys; b < 0: nothing.
struct Share {
  int b, S, part, parts;
};
// Workgroup w of `groups` for up to 64 streams (at most `groups`): stream i gets ceil(steps_i / per)
// of them, with the smallest per (in rounds of kWaves steps) that `groups` suffice for; each stream
// at least one.  The same in every wave.
__device__ __forceinline__ Share share_of(const DecodeQ8Args& a, int w, int lane) {
  const int S = lane < a.p.B ? keys_of(a, lane) : 0;
  const int rounds = lane < a.p.B ? max((S + kStep * kWaves - 1) / (kStep * kWaves), 1) : 0;
  const int total = __builtin_amdgcn_readlane(scan(rounds), 63);
  int per = (total + a.groups - 1) / a.groups, n, end;
  for (;; per += 1 + per / 16) {
    n = (rounds + per - 1) / per;
    end = scan(n);
    if (__builtin_amdgcn_readlane(end, 63) <= a.groups) break;  // at the latest at the longest's rounds
  }
  const uint64_t mask = __ballot(end > w);
  if (mask == 0) return {-1, 0, 0, 0};
  const int b = __builtin_ctzll(mask);
  const int parts = __builtin_amdgcn_readlane(n, b);
  return {b, __builtin_amdgcn_readlane(S, b), w - (__builtin_amdgcn_readlane(end, b) - parts), parts};
}

template <int DH, int NG>
__global__ __launch_bounds__(64 * kWaves, 2) void decode_q8_kernel(DecodeQ8Args a) {
  constexpr int R = 4 * NG;  // heads of a workgroup
  __shared__ float s_m[kWaves][R], s_l[kWaves][R];
  __shared__ float s_o[kWaves][R][DH];
  static_assert(R * kMaxGroups <= kWaves * R * DH, "the joining weights take the outputs' place");
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.y / a.chunks, chunk = blockIdx.y % a.chunks;
  const int G = a.p.Hq / a.p.Hkv;
  const int heads = min(G - chunk * R, R);
  Share sh;
  if (a.groups) {
    sh = share_of(a, blockIdx.x, lane);
    if (sh.b < 0) return;
  } else {
    sh = {static_cast<int>(blockIdx.z), keys_of(a, blockIdx.z), 0, 1};
  }
  const int b = sh.b, S = sh.S, part = sh.part, parts = sh.parts;
  const long row0 = static_cast<long>(b) * a.p.Hq + h * G + chunk * R;  // first (stream, q head)
  if (S == 0) {
    for (int i = tid; i < heads * DH; i += 64 * kWaves) a.p.out[row0 * DH + i] = 0.0f;
    return;
  }
  const int last_blk = (S - 1) >> 4;
  const int steps = (S + kStep - 1) / kStep, per = (steps + parts - 1) / parts;
  const int s_end = min((part + 1) * per, steps);
  int s = part * per + wave;
  RowState<DH, NG> st;
  Q8Step<DH> cur, nxt;
  StepBlocks blk{};
  if (s < s_end) {
    blk = step_blocks(a.map, b, h, s, last_blk, lane);
    load_step(cur, a.p, blk, lane);
    if (s + kWaves < s_end) blk = step_blocks(a.map, b, h, s + kWaves, last_blk, lane);
  }
  load_q<DH, NG>(st, a.p.q + row0 * DH, heads, a.scale_log2e, lane);
  while (s < s_end) {
    if (s + kWaves < s_end) {
      load_step(nxt, a.p, blk, lane);
      if (s + 2 * kWaves < s_end) blk = step_blocks(a.map, b, h, s + 2 * kWaves, last_blk, lane);
    }
    step<DH, NG>(st, cur, s, S, lane);
    s += kWaves;
    if (s >= s_end) break;
    if (s + kWaves < s_end) {
      load_step(cur, a.p, blk, lane);
      if (s + 2 * kWaves < s_end) blk = step_blocks(a.map, b, h, s + 2 * kWaves, last_blk, lane);
    }
    step<DH, NG>(st, nxt, s, S, lane);
    s += kWaves;
  }
  // ---- the waves' states joined in LDS ----
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float l = row_sum(st.l[g]);
    if (lane < 16 && (lane & 3) == 0) {
      s_m[wave][4 * g + (lane >> 2)] = st.m[g];
      s_l[wave][4 * g + (lane >> 2)] = l;
    }
#pragma unroll
    for (int n = 0; n < DH / 16; ++n)
      s_o[wave][4 * g + (lane >> 4)][16 * n + (lane & 15)] = st.acc[g][n];
  }
  __syncthreads();
  for (int i = tid; i < heads * DH; i += 64 * kWaves) {
    const int r = i / DH, d = i % DH;
    float M = -INFINITY, L = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_m[w][r]);
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float c = fast_exp2(s_m[w][r] - ref);
      L = fmaf(c, s_l[w][r], L);
      o = fmaf(c, s_o[w][r][d], o);
    }
    if (parts == 1) {
      a.p.out[row0 * DH + i] = L == 0.0f ? 0.0f : o / L;
    } else {
      const long at = (static_cast<long>(blockIdx.y) * a.groups + blockIdx.x) * R + r;
      store_dev(a.part_o + at * DH + d, o);
      if (d == 0) {
        store_dev(a.part_ml + 2 * at, M);
        store_dev(a.part_ml + 2 * at + 1, L);
      }
    }
  }
  if (parts == 1) return;
  // ---- the last workgroup of (stream, kv head, chunk) joins the ranges ----
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    unsigned* ctr = a.arrive + ((static_cast<long>(b) * a.p.Hkv + h) * a.chunks + chunk) * kCounterStride;
    const unsigned n = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = n + 1 == static_cast<unsigned>(parts);
    if (s_last) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  // a head's weights, divided by its sum: one wave a head, a range a lane
  float* weight = &s_o[0][0][0];  // [R][kMaxGroups]
  const long first = static_cast<long>(blockIdx.y) * a.groups + blockIdx.x - part;  // the stream's first
  for (int r = wave; r < heads; r += kWaves) {
    constexpr int N = kMaxGroups / 64;
    float m[N], l[N], M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = 64 * i + lane;
      const long at = ((first + min(j, parts - 1)) * R + r) * 2;
      m[i] = j < parts ? load_dev(a.part_ml + at) : -INFINITY;
      l[i] = j < parts ? load_dev(a.part_ml + at + 1) : 0.0f;
      M = fmaxf(M, m[i]);
    }
    M = wave_max(M);
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int i = 0; i < N; ++i) L = fmaf(fast_exp2(m[i] - ref), l[i], L);
    L = wave_sum(L);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (64 * i + lane < parts) weight[r * kMaxGroups + 64 * i + lane] = fast_exp2(m[i] - ref) * inv;
  }
  __syncthreads();
  for (int i = tid; i < heads * DH; i += 64 * kWaves) {
    const int r = i / DH;
    const float* from = a.part_o + (first * R + r) * DH + i % DH;
    constexpr int kBatch = 8;
    float o = 0.0f;
    for (int j0 = 0; j0 < parts; j0 += kBatch) {  // a batch of loads on the way at a time
      float x[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        x[j] = load_dev(from + static_cast<long>(min(j0 + j, parts - 1)) * R * DH);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (j0 + j < parts) o = fmaf(weight[r * kMaxGroups + j0 + j], x[j], o);
    }
    a.p.out[row0 * DH + i] = o;
  }
}

template <int DH, int NG>
int launch(const DecodeQ8Args& a, hipStream_t stream) {
  const dim3 grid(a.groups ? a.groups : 1, a.p.Hkv * a.chunks, a.groups ? 1 : a.p.B);
  hipLaunchKernelGGL((decode_q8_kernel<DH, NG>), grid, dim3(64 * kWaves), 0, stream, a);
  return check_launch("decode_q8_kernel");
}

}  // namespace

int launch_decode_q8(const KeysProblem& p, const Q8Map& map, hipStream_t stream) {
  const int G = p.Hq / p.Hkv;
  const int ng = G <= 4 ? 1 : G <= 8 ? 2 : 4;
  DecodeQ8Args a{};
  a.p = p;
  a.map = map;
  a.chunks = (G + 4 * ng - 1) / (4 * ng);
  a.scale_log2e = p.scale * 1.4426950408889634f;
  const long heads = static_cast<long>(p.Hkv) * a.chunks;
  if (heads > 65535) return fail(ORATOR_ERR_UNSUPPORTED, "gqa_decode_q8: too many heads");
  const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
  // no more than the streams can use: a round of steps each
  const long rounds = (static_cast<long>(map.capacity) + kStep * kWaves - 1) / (kStep * kWaves);
  const long groups = std::min(std::min<long>(2 * cus / heads, kMaxGroups), p.B * rounds);
  if (p.B <= 64 && p.B <= groups && p.B * heads <= kArriveCounters) {
    a.groups = static_cast<int>(groups);
    const size_t rows = static_cast<size_t>(heads) * groups * 4 * ng;
    char* ws = static_cast<char*>(workspace_graph(stream, rows * (p.Dh + 2) * sizeof(float), kWsKeys));
    if (!ws) return ORATOR_ERR_HIP;
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = a.part_o + rows * p.Dh;
    if (int rc = zeroed_counters(stream, kWsKeysArrive, &a.arrive, true)) return rc;
  }
  if (p.Dh == 128)
    return ng == 1 ? launch<128, 1>(a, stream) : ng == 2 ? launch<128, 2>(a, stream)
                                                         : launch<128, 4>(a, stream);
  return ng == 1 ? launch<64, 1>(a, stream) : ng == 2 ? launch<64, 2>(a, stream)
                                                      : launch<64, 4>(a, stream);
}

}  // namespace orator_hip
