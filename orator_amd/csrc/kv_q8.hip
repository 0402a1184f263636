// The KV cache in 8 bits: rows quantised as they are written, and read back.
//
// A row x of Dh values is held as scale = max|x| * fl(1 / 127) and codes = the integers nearest to
// x / scale.  The codes are exactly those of the real quotient: c = rint(x * (1 / scale)) is off
// by one at most, next to a border; the remainder r = x - c * scale is exact there (both terms are
// multiples of scale's last place over 2, and |r| is at most about scale / 2, so fma rounds
// nothing off), and 2 |r| against scale says on which side of the border x lies.
#include "kv_q8.hpp"

#include <string>

namespace orator_hip {
namespace {

struct WriteArgs {
  const float* k;
  const float* v;
  long kv_stride;
  int8_t* kq;
  float* ks;
  int8_t* vq;
  float* vs;
  Q8Map map;
  const int* pos0;
  int B, Tq, Dh;
};

// Code of x, in the low byte, for a scale with inv = 1 / scale; inv = 0 (a scale of 0 or NaN): any.
// |x / scale| is below 127.5 (scale is max|x| / 127 to two roundings), so no code needs clamping.
__device__ __forceinline__ uint32_t q8_code(float x, float scale, float inv) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: an integer added to it stands in its low bits
  const float y = fmaf(x, inv, kMagic);
  const float r = fmaf(kMagic - y, scale, x);
  const float r2 = fabsf(r + r);
  const uint32_t bits = __float_as_uint(y);
  // 1 towards r where x lies past the border, or on it with an odd code; no branches
  const uint32_t odd = bits << 31;
  const float edge = __uint_as_float(__float_as_uint(r2) | odd);  // negative for an odd code
  const uint32_t step = static_cast<uint32_t>(__float_as_int(r) >> 31) | 1u;
  uint32_t add = edge == -scale ? step : 0u;
  add = r2 > scale ? step : add;
  return bits + add;
}

// Scale of a row whose largest magnitude has the bits `amax` (as an integer: an infinity and a NaN
// are above every number): 0 where it would be subnormal, NaN for a row that is not finite.
__device__ __forceinline__ float q8_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const float s = __uint_as_float(amax) * (1.0f / 127.0f);
  return s >= 1.17549435e-38f ? s : 0.0f;
}

// About 1 / scale (1 ulp: q8_code mends what that does to a code); 0 for a scale of 0 or NaN.
__device__ __forceinline__ float q8_inverse(float scale) {
  return scale > 0.0f ? __builtin_amdgcn_rcpf(scale) : 0.0f;
}

__device__ __forceinline__ unsigned wave_item() {
  return __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
}

// Largest over the lanes of a group of `N` (16, 32 or 64).
template <int N>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  auto step = [&](uint32_t o) { v = max(v, o); };
  step(__builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false));   // xor 1
  step(__builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false));   // xor 2
  step(__builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));  // the other half of 8
  step(__builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, false));  // the other half of 16
  if constexpr (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  if constexpr (N >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  return v;
}

template <int N>
struct Floats {
  float v[N];
};
// N floats at any 4-byte address.
template <int N>
__device__ __forceinline__ Floats<N> load_floats(const float* p) {
  typedef float vec __attribute__((ext_vector_type(N), aligned(4)));
  Floats<N> f;
  if constexpr (N == 1) {
    f.v[0] = *p;
  } else {
    const vec x = __builtin_nontemporal_load(reinterpret_cast<const vec*>(p));
#pragma unroll
    for (int i = 0; i < N; ++i) f.v[i] = x[i];
  }
  return f;
}

// Where a wave of the block kernels works: one block of 16 positions of one stream and head, K or V.
struct BlockItem {
  int b, h, t0;     // rows t0 + 0 .. 15 of the call lie in the block
  int r0, r1;       // those in [r0, r1) exist
  long block;       // its number, -1: nothing to do
  bool is_v;
};
// Item `wave` (uniform) of stream blockIdx.y: block, head, K or V, the last the fastest.
__device__ __forceinline__ BlockItem block_item(const Q8Map& map, const int* pos0, unsigned item,
                                                int Tq, int blocks) {
  BlockItem w{};
  w.block = -1;
  w.is_v = item & 1u;
  item >>= 1;
  const unsigned i = item / static_cast<unsigned>(map.Hkv);
  w.h = static_cast<int>(item - i * map.Hkv);
  if (i >= static_cast<unsigned>(blocks)) return w;
  w.b = blockIdx.y;
  const long p0 = pos0[w.b];
  const long blk = (p0 >> 4) + i;  // rounds down for positions before 0
  w.t0 = static_cast<int>(blk * kQ8Block - p0);
  w.r0 = max(0, -w.t0);
  w.r1 = static_cast<int>(min(static_cast<long>(kQ8Block), static_cast<long>(Tq) - w.t0));
  if (blk >= 0 && blk < map.capacity / kQ8Block && w.r0 < w.r1)
    w.block = map.block(w.b, static_cast<int>(blk), w.h);
  return w;
}
// Prompts, Dh 64 and 128: one wave per block of 16 positions, head, and K or V.  Bound by VALU work
// beside the memory (5 Dh + 4 bytes per row and head, K and V apart): 2048 rows of 8 heads of 128 in 9.7
// us, 2.2 TB/s, with two waves per SIMD.  K: lanes across a row, 4 dims each, codes stored a
// dword a lane.  V: a lane has Dh / 64 dims of all 16 rows, so that its codes are 16 whole bytes of
// the transposed block each; a block that the call covers in part is stored byte by byte.
template <int DH>
__global__ __launch_bounds__(256) void kv_write_q8_block_kernel(WriteArgs a, int blocks) {
  const int lane = threadIdx.x & 63;
  const BlockItem w = block_item(a.map, a.pos0, wave_item(), a.Tq, blocks);
  if (w.block < 0) return;
  const float* src = (w.is_v ? a.v : a.k) + (static_cast<long>(w.b) * a.Tq + w.t0) * a.kv_stride +
                     static_cast<long>(w.h) * DH;
  float my_scale = 0.0f;  // of row `lane`
  if (w.is_v) {
    constexpr int E = DH / 64;
    Floats<E> x[kQ8Block];
#pragma unroll
    for (int r = 0; r < kQ8Block; ++r)
      // rows outside the call read its first or last one in the block
      x[r] = load_floats<E>(src + min(max(r, w.r0), w.r1 - 1) * a.kv_stride + E * lane);
    uint32_t out[E][4] = {};
#pragma unroll
    for (int r = 0; r < kQ8Block; ++r) {
      uint32_t amax = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) amax = max(amax, __float_as_uint(x[r].v[e]) & 0x7fffffffu);
      const float scale = q8_scale(group_max<64>(amax));
      const float inv = q8_inverse(scale);
      my_scale = lane == r ? scale : my_scale;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t c = q8_code(x[r].v[e], scale, inv) & 255u;
        out[e][r >> 2] |= (inv > 0.0f ? c : 0u) << (8 * (r & 3));
      }
    }
    int8_t* dst = a.vq + (w.block * DH + E * lane) * kQ8Block;
    if (w.r0 == 0 && w.r1 == kQ8Block) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        *reinterpret_cast<uint4*>(dst + e * kQ8Block) =
            make_uint4(out[e][0], out[e][1], out[e][2], out[e][3]);
    } else {
#pragma unroll
      for (int r = 0; r < kQ8Block; ++r)
        if (r >= w.r0 && r < w.r1) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            dst[e * kQ8Block + r] = static_cast<int8_t>(out[e][r >> 2] >> (8 * (r & 3)));
        }
    }
  } else {
    constexpr int LPR = DH / 4, RPI = 64 / LPR, N = kQ8Block / RPI;  // lanes per row, rows per load
    const int at = lane / LPR, d = 4 * (lane % LPR);
    Floats<4> x[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      x[i] = load_floats<4>(src + min(max(RPI * i + at, w.r0), w.r1 - 1) * a.kv_stride + d);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = RPI * i + at;
      uint32_t amax = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) amax = max(amax, __float_as_uint(x[i].v[e]) & 0x7fffffffu);
      const float scale = q8_scale(group_max<LPR>(amax));
      const float inv = q8_inverse(scale);
      uint32_t code = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) code |= (q8_code(x[i].v[e], scale, inv) & 255u) << (8 * e);
      code = inv > 0.0f ? code : 0u;
      if (r >= w.r0 && r < w.r1) {
        *reinterpret_cast<uint32_t*>(a.kq + (w.block * kQ8Block + r) * DH + d) = code;
        if (d == 0) a.ks[w.block * kQ8Block + r] = scale;
      }
    }
  }
  if (w.is_v && lane >= w.r0 && lane < w.r1) a.vs[w.block * kQ8Block + lane] = my_scale;
}

// Few rows, and any Dh: one wave per (token, head, K or V), lane l holds dims 4 l .. 4 l + 3.  A chain
// of three memory round trips (position, page, row): 16 streams' single rows of 8 heads in 3.3 us.
__global__ __launch_bounds__(256) void kv_write_q8_kernel(WriteArgs a) {
  const int lane = threadIdx.x & 63;
  const unsigned item = wave_item(), Hkv = a.map.Hkv;
  const bool is_v = item & 1u;
  const unsigned t = (item >> 1) / Hkv;
  const int h = static_cast<int>((item >> 1) - t * Hkv), b = blockIdx.y;
  if (t >= static_cast<unsigned>(a.Tq)) return;
  const long bt = static_cast<long>(b) * a.Tq + t;
  const long p = static_cast<long>(a.pos0[b]) + t;
  if (p < 0 || p >= a.map.capacity) return;
  const int blk = static_cast<int>(p >> 4), at = static_cast<int>(p & 15);
  const long block = a.map.block(b, blk, h);
  if (block < 0) return;
  const float* src = (is_v ? a.v : a.k) + bt * a.kv_stride + static_cast<long>(h) * a.Dh;
  const int d = 4 * lane;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (d < a.Dh)
    for (int i = 0; i < 4; ++i) x[i] = src[d + i];
  uint32_t amax = 0;
  for (int i = 0; i < 4; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
  for (int m = 1; m < 64; m <<= 1) amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), m)));
  const float scale = q8_scale(amax);
  const float inv = q8_inverse(scale);
  if (d < a.Dh) {
    uint32_t c[4];
    for (int i = 0; i < 4; ++i) c[i] = inv > 0.0f ? q8_code(x[i], scale, inv) & 255u : 0u;
    if (is_v) {
      int8_t* dst = a.vq + (block * a.Dh + d) * kQ8Block + at;
      for (int i = 0; i < 4; ++i) dst[i * kQ8Block] = static_cast<int8_t>(c[i]);
    } else {
      const uint32_t w = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
      *reinterpret_cast<uint32_t*>(a.kq + (block * kQ8Block + at) * a.Dh + d) = w;
    }
  }
  if (lane == 0) (is_v ? a.vs : a.ks)[block * kQ8Block + at] = scale;
}

struct ReadArgs {
  const int8_t* kq;
  const float* ks;
  const int8_t* vq;
  const float* vs;
  void* k;
  void* v;
  Q8Map map;
  const int* pos0;
  int B, Tq, Dh, out_bf16;
};

template <typename T>
__device__ __forceinline__ T value_as(float x) {
  return static_cast<T>(x);
}

// Dh 64 and 128: one wave per block of 16 positions, head, and K or V, as the write's block kernel;
// memory-bound, every load and store a whole line a row: 16 x 4096 rows of 8 heads of 128 into fp32 in
// 115 us, 5.9 TB/s (a wave per row: 476).
template <int DH, typename T>
__global__ __launch_bounds__(256) void kv_read_q8_block_kernel(ReadArgs a, int blocks) {
  const int lane = threadIdx.x & 63;
  const BlockItem w = block_item(a.map, a.pos0, wave_item(), a.Tq, blocks);
  if (w.block < 0) return;
  T* dst = static_cast<T*>(w.is_v ? a.v : a.k) +
           ((static_cast<long>(w.b) * a.Tq + w.t0) * a.map.Hkv + w.h) * DH;
  const long rs = static_cast<long>(a.map.Hkv) * DH;
  if (w.is_v) {
    constexpr int E = DH / 64;
    typedef T vec __attribute__((ext_vector_type(E)));
    const float4* sp = reinterpret_cast<const float4*>(a.vs + w.block * kQ8Block);
    float s[kQ8Block];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = sp[i];
      s[4 * i] = f.x, s[4 * i + 1] = f.y, s[4 * i + 2] = f.z, s[4 * i + 3] = f.w;
    }
    uint32_t c[E][4];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint4 x = load_nt(a.vq + (w.block * DH + E * lane + e) * kQ8Block);
      c[e][0] = x.x, c[e][1] = x.y, c[e][2] = x.z, c[e][3] = x.w;
    }
#pragma unroll
    for (int r = 0; r < kQ8Block; ++r) {
      if (r < w.r0 || r >= w.r1) continue;
      vec o;
#pragma unroll
      for (int e = 0; e < E; ++e)
        o[e] = value_as<T>(static_cast<float>(static_cast<int8_t>(c[e][r >> 2] >> (8 * (r & 3)))) * s[r]);
      __builtin_nontemporal_store(o, reinterpret_cast<vec*>(dst + r * rs + E * lane));
    }
  } else {
    constexpr int LPR = DH / 4, RPI = 64 / LPR, N = kQ8Block / RPI;
    typedef T vec __attribute__((ext_vector_type(4)));
    const int at = lane / LPR, d = 4 * (lane % LPR);
    uint32_t c[N];
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = *reinterpret_cast<const uint32_t*>(a.kq + (w.block * kQ8Block + RPI * i + at) * DH + d);
      s[i] = a.ks[w.block * kQ8Block + RPI * i + at];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = RPI * i + at;
      if (r < w.r0 || r >= w.r1) continue;
      vec o;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[e] = value_as<T>(static_cast<float>(static_cast<int8_t>(c[i] >> (8 * e))) * s[i]);
      __builtin_nontemporal_store(o, reinterpret_cast<vec*>(dst + r * rs + d));
    }
  }
}

// Few rows, and any Dh: one wave per (token, head, K or V), as the write.
__global__ __launch_bounds__(256) void kv_read_q8_kernel(ReadArgs a) {
  const int lane = threadIdx.x & 63;
  const unsigned item = wave_item(), Hkv = a.map.Hkv;
  const bool is_v = item & 1u;
  const unsigned t = (item >> 1) / Hkv;
  const int h = static_cast<int>((item >> 1) - t * Hkv), b = blockIdx.y;
  if (t >= static_cast<unsigned>(a.Tq)) return;
  const long row = (static_cast<long>(b) * a.Tq + t) * Hkv + h;
  const long p = static_cast<long>(a.pos0[b]) + t;
  if (p < 0 || p >= a.map.capacity) return;
  const int at = static_cast<int>(p & 15);
  const long block = a.map.block(b, static_cast<int>(p >> 4), h);
  const int d = 4 * lane;
  if (block < 0 || d >= a.Dh) return;
  const float s = (is_v ? a.vs : a.ks)[block * kQ8Block + at];
  const int8_t* src = is_v ? a.vq + (block * a.Dh + d) * kQ8Block + at
                           : a.kq + (block * kQ8Block + at) * a.Dh + d;
  const int step = is_v ? kQ8Block : 1;
  void* out = is_v ? a.v : a.k;
  for (int i = 0; i < 4; ++i) {
    const float x = static_cast<float>(src[i * step]) * s;
    if (a.out_bf16)
      static_cast<__bf16*>(out)[row * a.Dh + d + i] = static_cast<__bf16>(x);
    else
      static_cast<float*>(out)[row * a.Dh + d + i] = x;
  }
}

// Whether a call takes the block kernels: rows that fill their blocks (8 of 16 at least), and more
// of them than the chip holds waves of the row kernels, one per row, head, and K or V, at once (8 per
// SIMD; below that the row kernels' shorter chains win).  8 heads of 128, us, row / block kernel:
// writes of 16 x 16 rows 4.8 / 7.1, 16 x 32 7.0 / 7.3, 16 x 64 10.4 / 8.2, 1 x 64 3.5 / 6.1, 1 x 2048
// 22.3 / 9.7; reads of 16 x 16 rows 3.9 / 4.5, 16 x 32 5.2 / 5.1, 16 x 64 7.7 / 5.2.
bool by_blocks(int B, int Tq, int Hkv, int Dh) {
  const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
  return (Dh == 64 || Dh == 128) && Tq >= 8 && 2L * B * Tq * Hkv > 32 * cus;
}
// Blocks that Tq rows touch at most, from wherever they begin.
int most_blocks(int Tq) { return static_cast<int>((static_cast<long>(Tq) + 14) / kQ8Block + 1); }

// Grid of B streams of `waves` waves each, 4 to a workgroup.
int grid_of(long waves, int B, dim3* grid, const char* what) {
  if ((waves + 3) / 4 > kMaxGroups256 || B > 65535)
    return fail(ORATOR_ERR_UNSUPPORTED, std::string(what) + ": too many rows, or over 65535 streams");
  *grid = dim3(static_cast<unsigned>((waves + 3) / 4), B);
  return ORATOR_OK;
}

int launch_write(const char* what, const float* k, const float* v, long kv_stride, int8_t* kq,
                 float* ks, int8_t* vq, float* vs, const int* page_table, bool paged,
                 int max_pages, int page_size, int n_pages, int B, int Tq, int Hkv, int Dh,
                 const int* d_pos0, int capacity, hipStream_t stream) {
  if (B <= 0 || Tq <= 0 || Hkv <= 0 || Dh <= 0) return ORATOR_OK;
  if (!k || !v || !d_pos0) return fail(ORATOR_ERR_INVALID, std::string(what) + ": null pointer");
  if (int rc = q8_pointers(what, kq, ks, vq, vs)) return rc;
  WriteArgs a{k, v, kv_stride, kq, ks, vq, vs, {}, d_pos0, B, Tq, Dh};
  if (int rc = q8_map(&a.map, what, page_table, paged, max_pages, page_size, n_pages, Hkv, Dh,
                      capacity))
    return rc;
  if (kv_stride < static_cast<long>(Hkv) * Dh)
    return fail(ORATOR_ERR_INVALID, std::string(what) + ": kv_stride below Hkv * Dh");
  dim3 grid;
  if (by_blocks(B, Tq, Hkv, Dh)) {
    const int blocks = most_blocks(Tq);
    if (int rc = grid_of(2L * blocks * Hkv, B, &grid, what)) return rc;
    if (Dh == 128)
      hipLaunchKernelGGL(kv_write_q8_block_kernel<128>, grid, dim3(256), 0, stream, a, blocks);
    else
      hipLaunchKernelGGL(kv_write_q8_block_kernel<64>, grid, dim3(256), 0, stream, a, blocks);
    return check_launch(what);
  }
  if (int rc = grid_of(2L * Tq * Hkv, B, &grid, what)) return rc;
  hipLaunchKernelGGL(kv_write_q8_kernel, grid, dim3(256), 0, stream, a);
  return check_launch(what);
}

int launch_read(const char* what, const int8_t* kq, const float* ks, const int8_t* vq,
                const float* vs, const int* page_table, bool paged, int max_pages, int page_size,
                int n_pages, void* k, void* v, int out_bf16, int B, int Tq, int Hkv, int Dh,
                const int* d_pos0, int capacity, hipStream_t stream) {
  if (B <= 0 || Tq <= 0 || Hkv <= 0 || Dh <= 0) return ORATOR_OK;
  if (!k || !v || !d_pos0) return fail(ORATOR_ERR_INVALID, std::string(what) + ": null pointer");
  if (out_bf16 != 0 && out_bf16 != 1)
    return fail(ORATOR_ERR_INVALID, std::string(what) + ": out_bf16 must be 0 or 1");
  if (int rc = q8_pointers(what, kq, ks, vq, vs)) return rc;
  ReadArgs a{kq, ks, vq, vs, k, v, {}, d_pos0, B, Tq, Dh, out_bf16};
  if (int rc = q8_map(&a.map, what, page_table, paged, max_pages, page_size, n_pages, Hkv, Dh,
                      capacity))
    return rc;
  dim3 grid;
  // vector stores: outputs that are 16-byte aligned
  if (by_blocks(B, Tq, Hkv, Dh) && aligned_to(k, 16) && aligned_to(v, 16)) {
    const int blocks = most_blocks(Tq);
    if (int rc = grid_of(2L * blocks * Hkv, B, &grid, what)) return rc;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, a, blocks);
    };
    if (Dh == 128)
      out_bf16 ? launch(kv_read_q8_block_kernel<128, __bf16>) : launch(kv_read_q8_block_kernel<128, float>);
    else
      out_bf16 ? launch(kv_read_q8_block_kernel<64, __bf16>) : launch(kv_read_q8_block_kernel<64, float>);
    return check_launch(what);
  }
  if (int rc = grid_of(2L * Tq * Hkv, B, &grid, what)) return rc;
  hipLaunchKernelGGL(kv_read_q8_kernel, grid, dim3(256), 0, stream, a);
  return check_launch(what);
}

}  // namespace
}  // namespace orator_hip

using namespace orator_hip;

extern "C" {

int orator_kv_write_q8(const float* k, const float* v, long kv_stride, int8_t* kq, float* ks,
                       int8_t* vq, float* vs, int Tq, int Hkv, int Dh, const int* d_pos0,
                       int capacity, void* stream) {
  return guarded([&] {
    return launch_write("kv_write_q8", k, v, kv_stride, kq, ks, vq, vs, nullptr, false, 0, 0, 0, 1,
                        Tq, Hkv, Dh, d_pos0, capacity, static_cast<hipStream_t>(stream));
  });
}

int orator_kv_write_q8_paged(const float* k, const float* v, long kv_stride, int8_t* kq, float* ks,
                             int8_t* vq, float* vs, const int* page_table, int max_pages,
                             int page_size, int n_pages, int B, int Tq, int Hkv, int Dh,
                             const int* d_pos0, void* stream) {
  return guarded([&] {
    return launch_write("kv_write_q8_paged", k, v, kv_stride, kq, ks, vq, vs, page_table, true,
                        max_pages, page_size, n_pages, B, Tq, Hkv, Dh, d_pos0, 0,
                        static_cast<hipStream_t>(stream));
  });
}

int orator_kv_read_q8(const int8_t* kq, const float* ks, const int8_t* vq, const float* vs,
                      void* k, void* v, int out_bf16, int Tq, int Hkv, int Dh, const int* d_pos0,
                      int capacity, void* stream) {
  return guarded([&] {
    return launch_read("kv_read_q8", kq, ks, vq, vs, nullptr, false, 0, 0, 0, k, v, out_bf16, 1, Tq,
                       Hkv, Dh, d_pos0, capacity, static_cast<hipStream_t>(stream));
  });
}

int orator_kv_read_q8_paged(const int8_t* kq, const float* ks, const int8_t* vq, const float* vs,
                            const int* page_table, int max_pages, int page_size, int n_pages,
                            void* k, void* v, int out_bf16, int B, int Tq, int Hkv, int Dh,
                            const int* d_pos0, void* stream) {
  return guarded([&] {
    return launch_read("kv_read_q8_paged", kq, ks, vq, vs, page_table, true, max_pages, page_size,
                       n_pages, k, v, out_bf16, B, Tq, Hkv, Dh, d_pos0, 0,
                       static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
