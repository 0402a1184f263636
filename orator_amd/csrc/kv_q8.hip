// The KV cache in 8 bits: rows quantised as they are written, and read back.
//
// A row x of Dh values is held as scale = max|x| * fl(1 / 127) and codes = the integers nearest to
// x / scale.  The codes are exactly those of the real quotient: c = rint(x * fl(1 / scale)) is off
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

// Code of x for a scale with 1 / scale = inv; scale is normal, so inv and 2 r are finite.
__device__ __forceinline__ int q8_code(float x, float scale, float inv) {
  float c = rintf(x * inv);
  const float r2 = 2.0f * fmaf(-c, scale, x);
  const bool odd = static_cast<int>(c) & 1;
  if (r2 > scale || (r2 == scale && odd)) c += 1.0f;
  if (r2 < -scale || (r2 == -scale && odd)) c -= 1.0f;
  return static_cast<int>(fminf(fmaxf(c, -127.0f), 127.0f));
}

// Scale of a row whose largest magnitude has the bits `amax` (as an integer: an infinity and a NaN
// are above every number): 0 where it would be subnormal, NaN for a row that is not finite.
__device__ __forceinline__ float q8_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const float s = __uint_as_float(amax) * (1.0f / 127.0f);
  return s >= 1.17549435e-38f ? s : 0.0f;
}

// One wave per (token, head, K or V): lane l holds dims 4 l .. 4 l + 3.
__global__ __launch_bounds__(256) void kv_write_q8_kernel(WriteArgs a) {
  const int lane = threadIdx.x & 63;
  const long item = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int Hkv = a.map.Hkv;
  const long rows = static_cast<long>(a.B) * a.Tq * Hkv;
  if (item >= 2 * rows) return;
  const bool is_v = item >= rows;
  const long row = is_v ? item - rows : item;  // (b * Tq + t) * Hkv + h
  const int h = static_cast<int>(row % Hkv);
  const long bt = row / Hkv;
  const int b = static_cast<int>(bt / a.Tq);
  const long p = static_cast<long>(a.pos0[b]) + (bt - static_cast<long>(b) * a.Tq);
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
  const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;  // 0: a row of zeros, or one that is NaN
  if (d < a.Dh) {
    int c[4];
    for (int i = 0; i < 4; ++i) c[i] = inv > 0.0f ? q8_code(x[i], scale, inv) : 0;
    if (is_v) {
      int8_t* dst = a.vq + (block * a.Dh + d) * kQ8Block + at;
      for (int i = 0; i < 4; ++i) dst[i * kQ8Block] = static_cast<int8_t>(c[i]);
    } else {
      const uint32_t w = (c[0] & 255u) | (c[1] & 255u) << 8 | (c[2] & 255u) << 16 | (c[3] & 255u) << 24;
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

// One wave per (token, head, K or V), as the write.
__global__ __launch_bounds__(256) void kv_read_q8_kernel(ReadArgs a) {
  const int lane = threadIdx.x & 63;
  const long item = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int Hkv = a.map.Hkv;
  const long rows = static_cast<long>(a.B) * a.Tq * Hkv;
  if (item >= 2 * rows) return;
  const bool is_v = item >= rows;
  const long row = is_v ? item - rows : item;
  const int h = static_cast<int>(row % Hkv);
  const long bt = row / Hkv;
  const int b = static_cast<int>(bt / a.Tq);
  const long p = static_cast<long>(a.pos0[b]) + (bt - static_cast<long>(b) * a.Tq);
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

int blocks_of(long waves, unsigned* grid, const char* what) {
  const long n = (waves + 3) / 4;
  if (n > 0x7fffffffL) return fail(ORATOR_ERR_UNSUPPORTED, std::string(what) + ": too many rows");
  *grid = static_cast<unsigned>(n);
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
  unsigned grid = 0;
  if (int rc = blocks_of(2L * B * Tq * Hkv, &grid, what)) return rc;
  hipLaunchKernelGGL(kv_write_q8_kernel, dim3(grid), dim3(256), 0, stream, a);
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
  unsigned grid = 0;
  if (int rc = blocks_of(2L * B * Tq * Hkv, &grid, what)) return rc;
  hipLaunchKernelGGL(kv_read_q8_kernel, dim3(grid), dim3(256), 0, stream, a);
  return check_launch(what);
}

}  // namespace
}  // namespace orator_hip

using namespace orator_hip;

extern "C" {

int orator_kv_write_q8(const float* k, const float* v, long kv_stride, int8_t* kq, float* ks,
                       int8_t* vq, float* vs, int Tq, int Hkv, int Dh, const int* d_pos0,
                       int capacity, void* stream) {
  return launch_write("kv_write_q8", k, v, kv_stride, kq, ks, vq, vs, nullptr, false, 0, 0, 0, 1,
                      Tq, Hkv, Dh, d_pos0, capacity, static_cast<hipStream_t>(stream));
}

int orator_kv_write_q8_paged(const float* k, const float* v, long kv_stride, int8_t* kq, float* ks,
                             int8_t* vq, float* vs, const int* page_table, int max_pages,
                             int page_size, int n_pages, int B, int Tq, int Hkv, int Dh,
                             const int* d_pos0, void* stream) {
  return launch_write("kv_write_q8_paged", k, v, kv_stride, kq, ks, vq, vs, page_table, true,
                      max_pages, page_size, n_pages, B, Tq, Hkv, Dh, d_pos0, 0,
                      static_cast<hipStream_t>(stream));
}

int orator_kv_read_q8(const int8_t* kq, const float* ks, const int8_t* vq, const float* vs,
                      void* k, void* v, int out_bf16, int Tq, int Hkv, int Dh, const int* d_pos0,
                      int capacity, void* stream) {
  return launch_read("kv_read_q8", kq, ks, vq, vs, nullptr, false, 0, 0, 0, k, v, out_bf16, 1, Tq,
                     Hkv, Dh, d_pos0, capacity, static_cast<hipStream_t>(stream));
}

int orator_kv_read_q8_paged(const int8_t* kq, const float* ks, const int8_t* vq, const float* vs,
                            const int* page_table, int max_pages, int page_size, int n_pages,
                            void* k, void* v, int out_bf16, int B, int Tq, int Hkv, int Dh,
                            const int* d_pos0, void* stream) {
  return launch_read("kv_read_q8_paged", kq, ks, vq, vs, page_table, true, max_pages, page_size,
                     n_pages, k, v, out_bf16, B, Tq, Hkv, Dh, d_pos0, 0,
                     static_cast<hipStream_t>(stream));
}

}  // extern "C"
