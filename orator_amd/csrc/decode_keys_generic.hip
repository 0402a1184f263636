// Decode attention over an 8-bit or bf16 paged cache, with an optional shared prefix, for any head
// size that is a multiple of 16 (up to 256) and any group, and the entry points of both.
//
// One wave per (split of the keys, q head, stream): a lane scores one key of 64 with q in LDS, the
// wave's softmax state is updated once per 64 keys, and for the values each lane owns dims lane,
// lane + 64, ... .  Splits are joined by their maxima and sums in a second kernel.
#include <algorithm>
#include <string>

#include "kv_q8.hpp"

namespace orator_hip {
namespace {

constexpr int kGenSplit = 256;      // keys of a split, at least
constexpr int kGenMaxSplits = 64;   // splits of a stream: what the joining scratch is sized by

struct KeysArgs {
  KeysProblem p;
  Q8Map map;
  int n_splits, split_len;  // a multiple of 64
  float scale_log2e;
  float* part_o;   // [B * Hq][n_splits][Dh]
  float* part_ml;  // [B * Hq][n_splits][2]
};

__device__ __forceinline__ int keys_of(const KeysArgs& a, int b) {
  const int pos = a.p.pos[b];
  return pos < 0 ? 0 : min(pos, a.map.capacity - 1) + 1;
}

template <bool Q8>
__global__ __launch_bounds__(64) void keys_generic_kernel(KeysArgs a) {
  __shared__ float sq[kQ8MaxDh];
  __shared__ float sp[64];
  __shared__ long sv[64];
  const int lane = threadIdx.x;
  const int split = blockIdx.x, hq = blockIdx.y, b = blockIdx.z;
  const int Dh = a.p.Dh, Hkv = a.p.Hkv, h = hq / (a.p.Hq / Hkv);
  const int S = keys_of(a, b);
  const long bh = static_cast<long>(b) * a.p.Hq + hq;
  const long from = static_cast<long>(split) * a.split_len;
  const int j0 = static_cast<int>(min(from, static_cast<long>(S)));
  const int j1 = static_cast<int>(min(from + a.split_len, static_cast<long>(S)));
  float m = -INFINITY, l = 0.0f, acc[kQ8MaxDh / 64] = {};
  for (int d = lane; d < Dh; d += 64) sq[d] = a.p.q[bh * Dh + d];
  __syncthreads();
  for (int c = j0; c < j1; c += 64) {
    const int j = c + lane;
    // where the key lies: its block's number in the 8-bit cache, its page in the bf16 pool
    const int tb = j < a.p.shared_len ? 0 : b;
    long block = -1;
    if (j < j1) {
      if constexpr (Q8)
        block = a.map.block(tb, j >> 4, h);
      else
        block = a.map.page(tb, j >> 4);
    }
    float s = -INFINITY;
    long v = -1;
    if (block >= 0) {
      float dot = 0.0f;
      if constexpr (Q8) {
        const int8_t* k = a.p.kq + (block * kQ8Block + (j & 15)) * Dh;
        for (int d = 0; d < Dh; ++d) dot = fmaf(sq[d], static_cast<float>(k[d]), dot);
        s = dot * a.p.ks[block * kQ8Block + (j & 15)] * a.scale_log2e;
        v = block;
      } else {
        const int ps = a.map.block_shift + 4;
        v = (((block << ps) + (j & ((1 << ps) - 1))) * Hkv + h) * Dh;
        const uint16_t* k = a.p.kpool + v;
        for (int d = 0; d < Dh; ++d) dot = fmaf(sq[d], bf16_to_f32(k[d]), dot);
        s = dot * a.scale_log2e;
      }
    }
    const float mn = fmaxf(m, wave_max(s));
    const float ref = mn == -INFINITY ? 0.0f : mn;  // no key yet
    const float corr = fast_exp2(m - ref);
    const float p = block >= 0 ? fast_exp2(s - ref) : 0.0f;
    m = mn;
    l = l * corr + wave_sum(p);
    for (float& x : acc) x *= corr;
    __syncthreads();
    sp[lane] = Q8 && block >= 0 ? p * a.p.vs[block * kQ8Block + (j & 15)] : p;
    sv[lane] = v;
    __syncthreads();
    for (int i = 0; i < min(64, j1 - c); ++i) {
      const long at = sv[i];
      if (at < 0) continue;
      const float w = sp[i];
      for (int e = 0; e < kQ8MaxDh / 64; ++e) {
        const int d = 64 * e + lane;
        if (d >= Dh) break;
        float x;
        if constexpr (Q8)
          x = static_cast<float>(a.p.vq[(at * Dh + d) * kQ8Block + ((c + i) & 15)]);
        else
          x = bf16_to_f32(a.p.vpool[at + d]);
        acc[e] = fmaf(w, x, acc[e]);
      }
    }
  }
  const long ps = bh * a.n_splits + split;
  for (int e = 0; e < kQ8MaxDh / 64; ++e)
    if (64 * e + lane < Dh) a.part_o[ps * Dh + 64 * e + lane] = acc[e];
  if (lane == 0) {
    a.part_ml[2 * ps] = m;
    a.part_ml[2 * ps + 1] = l;
  }
}

// out[bh][d] = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s; no key at all: zeros.
__global__ __launch_bounds__(256) void keys_merge_kernel(KeysArgs a) {
  const long bh = blockIdx.x;
  const int Dh = a.p.Dh;
  const int d = threadIdx.x;
  if (d >= Dh) return;
  float M = -INFINITY, L = 0.0f, o = 0.0f;
  for (int s = 0; s < a.n_splits; ++s) M = fmaxf(M, a.part_ml[2 * (bh * a.n_splits + s)]);
  const float ref = M == -INFINITY ? 0.0f : M;
  for (int s = 0; s < a.n_splits; ++s) {
    const long ps = bh * a.n_splits + s;
    const float w = fast_exp2(a.part_ml[2 * ps] - ref);
    L = fmaf(w, a.part_ml[2 * ps + 1], L);
    o = fmaf(w, a.part_o[ps * Dh + d], o);
  }
  a.p.out[bh * Dh + d] = L == 0.0f ? 0.0f : o / L;
}

}  // namespace

int launch_keys_generic(const KeysProblem& p, const Q8Map& map, hipStream_t stream) {
  const long cap = map.capacity;
  const long len = std::max<long>(kGenSplit, ((cap + kGenMaxSplits - 1) / kGenMaxSplits + 63) / 64 * 64);
  const long splits = (cap + len - 1) / len;
  const size_t rows = static_cast<size_t>(p.B) * p.Hq * splits;
  char* ws = static_cast<char*>(workspace_graph(stream, rows * (p.Dh + 2) * sizeof(float), kWsKeys));
  if (!ws) return ORATOR_ERR_HIP;
  KeysArgs a{p, map, static_cast<int>(splits), static_cast<int>(len), p.scale * 1.4426950408889634f,
             reinterpret_cast<float*>(ws), reinterpret_cast<float*>(ws) + rows * p.Dh};
  const dim3 grid(static_cast<unsigned>(splits), p.Hq, p.B);
  if (p.bf16)
    hipLaunchKernelGGL(keys_generic_kernel<false>, grid, dim3(64), 0, stream, a);
  else
    hipLaunchKernelGGL(keys_generic_kernel<true>, grid, dim3(64), 0, stream, a);
  if (int rc = check_launch("keys_generic_kernel")) return rc;
  hipLaunchKernelGGL(keys_merge_kernel, dim3(static_cast<unsigned>(p.B) * p.Hq), dim3(256), 0, stream,
                     a);
  return check_launch("keys_merge_kernel");
}

namespace {

// Checks and runs a decode over keys; what: the entry's name.
int decode_keys(const char* what, const KeysProblem& p, bool paged, hipStream_t stream) {
  if (p.B <= 0 || p.Hq <= 0 || p.Hkv <= 0 || p.Dh <= 0) return ORATOR_OK;
  const std::string who(what);
  if (!p.q || !p.pos || !p.out) return fail(ORATOR_ERR_INVALID, who + ": null pointer");
  if (p.bf16) {
    if (!p.kpool || !p.vpool) return fail(ORATOR_ERR_INVALID, who + ": null cache");
    if (!aligned_to(p.kpool, 16) || !aligned_to(p.vpool, 16))
      return fail(ORATOR_ERR_INVALID, who + ": caches must be 16-byte aligned");
  } else if (int rc = q8_pointers(what, p.kq, p.ks, p.vq, p.vs)) {
    return rc;
  }
  if (p.Hq % p.Hkv) return fail(ORATOR_ERR_INVALID, who + ": Hq must be a multiple of Hkv");
  if (p.B > 65535 || p.Hq > 65535 || static_cast<long>(p.B) * p.Hq > kMaxGroups256)
    return fail(ORATOR_ERR_UNSUPPORTED, who + ": too many streams or q heads");
  Q8Map map;
  if (int rc = q8_map(&map, what, p.page_table, paged, p.max_pages, p.page_size, p.n_pages, p.Hkv,
                      p.Dh, p.capacity))
    return rc;
  if (p.shared_len < 0) return fail(ORATOR_ERR_INVALID, who + ": shared_len must be >= 0");
  if (p.shared_len > map.capacity)
    return fail(ORATOR_ERR_CAPACITY, who + ": shared_len exceeds max_pages * page_size");
  if (p.Dh != 64 && p.Dh != 128) return launch_keys_generic(p, map, stream);
  if (!p.bf16 && p.shared_len == 0) return launch_decode_q8(p, map, stream);
  return launch_shared_prefix(p, map, stream);
}

KeysProblem keys_problem(const float* q, const int* d_pos, float* out, int B, int Hq, int Hkv,
                         int Dh, float scale) {
  KeysProblem p{};
  p.q = q;
  p.pos = d_pos;
  p.out = out;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.Dh = Dh;
  p.scale = scale;
  return p;
}

void q8_cache(KeysProblem* p, const int8_t* kq, const float* ks, const int8_t* vq,
              const float* vs) {
  p->kq = kq;
  p->ks = ks;
  p->vq = vq;
  p->vs = vs;
}

void pages(KeysProblem* p, const int* page_table, int max_pages, int page_size, int n_pages) {
  p->page_table = page_table;
  p->max_pages = max_pages;
  p->page_size = page_size;
  p->n_pages = n_pages;
}

}  // namespace
}  // namespace orator_hip

using namespace orator_hip;

extern "C" {

int orator_gqa_decode_q8(const float* q, const int8_t* kq, const float* ks, const int8_t* vq,
                         const float* vs, float* out, int Hq, int Hkv, int Dh, const int* d_pos,
                         int capacity, float scale, void* stream) {
  return guarded([&] {
    KeysProblem p = keys_problem(q, d_pos, out, 1, Hq, Hkv, Dh, scale);
    q8_cache(&p, kq, ks, vq, vs);
    p.capacity = capacity;
    return decode_keys("gqa_decode_q8", p, false, static_cast<hipStream_t>(stream));
  });
}

int orator_gqa_decode_q8_paged(const float* q, const int8_t* kq, const float* ks, const int8_t* vq,
                               const float* vs, const int* page_table, int max_pages,
                               int page_size, int n_pages, const int* d_pos, float* out, int B,
                               int Hq, int Hkv, int Dh, float scale, void* stream) {
  return guarded([&] {
    KeysProblem p = keys_problem(q, d_pos, out, B, Hq, Hkv, Dh, scale);
    q8_cache(&p, kq, ks, vq, vs);
    pages(&p, page_table, max_pages, page_size, n_pages);
    return decode_keys("gqa_decode_q8_paged", p, true, static_cast<hipStream_t>(stream));
  });
}

int orator_gqa_decode_shared_paged(const float* q, const uint16_t* kpool, const uint16_t* vpool,
                                   const int* page_table, int max_pages, int page_size,
                                   int n_pages, const int* d_pos, int shared_len, float* out,
                                   int B, int Hq, int Hkv, int Dh, float scale, void* stream) {
  return guarded([&] {
    KeysProblem p = keys_problem(q, d_pos, out, B, Hq, Hkv, Dh, scale);
    p.bf16 = true;
    p.kpool = kpool;
    p.vpool = vpool;
    pages(&p, page_table, max_pages, page_size, n_pages);
    p.shared_len = shared_len;
    return decode_keys("gqa_decode_shared_paged", p, true, static_cast<hipStream_t>(stream));
  });
}

int orator_gqa_decode_shared_q8_paged(const float* q, const int8_t* kq, const float* ks,
                                      const int8_t* vq, const float* vs, const int* page_table,
                                      int max_pages, int page_size, int n_pages, const int* d_pos,
                                      int shared_len, float* out, int B, int Hq, int Hkv, int Dh,
                                      float scale, void* stream) {
  return guarded([&] {
    KeysProblem p = keys_problem(q, d_pos, out, B, Hq, Hkv, Dh, scale);
    q8_cache(&p, kq, ks, vq, vs);
    pages(&p, page_table, max_pages, page_size, n_pages);
    p.shared_len = shared_len;
    return decode_keys("gqa_decode_shared_q8_paged", p, true, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
