// Decode attention of a batch whose streams share a prefix, over the bf16 pool or the 8-bit cache:
// the prefix's keys are read once for all streams, gfx950.
//
// For one kv head, the B G query rows of the batch against the prefix are a matrix product; a stream's
// G rows against its own keys use few columns of one, and their time is their memory's.  One kernel
// does both, in two kinds of units:
//  * prefix units, a workgroup each: columns are 32 rows (stream, head) b G + g of the batch, keys a
//    range of [0, P) through page-table row 0, which the waves take tile by tile in turn;
//  * own units, a wave each: columns are up to 8 heads of one stream, keys every n_own-th tile of
//    [P, S_b) through its own row.  A stream with fewer keys than the prefix has none there and is no
//    column of a prefix unit: its units take keys [0, S_b) of row 0.  So a unit's columns all attend
//    the same keys, and a value that is not finite reaches no stream that does not attend it (0 * inf
//    in a product is NaN).
//
// Per 32-key tile of a wave, S^T = K Q^T and O^T += V^T W^T on mfma_f32_32x32x16_bf16:
//  * q and the weights w enter as three bf16 terms (the top 8, middle 8 and last 8 bits of the
//    fp32 significand, split by truncation: exact), K and V as they are (bf16, or int8 codes,
//    which bf16 holds exactly): fp32 accuracy for 3 MFMAs per product.  In an own unit a head's
//    terms are the columns of a quad instead, and one MFMA does all: scores are the quad's sums, the
//    outputs' terms are summed at the end.
//  * a lane has one query column, and scores of 16 consecutive keys: tile row 8 a + 4 h + i is key
//    16 h + 4 a + i, so lane half h holds block h of the tile and its registers are the B operand
//    of the second product as they are.
//  * bf16 rows are loaded as whole lines and go through LDS: K, then V in its place (V^T by the
//    transposing read).  8-bit codes go from memory into the operands: K a half line of a row, V as
//    it lies transposed.
//  * softmax with a reference that follows the running maximum once it is 8 (log2) behind.
// A prefix unit's waves are joined in LDS; the units' partials of a (stream, head) by a second kernel
// (joined by the last unit to finish, in the same launch, the one that completes a block of columns
// joins 32 rows alone: B = 64, prefix 4096 measured 52 us instead of 41, B = 16 over the 8-bit cache 30
// instead of 15).
//
// Measured, 16 q / 8 kv heads of 128, both launches: 64 streams behind 4096 keys with 1 to 512 of their
// own, bf16, 28.4 us (85 MB: 16.5 us at a copy's rate; own keys by workgroups of four waves with three
// MFMAs a product 37.9; with written lines in the caches, 256 streams of up to 128 keys behind 1024 42
// us instead of 56, 16 streams of 32 q heads on 2 kv heads 20.8 instead of 19.9); 16 behind 2048, 8-bit, 15.1 us; 6 behind 503, bf16, 10.7 us.  A prefix tile is
// 48 MFMAs (0.7 us) and some 430 VALU instructions, one wave after another 1.3 us per SIMD; the rest is
// the chain page -> rows -> products -> partials -> join of two launches.
#include <algorithm>
#include <string>

#include "kv_q8.hpp"
#include "mfma_tile.hpp"

namespace orator_hip {
namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;     // keys per wave tile
constexpr int kCols = 32;     // query columns of a unit
constexpr int kOwnHeads = 8;  // heads of an own unit: 4 columns each
constexpr int kMaxOwn = 128;  // own units per stream, at most: a wave of the second kernel joins them
constexpr float kSlack = 8.0f;
// instruction kinds of __builtin_amdgcn_sched_group_barrier
constexpr int kMfma = 0x008, kDsRead = 0x100;

struct SharedArgs {
  KeysProblem p;
  Q8Map map;
  float scale_log2e;
  int G;
  int col_blocks;   // blocks of 32 rows of the batch
  int n_pre;        // prefix units per (kv head, column block)
  int pre_tiles;    // tiles per prefix unit
  int n_own;        // own units (waves) per (stream, kv head, chunk of kOwnHeads heads)
  int own_chunks;
  int slots;        // n_pre + n_own: partials per (stream, head)
  float* part_o;    // [B * Hq][slots][Dh]
  float* part_ml;   // [B * Hq][slots][2]
};

__device__ __forceinline__ int stream_len(const SharedArgs& a, int b) {
  const int pos = a.p.pos[b];
  return pos < 0 ? 0 : min(pos, a.map.capacity - 1) + 1;
}

// Two fp32 to one dword of their upper halves (the bf16 that truncation gives).
__device__ __forceinline__ uint32_t upper2(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float drop_upper(float x) {
  return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}

// 8 fp32 as three bf16 terms; exact but for an infinity (NaN).
__device__ __forceinline__ void split3(const float (&x)[8], uint4 (&t)[3]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    t[k] = make_uint4(upper2(r[0], r[1]), upper2(r[2], r[3]), upper2(r[4], r[5]), upper2(r[6], r[7]));
    if (k < 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = drop_upper(r[i]);
    }
  }
}

// 8 int8 codes (two dwords) as bf16, exact.
__device__ __forceinline__ uint4 codes_bf16(uint32_t lo, uint32_t hi) {
  asm volatile("" : "+v"(lo), "+v"(hi));  // converted where it stands, not with the others at once
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = static_cast<float>(static_cast<int8_t>(lo >> (8 * i)));
    f[4 + i] = static_cast<float>(static_cast<int8_t>(hi >> (8 * i)));
  }
  return make_uint4(upper2(f[0], f[1]), upper2(f[2], f[3]), upper2(f[4], f[5]), upper2(f[6], f[7]));
}

template <bool Q8, int DH>
struct Tile {
  static constexpr int NK = Q8 ? DH / 32 : DH / 16;  // 16-byte loads of K, and of V
  u32x4_t k[NK], v[NK];  // plain vectors: they have to stay in registers
  float4 ks[Q8 ? 4 : 1], vs[Q8 ? 4 : 1];
  bool mapped0, mapped1;  // the tile's two blocks
};

// The page-table entries of a wave's tiles, 32 tiles at a time: lane 2 j + i holds the entry of block i
// of tile first + j * stride, so that a tile's loads go out without a look-up before them.
struct TilePages {
  int entry;
  int at = 0;  // j of the next tile

  __device__ __forceinline__ void fetch(const Q8Map& m, int row_b, int first, int stride, int lane) {
    const long blk = 2 * (first + static_cast<long>(lane >> 1) * stride) + (lane & 1);
    entry = m.page(row_b, static_cast<int>(min(blk, static_cast<long>(m.capacity / kQ8Block - 1))));
    at = 0;
  }
  // Pages of tile `tile`, which follows the one asked for last; -1: unmapped.
  __device__ __forceinline__ void next(const Q8Map& m, int row_b, int tile, int stride, int lane, int* p0,
                                       int* p1) {
    if (at == 32) fetch(m, row_b, tile, stride, lane);
    *p0 = __builtin_amdgcn_readlane(entry, 2 * at);
    *p1 = __builtin_amdgcn_readlane(entry, 2 * at + 1);
    ++at;
  }
};

// The rows of a bf16 tile in the pool.
struct TileRows {
  long r0, r1;            // of its two blocks' first keys
  bool mapped0, mapped1;  // (unmapped: rows of page 0, which are masked)
};
__device__ __forceinline__ TileRows tile_rows(const Q8Map& m, int p0, int p1, int tile) {
  const int bs = m.block_shift, msk = (1 << bs) - 1;
  return {((static_cast<long>(max(p0, 0)) << bs) + (2 * tile & msk)) << 4,
          ((static_cast<long>(max(p1, 0)) << bs) + ((2 * tile + 1) & msk)) << 4, p0 >= 0, p1 >= 0};
}
// Rows that one unit reads (NT) are loaded past the caches' other lines: behind a kernel that left 256
// MB of written lines there, 64 streams of 1 to 512 keys 20.8 us instead of 33.6 (of 8-bit codes, V
// alone, whose lines a load covers: 28.6 instead of 30.2); no difference with clean caches.
// A bf16 tile of K or V, rows as they lie, whole lines: DH / 8 lanes per row, rows in order.
template <int DH, bool NT>
__device__ __forceinline__ void load_rows(u32x4_t (&r)[DH / 16], const uint16_t* pool,
                                          const TileRows& t, long rs, int kvh, int lane) {
  constexpr int LPR = DH / 8, RPI = 64 / LPR;  // lanes per row, rows per load
  const uint32_t off = static_cast<uint32_t>(lane / LPR) * static_cast<uint32_t>(rs) + 8 * (lane % LPR);
#pragma unroll
  for (int i = 0; i < DH / 16; ++i) {
    const int row = RPI * i;  // a load's rows lie in one block (RPI divides 16): a uniform base
    const uint16_t* at = pool + ((row < 16 ? t.r0 : t.r1) + (row & 15)) * rs + kvh * DH;
    const u32x4_t* from = reinterpret_cast<const u32x4_t*>(at + off);
    r[i] = NT ? __builtin_nontemporal_load(from) : *from;
  }
}

// The dims of k-step s, lane half h, element e: bf16 K is loaded 8 dims at a time, the 8-bit codes
// 16 at a time, which serve two k-steps.
template <bool Q8>
__device__ __forceinline__ int dim_of(int s, int h) {
  return Q8 ? 32 * (s >> 1) + 16 * h + 8 * (s & 1) : 16 * s + 8 * h;
}

// An 8-bit tile of pages p0 and p1.
template <int DH, bool NT>
__device__ __forceinline__ void load_tile(Tile<true, DH>& t, const SharedArgs& a, int p0, int p1, int kvh,
                                          int tile, int lane) {
  const int h = lane >> 5;
  const bool second = lane & 4;                       // K: the block of tile row lane & 31
  const int at = 4 * ((lane >> 3) & 3) + (lane & 3);  // and its place there
  t.mapped0 = p0 >= 0;
  t.mapped1 = p1 >= 0;
  // unmapped: a block of page 0 is read, its keys are masked
  const int bs = a.map.block_shift, msk = (1 << bs) - 1;
  const long n0 = ((static_cast<long>(max(p0, 0)) * a.p.Hkv + kvh) << bs) + (2 * tile & msk);
  const long n1 = ((static_cast<long>(max(p1, 0)) * a.p.Hkv + kvh) << bs) + ((2 * tile + 1) & msk);
  const int8_t* k = a.p.kq + ((second ? n1 : n0) * kQ8Block + at) * DH + 16 * h;
  const long nv = h ? n1 : n0;
  const int8_t* v = a.p.vq + (nv * DH + (lane & 31)) * kQ8Block;
#pragma unroll
  for (int i = 0; i < DH / 32; ++i) t.k[i] = *reinterpret_cast<const u32x4_t*>(k + 32 * i);
#pragma unroll
  for (int i = 0; i < DH / 32; ++i) {
    const u32x4_t* from = reinterpret_cast<const u32x4_t*>(v + 32 * i * kQ8Block);
    t.v[i] = NT ? __builtin_nontemporal_load(from) : *from;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t.ks[i] = *reinterpret_cast<const float4*>(a.p.ks + nv * kQ8Block + 4 * i);
    t.vs[i] = *reinterpret_cast<const float4*>(a.p.vs + nv * kQ8Block + 4 * i);
  }
}

template <int DH>
constexpr int kVStride = DH + 16;  // bf16 elements of a V row in LDS
template <int DH>
constexpr int kKStride = DH + 8;   // of a K row
template <int DH>
constexpr int kQStride = DH + 8;   // and of a q row

// A wave's softmax state and sums: of query column lane & 31, dims 32 n + 8 (r >> 2) + 4 (lane >> 5) +
// (r & 3) in o[n][r]; l is this lane's share.
template <int DH>
struct ColState {
  float m = -INFINITY, l = 0.0f;
  f32x16_t o[DH / 32] = {};
};

// A wave's tiles `tile`, tile + stride, ... of keys [lo, hi) through table row row_b; pages: theirs.
// prepare() runs once the first tile's loads are on the way, and makes q ready for `q`: with OWN k-step
// s's operand is q.at(s), one term a column, else q.at(s, term).  vt: the wave's buffer for a bf16 tile
// in LDS.
template <bool Q8, int DH, bool OWN, typename Query, typename Prepare>
__device__ __forceinline__ void attend_tiles(ColState<DH>& st, const SharedArgs& a, int row_b, int kvh,
                                             int lo, int hi, int tile, int stride, TilePages& pages,
                                             uint16_t* vt, int lane, const Query& q, Prepare&& prepare) {
  constexpr int NS = DH / 16;  // k-steps of the first product
  constexpr int ND = DH / 32;  // dim blocks of the second
  constexpr int NT = OWN ? 1 : 3;  // products of an operand pair
  const int h = lane >> 5;
  const int t_end = hi > lo ? (hi + kTile - 1) / kTile : 0;
  Tile<Q8, DH> nxt;
  const long rs = static_cast<long>(a.p.Hkv) * DH;
  TileRows rows{};  // bf16: of the tile in nxt
  auto load_codes = [&](auto& t, int at) {
    int p0, p1;
    pages.next(a.map, row_b, at, stride, lane, &p0, &p1);
    load_tile<DH, OWN>(t, a, p0, p1, kvh, at, lane);
  };
  auto find_rows = [&](int at) {
    int p0, p1;
    pages.next(a.map, row_b, at, stride, lane, &p0, &p1);
    return tile_rows(a.map, p0, p1, at);
  };
  if (tile < t_end) {
    if constexpr (Q8) {
      load_codes(nxt, tile);
    } else {
      rows = find_rows(tile);
      load_rows<DH, OWN>(nxt.k, a.p.kpool, rows, rs, kvh, lane);
      load_rows<DH, OWN>(nxt.v, a.p.vpool, rows, rs, kvh, lane);
    }
  }
  prepare(tile < t_end);
  // OWN: which of w's terms this lane's column holds: w less its first (1), and less its second (2)
  const uint32_t drop1 = OWN && (lane & 3) >= 1 ? 0xffff0000u : 0u;
  const uint32_t drop2 = OWN && (lane & 3) >= 2 ? 0xffff0000u : 0u;

  auto work = [&](Tile<Q8, DH>& cur) __attribute__((always_inline)) {
    const int key0 = kTile * tile + 16 * h;  // this lane's 16 keys
    const bool mapped0 = Q8 ? cur.mapped0 : rows.mapped0, mapped1 = Q8 ? cur.mapped1 : rows.mapped1;
    // Keeps y of the lane's keys that are attended, puts `none` for the others; one compare each, no
    // branches.
    auto mask = [&](float (&y)[16], float none) {
      const int first = max(lo - key0, 0);
      const uint32_t n = (h ? mapped1 : mapped0) ? static_cast<uint32_t>(max(hi - key0 - first, 0)) : 0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = static_cast<uint32_t>(i - first) < n ? y[i] : none;
    };
    const bool whole = mapped0 && mapped1 && kTile * tile >= lo && kTile * (tile + 1) <= hi;
    const bool more = tile + stride < t_end;  // bf16: the next tile takes this one's registers
    constexpr int LPR = DH / 8, RPI = 64 / LPR;
    if constexpr (!Q8) {
#pragma unroll
      for (int i = 0; i < DH / 16; ++i)
        *reinterpret_cast<u32x4_t*>(vt + (RPI * i + lane / LPR) * kKStride<DH> + 8 * (lane % LPR)) =
            cur.k[i];
      if (!whole) {
        // rows that are not attended go in as zeros: their weights are 0, and 0 * inf is NaN
#pragma unroll
        for (int i = 0; i < DH / 16; ++i) {
          const int key = kTile * tile + RPI * i + lane / LPR;
          const bool in = (RPI * i < 16 ? mapped0 : mapped1) & (key >= lo) & (key < hi);
          cur.v[i] &= in ? ~0u : 0u;
        }
      }
      if (more) {
        rows = find_rows(tile + stride);
        load_rows<DH, OWN>(cur.k, a.p.kpool, rows, rs, kvh, lane);
      }
      wave_lds_sync();
    }
    // tile row lane & 31: key 16 h + 4 a + i for row 8 a + 4 h + i
    const uint16_t* krow =
        vt + (4 * (lane & 4) + 4 * ((lane >> 3) & 3) + (lane & 3)) * kKStride<DH> + 8 * h;
    f32x16_t sc = {};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      uint4 kf;
      if constexpr (Q8) {
        // codes become bf16 as they are needed: all at once are too many registers
        if (s % 2 == 0) __builtin_amdgcn_sched_barrier(0);
        const u32x4_t c = cur.k[s >> 1];
        kf = (s & 1) ? codes_bf16(c.z, c.w) : codes_bf16(c.x, c.y);
      } else {
        kf = *reinterpret_cast<const uint4*>(krow + 16 * s);
      }
#pragma unroll
      for (int k = NT - 1; k >= 0; --k) sc = mfma32(as_bf16x8(kf), as_bf16x8(q.at(s, k)), sc);
    }
    if constexpr (!Q8) {
      if constexpr (!OWN) {
        // a k-step's operands are read ahead of the products of the one before
        __builtin_amdgcn_sched_group_barrier(kDsRead, 8, 0);
#pragma unroll
        for (int s = 0; s < NS - 2; ++s) {
          __builtin_amdgcn_sched_group_barrier(kMfma, 3, 0);
          __builtin_amdgcn_sched_group_barrier(kDsRead, 4, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kMfma, 6, 0);
      }
      // V takes K's place
      wave_lds_sync();
#pragma unroll
      for (int i = 0; i < DH / 16; ++i)
        *reinterpret_cast<u32x4_t*>(vt + (RPI * i + lane / LPR) * kVStride<DH> + 8 * (lane % LPR)) =
            cur.v[i];
      if (more) load_rows<DH, OWN>(cur.v, a.p.vpool, rows, rs, kvh, lane);
    }
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = sc[i];
      if constexpr (OWN) x[i] = quad_sum(x[i]);  // a head's terms are its quad's columns
      if constexpr (Q8) x[i] *= reinterpret_cast<const float*>(cur.ks)[i];
    }
    if (!whole) mask(x, -INFINITY);
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    mx = xor32_max(mx);
    if (__any(mx > st.m + kSlack)) {  // m is -infinity before the first key
      const float mn = fmaxf(st.m, mx);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      const float c = fast_exp2(st.m - ref);
      st.l *= c;
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[n][i] *= c;
      st.m = mn;
    }
    const float ref = st.m == -INFINITY ? 0.0f : st.m;
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      w[i] = fast_exp2(x[i] - ref);
      st.l += w[i];
      if constexpr (Q8) w[i] *= reinterpret_cast<const float*>(cur.vs)[i];
    }
    if (Q8 && !whole) mask(w, 0.0f);  // a scale behind the last key may be anything
    uint4 wt[2][NT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = w[8 * s + i];
        if constexpr (OWN) {
          y[i] -= __uint_as_float(__float_as_uint(y[i]) & drop1);
          y[i] -= __uint_as_float(__float_as_uint(y[i]) & drop2);
        }
      }
      if constexpr (OWN)
        wt[s][0] = make_uint4(upper2(y[0], y[1]), upper2(y[2], y[3]), upper2(y[4], y[5]), upper2(y[6], y[7]));
      else
        split3(y, wt[s]);
    }
    if constexpr (!Q8) wave_lds_sync();
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      if constexpr (Q8) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint4 vf;
        if constexpr (Q8) {
          const u32x4_t c = cur.v[n];
          vf = s ? codes_bf16(c.z, c.w) : codes_bf16(c.x, c.y);
        } else {
          // keys 16 h + 8 s + 0..3 and + 4..7 of dim 32 n + (lane & 31)
          const uint16_t* at = vt + (16 * h + 8 * s + ((lane & 15) >> 2)) * kVStride<DH> + 32 * n +
                               (lane & 16) + 4 * (lane & 3);
          const uint2 x0 = lds_read_tr16(at), x1 = lds_read_tr16(at + 4 * kVStride<DH>);
          vf = make_uint4(x0.x, x0.y, x1.x, x1.y);
        }
#pragma unroll
        for (int k = NT - 1; k >= 0; --k) st.o[n] = mfma32(as_bf16x8(vf), as_bf16x8(wt[s][k]), st.o[n]);
      }
    }
    if constexpr (!Q8) wave_lds_sync();  // the tile's buffer is written again
  };
  if constexpr (Q8) {
    // two tiles' registers in turn: the next one is loaded while one is worked on
    Tile<Q8, DH> other;
    while (tile < t_end) {
      if (tile + stride < t_end) load_codes(other, tile + stride);
      work(nxt);
      tile += stride;
      if (tile >= t_end) break;
      if (tile + stride < t_end) load_codes(nxt, tile + stride);
      work(other);
      tile += stride;
    }
  } else {
    for (; tile < t_end; tile += stride) work(nxt);
  }
  st.l = xor32_sum(st.l);
}

// q of an own unit: column 4 g + t holds term t of head g (t = 3: zeros).  Held in registers; beside
// two tiles of the 8-bit cache there is no room, each lane keeps its operands in LDS.
template <bool Q8, int DH>
struct OwnQuery {
  uint4 f[Q8 ? 1 : DH / 16];
  uint4* mine;  // Q8: this lane's, 64 apart

  __device__ __forceinline__ uint4 at(int s, int) const {
    if constexpr (Q8)
      return mine[64 * s];
    else
      return f[s];
  }
  // row: the first head's q
  __device__ __forceinline__ void load(const float* row, int heads, float scale, int lane) {
    const int g = (lane & 31) >> 2, t = lane & 3, h = lane >> 5;
    const uint32_t drop1 = t >= 1 ? 0xffff0000u : 0u, drop2 = t >= 2 ? 0xffff0000u : 0u;
    const bool in = g < heads && t < 3;
    const float* from = row + static_cast<long>(min(g, heads - 1)) * DH;
    // all of it on its way before any is worked on, and no branch between
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    f4 raw[DH / 8];
#pragma unroll
    for (int i = 0; i < DH / 8; ++i)
      raw[i] = *reinterpret_cast<const f4*>(from + dim_of<Q8>(i >> 1, h) + 4 * (i & 1));
#pragma unroll
    for (int s = 0; s < DH / 16; ++s) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = in ? raw[2 * s + (e >> 2)][e & 3] * scale : 0.0f;
        x[e] -= __uint_as_float(__float_as_uint(x[e]) & drop1);
        x[e] -= __uint_as_float(__float_as_uint(x[e]) & drop2);
      }
      const uint4 op = make_uint4(upper2(x[0], x[1]), upper2(x[2], x[3]), upper2(x[4], x[5]),
                                  upper2(x[6], x[7]));
      if constexpr (Q8)
        mine[64 * s] = op;
      else
        f[s] = op;
    }
  }
};

// An own unit: one wave, up to 8 heads of one stream, a range of its keys.
template <bool Q8, int DH>
__device__ __forceinline__ void own_unit(const SharedArgs& a, long unit, uint16_t* vt, uint4* lds_q,
                                         int lane) {
  // units beside each other are the heads of one range: what they read lies side by side
  const int chunk = static_cast<int>(unit % a.own_chunks);
  unit /= a.own_chunks;
  const int kvh = static_cast<int>(unit % a.p.Hkv);
  unit /= a.p.Hkv;
  const int part = static_cast<int>(unit % a.n_own);
  if (unit / a.n_own >= a.p.B) return;
  const int b = static_cast<int>(unit / a.n_own);
  // every n_own-th tile from the one that the prefix ends in: where the wave begins does not depend on
  // the stream's length, which comes from memory with the pages
  const int P = a.p.shared_len;
  int first = P, row_b = b, tile = P / kTile + part;
  TilePages pages;
  pages.fetch(a.map, row_b, tile, a.n_own, lane);
  const int S = stream_len(a, b);
  if (S < P) {  // uniform
    first = 0, row_b = 0, tile = part;
    pages.fetch(a.map, row_b, tile, a.n_own, lane);
  }
  const int heads = min(a.G - chunk * kOwnHeads, kOwnHeads);
  const long head0 = static_cast<long>(b) * a.p.Hq + kvh * a.G + chunk * kOwnHeads;
  ColState<DH> st;
  OwnQuery<Q8, DH> q;
  q.mine = lds_q + lane;
  attend_tiles<Q8, DH, true>(st, a, row_b, kvh, first, S, tile, a.n_own, pages, vt, lane, q, [&](bool any) {
    if (any) q.load(a.p.q + head0 * DH, heads, a.scale_log2e, lane);
  });
  const int g = (lane & 31) >> 2, t = lane & 3, h = lane >> 5;
  const long ps = (head0 + g) * a.slots + a.n_pre + part;
#pragma unroll
  for (int i = 0; i < DH / 32; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = quad_sum(t == 3 ? 0.0f : st.o[i][4 * r + e]);
      if (t == r && g < heads)
        *reinterpret_cast<float4*>(a.part_o + ps * DH + 32 * i + 8 * r + 4 * h) =
            make_float4(x[0], x[1], x[2], x[3]);
    }
  if (lane < 32 && t == 0 && g < heads) {
    a.part_ml[2 * ps] = st.m;
    a.part_ml[2 * ps + 1] = st.l;
  }
}

// q of a prefix unit's columns as three terms in LDS.
template <bool Q8, int DH>
struct PrefixQuery {
  static constexpr size_t kTerm = kCols * kQStride<DH>;  // elements of a term
  const uint16_t* col;  // this lane's column
  int h;
  __device__ __forceinline__ uint4 at(int s, int k) const {
    return *reinterpret_cast<const uint4*>(col + k * kTerm + dim_of<Q8>(s, h));
  }
};

template <bool Q8, int DH>
__global__ __launch_bounds__(64 * kWaves, 2) void shared_attn_kernel(SharedArgs a) {
  constexpr int ND = DH / 32;
  constexpr int OS = DH + 4;   // floats of an output row in LDS
  constexpr size_t kQTerm = PrefixQuery<Q8, DH>::kTerm;
  constexpr size_t kQBytes = 3 * kQTerm * 2;
  constexpr size_t kVBytes = Q8 ? 0 : kTile * kVStride<DH> * 2;
  constexpr size_t kOBytes = kCols * OS * 4;
  // q's terms and the waves' bf16 tiles; then the waves' outputs
  constexpr size_t kWork = kQBytes + kWaves * kVBytes;
  __shared__ __align__(16) unsigned char smem[kWork > kWaves * kOBytes ? kWork : kWaves * kOBytes];
  __shared__ float s_m[kWaves][kCols], s_l[kWaves][kCols];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, col = lane & 31;
  const int G = a.G, Hq = a.p.Hq, Hkv = a.p.Hkv, P = a.p.shared_len;
  uint16_t* vt = reinterpret_cast<uint16_t*>(smem + kQBytes + wave * kVBytes);

  // ---- the unit: the prefix's first, they are the longer ones ----
  const unsigned n_prefix = static_cast<unsigned>(a.col_blocks) * a.n_pre * Hkv;
  if (blockIdx.x >= n_prefix) {
    constexpr int kOps = 64 * (DH / 16);  // 16-byte operands of a wave's q
    static_assert(!Q8 || kWaves * kOps * 16 <= sizeof(smem), "the waves' q take the outputs' place");
    own_unit<Q8, DH>(a, static_cast<long>(blockIdx.x - n_prefix) * kWaves + wave, vt,
                     reinterpret_cast<uint4*>(smem) + wave * kOps, lane);
    return;
  }
  const int kvh = blockIdx.x % Hkv, u = blockIdx.x / Hkv;
  const int part = u / a.col_blocks, first_row = (u % a.col_blocks) * kCols;
  // (in 64 bits: the last range's end may pass 2^31)
  const long from = static_cast<long>(part) * a.pre_tiles * kTile;
  const int lo = static_cast<int>(min(from, static_cast<long>(P)));
  const int hi = static_cast<int>(min(from + static_cast<long>(a.pre_tiles) * kTile, static_cast<long>(P)));
  // stream and head (of the kv head's G) of column c; false: there is none
  auto column = [&](int c, int* b, int* g) {
    *b = (first_row + c) / G;
    *g = (first_row + c) % G;
    return *b < a.p.B;
  };
  ColState<DH> st;
  uint16_t* qt = reinterpret_cast<uint16_t*>(smem);
  const PrefixQuery<Q8, DH> q{qt + col * kQStride<DH>, h};
  const int tile = lo / kTile + wave;
  TilePages pages;
  pages.fetch(a.map, 0, tile, kWaves, lane);
  attend_tiles<Q8, DH, false>(st, a, 0, kvh, lo, hi, tile, kWaves, pages, vt, lane, q, [&](bool) {
    // rows of columns; columns that there are not hold zeros.  Every load is on its way before the first
    // is waited for
    constexpr int N = kCols * (DH / 8) / (64 * kWaves);
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    f4 raw[N][2];
    bool in[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = tid + j * 64 * kWaves;
      int b, g;
      in[j] = column(i / (DH / 8), &b, &g);
      const float* row = a.p.q + (static_cast<long>(min(b, a.p.B - 1)) * Hq + kvh * G + g) * DH +
                         8 * (i % (DH / 8));
      raw[j][0] = *reinterpret_cast<const f4*>(row);
      raw[j][1] = *reinterpret_cast<const f4*>(row + 4);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = tid + j * 64 * kWaves, c = i / (DH / 8), d = 8 * (i % (DH / 8));
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = in[j] ? raw[j][e >> 2][e & 3] * a.scale_log2e : 0.0f;
      uint4 t[3];
      split3(x, t);
#pragma unroll
      for (int k = 0; k < 3; ++k)
        *reinterpret_cast<uint4*>(qt + k * kQTerm + c * kQStride<DH> + d) = t[k];
    }
    lds_barrier();  // the first tile's loads stay on the way
  });

  // ---- the waves joined in LDS ----
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem + wave * kOBytes);
  if (h == 0) {
    s_m[wave][col] = st.m;
    s_l[wave][col] = st.l;
  }
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<float4*>(so + col * OS + 32 * n + 8 * r + 4 * h) =
          make_float4(st.o[n][4 * r], st.o[n][4 * r + 1], st.o[n][4 * r + 2], st.o[n][4 * r + 3]);
  __syncthreads();
  const float* all = reinterpret_cast<const float*>(smem);
  for (int i = tid; i < kCols * (DH / 4); i += 64 * kWaves) {
    const int c = i / (DH / 4), d = 4 * (i % (DH / 4));
    int b, g;
    if (!column(c, &b, &g)) continue;
    float M = -INFINITY, L = 0.0f;
    float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_m[w][c]);
    // a stream that is no column of the prefix leaves nothing there
    const bool none = stream_len(a, b) < P;
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = fast_exp2(s_m[w][c] - ref);
      const float4 x = *reinterpret_cast<const float4*>(all + w * (kOBytes / 4) + c * OS + d);
      L = fmaf(f, s_l[w][c], L);
      r.x = fmaf(f, x.x, r.x);
      r.y = fmaf(f, x.y, r.y);
      r.z = fmaf(f, x.z, r.z);
      r.w = fmaf(f, x.w, r.w);
    }
    const long ps = (static_cast<long>(b) * Hq + kvh * G + g) * a.slots + part;
    if (none) {
      M = -INFINITY;
      L = 0.0f;
      r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    *reinterpret_cast<float4*>(a.part_o + ps * DH + d) = r;
    if (d == 0) {
      a.part_ml[2 * ps] = M;
      a.part_ml[2 * ps + 1] = L;
    }
  }
}

// One wave per (stream, head): out = sum_j 2^(m_j - M) o_j / sum_j 2^(m_j - M) l_j over its slots.
template <int DH>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a) {
  const int lane = threadIdx.x & 63;
  const long row = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= static_cast<long>(a.p.B) * a.p.Hq) return;
  constexpr int E = DH / 64, kBatch = 16;
  float M = -INFINITY, L = 0.0f, o[E] = {};
  for (int s0 = 0; s0 < a.slots; s0 += 64) {
    const bool in = s0 + lane < a.slots;
    const long ps = row * a.slots + s0 + lane;
    const float m = in ? a.part_ml[2 * ps] : -INFINITY;
    const float l = in ? a.part_ml[2 * ps + 1] : 0.0f;
    const float mn = fmaxf(M, wave_max(m));
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float c = fast_exp2(M - ref), w = fast_exp2(m - ref);
    M = mn;
    L = fmaf(L, c, wave_sum(w * l));
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= c;
    const int n = min(64, a.slots - s0);
    for (int j0 = 0; j0 < n; j0 += kBatch) {  // a batch of loads on the way at a time
      float x[kBatch][E];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e)
          x[j][e] = a.part_o[(row * a.slots + s0 + min(j0 + j, n - 1)) * DH + 64 * e + lane];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const float wj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), min(j0 + j, n - 1)));
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (j0 + j < n) o[e] = fmaf(wj, x[j][e], o[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.p.out[row * DH + 64 * e + lane] = L == 0.0f ? 0.0f : o[e] / L;
}

template <bool Q8, int DH>
int launch(const SharedArgs& a, unsigned grid, hipStream_t stream) {
  hipLaunchKernelGGL((shared_attn_kernel<Q8, DH>), dim3(grid), dim3(64 * kWaves), 0, stream, a);
  if (int rc = check_launch("shared_attn_kernel")) return rc;
  const long rows = static_cast<long>(a.p.B) * a.p.Hq;
  hipLaunchKernelGGL((shared_merge_kernel<DH>), dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0,
                     stream, a);
  return check_launch("shared_merge_kernel");
}

}  // namespace

int launch_shared_prefix(const KeysProblem& p, const Q8Map& map, hipStream_t stream) {
  SharedArgs a{};
  a.p = p;
  a.map = map;
  a.scale_log2e = p.scale * 1.4426950408889634f;
  a.G = p.Hq / p.Hkv;
  const long rows = static_cast<long>(p.B) * a.G;
  a.col_blocks = static_cast<int>((rows + kCols - 1) / kCols);
  a.own_chunks = (a.G + kOwnHeads - 1) / kOwnHeads;
  const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
  // Prefix units of at least one tile per wave, up to one workgroup per CU; own units, a wave each, of
  // at least a tile, as many as fill what is left of the two workgroups per CU that run at once.
  const long tiles = (p.shared_len + kTile - 1) / kTile;
  const long pre_units = static_cast<long>(a.col_blocks) * p.Hkv;
  long n_pre = tiles == 0 ? 0 : std::clamp(cus / pre_units, 1L, (tiles + kWaves - 1) / kWaves);
  a.pre_tiles = n_pre ? static_cast<int>((tiles + n_pre - 1) / n_pre) : 0;
  a.n_pre = a.pre_tiles ? static_cast<int>((tiles + a.pre_tiles - 1) / a.pre_tiles) : 0;
  const long own = (static_cast<long>(map.capacity) - p.shared_len + kTile - 1) / kTile + 1;
  const long own_units = static_cast<long>(p.B) * a.own_chunks;
  const long room = kWaves * (2 * cus - pre_units * a.n_pre);
  a.n_own = static_cast<int>(std::clamp(room / (own_units * p.Hkv), 1L, std::min<long>(own, kMaxOwn)));
  a.slots = a.n_pre + a.n_own;
  const long grid = pre_units * a.n_pre + (own_units * p.Hkv * a.n_own + kWaves - 1) / kWaves;
  if (grid > kMaxGroups256)
    return fail(ORATOR_ERR_UNSUPPORTED, "gqa_decode_shared: too many streams and heads");
  const size_t parts = static_cast<size_t>(p.B) * p.Hq * a.slots;
  char* ws = static_cast<char*>(workspace_graph(stream, parts * (p.Dh + 2) * sizeof(float), kWsKeys));
  if (!ws) return ORATOR_ERR_HIP;
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = a.part_o + parts * p.Dh;
  const unsigned g = static_cast<unsigned>(grid);
  if (p.bf16) return p.Dh == 128 ? launch<false, 128>(a, g, stream) : launch<false, 64>(a, g, stream);
  return p.Dh == 128 ? launch<true, 128>(a, g, stream) : launch<true, 64>(a, g, stream);
}

}  // namespace orator_hip
