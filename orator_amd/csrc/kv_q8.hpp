// The KV cache in 8 bits: where its codes and scales lie (kernels), and the checks of its
// arguments (launchers).
//
// A page holds page_size positions of every kv head, in blocks of 16 positions:
//   K codes [page][Hkv][page_size / 16][16][Dh]   a block's rows, one after the other
//   V codes [page][Hkv][page_size / 16][Dh][16]   a block with the dims outside
//   scales  [page][Hkv][page_size / 16][16]
// so block number (page * Hkv + head) * blocks_per_page + block_in_page gives all four addresses.
// V is held transposed because the attention sums over positions: 16 positions of one dim are
// then 16 consecutive bytes, one lane's operand of the 64-deep int8 MFMA, and no kernel
// transposes V.  Scales are apart from the codes, a block's 16 together: 64 bytes per block and
// head, where one scale per [row][head] would spread them over 16 lines.
#pragma once

#include "common.hpp"
#include "internal.hpp"

namespace orator_hip {

constexpr int kQ8Block = 16;   // positions per block
constexpr int kQ8MaxDh = 256;

struct Q8Map {
  const int* page_table;  // nullptr: contiguous, one page
  int max_pages;
  int block_shift;        // log2 of the blocks per page (paged)
  int n_pages;
  int Hkv;
  int capacity;           // positions a stream can hold

  // Page of stream b's block `blk` (blk * 16 < capacity), paged caches; -1 if it is unmapped.
  __device__ __forceinline__ int page(int b, int blk) const {
    const int pg = page_table[static_cast<long>(b) * max_pages + (blk >> block_shift)];
    return pg < 0 || pg >= n_pages ? -1 : pg;
  }
  // Number of stream b's block `blk` of head h; -1 if its page is unmapped.
  __device__ __forceinline__ long block(int b, int blk, int h) const {
    if (!page_table) return static_cast<long>(h) * (capacity / kQ8Block) + blk;
    const int pg = page(b, blk);
    if (pg < 0) return -1;
    return ((static_cast<long>(pg) * Hkv + h) << block_shift) + (blk & ((1 << block_shift) - 1));
  }
};

inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Largest capacity a launch takes: positions and their successors stay ints.
constexpr long kQ8MaxCapacity = 0x7fffff00L;

// Workgroups of 256 threads in one dimension of a grid, which holds fewer than 2^32 threads.
constexpr long kMaxGroups256 = (1L << 24) - 1;

// Checks a cache's shape and fills the map (page_table null: contiguous); what: the entry's name.
inline int q8_map(Q8Map* m, const char* what, const int* page_table, bool paged, int max_pages,
                  int page_size, int n_pages, int Hkv, int Dh, int capacity) {
  const std::string who(what);
  if (Dh % kQ8Block || Dh > kQ8MaxDh)
    return fail(ORATOR_ERR_UNSUPPORTED, who + ": Dh must be a multiple of 16, at most 256");
  m->page_table = paged ? page_table : nullptr;
  m->Hkv = Hkv;
  m->max_pages = max_pages;
  m->n_pages = n_pages;
  m->block_shift = 0;
  if (paged) {
    if (!page_table) return fail(ORATOR_ERR_INVALID, who + ": null page table");
    const int shift = ilog2_exact(page_size);
    if (shift < 4) return fail(ORATOR_ERR_INVALID, who + ": page_size must be a power of two >= 16");
    if (max_pages <= 0 || n_pages <= 0)
      return fail(ORATOR_ERR_INVALID, who + ": max_pages and n_pages must be > 0");
    m->block_shift = shift - 4;
    const long cap = static_cast<long>(max_pages) << shift;
    m->capacity = static_cast<int>(cap < kQ8MaxCapacity ? cap : kQ8MaxCapacity);
  } else {
    if (capacity <= 0 || capacity % kQ8Block || capacity > kQ8MaxCapacity)
      return fail(ORATOR_ERR_INVALID, who + ": capacity must be a positive multiple of 16");
    m->capacity = capacity;
  }
  return ORATOR_OK;
}

inline int q8_pointers(const char* what, const void* kq, const void* ks, const void* vq,
                       const void* vs) {
  if (!kq || !ks || !vq || !vs) return fail(ORATOR_ERR_INVALID, std::string(what) + ": null cache");
  if (!aligned_to(kq, 16) || !aligned_to(ks, 16) || !aligned_to(vq, 16) || !aligned_to(vs, 16))
    return fail(ORATOR_ERR_INVALID, std::string(what) + ": caches must be 16-byte aligned");
  return ORATOR_OK;
}

}  // namespace orator_hip
