// The paged KV cache of the generation path: what its kernels share.
//
// k_pages / v_pages: bf16 [n_pages][n_kv_heads][page_size][head_dim], pages `ld_page` elements apart. The rows of one head of one page are
// contiguous (page_size * head_dim * 2 bytes: 16 KiB for 64 tokens of width 128), so a key tile of the attention kernels is one straight
// piece of memory. Token j of sample b lies in page block_table[b][j / page_size], row j % page_size; page_size is a power of two >= 16.
// A table entry outside [0, n_pages) is a page that is not there: nothing is read or written through it and its tokens are masked.
#pragma once
#include <atomic>
#include "vm_common.hpp"

typedef __attribute__((ext_vector_type(4))) unsigned u32x4_t;

struct PagedKV {
  const unsigned short* k;
  const unsigned short* v;
  int64_t ld_page;
  const int32_t* table;
  int64_t ld_table;
  int n_pages, max_pages;
  int shift, mask;            // page_size = 1 << shift = mask + 1
  int n_kv_heads;
};

__device__ __forceinline__ bool page_ok(int page, int n_pages) { return (unsigned)page < (unsigned)n_pages; }

// element offset of row `row` of head `hk` of page `page` (64 bits: a pool may hold more than 2^31 elements)
__device__ __forceinline__ int64_t page_row(int page, int64_t ld_page, int hk, int row, int shift, int head_dim) {
  return (int64_t)page * ld_page + (((int64_t)hk << shift) + row) * head_dim;
}

// the page numbers of a sample, through the scalar cache (the table does not change while a kernel runs)
typedef const __attribute__((address_space(4))) int32_t* table_ptr;
__device__ __forceinline__ table_ptr table_of(const PagedKV& c, int seq) { return (table_ptr)(uintptr_t)(c.table + (int64_t)seq * c.ld_table); }

// (byte offset in 32 bits: one scalar load and no 64-bit address arithmetic; a sample's table is shorter than 2^29 bytes)
__device__ __forceinline__ int table_at(table_ptr t, int i) { return *(table_ptr)((const __attribute__((address_space(4))) char*)t + (unsigned)i * 4u); }

inline int paged_shift(int page_size) {          // log2 of a legal page size, -1 otherwise
  for (int s = 4; s <= 10; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

// allows `fn` that much dynamic LDS on the current device; once per device (`done`: a bit for each of the first 64)
inline bool allow_lds(const void* fn, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

inline bool misaligned16(const void* a) { return ((uintptr_t)a & 15) != 0; }

// the checks that every entry on the cache shares; fills `c`
inline int paged_cache(const vm_paged_kv* a, PagedKV& c) {
  if (!a || !a->k_pages || !a->v_pages || a->n_seq < 0 || (a->n_seq > 0 && !a->block_table)) return VM_ERR_BAD_ARG;
  if (a->n_pages <= 0 || a->max_pages <= 0 || a->n_kv_heads <= 0) return VM_ERR_BAD_ARG;
  if (a->head_dim != 32 && a->head_dim != 64 && a->head_dim != 128) return VM_ERR_UNSUPPORTED;
  const int shift = paged_shift(a->page_size);
  if (shift < 0) return VM_ERR_UNSUPPORTED;
  if (misaligned16(a->k_pages) || misaligned16(a->v_pages) || (a->ld_page & 7)) return VM_ERR_BAD_ARG;
  if (a->ld_page < (((int64_t)a->n_kv_heads << shift) * a->head_dim) || a->ld_table < a->max_pages) return VM_ERR_BAD_ARG;
  if (((int64_t)a->max_pages << shift) > 0x7FFFFFFF - 4096) return VM_ERR_UNSUPPORTED;
  c.k = (const unsigned short*)a->k_pages; c.v = (const unsigned short*)a->v_pages; c.ld_page = a->ld_page;
  c.table = a->block_table; c.ld_table = a->ld_table;
  c.n_pages = a->n_pages; c.max_pages = a->max_pages; c.shift = shift; c.mask = a->page_size - 1; c.n_kv_heads = a->n_kv_heads;
  return VM_OK;
}
