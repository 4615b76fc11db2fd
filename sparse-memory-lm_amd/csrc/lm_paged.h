// The pages of a key-value cache as the kernels see them.
#pragma once

#include "pkm_common.h"

namespace smlm {

struct KVPages {
  void *k, *v, *k_scale, *v_scale;   // (pages, kv_heads, page, row); scales (pages, kv_heads, page) of bf16 step | lo << 16
  int64_t num_pages;
  int page_shift, kv_heads;

  // index of the row that holds kv head h of slot page id * page + offset
  __device__ __forceinline__ int64_t row(int64_t slot, uint32_t h) const {
    const int64_t page = slot >> page_shift;
    return ((page * kv_heads + h) << page_shift) + (slot - (page << page_shift));
  }
};

// Checks the pages of an entry point `name` and fills in what the kernels need; a status code.
int kv_pages(const char *name, const smlm_kv_pages *p, KVPages *out);

}  // namespace smlm
