// Paged KV cache (b2d_paged_kv): argument checks and the page lookup shared by csrc/paged_append.cu and
// csrc/paged_attention.cu.
#pragma once

#include "common.cuh"

namespace b2d {

constexpr int kMaxPageSize = 1024;

// An int32 from L2, in its place among the waits: lengths and page tables may be written on the device (b2d_page_plan) by a kernel
// that had not begun when this one, behind other dependent launches, became resident, which the read-only path and lines that this
// SM's L1 holds from before need not show.
__device__ __forceinline__ int load_l2(const int32_t* p) {
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];\n" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Position -> (page index, slot). Pages of a power of two take a shift; the others a division.
struct PageDiv {
  int size, shift;   // shift < 0: not a power of two
  __device__ __forceinline__ int page(int pos) const { return shift >= 0 ? pos >> shift : pos / size; }
  __device__ __forceinline__ int slot(int pos, int page) const { return pos - page * size; }
};

inline PageDiv page_div(int size) {
  int shift = -1;
  if ((size & (size - 1)) == 0)
    for (shift = 0; (1 << shift) < size; ++shift) {}
  return PageDiv{size, shift};
}

inline int check_paged_kv(const b2d_paged_kv* kv) {
  if (!kv || kv->num_pages < 0 || kv->KVH < 0 || kv->D < 0) return B2D_ERR_ARG;
  if (kv->dtype != B2D_F16 && kv->dtype != B2D_BF16) return B2D_ERR_DTYPE;
  if (kv->page_size < 1 || kv->page_size > kMaxPageSize || kv->KVH == 0) return B2D_ERR_SHAPE;
  if (kv->num_pages > 0 && (!kv->k || !kv->v)) return B2D_ERR_ARG;
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16) ||
      (kv->sk_p | kv->sk_h | kv->sk_s | kv->sv_p | kv->sv_h | kv->sv_s) % 8)
    return B2D_ERR_ALIGN;
  return B2D_OK;
}

}  // namespace b2d
