// Paged KV cache in 4 bits (b2d_int4_kv): the layout of a tile, argument checks, and (de)quantisation shared by
// csrc/int4_append.cu and csrc/int4_attention.cu.
//
// A tile holds 16 positions of one head, laid out as the attention's matrix fragments read it (mma.sync m16n8k16,
// lane = 4 g + t), so that a lane's operands are whole 16-byte words and every nibble becomes one half of a register by a
// mask alone: a nibble c in bits 0..3 of a half is the fp16 subnormal c 2^-24, in bits 4..7 it is c 2^-20, and the
// tensor cores take subnormals exactly. The powers of two are undone in fp32.
//   keys    row r (D / 2 bytes at r D / 2): lane t's D / 8 bytes are 32-bit words, each for two steps of 16 elements; step j's
//           elements 16 j + 4 t + e sit in half e & 1 of word j / 2, byte j & 1 of that half, low nibble for e < 2 and
//           high for e >= 2 (whose query factor carries the missing 2^-4).
//   values  words [D / 64][lane][4]: word of elements 16 mb + g (low nibbles) and 16 mb + g + 8 (high), whose bytes are the
//           positions 2 t, 2 t + 8, 2 t + 1, 2 t + 9.
//   {s, m}  of the keys, [position][run of `group` elements], then of the values.
#pragma once

#include "common.cuh"
#include "paged.cuh"

namespace b2d {

constexpr int kTileKeys = 16;

__host__ __device__ constexpr int int4_tile_bytes(int D, int runs) { return 16 * D + 128 * runs; }
__host__ __device__ constexpr int int4_v_off(int D) { return 8 * D; }
__host__ __device__ constexpr int int4_ks_off(int D) { return 16 * D; }
__host__ __device__ constexpr int int4_vs_off(int D, int runs) { return 16 * D + 64 * runs; }

inline bool int4_sizes(int page_size, int D, int group) {
  return (D == 64 || D == 128) && (group == 32 || group == 64) && page_size >= kTileKeys &&
         page_size <= kMaxPageSize && page_size % kTileKeys == 0;
}

inline int check_int4_kv(const b2d_int4_kv* kv) {
  if (!kv || kv->num_pages < 0 || kv->KVH < 0 || kv->D < 0) return B2D_ERR_ARG;
  if (kv->dtype != B2D_F16 && kv->dtype != B2D_BF16) return B2D_ERR_DTYPE;
  if (!int4_sizes(kv->page_size, kv->D, kv->group) || kv->KVH == 0 || kv->KVH > 65535) return B2D_ERR_SHAPE;
  if (kv->num_pages > 0 && !kv->pages) return B2D_ERR_ARG;
  if (!aligned(kv->pages, 16) || (kv->sp_p | kv->sp_h) % 16) return B2D_ERR_ALIGN;
  return B2D_OK;
}

// {s, m} as stored -> fp32
template <typename T>
__device__ __forceinline__ float2 unpack_sm(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack_sm<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack_sm<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

}  // namespace b2d
