// Append to the 4-bit paged cache (norm, rotation, quantisation) and the read back of its values (sm_100a); the layout is in
// int4_kv.cuh, the 16-bit counterpart in paged_append.cu.
//
// D / 16 neighbouring lanes own a head, 16 elements each as two chunks of 8 that hold whole rotation pairs: [8 j, 8 j + 8) and
// [R / 2 + 8 j, ...) for the half layout's turning elements, 16 neighbouring ones otherwise. A warp takes a token (or, for few
// tokens, a part of one): its query heads four (D = 128) or eight at a time, then the keys, then the values.
// The next heads' loads are issued before the present ones are worked on; the tables' factors of a token are loaded once.
//  * q: fp32, one rounding.
//  * k: the mean in 64 bits and every product and sum rounded as the definition says (no contraction), so that a code is the
//    formula's and not its neighbour; the row passes through shared memory to the order of the runs, 16 neighbouring
//    elements a lane, where a run's extrema are one or two shuffles and the codes of a lane are a step of the fragment order.
//  * v: loaded in that order at once. A position's codes lie in single bytes (the other bytes of a word are other
//    positions'), which L2 merges.
#include "int4_kv.cuh"

namespace b2d {
namespace {

struct Int4AppendArgs {
  const void* q; int64_t sq_n, sq_h;
  const void* k; int64_t sk_n, sk_h;
  const void* v; int64_t sv_n, sv_h;
  const int64_t* positions;
  const int32_t* seq_ids;
  const int32_t* table; int64_t ld_table;
  const void* cos; const void* sin; int64_t ld_cs;
  const void* q_weight; const void* k_weight;
  float eps;
  void* q_out; int64_t sqo_n, sqo_h;
  b2d_int4_kv kv;
  PageDiv div;
  int N, H, B, per_seq, pages_per_seq, rotary, interleaved, parts;
  int64_t limit;   // positions from here on are padding
};

constexpr int kWarps = 4;

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float* f) {
  const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = Dt<T>::to_f32(h[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(Dt<T>::pack2(f[0], f[1]), Dt<T>::pack2(f[2], f[3]), Dt<T>::pack2(f[4], f[5]), Dt<T>::pack2(f[6], f[7]));
}
template <typename C>
__device__ __forceinline__ void load8(const C* p, float* f) {
  if constexpr (sizeof(C) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    unpack8<C>(__ldg(reinterpret_cast<const uint4*>(p)), f);
  }
}

struct Chunks {
  uint4 a, b;
};

// A token's rotation factors of a lane's eight pairs.
struct Turn {
  float c[8], s[8];
};

// (a, b) -> (a c - b s, b c + a s) for a lane's pairs; EXACT: every product and sum rounded by itself
template <bool EXACT>
__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
  const float a0 = a, b0 = b;
  if constexpr (EXACT) {
    a = __fsub_rn(__fmul_rn(a0, c), __fmul_rn(b0, s));
    b = __fadd_rn(__fmul_rn(b0, c), __fmul_rn(a0, s));
  } else {
    a = fmaf(a0, c, -b0 * s);
    b = fmaf(b0, c, a0 * s);
  }
}
template <bool EXACT>
__device__ __forceinline__ void turn(float (&x)[16], const Turn& t, bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < 8; ++e) turn_pair<EXACT>(x[2 * e], x[2 * e + 1], t.c[e], t.s[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) turn_pair<EXACT>(x[e], x[8 + e], t.c[e], t.s[e]);
  }
}

// 16 neighbouring elements of a run's lanes -> {s, m} and the codes
template <typename T>
__device__ __forceinline__ uint32_t quantise(const float (&x)[16], int run_lanes, uint32_t (&code)[16]) {
  float lo = x[0], hi = x[0], odd = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    odd = fmaf(x[e], 0.f, odd);   // NaN once an element is infinite or NaN
  }
  for (int o = 1; o < run_lanes; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    odd += __shfl_xor_sync(0xffffffffu, odd, o);
  }
  const T mt = Dt<T>::from_f32(lo);
  const float m = Dt<T>::to_f32(mt);
  const T st = Dt<T>::from_f32(fmaxf(__fdiv_rn(__fsub_rn(hi, m), 15.f), 0.f));
  const float s = Dt<T>::to_f32(st);
  const bool sound = odd == 0.f && fabsf(m) < INFINITY && s < INFINITY;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float c = s > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[e], m), s)) : 0.f;
    code[e] = sound ? static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f)) : 0u;
  }
  if (!sound) return Dt<T>::pack2(NAN, NAN);
  return Dt<T>::pack2(s, m);
}

// T: cache and activation dtype, C: the tables' type
template <typename T, typename C, int D>
__global__ void __launch_bounds__(kWarps * 32) int4_append_kernel(const __grid_constant__ Int4AppendArgs a) {
  constexpr int LANES = D / 16, HPW = 32 / LANES;   // lanes of a head, heads of a warp
  __shared__ __align__(16) float s_row[kWarps][HPW][D];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = lane % LANES, sub = lane / LANES;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  const int64_t n = unit / a.parts;
  const int part = static_cast<int>(unit - n * a.parts);
  if (n >= a.N) return;
  const int64_t pos = a.positions[n];
  const int seq = a.seq_ids ? a.seq_ids[n] : static_cast<int>(n) / a.per_seq;
  if (seq < 0 || seq >= a.B || pos < 0 || pos >= a.limit) return;   // padding
  const int KVH = a.kv.KVH, run_lanes = a.kv.group / 16, runs = D / a.kv.group;
  const int q_items = a.q ? (a.H + HPW - 1) / HPW : 0, kv_items = (KVH + HPW - 1) / HPW, items = q_items + 2 * kv_items;
  // the lane's chunks: of the turning elements, of the rest
  const bool turns = a.cos && 16 * j < a.rotary, halves = turns && !a.interleaved;
  const int o1 = halves ? 8 * j : 16 * j, o2 = halves ? a.rotary / 2 + 8 * j : 16 * j + 8;

  auto load = [&](int item) {
    Chunks x{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (item < q_items) {
      const int h = item * HPW + sub;
      if (h < a.H) {
        const T* p = static_cast<const T*>(a.q) + n * a.sq_n + h * a.sq_h;
        x.a = *reinterpret_cast<const uint4*>(p + o1);
        x.b = *reinterpret_cast<const uint4*>(p + o2);
      }
    } else if (item < items) {
      const bool key = item < q_items + kv_items;
      const int h = (item - q_items - (key ? 0 : kv_items)) * HPW + sub;
      if (h < KVH) {
        const T* p = key ? static_cast<const T*>(a.k) + n * a.sk_n + h * a.sk_h : static_cast<const T*>(a.v) + n * a.sv_n + h * a.sv_h;
        x.a = __ldg(reinterpret_cast<const uint4*>(p + (key ? o1 : 16 * j)));
        x.b = __ldg(reinterpret_cast<const uint4*>(p + (key ? o2 : 16 * j + 8)));
      }
    }
    return x;
  };
  Chunks next = load(part);
  // where the token's entries go
  int page = -1, tile_row = 0;
  const uint8_t* head0 = nullptr;
  if (pos < static_cast<int64_t>(a.pages_per_seq) * a.kv.page_size) {
    const int p = static_cast<int>(pos), pi = a.div.page(p);
    page = a.table[static_cast<int64_t>(seq) * a.ld_table + pi];
    if (page >= a.kv.num_pages) page = -1;
    if (page >= 0) {
      const int slot = a.div.slot(p, pi);
      tile_row = slot % kTileKeys;
      head0 = a.kv.pages + page * a.kv.sp_p + static_cast<int64_t>(slot / kTileKeys) * int4_tile_bytes(D, runs);
    }
  }
  Turn t;
  if (turns) {
    load8(static_cast<const C*>(a.cos) + pos * a.ld_cs + 8 * j, t.c);
    load8(static_cast<const C*>(a.sin) + pos * a.ld_cs + 8 * j, t.s);
  }
  float w[16];
  const void* loaded = nullptr;   // the weights in w
  for (int item = part; item < items; item += a.parts) {
    const Chunks now = next;
    next = load(item + a.parts);
    float x[16];
    unpack8<T>(now.a, x);
    unpack8<T>(now.b, x + 8);
    if (item < q_items + kv_items) {   // norm and rotation
      const bool key = item >= q_items;
      const void* weight = key ? a.k_weight : a.q_weight;
      if (weight) {
        if (weight != loaded) {
          load8(static_cast<const T*>(weight) + o1, w);
          load8(static_cast<const T*>(weight) + o2, w + 8);
          loaded = weight;
        }
        float r;
        if (key) {
          double ss = 0.0;
#pragma unroll
          for (int e = 0; e < 16; ++e) ss = fma(static_cast<double>(x[e]), static_cast<double>(x[e]), ss);
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          r = static_cast<float>(rsqrt(ss / D + static_cast<double>(a.eps)));
        } else {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          r = rsqrtf(fmaf(ss, 1.f / D, a.eps));
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], r), w[e]);
      }
      if (!key) {
        if (turns) turn<false>(x, t, a.interleaved);
        const int h = item * HPW + sub;
        if (h < a.H) {
          T* p = static_cast<T*>(a.q_out) + n * a.sqo_n + h * a.sqo_h;
          *reinterpret_cast<uint4*>(p + o1) = pack8<T>(x);
          *reinterpret_cast<uint4*>(p + o2) = pack8<T>(x + 8);
        }
        continue;
      }
      if (turns) turn<true>(x, t, a.interleaved);
    }
    if (page < 0) continue;   // the whole warp
    const bool key = item < q_items + kv_items;
    const int h = (item - q_items - (key ? 0 : kv_items)) * HPW + sub;
    uint8_t* const tile = const_cast<uint8_t*>(head0) + h * a.kv.sp_h;
    uint32_t code[16];
    if (key) {
      if (a.cos && !a.interleaved) {   // into neighbouring elements
        float* row = s_row[warp][sub];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          *reinterpret_cast<float4*>(row + o1 + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
          *reinterpret_cast<float4*>(row + o2 + e) = make_float4(x[8 + e], x[9 + e], x[10 + e], x[11 + e]);
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 y = *reinterpret_cast<const float4*>(row + 16 * j + e);
          x[e] = y.x; x[e + 1] = y.y; x[e + 2] = y.z; x[e + 3] = y.w;
        }
        __syncwarp();
      }
      const uint32_t sm = quantise<T>(x, run_lanes, code);
      // lane j has step j: one byte of each half of the words (t', j / 2), t' = 0..3; the pair of lanes joins them
      uint32_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        v[u] = code[4 * u] | code[4 * u + 2] << 4 | code[4 * u + 1] << 16 | code[4 * u + 3] << 20;
      const bool upper = j & 1;
      const uint32_t r0 = __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[2], 1);
      const uint32_t r1 = __shfl_xor_sync(0xffffffffu, upper ? v[1] : v[3], 1);
      if (h < KVH) {
        uint8_t* row = tile + tile_row * (D / 2) + (upper ? 2 : 0) * (D / 8) + 4 * (j / 2);
        *reinterpret_cast<uint32_t*>(row) = upper ? r0 | v[2] << 8 : v[0] | r0 << 8;
        *reinterpret_cast<uint32_t*>(row + D / 8) = upper ? r1 | v[3] << 8 : v[1] | r1 << 8;
        if (j % run_lanes == 0)
          *reinterpret_cast<uint32_t*>(tile + int4_ks_off(D) + (tile_row * runs + j / run_lanes) * 4) = sm;
      }
    } else {
      const uint32_t sm = quantise<T>(x, run_lanes, code);
      if (h < KVH) {
        uint8_t* p = tile + int4_v_off(D) + (j / 4) * 512 + ((tile_row % 8) / 2) * 16 + (j % 4) * 4 + (tile_row & 1) * 2 + tile_row / 8;
#pragma unroll
        for (int g = 0; g < 8; ++g) p[g * 64] = static_cast<uint8_t>(code[g] | code[g + 8] << 4);
        if (j % run_lanes == 0)
          *reinterpret_cast<uint32_t*>(tile + int4_vs_off(D, runs) + (tile_row * runs + j / run_lanes) * 4) = sm;
      }
    }
  }
}

struct Int4ReadArgs {
  const int64_t* positions;
  const int32_t* seq_ids;
  const int32_t* table; int64_t ld_table;
  void* k; int64_t sk_n, sk_h;
  void* v; int64_t sv_n, sv_h;
  b2d_int4_kv kv;
  PageDiv div;
  int N, B, per_seq, pages_per_seq, parts;
};

// The inverse, lane for lane: 16 neighbouring elements of a head from the step's bytes. O: output type.
template <typename T, typename O, int D>
__global__ void __launch_bounds__(kWarps * 32) int4_read_kernel(const __grid_constant__ Int4ReadArgs a) {
  constexpr int LANES = D / 16, HPW = 32 / LANES;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = lane % LANES, sub = lane / LANES;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  const int64_t n = unit / a.parts;
  const int part = static_cast<int>(unit - n * a.parts);
  if (n >= a.N) return;
  const int64_t pos = a.positions[n];
  const int seq = a.seq_ids ? a.seq_ids[n] : static_cast<int>(n) / a.per_seq;
  if (seq < 0 || seq >= a.B || pos < 0 || pos >= static_cast<int64_t>(a.pages_per_seq) * a.kv.page_size) return;
  const int KVH = a.kv.KVH, run_lanes = a.kv.group / 16, runs = D / a.kv.group;
  const int k_items = a.k ? (KVH + HPW - 1) / HPW : 0, items = k_items + (a.v ? (KVH + HPW - 1) / HPW : 0);
  const int p = static_cast<int>(pos), pi = a.div.page(p), slot = a.div.slot(p, pi), row = slot % kTileKeys;
  const int page = a.table[static_cast<int64_t>(seq) * a.ld_table + pi];
  const bool there = page >= 0 && page < a.kv.num_pages;
  const uint8_t* head0 = a.kv.pages + (there ? page * a.kv.sp_p + static_cast<int64_t>(slot / kTileKeys) * int4_tile_bytes(D, runs) : 0);
  for (int item = part; item < items; item += a.parts) {
    const bool key = item < k_items;
    const int h = (item - (key ? 0 : k_items)) * HPW + sub;
    if (h >= KVH) continue;
    float x[16];
    if (there) {
      const uint8_t* tile = head0 + h * a.kv.sp_h;
      uint32_t code[16];
      const uint32_t sm = __ldg(reinterpret_cast<const uint32_t*>(tile + (key ? int4_ks_off(D) : int4_vs_off(D, runs)) + (row * runs + j / run_lanes) * 4));
      if (key) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(tile + row * (D / 2) + u * (D / 8) + 4 * (j / 2))) >> 8 * (j & 1);
          code[4 * u] = w & 15;
          code[4 * u + 1] = w >> 16 & 15;
          code[4 * u + 2] = w >> 4 & 15;
          code[4 * u + 3] = w >> 20 & 15;
        }
      } else {
        const uint8_t* b = tile + int4_v_off(D) + (j / 4) * 512 + ((row % 8) / 2) * 16 + (j % 4) * 4 + (row & 1) * 2 + row / 8;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const uint32_t w = __ldg(b + g * 64);
          code[g] = w & 15;
          code[g + 8] = w >> 4;
        }
      }
      const float2 f = unpack_sm<T>(sm);
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = fmaf(f.x, static_cast<float>(code[e]), f.y);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 0.f;
    }
    O* o = static_cast<O*>(key ? a.k : a.v) + n * (key ? a.sk_n : a.sv_n) + h * (key ? a.sk_h : a.sv_h) + 16 * j;
    if constexpr (sizeof(O) == 4) {
#pragma unroll
      for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(o + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
    } else {
      *reinterpret_cast<uint4*>(o) = pack8<O>(x);
      *reinterpret_cast<uint4*>(o + 8) = pack8<O>(x + 8);
    }
  }
}

// Warps a token: enough for a few per scheduler, at most one per item.
int warps_per_token(int64_t N, int items, int sm) {
  int parts = 1;
  while (parts < items && N * parts < static_cast<int64_t>(sm) * 128) parts *= 2;
  return parts < items ? parts : items;
}

template <typename T, typename C, int D>
int launch_append(Int4AppendArgs& a, int sm, bool pdl, cudaStream_t s) {
  constexpr int HPW = 512 / D;
  const int items = (a.q ? (a.H + HPW - 1) / HPW : 0) + 2 * ((a.kv.KVH + HPW - 1) / HPW);
  a.parts = warps_per_token(a.N, items, sm);
  const int64_t blocks = (static_cast<int64_t>(a.N) * a.parts + kWarps - 1) / kWarps;
  if (blocks > INT32_MAX) return B2D_ERR_SHAPE;
  return launch_kernel(int4_append_kernel<T, C, D>, dim3(static_cast<unsigned>(blocks)), dim3(kWarps * 32), 0, s, pdl, a);
}
template <typename T, typename O, int D>
int launch_read(Int4ReadArgs& a, int sm, bool pdl, cudaStream_t s) {
  constexpr int HPW = 512 / D;
  a.parts = warps_per_token(a.N, ((a.k ? 1 : 0) + (a.v ? 1 : 0)) * ((a.kv.KVH + HPW - 1) / HPW), sm);
  const int64_t blocks = (static_cast<int64_t>(a.N) * a.parts + kWarps - 1) / kWarps;
  if (blocks > INT32_MAX) return B2D_ERR_SHAPE;
  return launch_kernel(int4_read_kernel<T, O, D>, dim3(static_cast<unsigned>(blocks)), dim3(kWarps * 32), 0, s, pdl, a);
}

int check_tokens(const b2d_int4_kv* kv, const int32_t* seq_ids, int N, int B, int64_t ld_table, int pages_per_seq) {
  if (B == 0 || (!seq_ids && N % B != 0) || ld_table < 0) return B2D_ERR_SHAPE;
  if (static_cast<int64_t>(pages_per_seq) * kv->page_size > (int64_t(1) << 31) - 1024) return B2D_ERR_SHAPE;
  return B2D_OK;
}

}  // namespace
}  // namespace b2d

using namespace b2d;

extern "C" size_t b2d_int4_page_bytes(int page_size, int D, int group) {
  return int4_sizes(page_size, D, group) ? static_cast<size_t>(page_size / kTileKeys) * int4_tile_bytes(D, D / group) : 0;
}

extern "C" int b2d_int4_append(const b2d_int4_kv* kv, const void* q, int64_t sq_n, int64_t sq_h, const void* k, int64_t sk_n,
                               int64_t sk_h, const void* v, int64_t sv_n, int64_t sv_h, const int64_t* positions,
                               const int32_t* seq_ids, const int32_t* page_table, int64_t ld_table, int pages_per_seq, int B,
                               const void* cos, const void* sin, int64_t ld_cs, int S_max, int cs_dtype, int rotary_dim,
                               int interleaved, const void* q_weight, const void* k_weight, float eps, void* q_out,
                               int64_t sqo_n, int64_t sqo_h, int N, int H, int flags, void* stream) {
  int st;
  if ((st = check_int4_kv(kv)) != B2D_OK) return st;
  if (N < 0 || H < 0 || B < 0 || pages_per_seq < 0 || (cos && (S_max < 0 || rotary_dim < 0))) return B2D_ERR_ARG;
  if (cos && cs_dtype != kv->dtype && cs_dtype != B2D_F32) return B2D_ERR_DTYPE;
  if (q && (H % kv->KVH != 0 || H > 65535)) return B2D_ERR_SHAPE;
  if (cos && (rotary_dim % 16 != 0 || rotary_dim < 16 || rotary_dim > kv->D)) return B2D_ERR_SHAPE;
  if (N == 0) return B2D_OK;
  if ((st = check_tokens(kv, seq_ids, N, B, ld_table, pages_per_seq)) != B2D_OK) return st;
  if (!k || !v || !positions || (!page_table && pages_per_seq > 0) || !cos != !sin || (q && !q_out) || (cos && ld_cs < 0)) return B2D_ERR_ARG;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) || !aligned(cos, 16) || !aligned(sin, 16) ||
      !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(positions, 8) || !aligned(page_table, 4) ||
      !aligned(seq_ids, 4) || (sk_n | sk_h | sv_n | sv_h) % 8 || (q && (sq_n | sq_h | sqo_n | sqo_h) % 8) ||
      (cos && ld_cs % (cs_dtype == B2D_F32 ? 4 : 8)))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  if ((st = device_info(&di)) != B2D_OK) return st;
  Int4AppendArgs a{q, sq_n, sq_h, k, sk_n, sk_h, v, sv_n, sv_h, positions, seq_ids, page_table, ld_table, cos, sin, ld_cs,
                   q_weight, k_weight, eps, q_out, sqo_n, sqo_h, *kv, page_div(kv->page_size), N, H, B, seq_ids ? 1 : N / B,
                   pages_per_seq, cos ? rotary_dim : 0, interleaved != 0, 1, cos ? S_max : INT64_MAX};
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0, f32 = cos && cs_dtype == B2D_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sm = di.sm_count;
  if (kv->dtype == B2D_F16) {
    if (kv->D == 64) return f32 ? launch_append<__half, float, 64>(a, sm, pdl, s) : launch_append<__half, __half, 64>(a, sm, pdl, s);
    return f32 ? launch_append<__half, float, 128>(a, sm, pdl, s) : launch_append<__half, __half, 128>(a, sm, pdl, s);
  }
  if (kv->D == 64)
    return f32 ? launch_append<__nv_bfloat16, float, 64>(a, sm, pdl, s) : launch_append<__nv_bfloat16, __nv_bfloat16, 64>(a, sm, pdl, s);
  return f32 ? launch_append<__nv_bfloat16, float, 128>(a, sm, pdl, s) : launch_append<__nv_bfloat16, __nv_bfloat16, 128>(a, sm, pdl, s);
}

extern "C" int b2d_int4_read(const b2d_int4_kv* kv, const int64_t* positions, const int32_t* seq_ids, const int32_t* page_table,
                             int64_t ld_table, int pages_per_seq, int B, void* k_out, int64_t sk_n, int64_t sk_h, void* v_out,
                             int64_t sv_n, int64_t sv_h, int out_dtype, int N, int flags, void* stream) {
  int st;
  if ((st = check_int4_kv(kv)) != B2D_OK) return st;
  if (N < 0 || B < 0 || pages_per_seq < 0) return B2D_ERR_ARG;
  if (out_dtype != kv->dtype && out_dtype != B2D_F32) return B2D_ERR_DTYPE;
  if (N == 0 || (!k_out && !v_out)) return B2D_OK;
  if ((st = check_tokens(kv, seq_ids, N, B, ld_table, pages_per_seq)) != B2D_OK) return st;
  if (!positions || (!page_table && pages_per_seq > 0)) return B2D_ERR_ARG;
  if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(positions, 8) || !aligned(page_table, 4) || !aligned(seq_ids, 4) ||
      (k_out && (sk_n | sk_h) % 8) || (v_out && (sv_n | sv_h) % 8))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  if ((st = device_info(&di)) != B2D_OK) return st;
  Int4ReadArgs a{positions, seq_ids, page_table, ld_table, k_out, sk_n, sk_h, v_out, sv_n, sv_h, *kv,
                 page_div(kv->page_size), N, B, seq_ids ? 1 : N / B, pages_per_seq, 1};
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0, f32 = out_dtype == B2D_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sm = di.sm_count;
  if (kv->dtype == B2D_F16) {
    if (kv->D == 64) return f32 ? launch_read<__half, float, 64>(a, sm, pdl, s) : launch_read<__half, __half, 64>(a, sm, pdl, s);
    return f32 ? launch_read<__half, float, 128>(a, sm, pdl, s) : launch_read<__half, __half, 128>(a, sm, pdl, s);
  }
  if (kv->D == 64) return f32 ? launch_read<__nv_bfloat16, float, 64>(a, sm, pdl, s) : launch_read<__nv_bfloat16, __nv_bfloat16, 64>(a, sm, pdl, s);
  return f32 ? launch_read<__nv_bfloat16, float, 128>(a, sm, pdl, s) : launch_read<__nv_bfloat16, __nv_bfloat16, 128>(a, sm, pdl, s);
}
