// Rotary embedding of new tokens (optionally behind an RMS norm of each query and key head) and the append
// of their keys and values to a paged cache, one pass (sm_100a). The contiguous-cache counterpart is
// rope_kv_append_kernel in decode_glue.cu, which reproduces the torch ops' intermediate roundings; here
// every intermediate stays in fp32 and the result is rounded once.
//
// Per head x of D elements: x' = x * rsqrt(mean(x^2) + eps) * w; y = x' * cos + rotate_half(x') * sin.
// D/16 neighbouring threads own a head: thread j holds elements [8j, 8j + 8) and [D/2 + 8j, D/2 + 8j + 8),
// the two halves that the rotation pairs, in two 16-byte loads; the mean is a shuffle over the group.
// Bound by bytes (2 (H + 2 KVH) D elements a token), by latency for a few tokens.
#include "paged.cuh"

namespace b2d {
namespace {

struct PagedAppendArgs {
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
  b2d_paged_kv kv;
  PageDiv div;
  int N, H, B, per_seq, pages_per_seq, S_max;
};

constexpr int kAppendThreads = 128;

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = Dt<T>::to_f32(h[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Dt<T>::pack2(f[0], f[1]), Dt<T>::pack2(f[2], f[3]), Dt<T>::pack2(f[4], f[5]),
                    Dt<T>::pack2(f[6], f[7]));
}
// 8 table values (the rotary tables are in the cache's dtype or in fp32)
template <typename C>
__device__ __forceinline__ void load8(const C* p, float (&f)[8]) {
  if constexpr (sizeof(C) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    unpack8<C>(__ldg(reinterpret_cast<const uint4*>(p)), f);
  }
}

// T: cache and activation dtype, C: rotary table type, GROUP: threads of a head (a power of two >= D/16)
template <typename T, typename C, int GROUP>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedAppendArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int heads = a.H + 2 * a.kv.KVH;
  const int64_t item = (blockIdx.x * static_cast<int64_t>(kAppendThreads) + threadIdx.x) / GROUP;
  const int j = threadIdx.x % GROUP;
  const int64_t n = item / heads;
  const int hd = static_cast<int>(item - n * heads);
  const int D = a.kv.D, half = D / 2;
  bool live = n < a.N && 8 * j < half;
  int64_t seq = -1, pos = -1;
  if (live) {
    pos = a.positions[n];
    seq = a.seq_ids ? a.seq_ids[n] : n / a.per_seq;
    live = seq >= 0 && seq < a.B && pos >= 0 && pos < a.S_max;
  }
  const bool is_q = hd < a.H, is_k = !is_q && hd < a.H + a.kv.KVH;
  const int h = is_q ? hd : is_k ? hd - a.H : hd - a.H - a.kv.KVH;
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  T* dst = nullptr;
  if (live) {
    const T* src = is_q   ? static_cast<const T*>(a.q) + n * a.sq_n + h * a.sq_h
                   : is_k ? static_cast<const T*>(a.k) + n * a.sk_n + h * a.sk_h
                          : static_cast<const T*>(a.v) + n * a.sv_n + h * a.sv_h;
    lo = *reinterpret_cast<const uint4*>(src + 8 * j);
    hi = *reinterpret_cast<const uint4*>(src + half + 8 * j);
    if (is_q) {
      dst = static_cast<T*>(a.q_out) + n * a.sqo_n + h * a.sqo_h;
    } else {
      const int p = static_cast<int>(pos), pi = a.div.page(p);
      const int page = pi < a.pages_per_seq ? a.table[seq * a.ld_table + pi] : -1;
      if (page >= 0 && page < a.kv.num_pages) {
        const int slot = a.div.slot(p, pi);
        dst = is_k ? static_cast<T*>(a.kv.k) + page * a.kv.sk_p + h * a.kv.sk_h + slot * a.kv.sk_s
                   : static_cast<T*>(a.kv.v) + page * a.kv.sv_p + h * a.kv.sv_h + slot * a.kv.sv_s;
      }
    }
  }
  float x1[8], x2[8];
  unpack8<T>(lo, x1);
  unpack8<T>(hi, x2);
  const T* weight = static_cast<const T*>(is_q ? a.q_weight : is_k ? a.k_weight : nullptr);
  if (a.q_weight || a.k_weight) {   // uniform over the launch: every lane takes the shuffles
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x1[i], x1[i], fmaf(x2[i], x2[i], ss));
#pragma unroll
    for (int o = GROUP / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (weight && live) {
      const float rstd = rsqrtf(ss / static_cast<float>(D) + a.eps);
      float w1[8], w2[8];
      load8(weight + 8 * j, w1);
      load8(weight + half + 8 * j, w2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x1[i] *= rstd * w1[i];
        x2[i] *= rstd * w2[i];
      }
    }
  }
  if (!dst) return;
  if (is_q || is_k) {
    float c1[8], c2[8], s1[8], s2[8];
    const C* cs = static_cast<const C*>(a.cos) + pos * a.ld_cs + 8 * j;
    const C* sn = static_cast<const C*>(a.sin) + pos * a.ld_cs + 8 * j;
    load8(cs, c1);
    load8(cs + half, c2);
    load8(sn, s1);
    load8(sn + half, s2);
    float y1[8], y2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y1[i] = fmaf(x1[i], c1[i], -x2[i] * s1[i]);
      y2[i] = fmaf(x2[i], c2[i], x1[i] * s2[i]);
    }
    lo = pack8<T>(y1);
    hi = pack8<T>(y2);
  }
  *reinterpret_cast<uint4*>(dst + 8 * j) = lo;
  *reinterpret_cast<uint4*>(dst + half + 8 * j) = hi;
}

template <typename T, typename C>
int launch_append(const PagedAppendArgs& a, bool pdl, cudaStream_t s) {
  const int group = a.kv.D <= 64 ? 4 : a.kv.D <= 128 ? 8 : 16;
  const int64_t threads = static_cast<int64_t>(a.N) * (a.H + 2 * a.kv.KVH) * group;
  const int64_t blocks = (threads + kAppendThreads - 1) / kAppendThreads;
  if (blocks > (int64_t(1) << 31) - 1) return B2D_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(blocks)), block(kAppendThreads);
  if (group == 4) return launch_kernel(paged_append_kernel<T, C, 4>, grid, block, 0, s, pdl, a);
  if (group == 8) return launch_kernel(paged_append_kernel<T, C, 8>, grid, block, 0, s, pdl, a);
  return launch_kernel(paged_append_kernel<T, C, 16>, grid, block, 0, s, pdl, a);
}

}  // namespace
}  // namespace b2d

using namespace b2d;

extern "C" int b2d_paged_rope_append(const b2d_paged_kv* kv, const void* q, int64_t sq_n, int64_t sq_h,
                                     const void* k, int64_t sk_n, int64_t sk_h, const void* v, int64_t sv_n,
                                     int64_t sv_h, const int64_t* positions, const int32_t* seq_ids,
                                     const int32_t* page_table, int64_t ld_table, int pages_per_seq, int B,
                                     const void* cos, const void* sin, int64_t ld_cs, int S_max, int cs_dtype,
                                     const void* q_weight, const void* k_weight, float eps, void* q_out,
                                     int64_t sqo_n, int64_t sqo_h, int N, int H, int flags, void* stream) {
  int st;
  if ((st = check_paged_kv(kv)) != B2D_OK) return st;
  if (N < 0 || H < 0 || B < 0 || S_max < 0 || pages_per_seq < 0) return B2D_ERR_ARG;
  if (cs_dtype != kv->dtype && cs_dtype != B2D_F32) return B2D_ERR_DTYPE;
  if (kv->D % 16 != 0 || kv->D < 16 || kv->D > 256 || H % kv->KVH != 0) return B2D_ERR_SHAPE;
  if (N == 0) return B2D_OK;
  if (B == 0 || (!seq_ids && N % B != 0) || ld_table < 0 || ld_cs < 0) return B2D_ERR_SHAPE;
  if (!q || !k || !v || !positions || !page_table || !cos || !sin || !q_out) return B2D_ERR_ARG;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) || !aligned(cos, 16) ||
      !aligned(sin, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(positions, 8) ||
      !aligned(page_table, 4) || !aligned(seq_ids, 4) ||
      (sq_n | sq_h | sk_n | sk_h | sv_n | sv_h | sqo_n | sqo_h | ld_cs) % 8)
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  if ((st = device_info(&di)) != B2D_OK) return st;
  PagedAppendArgs a{q, sq_n, sq_h, k, sk_n, sk_h, v, sv_n, sv_h, positions, seq_ids, page_table, ld_table, cos, sin,
                    ld_cs, q_weight, k_weight, eps, q_out, sqo_n, sqo_h, *kv, page_div(kv->page_size), N, H, B,
                    seq_ids ? 1 : N / B, pages_per_seq, S_max};
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0, f32 = cs_dtype == B2D_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kv->dtype == B2D_F16)
    return f32 ? launch_append<__half, float>(a, pdl, s) : launch_append<__half, __half>(a, pdl, s);
  return f32 ? launch_append<__nv_bfloat16, float>(a, pdl, s) : launch_append<__nv_bfloat16, __nv_bfloat16>(a, pdl, s);
}
