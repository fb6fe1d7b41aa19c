// Rotary embedding of new tokens (optionally behind an RMS norm of each query and key head) and the append
// of their keys and values to a paged cache, one pass (sm_100a). The contiguous-cache counterpart is
// rope_kv_append_kernel in decode_glue.cu, which reproduces the torch ops' intermediate roundings; here
// every intermediate stays in fp32 and the result is rounded once.
//
// Per head x of D elements: x' = x * rsqrt(mean(x^2) + eps) * w; y = x' * cos + rotate_half(x') * sin.
// D/16 neighbouring threads own a head: thread j holds elements [8j, 8j + 8) and [D/2 + 8j, D/2 + 8j + 8),
// the two halves that the rotation pairs, as two 16-byte chunks; the mean is a shuffle over the group. A block of
// 64 threads takes one token after another (for few tokens: a part of one token's heads). The next token's
// heads are always under way: every thread copies its own chunks through two private stages of shared memory
// (16-byte cp.async), so no thread waits for another. The products w * cos and w * sin are formed once per
// thread and token and serve all of its heads.
// Measured on B200: 8168 tokens of 32 + 8 + 8 heads of 128 with norms, bf16: 46.3 us, 4.35 TB/s of read and written
// bytes (copy rate 6.55; without the look at the sums of squares 45.1); 320 tokens 4.9 us; one token 2.4 us (launch and latency). Bound by bytes in the limit,
// 2 (H + 2 KVH) D elements a token. What is left at 8168 tokens is latency: 16.7 warps per SM are active (shared
// memory allows 9 blocks) and issue in half of the slots. One head per thread took 49 us, three stages 51, four-element
// halves 58 to 63 with 80 % of the slots issuing.
#include <type_traits>

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

constexpr int kAppendThreads = 64;
constexpr int kAppendStages = 2;

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
// 8 values of a rotary table (the cache's dtype or fp32) or of a weight. No kernel of the library, which alone start their dependents
// early, writes those: the read-only path may take them (by ordinary loads 8 x 1021 tokens 46.3 -> 48.8 us).
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

// y1 = r (x1 a1 - x2 b1), y2 = r (x2 a2 + x1 b2), r the norm's factor
struct Turn {
  float a1[8], b1[8], a2[8], b2[8];
};
template <typename T, typename C>
__device__ __forceinline__ void load_turn(const PagedAppendArgs& a, int64_t pos, int j, const void* weight, Turn& t) {
  const int half = a.kv.D / 2;
  const C* cs = static_cast<const C*>(a.cos) + pos * a.ld_cs + 8 * j;
  const C* sn = static_cast<const C*>(a.sin) + pos * a.ld_cs + 8 * j;
  load8(cs, t.a1);
  load8(cs + half, t.a2);
  load8(sn, t.b1);
  load8(sn + half, t.b2);
  if (weight) {
    float w1[8], w2[8];
    load8(static_cast<const T*>(weight) + 8 * j, w1);
    load8(static_cast<const T*>(weight) + half + 8 * j, w2);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t.a1[e] *= w1[e];
      t.b1[e] *= w2[e];
      t.a2[e] *= w2[e];
      t.b2[e] *= w1[e];
    }
  }
}

// One head's pair of 16-byte chunks.
struct Pair {
  uint4 lo, hi;
};
template <typename T>
__device__ __forceinline__ Pair load_pair(const T* head, int j, int half) {
  return Pair{*reinterpret_cast<const uint4*>(head + 8 * j), *reinterpret_cast<const uint4*>(head + half + 8 * j)};
}
template <typename T>
__device__ __forceinline__ void store_pair(const Pair& p, T* head, int j, int half) {
  *reinterpret_cast<uint4*>(head + 8 * j) = p.lo;
  *reinterpret_cast<uint4*>(head + half + 8 * j) = p.hi;
}
// Norm (every lane of the warp takes part in the shuffles) and rotation.
template <typename T, int GROUP>
__device__ __forceinline__ Pair turn_pair(const Pair& p, const Turn& t, bool norm, float inv_d, float eps) {
  float x1[8], x2[8], r = 1.f;
  unpack8<T>(p.lo, x1);
  unpack8<T>(p.hi, x2);
  if (norm) {
    auto squares = [&] {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x1[e], x1[e], fmaf(x2[e], x2[e], ss));
#pragma unroll
      for (int o = GROUP / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      return ss;
    };
    float ss = squares();
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      // squares that leave fp32 (elements of 2^60 and more, or none above 2^-40 and no eps to speak of): the head times 2^-70 or 2^80
      const float least = eps < 0x1p-60f ? 0x1p-80f : 0.f;
      if (__any_sync(0xffffffffu, !(ss >= least && ss <= 0x1p120f))) {
        const float f = ss > 0x1p120f ? 0x1p-70f : ss < least ? 0x1p80f : 1.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x1[e] *= f;
          x2[e] *= f;
        }
        ss = squares();
        eps = eps * f * f;
      }
    }
    r = rsqrtf(fmaf(ss, inv_d, eps));
  }
  float y1[8], y2[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y1[e] = fmaf(x1[e], t.a1[e], -x2[e] * t.b1[e]) * r;
    y2[e] = fmaf(x2[e], t.a2[e], x1[e] * t.b2[e]) * r;
  }
  return Pair{pack8<T>(y1), pack8<T>(y2)};
}

// T: cache and activation dtype, C: rotary table type, GROUP: threads of a head (a power of two >= D/16),
// HEADS: query heads of a thread that are staged (0: a block has one token, whose first heads are loaded straight
// into registers: 2.4 against 3.3 us for a single token). The groups of a token's blocks (blockIdx.y) take the query
// heads in turn; the first groups also the keys, the last ones the values. Heads past the staged ones are
// loaded when their turn comes.
template <typename T, typename C, int GROUP, int HEADS>
__global__ void __launch_bounds__(kAppendThreads, HEADS == 0 ? 4 : 9) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
  constexpr int GROUPS = kAppendThreads / GROUP, CHUNKS = 2 * (HEADS + 2);   // staged chunks: queries, key, value
  constexpr int TRIP = HEADS > 0 ? HEADS : 1;
  extern __shared__ uint4 s_chunk[];                                        // [stage][chunk][thread]
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, j = tid % GROUP, step = GROUPS * gridDim.y;
  const int group = static_cast<int>(blockIdx.y) * GROUPS + tid / GROUP, vgroup = step - 1 - group;
  const int KVH = a.kv.KVH, half = a.kv.D / 2;
  const bool on = 8 * j < half;
  const float inv_d = 1.f / static_cast<float>(a.kv.D);
  const int64_t hop = gridDim.x;
  // this thread's chunks of the token that is fetched next
  const T* qf = static_cast<const T*>(a.q) + blockIdx.x * a.sq_n + group * a.sq_h + 8 * j;
  const T* kf = static_cast<const T*>(a.k) + blockIdx.x * a.sk_n + group * a.sk_h + 8 * j;
  const T* vf = static_cast<const T*>(a.v) + blockIdx.x * a.sv_n + vgroup * a.sv_h + 8 * j;
  const int64_t q_step = step * a.sq_h;
  uint4* const chunk = s_chunk + tid;   // + (stage CHUNKS + c) kAppendThreads
  Pair direct[3] = {};   // query, key, value of the only token
  if constexpr (HEADS == 0) {
    if (on && group < a.H) direct[0] = Pair{*reinterpret_cast<const uint4*>(qf), *reinterpret_cast<const uint4*>(qf + half)};
    if (on && group < KVH) direct[1] = Pair{*reinterpret_cast<const uint4*>(kf), *reinterpret_cast<const uint4*>(kf + half)};
    if (on && vgroup < KVH) direct[2] = Pair{*reinterpret_cast<const uint4*>(vf), *reinterpret_cast<const uint4*>(vf + half)};
  }
  if (HEADS > 0 && !on)   // lanes past the head's end add zeros to its mean
    for (int c = 0; c < kAppendStages * CHUNKS; ++c) chunk[c * kAppendThreads] = make_uint4(0, 0, 0, 0);
  auto fetch = [&](int stage, bool any) {   // heads that do not exist leave their chunks as they are
    if (on && any) {
      const uint32_t dst = smem_u32(chunk + stage * CHUNKS * kAppendThreads);
      auto pair = [&](int slot, const T* src) {
        cp_async16(dst + (2 * slot) * kAppendThreads * 16, src);
        cp_async16(dst + (2 * slot + 1) * kAppendThreads * 16, src + half);
      };
#pragma unroll
      for (int i = 0; i < HEADS; ++i)
        if (group + i * step < a.H) pair(i, qf + i * q_step);
      if (group < KVH) pair(HEADS, kf);
      if (vgroup < KVH) pair(HEADS + 1, vf);
      qf += hop * a.sq_n;
      kf += hop * a.sk_n;
      vf += hop * a.sv_n;
    }
    cp_async_commit();
  };
  int64_t next_pos = a.positions[blockIdx.x];
  if constexpr (HEADS > 0) fetch(0, true);
  int stage = 0;
  for (int64_t n = blockIdx.x; n < a.N; n += hop, stage ^= 1) {
    const int64_t pos = next_pos;
    const int seq = a.seq_ids ? a.seq_ids[n] : static_cast<int>(n) / a.per_seq;
    const bool more = n + hop < a.N;
    if (more) next_pos = a.positions[n + hop];
    if constexpr (HEADS > 0) {
      fetch(stage ^ 1, more);
      cp_async_wait<1>();   // this thread's own copies of token n
    }
    const uint4* const now = chunk + stage * CHUNKS * kAppendThreads;
    auto staged = [&](int slot) {
      if constexpr (HEADS == 0) return direct[slot];
      else return Pair{now[2 * slot * kAppendThreads], now[(2 * slot + 1) * kAppendThreads]};
    };
    if (seq < 0 || seq >= a.B || pos < 0 || pos >= a.S_max) continue;   // padding: the whole block
    const int p = static_cast<int>(pos), pi = a.div.page(p), slot = a.div.slot(p, pi);
    const int page = pi < a.pages_per_seq ? a.table[static_cast<int64_t>(seq) * a.ld_table + pi] : -1;
    const bool paged = page >= 0 && page < a.kv.num_pages;
    Turn t;
    if (on) load_turn<T, C>(a, pos, j, a.q_weight, t);
    T* const qd = static_cast<T*>(a.q_out) + n * a.sqo_n;
    for (int h0 = 0; h0 < a.H; h0 += TRIP * step) {   // the same trips for every lane
#pragma unroll
      for (int i = 0; i < TRIP; ++i) {
        const int h = h0 + group + i * step;
        Pair x = staged(i);
        if (h0 > 0 && on && h < a.H) x = load_pair(static_cast<const T*>(a.q) + n * a.sq_n + h * a.sq_h, j, half);
        const Pair y = turn_pair<T, GROUP>(x, t, a.q_weight != nullptr, inv_d, a.eps);
        if (on && h < a.H) store_pair(y, qd + h * a.sqo_h, j, half);
      }
    }
    if (!paged) continue;
    if (on) {
      T* const vd = static_cast<T*>(a.kv.v) + page * a.kv.sv_p + slot * a.kv.sv_s;
      for (int h = vgroup; h < KVH; h += step)
        store_pair(h == vgroup ? staged(TRIP + 1) : load_pair(static_cast<const T*>(a.v) + n * a.sv_n + h * a.sv_h, j, half),
                   vd + h * a.kv.sv_h, j, half);
    }
    const int warp_first = group - (tid & 31) / GROUP;   // uniform for the warp's lanes
    if (warp_first >= KVH) continue;
    if (on && a.k_weight != a.q_weight) load_turn<T, C>(a, pos, j, a.k_weight, t);
    T* const kd = static_cast<T*>(a.kv.k) + page * a.kv.sk_p + slot * a.kv.sk_s;
    for (int h0 = warp_first; h0 < KVH; h0 += step) {
      const int h = h0 + group - warp_first;
      Pair x = staged(TRIP);
      if (h0 > warp_first && on && h < KVH) x = load_pair(static_cast<const T*>(a.k) + n * a.sk_n + h * a.sk_h, j, half);
      const Pair y = turn_pair<T, GROUP>(x, t, a.k_weight != nullptr, inv_d, a.eps);
      if (on && h < KVH) store_pair(y, kd + h * a.kv.sk_h, j, half);
    }
  }
  if constexpr (HEADS > 0) cp_async_wait<0>();
}

template <typename T, typename C, int GROUP, int HEADS>
int launch_kernel_of(const PagedAppendArgs& a, dim3 grid, bool pdl, cudaStream_t s) {
  constexpr size_t bytes = HEADS == 0 ? 0 : static_cast<size_t>(kAppendStages) * 2 * (HEADS + 2) * kAppendThreads * 16;   // <= 24 KB
  return launch_kernel(paged_append_kernel<T, C, GROUP, HEADS>, grid, dim3(kAppendThreads), bytes, s, pdl, a);
}
template <typename T, typename C, int GROUP>
int launch_group(const PagedAppendArgs& a, int sm, bool pdl, cudaStream_t s) {
  constexpr int GROUPS = kAppendThreads / GROUP;
  int parts = (a.H + GROUPS - 1) / GROUPS;
  if (parts < 1) parts = 1;
  // few tokens: a token's heads over several blocks, one query head a thread (one token 2.4 us against 3.3 staged, 320 tokens
  // of 32 heads 4.85 against 5.05; 8168 tokens staged 45, direct 50)
  if (static_cast<int64_t>(a.N) * parts <= 24 * sm) return launch_kernel_of<T, C, GROUP, 0>(a, dim3(a.N, parts), pdl, s);
  if (parts == 1) return launch_kernel_of<T, C, GROUP, 1>(a, dim3(a.N < 16 * sm ? a.N : 16 * sm), pdl, s);
  if (parts == 2) return launch_kernel_of<T, C, GROUP, 2>(a, dim3(a.N < 12 * sm ? a.N : 12 * sm), pdl, s);
  return launch_kernel_of<T, C, GROUP, 4>(a, dim3(a.N < 9 * sm ? a.N : 9 * sm), pdl, s);
}
template <typename T, typename C>
int launch_append(const PagedAppendArgs& a, int sm, bool pdl, cudaStream_t s) {
  if (a.kv.D <= 64) return launch_group<T, C, 4>(a, sm, pdl, s);
  if (a.kv.D <= 128) return launch_group<T, C, 8>(a, sm, pdl, s);
  return launch_group<T, C, 16>(a, sm, pdl, s);
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
  if (kv->D % 16 != 0 || kv->D < 16 || kv->D > 256 || H % kv->KVH != 0 || H > 65535) return B2D_ERR_SHAPE;
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
    return f32 ? launch_append<__half, float>(a, di.sm_count, pdl, s)
               : launch_append<__half, __half>(a, di.sm_count, pdl, s);
  return f32 ? launch_append<__nv_bfloat16, float>(a, di.sm_count, pdl, s)
             : launch_append<__nv_bfloat16, __nv_bfloat16>(a, di.sm_count, pdl, s);
}
