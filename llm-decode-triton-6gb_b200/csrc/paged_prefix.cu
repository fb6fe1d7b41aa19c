// Attention over a prefix that the whole batch shares, on the 5th-generation tensor cores (sm_100a): the
// queries of all sequences that read one KV head form one row axis, so the prefix is read once for up to 256
// rows and the two products are 128 x 128 x 128 matrix products. Used from more than 32 rows on (below, the
// mma.sync kernel of csrc/paged_attention.cu is bound by the same bytes); leaves (O, m, l) per row and split
// of the keys, which that file's per-sequence kernel takes in.
//
// A CTA owns (256 rows as two tiles of 128, KV head, split). Per tile of 128 keys and row tile:
//   S = Q K^T     tcgen05.mma kind::f16, M = N = 128, both operands K-major in shared memory, S in TMEM
//   softmax       one warpgroup per row tile, one thread per row (tcgen05.ld brings the row's 128 scores into
//                 registers); P is rounded to the cache's dtype and overwrites S in TMEM
//   O += P V      P from TMEM, V from shared memory (MN-major), O in TMEM
// One elected thread issues all products; while it works for one row tile, the other tile's warpgroup is in
// its softmax. With 128 rows or fewer both warpgroups take the same rows and alternate over the key tiles.
// The running maximum moves only when a score exceeds it by 2^8 (weights up to 256 are as exact in fp32 and
// in both 16-bit types), so O in TMEM is rarely rescaled. K and V come as 128-byte-swizzled tensor copies,
// page by page, through a ring of four 128-key tiles.
// TMEM columns: S/P of the two warpgroups at 0 and 128, their O at 256 and 256 + D.
#include <type_traits>

#include "paged_attention.cuh"
#include "pipeline.cuh"

namespace b2d {
namespace {

constexpr int kTile = 128;                  // keys of a tile, rows of a row tile
constexpr int kSoftmax = 256;               // softmax threads (two warpgroups)
constexpr int kProducer = 8, kIssuer = 9;   // warps
constexpr int kPrefixThreads = 384;         // the third warpgroup: producer, issuer, two idle warps
constexpr int kRing = 4;                    // K or V tiles in flight
constexpr uint32_t kTmemCols = 512;
constexpr float kLazy = 8.f;                // log2 of the largest weight before the maximum moves

__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
// 32 TMEM columns of this thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Shared-memory operand descriptors, 128-byte swizzle (layout type 2), descriptor version 1, tiles of
// 128-byte rows on 1024-byte boundaries. K-major: 8-row groups 1024 bytes apart. MN-major: the rows are the
// reduction axis in 8-row groups 1024 bytes apart, and columns of 64 elements are `column` bytes apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr, uint32_t column) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(column >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// kind::f16 instruction descriptor: fp32 accumulator, A and B of T, M = 128; A K-major, B K- or MN-major
template <typename T, int N, bool B_MN>
__host__ __device__ constexpr uint32_t idesc() {
  return (1u << 4) | ((std::is_same<T, __half>::value ? 0u : 1u) << 7) |
         ((std::is_same<T, __half>::value ? 0u : 1u) << 10) | ((B_MN ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
      : "memory");
}

template <int D>
constexpr uint32_t tile_bytes() { return kTile * D * 2; }
template <int D>
constexpr uint32_t prefix_smem() { return (2 + kRing) * tile_bytes<D>() + 1024; }

template <typename T, int D>
__global__ void __launch_bounds__(kPrefixThreads, 1) paged_prefix_kernel(const __grid_constant__ PoolMaps maps,
                                                                         const __grid_constant__ PagedAttnArgs a) {
  constexpr uint32_t TILEB = kTile * D * 2, COLB = kTile * 128;   // a K, V or Q tile; its 64-element column
  constexpr int HALVES = D / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * kRing + 7];
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* const smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  const uint32_t q_s = smem_u32(smem), ring = q_s + 2 * TILEB;
  const uint32_t full = smem_u32(s_bar), empty = full + 8 * kRing, s_full = empty + 8 * kRing, p_full = s_full + 16,
                 o_full = p_full + 16, q_full = o_full + 16;

  const int rows = a.B * a.rows;
  const bool pair = rows > kTile;          // two row tiles; else one, whose key tiles the warpgroups share
  const int kvh = blockIdx.y, split = blockIdx.x % a.splits, row0 = static_cast<int>(blockIdx.x) / a.splits * (2 * kTile);
  const int ktiles = (a.shared + kTile - 1) / kTile;
  const int t0 = ktiles * split / a.splits, n = ktiles * (split + 1) / a.splits - t0;   // this split's key tiles
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(s_full + 8 * w, 1);
      mbar_init(p_full + 8 * w, kTile);
      mbar_init(o_full + 8 * w, 1);
    }
    mbar_init(q_full, kSoftmax);
    fence_mbar_init();
  }
  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)),
                 "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (tid == 32 * kProducer) {
    prefetch_tensormap(&maps.k);
    prefetch_tensormap(&maps.v);
  }
  pdl_wait();
  pdl_launch_dependents();   // the dependent reads the same inputs: it starts once they are complete
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  // Registers: 168 a thread at launch (64,512 in all); the softmax takes 208 and the rest 80 (63,488).
  if (warp >= kProducer) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;\n");
  if (warp > kIssuer) {
  } else if (warp == kProducer) {
    // ---- K and V tiles in the order in which the issuer uses them; a lane per (64-element column, box)
    const int bp = a.box_rows, boxes = kTile / bp, col = lane / boxes, box = lane - col * boxes;
    int unit = 0;
    bool ok = true;
    auto load = [&](bool is_v, int tile) {
      const int tok = (t0 + tile) * kTile + box * bp, slot = unit % kRing;
      const bool live = col < HALVES && tok < a.shared;
      const int page = live ? __ldg(a.prefix_table + a.div.page(tok)) : -1;
      if (unit >= kRing) ok = ok && __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, (unit / kRing - 1) & 1));
      if (!ok) return;
      const uint32_t dst = ring + slot * TILEB + col * COLB + box * bp * 128;
      const bool copy = live && page >= 0 && page < a.kv.num_pages;
      if (live && !copy) {   // a page id outside the pool: zeros
        for (int i = 0; i < bp * 8; ++i)
          *reinterpret_cast<uint4*>(smem + (dst - q_s) + 16 * i) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();   // the tensor core reads them through the async proxy
      }
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, copy)) * bp * 128;
      __syncwarp();
      if (lane == 0) mbar_expect_tx(full + 8 * slot, bytes);
      __syncwarp();
      if (copy)
        tma_load_4d(dst, is_v ? &maps.v : &maps.k, 64 * col, a.div.slot(tok, a.div.page(tok)), kvh, page, full + 8 * slot);
      ++unit;
    };
    const int ahead = pair ? 1 : 2;   // score products that run ahead of the first P V
    for (int i = 0; i < ahead && i < n; ++i) load(false, i);
    for (int i = 0; i < n; ++i) {
      load(true, i);
      if (i + ahead < n) load(false, i + ahead);
    }
  } else if (warp == kIssuer) {
    if (lane == 0 && n > 0) {
      constexpr uint32_t ID_S = idesc<T, kTile, false>(), ID_O = idesc<T, D, true>();
      int unit = 0, done[2] = {0, 0};   // ring position; tiles whose P V is issued, per warpgroup
      auto take = [&]() -> uint32_t {
        const uint32_t slot = unit % kRing;
        mbar_wait(full + 8 * slot, (unit / kRing) & 1);
        ++unit;
        return slot;
      };
      auto scores = [&](int w, uint32_t slot) {   // S_w = Q K^T
        const uint32_t qa = q_s + (pair ? w * TILEB : 0u), kb = ring + slot * TILEB;
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
          mma_ss(tmem + 128 * w, desc_k_major(qa + (j >> 2) * COLB + (j & 3) * 32),
                 desc_k_major(kb + (j >> 2) * COLB + (j & 3) * 32), ID_S, j != 0);
        mma_commit(s_full + 8 * w);
      };
      auto values = [&](int w, uint32_t slot, int tile) {   // O_w += P_w V
        mbar_wait(p_full + 8 * w, done[w] & 1);
        tc_fence_after();
        const uint32_t vb = ring + slot * TILEB;
        const int steps = min(kTile, a.shared - (t0 + tile) * kTile) / 16;
        for (int j = 0; j < steps; ++j)
          mma_ts(tmem + 256 + D * w, tmem + 128 * w + 8 * j, desc_mn_major(vb + 2048 * j, COLB), ID_O,
                 done[w] != 0 || j != 0);
        ++done[w];
      };
      mbar_wait(q_full, 0);
      tc_fence_after();
      if (pair) {
        uint32_t ks = take();
        scores(0, ks);
        scores(1, ks);
        mma_commit(empty + 8 * ks);
        for (int i = 0; i < n; ++i) {
          const uint32_t vs = take();
          const bool more = i + 1 < n;
          values(0, vs, i);
          if (more) {
            ks = take();
            scores(0, ks);
          }
          values(1, vs, i);
          mma_commit(empty + 8 * vs);
          if (more) {
            scores(1, ks);
            mma_commit(empty + 8 * ks);
          }
        }
      } else {
        for (int i = 0; i < 2 && i < n; ++i) {
          const uint32_t ks = take();
          scores(i, ks);
          mma_commit(empty + 8 * ks);
        }
        for (int i = 0; i < n; ++i) {
          const uint32_t vs = take();
          values(i & 1, vs, i);
          mma_commit(empty + 8 * vs);
          if (i + 2 < n) {
            const uint32_t ks = take();
            scores(i & 1, ks);
            mma_commit(empty + 8 * ks);
          }
        }
      }
      mma_commit(o_full);
      mma_commit(o_full + 8);
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n");
    // ---- softmax: warpgroup w, thread = row (TMEM lane)
    const int w = warp >> 2, r = tid & (kTile - 1);
    const int row = row0 + (pair ? w * kTile : 0) + r;
    const bool live = row < rows;
    const int qb = row / a.rows, qr = row - qb * a.rows, t = qr / a.G, head = kvh * a.G + qr - t * a.G;
    if (pair || w == 0) {
      // this thread's row of Q into the K-major tile; a negative scale is moved into Q's sign
      const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + qb * a.sq_b + t * a.sq_t +
                                                        static_cast<int64_t>(head) * a.sq_h);
      uint8_t* dst = smem + (pair ? w * TILEB : 0u) + r * 128;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint4 x = live ? src[c] : make_uint4(0, 0, 0, 0);
        x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
        *reinterpret_cast<uint4*>(dst + (c >> 3) * COLB + (((c & 7) ^ (r & 7)) << 4)) = x;
      }
      fence_proxy_async();
    }
    mbar_arrive(q_full);
    const float scale = fabsf(a.scale_log2);
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t st = tmem + lanes + 128 * w, ot = tmem + lanes + 256 + D * w;
    const int mine = pair ? n : (n + 1 - w) / 2;   // key tiles of this warpgroup
    float m_run = 0.f, l[4] = {0.f, 0.f, 0.f, 0.f};
    bool landed = true;
    for (int i = 0; i < mine; ++i) {
      const int tile = pair ? i : 2 * i + w;
      const int valid = min(kTile, a.shared - (t0 + tile) * kTile);
      landed = mbar_wait(s_full + 8 * w, i & 1) && landed;
      __syncwarp();
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(st + 32 * c, s[c]);
      tmem_wait_ld();
      if (valid < kTile) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (32 * c + j >= valid) s[c][j] = __float_as_uint(-INFINITY);
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 32; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][j]));
      const float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
      if (i == 0) {
        m_run = m_new == -INFINITY ? 0.f : m_new;
      } else if (__any_sync(0xffffffffu, m_new > m_run + kLazy)) {
        // the products into O have completed: the commit behind S covers them
        const float alpha = m_new > m_run + kLazy ? exp2_fast(m_run - m_new) : 1.f;
        if (m_new > m_run + kLazy) m_run = m_new;
#pragma unroll
        for (int c = 0; c < 4; ++c) l[c] *= alpha;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t x[16];
          tmem_ld16(ot + 16 * c, x);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * alpha);
          tmem_st16(ot + 16 * c, x);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {   // 32 scores -> 16 columns of P
        uint32_t p[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float p0 = exp2_fast(fmaf(__uint_as_float(s[c][j]), scale, -m_run));
          const float p1 = exp2_fast(fmaf(__uint_as_float(s[c][j + 1]), scale, -m_run));
          l[j & 2] += p0;
          l[(j & 2) + 1] += p1;
          p[j / 2] = Dt<T>::pack2(p0, p1);
        }
        tmem_st16(st + 16 * c, p);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full + 8 * w);
    }
    if (mine > 0) {
      landed = mbar_wait(o_full + 8 * w, 0) && landed;
      __syncwarp();
      tc_fence_after();
    }
    const int64_t all_rows = static_cast<int64_t>(a.B) * a.T * a.H;
    const int64_t out = (static_cast<int64_t>(pair ? split : 2 * split + w)) * all_rows +
                        (static_cast<int64_t>(qb) * a.T + t) * a.H + head;
    float sum = (l[0] + l[1]) + (l[2] + l[3]);
    if (!landed) sum = NAN;
    if (live) *reinterpret_cast<float2*>(a.ml + out * 2) = make_float2(mine > 0 ? m_run : -INFINITY, sum);
    if (mine > 0) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t x[32];
        tmem_ld32(ot + 32 * c, x);
        tmem_wait_ld();
        if (live) {
          uint4* dst = reinterpret_cast<uint4*>(a.acc + out * D + 32 * c);
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[j] = make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
        }
      }
    } else if (live) {   // an entry that never counts, but is multiplied by zero
      for (int c = 0; c < D / 4; ++c) reinterpret_cast<uint4*>(a.acc + out * D)[c] = make_uint4(0, 0, 0, 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <typename T, int D>
int launch(const PoolMaps& maps, const PagedAttnArgs& a, bool pdl, cudaStream_t s) {
  auto kern = paged_prefix_kernel<T, D>;
  constexpr uint32_t bytes = prefix_smem<D>();
  static bool configured[64] = {};   // per device; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != cudaSuccess) {
      set_cuda_error(e);
      return B2D_ERR_LAUNCH;
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const unsigned row_pairs = (a.B * a.rows + 2 * kTile - 1) / (2 * kTile);
  return launch_kernel(kern, dim3(row_pairs * a.splits, a.kv.KVH), dim3(kPrefixThreads), bytes, s, pdl, maps, a);
}

}  // namespace

int launch_prefix_tc5(const PoolMaps& maps, const PagedAttnArgs& a, bool pdl, cudaStream_t s) {
  if (a.kv.dtype == B2D_F16) return a.kv.D == 64 ? launch<__half, 64>(maps, a, pdl, s) : launch<__half, 128>(maps, a, pdl, s);
  return a.kv.D == 64 ? launch<__nv_bfloat16, 64>(maps, a, pdl, s) : launch<__nv_bfloat16, 128>(maps, a, pdl, s);
}

}  // namespace b2d
