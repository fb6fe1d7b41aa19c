// Attention over a prefix that the whole batch shares, on the 5th-generation tensor cores (sm_100a): the
// queries of all sequences that read one KV head form one row axis, so the prefix is read once for up to 256
// rows and its products are matrix products of 128 rows: 128 x 64 x D for the scores, 128 x D x 64 for the values. Used
// from more than 32 rows on (below, the mma.sync kernel of csrc/paged_attention.cu is bound by the same bytes);
// leaves (O, m, l) per row and split of the keys. The combine launch of that file merges them with the sequences' own
// parts: it waits for the streaming launch, which runs beside this one and waits for it at its end.
//
// A CTA owns (256 rows as two tiles of 128, KV head, split). Per 64 keys and row tile:
//   S = Q K^T     tcgen05.mma kind::f16, M = 128, N = 64, both operands K-major in shared memory, S in TMEM
//   softmax       one warpgroup per row tile, one thread per row (tcgen05.ld brings the row's 64 scores into
//                 registers); P is rounded to the cache's dtype and overwrites S in TMEM
//   O += P V      P from TMEM, V from shared memory (MN-major), O in TMEM
// Each warpgroup has two S buffers, so the product for the next 64 keys is under way while it works: with one
// buffer of 128 keys the warpgroup waited as long as it worked (2.33 us per 128 keys and 256 rows, by time stamps).
// A warp per warpgroup issues its products. With 128 rows or fewer both warpgroups take the same rows and alternate over the
// key tiles. The running maximum moves only when a score exceeds it by 2^8 (weights up to 256 are as exact in
// fp32 and in both 16-bit types), so O in TMEM is rarely rescaled. K and V come as 128-byte-swizzled tensor
// copies, page by page, through a ring of four 128-key tiles.
// Measured on B200 (32 sequences x 4 drafts, 32 / 8 heads of 128, 16384 shared keys, bf16; 34.4 GFLOP): the call
// takes 65 to 66 us by graph replay; with cold caches this kernel is 44.5 us of it, the sequences' own keys 28.9, the
// combine 12.9. One product of 64 keys and 256 rows after another took about 1.1 us with time stamps in the
// kernel, which lengthen it; their shared-memory reads alone are estimated at 0.7 and the exponentials at 0.55.
// The call took 168 us with mma.sync, 83 with the first tcgen05 form. Merging the splits through distributed
// shared memory before the write: 67.8 against 64.8, not kept.
// TMEM columns: S/P buffers of the two warpgroups at 0, 64 and 128, 192, their O at 256 and 256 + D.
#include <cfloat>
#include <type_traits>

#include "paged_attention.cuh"
#include "pipeline.cuh"

namespace b2d {
namespace {

constexpr int kTile = 128;                  // keys of a copied tile, rows of a row tile
constexpr int kSub = 64;                    // keys of a product
constexpr int kSoftmax = 256;               // softmax threads (two warpgroups)
constexpr int kProducer = 8, kIssuer = 9;   // warps: one producer, an issuer per warpgroup
constexpr int kPrefixThreads = 352;
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
// One lane of a converged warp. The issuing code runs warp-uniformly around it, so that descriptors and addresses
// stay in uniform registers: from a single divergent lane a product took 90 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}\n" : "=r"(p));
  return p != 0;
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
// D (+)= A B; A from shared memory (ss) or TMEM (ts)
template <bool ADD>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
      ::"r"(d), "l"(a), "l"(b), "r"(id), "n"(ADD ? 1 : 0)
      : "memory");
}
template <bool ADD>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d), "r"(a), "l"(b), "r"(id), "n"(ADD ? 1 : 0)
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
  constexpr uint32_t SUBB = kSub * 128;                           // 64 keys of a column
  constexpr int HALVES = D / 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * kRing + 12];
  __shared__ uint32_t s_tmem;
  __shared__ int64_t s_q[kSoftmax];   // per row: offset of its query, -1 past the end
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* const smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  const uint32_t q_s = smem_u32(smem), ring = q_s + 2 * TILEB;
  // barriers: ring slots full / empty; scores ready and weights ready per warpgroup and buffer; products into O
  const uint32_t full = smem_u32(s_bar), empty = full + 8 * kRing, s_full = empty + 8 * kRing, p_full = s_full + 32,
                 o_full = p_full + 32, q_full = o_full + 16, done = q_full + 8;

  const int rows = a.B * a.rows;
  const bool pair = rows > kTile;          // two row tiles; else one, whose key tiles the warpgroups share
  const int kvh = blockIdx.y, split = blockIdx.x % a.splits, row0 = static_cast<int>(blockIdx.x) / a.splits * (2 * kTile);
  const int ktiles = (a.shared + kTile - 1) / kTile;
  const int t0 = ktiles * split / a.splits, n = ktiles * (split + 1) / a.splits - t0;   // this split's key tiles
  const int subs = min(2 * n, a.shared / kSub - 2 * t0);                                // and steps of 64 keys
  // steps of warpgroup w: tile of step u, and how many
  auto tile_of = [&](int w, int u) { return pair ? u >> 1 : 2 * (u >> 1) + w; };
  auto steps_of = [&](int w) {
    if (pair) return subs;
    const int tiles = (n + 1 - w) / 2;   // tiles w, w + 2, ...
    return 2 * tiles - (tiles > 0 && 2 * tile_of(w, 2 * tiles - 1) + 1 >= subs ? 1 : 0);
  };
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, pair ? 2 : 1);   // the issuers that use a slot
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, kTile);
    }
    mbar_init(o_full, 1);
    mbar_init(o_full + 8, 1);
    mbar_init(q_full, kSoftmax);
    mbar_init(done, 2);
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
  // All of TMEM is this CTA's, so its base is column 0: a constant, which keeps the products' addresses in
  // uniform registers (were it ever another, the rows would be NaN)
  constexpr uint32_t tmem = 0;

  if (warp == kProducer) {
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
    // behind the first tile the copies wait for Q: ahead of its loads they would hold them up (8 us)
    const int ahead = pair ? 1 : 2;   // tiles of scores that run ahead of the first P V
    for (int i = 0; i < ahead && i < n; ++i) {
      load(false, i);
      if (i == 0) ok = ok && __all_sync(0xffffffffu, mbar_wait(q_full, 0));
    }
    for (int i = 0; i < n; ++i) {
      load(true, i);
      if (i + ahead < n) load(false, i + ahead);
    }
  } else if (warp >= kIssuer) {
    // ---- the products of warpgroup w, in the order that its buffers need: P V of a step, then the scores of the
    // step after the next, which overwrite that P (the tensor core takes a thread's products in order). After a wait
    // that ran out `done` never completes, and the softmax warps give NaN: the waits hand on the number of tries that
    // they have left. (A flag in shared memory instead: 70 us for the call of the header, not 65.)
    const int w = warp - kIssuer, steps = steps_of(w);
    constexpr uint32_t ID_S = idesc<T, kSub, false>(), ID_O = idesc<T, D, true>();
    const int ahead = pair ? 1 : 2;
    int tries = kMbarTries;
    // the producer's position of a K or V tile
    auto unit_k = [&](int tile) { return tile < ahead ? tile : 2 * tile - ahead + 1; };
    auto unit_v = [&](int tile) { return min(tile + ahead, n) + tile; };
    auto ready = [&](int unit) {
      tries = mbar_wait_tries(full + 8 * (unit % kRing), (unit / kRing) & 1, tries);
      return static_cast<uint32_t>(unit % kRing);
    };
    auto scores = [&](int u) {   // S_w[u & 1] = Q K^T for step u
      const uint32_t slot = ready(unit_k(tile_of(w, u)));
      const uint32_t qa = q_s + (pair ? w * TILEB : 0u), kb = ring + slot * TILEB + (u & 1) * SUBB;
      if (elect_one()) {
        const uint32_t d = tmem + 128 * w + 64 * (u & 1);
        const uint64_t qd = desc_k_major(qa), kd = desc_k_major(kb);   // addresses count 16 bytes: + offset / 16
        mma_ss<false>(d, qd, kd, ID_S);
#pragma unroll
        for (int j = 1; j < D / 16; ++j) {
          const uint32_t off = ((j >> 2) * COLB + (j & 3) * 32) >> 4;
          mma_ss<true>(d, qd + off, kd + off, ID_S);
        }
        mma_commit(s_full + 16 * w + 8 * (u & 1));
        if (u % 2 == 1 || u == steps - 1) mma_commit(empty + 8 * slot);   // the tile's last use
      }
      __syncwarp();
    };
    auto values = [&](int u) {   // O_w += P_w V for step u
      const uint32_t slot = ready(unit_v(tile_of(w, u)));
      tries = mbar_wait_tries(p_full + 16 * w + 8 * (u & 1), (u >> 1) & 1, tries);
      tc_fence_after();
      const uint32_t vb = ring + slot * TILEB + (u & 1) * SUBB;
      if (elect_one()) {
        const uint32_t d = tmem + 256 + D * w, p = tmem + 128 * w + 64 * (u & 1);
        const uint64_t vd = desc_mn_major(vb, COLB);
        if (u == 0) mma_ts<false>(d, p, vd, ID_O);
        else mma_ts<true>(d, p, vd, ID_O);
#pragma unroll
        for (int j = 1; j < kSub / 16; ++j) mma_ts<true>(d, p + 8 * j, vd + (2048 * j >> 4), ID_O);
        mma_commit(o_full + 8 * w);
        if (u % 2 == 1 || u == steps - 1) mma_commit(empty + 8 * slot);
      }
      __syncwarp();
    };
    if (n > 0) {
      tries = mbar_wait_tries(q_full, 0, tries);
      tc_fence_after();
      for (int u = 0; u < 2 && u < steps; ++u) scores(u);
      for (int u = 0; u < steps; ++u) {
        values(u);
        if (u + 2 < steps) scores(u + 2);
      }
      if (__all_sync(0xffffffffu, tries > 0) && elect_one()) mma_commit(done);
    }
    __syncwarp();
  } else {
    // ---- softmax: warpgroup w, thread = row (TMEM lane)
    const int w = warp >> 2, r = tid & (kTile - 1);
    {
      // Q into the K-major tiles, 16 bytes a copy
      constexpr int CH = D / 8;
      const int tile_rows = pair ? 2 * kTile : kTile;
      {
        const int row = row0 + tid, qb = row / a.rows, qr = row - qb * a.rows, t = qr * a.inv_g >> 16;
        s_q[tid] = row < rows ? qb * a.sq_b + t * a.sq_t + static_cast<int64_t>(kvh * a.G + qr - t * a.G) * a.sq_h : -1;
      }
      named_sync<1, kSoftmax>();
#pragma unroll 1
      for (int i = tid; i < tile_rows * CH; i += kSoftmax) {
        const int qrow = i / CH, c = i % CH, tr = qrow & (kTile - 1);
        const int64_t off = s_q[qrow];
        cp_async16_zfill(q_s + (qrow >> 7) * TILEB + (c >> 3) * COLB + tr * 128 + (((c & 7) ^ (tr & 7)) << 4),
                         static_cast<const T*>(a.q) + (off < 0 ? 0 : off + c * 8), off >= 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
      fence_proxy_async();
    }
    mbar_arrive(q_full);
    const float scale = a.scale_log2;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t st = tmem + lanes + 128 * w, ot = tmem + lanes + 256 + D * w;
    const int steps = steps_of(w);
    float m_run = 0.f, l[4] = {0.f, 0.f, 0.f, 0.f};
    bool landed = s_tmem == tmem;
    for (int u = 0; u < steps; ++u) {
      const uint32_t sb = st + 64 * (u & 1);
      landed = landed && mbar_wait(s_full + 16 * w + 8 * (u & 1), (u >> 1) & 1);
      __syncwarp();
      tc_fence_after();
      uint32_t s[2][32];
      tmem_ld32(sb, s[0]);
      tmem_ld32(sb + 32, s[1]);
      tmem_wait_ld();
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 32; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) mx[2 * c + (j & 1)] = fmaxf(mx[2 * c + (j & 1)], __uint_as_float(s[c][j]));
      if (scale < 0.f) {   // the largest product has the smallest score
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = INFINITY;
#pragma unroll
        for (int j = 0; j < 32; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) mx[2 * c + (j & 1)] = fminf(mx[2 * c + (j & 1)], __uint_as_float(s[c][j]));
        mx[0] = fminf(fminf(mx[0], mx[1]), fminf(mx[2], mx[3]));
        mx[1] = mx[2] = mx[3] = mx[0];
      }
      const float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
      if (u == 0) {
        m_run = fmaxf(m_new, -FLT_MAX);   // -infinity everywhere: the first other score moves it (inf - inf is none)
      } else if (__any_sync(0xffffffffu, m_new > m_run + kLazy)) {
        landed = landed && mbar_wait(o_full + 8 * w, (u - 1) & 1);   // the products into O so far
        __syncwarp();
        tc_fence_after();
        const bool move = m_new > m_run + kLazy;
        const float alpha = move ? exp2_fast(m_run - m_new) : 1.f;
        if (move) m_run = m_new;
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
      for (int c = 0; c < 2; ++c) {   // 32 scores -> 16 columns of P
        uint32_t p[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float p0 = exp2_fast(fmaf(__uint_as_float(s[c][j]), scale, -m_run));
          const float p1 = exp2_fast(fmaf(__uint_as_float(s[c][j + 1]), scale, -m_run));
          l[j & 2] += p0;
          l[(j & 2) + 1] += p1;
          p[j / 2] = Dt<T>::pack2(p0, p1);
        }
        tmem_st16(sb + 16 * c, p);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full + 16 * w + 8 * (u & 1));
    }
    // ---- the partials. Both warpgroups' products are done, so the ring is free: rows pass through it (16-byte
    // chunk c of row r at c ^ r) and leave as whole lines
    if (n > 0) landed = landed && mbar_wait(done, 0);
    __syncwarp();
    tc_fence_after();
    const int64_t all = static_cast<int64_t>(a.B) * a.T * a.H;
    const int row = row0 + (pair ? w * kTile : 0) + r;
    const int qb = row / a.rows, qr = row - qb * a.rows, t = qr * a.inv_g >> 16;
    const int64_t out = row >= rows ? -1 : static_cast<int64_t>(pair ? split : 2 * split + w) * all +
                                              (static_cast<int64_t>(qb) * a.T + t) * a.H + kvh * a.G + qr - t * a.G;
    float sum = (l[0] + l[1]) + (l[2] + l[3]);
    if (!landed) sum = NAN;
    if (out >= 0) *reinterpret_cast<float2*>(a.ml + out * 2) = make_float2(steps > 0 ? m_run : -INFINITY, sum);
    constexpr int OC = D / 4;   // 16-byte chunks of a row
    uint8_t* const stage = smem + 2 * TILEB + warp * (32 * D * 4);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      uint32_t x[32];
      if (steps > 0) {
        tmem_ld32(ot + 32 * c, x);
        tmem_wait_ld();
      } else {   // an entry that never counts, but is multiplied by zero
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = 0;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<uint4*>(stage + lane * (D * 4) + (((8 * c + j) ^ (lane & (OC - 1))) << 4)) =
            make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
    }
    __syncwarp();
#pragma unroll 8
    for (int i = 0; i < OC; ++i) {   // 32 chunks a step: 32 / OC rows
      const int rr = i * (32 / OC) + lane / OC, c = lane % OC;
      const int64_t to = __shfl_sync(0xffffffffu, out, rr);
      if (to >= 0)
        *reinterpret_cast<uint4*>(a.acc + to * D + 4 * c) =
            *reinterpret_cast<const uint4*>(stage + rr * (D * 4) + ((c ^ (rr & (OC - 1))) << 4));
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
