// Attention of the newest tokens of every sequence over a paged KV cache, causal among themselves, with an
// optional prefix shared by the whole batch (sm_100a). The contiguous one-token counterpart is
// csrc/gqa_decode.cu (reference: profiling/kernels/decode_attention.py:18-91).
//
// o[b, t, h] = sum_{j < limit} softmax_j(scale q.k_j) v_j, limit = seqlens[b] - T + 1 + t. Key j lies in
// prefix_table's pages for j < prefix_len and in page_table[b]'s behind.
//
// A CTA owns one (sequence, KV head, tile of 16 RW rows, split of the keys): rows are the T x G query vectors
// that read this KV head (row = t G + g), so K and V are read once for all of them. A producer warp streams
// 32 KB stages (64 keys of 128, 128 keys of 64) through a 3-stage shared-memory ring: its lanes look the
// pages up one stage ahead and issue one tensor copy per (page, 64 elements, K or V), 128-byte swizzled, so
// that the ldmatrix reads hit 8 distinct bank groups; completion on mbarriers. Pages that tensor copies do
// not fit (sizes that neither divide nor are divided by 64, ...) take 16-byte cp.async from the same warp.
// S = Q K^T and O += P V by mma.sync m16n8k16 (fp32 accumulate): consumer warp (rw, kw) takes rows
// [16 rw, 16 rw + 16) and its share of each stage's keys; online softmax in the log2 domain; the key warps
// meet in shared memory. P is rounded to the cache's dtype for the second product, as its V operand is; the
// sum of the weights is taken before that rounding, in fp32. Value rows at or past the length are set to
// zero in shared memory before they are multiplied (a zero weight times a stale NaN would not be zero).
//
// Splits: the sequence's own length on the device is divided evenly over the splits, so a ragged batch needs
// no host knowledge of its lengths. The splits of one (sequence, KV head, row tile) form a thread-block
// cluster of up to 8 CTAs that meet through distributed shared memory, so the common case is one launch
// without scratch; longer work takes several clusters, which leave (unnormalised O, m, l) in the workspace
// for a small combine kernel.
//
// Shared prefix: a first launch (PREFIX) takes all sequences' rows as one row axis, [0, B T G), over the
// prefix's pages, and leaves (O, m, l) per row and split; the per-sequence kernel starts behind the prefix
// and takes those partials in at its end. It is launched as a programmatic dependent and waits for the
// prefix launch only there. A sequence with a query that does not see the whole prefix is computed by the
// per-sequence kernel alone, from position 0.
#include <mutex>
#include <type_traits>

#include "paged_attention.cuh"
#include "pipeline.cuh"

namespace b2d {
namespace {

constexpr int kWarps = 4;                       // consumer warps
constexpr int kConsumers = kWarps * 32;
constexpr int kThreads = kConsumers + 32;       // and the producer warp
constexpr int kStageBytes = 32 * 1024;          // K and V of a stage
constexpr int kStages = 3;
constexpr int kMaxT = 16, kMaxG = 16;
constexpr float kLog2e = 1.4426950408889634f;

constexpr int kMaxCluster = 8;     // portable size

constexpr size_t kRingBytes = static_cast<size_t>(kStages) * kStageBytes;
template <int D>
__host__ __device__ constexpr int stage_keys() { return kStageBytes / (2 * D * 2); }

__device__ __forceinline__ uint32_t map_cluster(uint32_t local, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
// any infinity or NaN among 8 values
template <typename T>
__device__ __forceinline__ bool nonfinite8(const uint4& u) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;   // exponent bits
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & e) == e || (w[i] >> 16 & e) == e;
  return bad;
}

template <typename T>
__device__ __forceinline__ void store_out(const PagedAttnArgs& a, int64_t off, float v) {
  if (a.out_f32) static_cast<float*>(a.out)[off] = v;
  else static_cast<T*>(a.out)[off] = Dt<T>::from_f32(v);
}

template <typename T, int D, int RW, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 2) paged_attention_kernel(const __grid_constant__ PoolMaps maps,
                                                                      const __grid_constant__ PagedAttnArgs a) {
  constexpr int KEYS = stage_keys<D>();
  constexpr int KW = kWarps / RW;       // warps that share a row tile and split a stage's keys
  constexpr int WK = KEYS / KW;         // keys of a stage that a warp takes,
  constexpr int WB = WK < 32 ? WK : 32; // at most 32 at a time
  constexpr int ROWS = 16 * RW;
  constexpr int KSTEPS = D / 16, NTILES = D / 8, CH = D / 8, HALVES = D / 64;
  constexpr uint32_t HALFB = KEYS * 128, TILEB = HALVES * HALFB;   // a stage's 64-element column; its K (or V)
  constexpr int OPAD = D + 8;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ float s_m[kWarps][16], s_l[kWarps][16];
  __shared__ float2 s_ml[ROWS];         // this CTA's (m, l) per row, read by the cluster
  __shared__ uint32_t s_bad[2][KEYS / 32];
  __shared__ __align__(8) uint64_t s_bar[2 * kStages];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* const smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  const uint32_t sbase = smem_u32(smem), full = smem_u32(s_bar), empty = full + 8 * kStages;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + 8 * i, a.box_rows ? 1 : 32);
      mbar_init(empty + 8 * i, kWarps);
    }
    fence_mbar_init();
  }
  if (tid < 2 * KEYS / 32) s_bad[0][tid] = 0;
  if (a.box_rows && tid == kConsumers) {
    prefetch_tensormap(&maps.k);
    prefetch_tensormap(&maps.v);
  }
  if constexpr (PREFIX) {   // the dependent launch reads the same inputs: it starts once they are complete
    pdl_wait();
    pdl_launch_dependents();
  } else {
    if (!a.after_prefix) pdl_wait();
    pdl_launch_dependents();
  }
  const int nsplit = a.cs * a.ncl;
  const int split = static_cast<int>(blockIdx.x) % nsplit, tile = static_cast<int>(blockIdx.x) / nsplit;
  const int rank = split % a.cs;
  const int row0 = tile * ROWS, kvh = blockIdx.y, b = PREFIX ? 0 : blockIdx.z;
  const int rows = PREFIX ? a.B * a.rows : a.rows;
  const int row_end = min(rows, row0 + ROWS);
  const int32_t* table = PREFIX ? a.prefix_table : a.table + b * a.ld_table;

  // keys of the tile's rows [k_begin, k_end) and this split's share [t_begin, t_end)
  int len = 0, k_begin = 0, k_end = a.shared, lim_min = a.shared;
  bool shares = false;
  if constexpr (!PREFIX) {
    const int64_t reach = static_cast<int64_t>(a.pages_per_seq) * a.kv.page_size;
    len = max(a.seqlens[b], 0);
    if (len > reach) len = max(static_cast<int>(reach), a.prefix_len);
    shares = len - a.T + 1 >= a.shared && len > 0;
    k_begin = shares ? a.shared : 0;
    k_end = max(0, len - a.T + 1 + (row_end - 1) / a.G);
    lim_min = len - a.T + 1 + row0 / a.G;   // below it no row is masked
  }
  const int stages = (max(0, k_end - k_begin) + KEYS - 1) / KEYS;
  const int st0 = static_cast<int>(static_cast<int64_t>(stages) * split / nsplit);
  const int nst = static_cast<int>(static_cast<int64_t>(stages) * (split + 1) / nsplit) - st0;
  const int t_begin = k_begin + st0 * KEYS, t_end = min(k_end, t_begin + nst * KEYS);
  __syncthreads();   // barriers and s_bad are set

  if (warp == kWarps) {
    // ---- producer
    if (a.box_rows) {
      // lane -> (K or V, 64-element column, page of the stage): 32 lanes are enough from boxes of 8 rows on
      const int bp = a.box_rows, boxes = KEYS / bp, per = HALVES * boxes;
      const int kv = lane / per, rest = lane - kv * per, col = rest / boxes, pg = rest - col * boxes;
      const bool mine = lane < 2 * per;
      const CUtensorMap* map = kv ? &maps.v : &maps.k;
      auto lookup = [&](int it) {
        const int tok = t_begin + it * KEYS + pg * bp;
        return mine && tok < t_end ? __ldg((PREFIX || tok >= a.prefix_len ? table : a.prefix_table) + a.div.page(tok)) : -1;
      };
      int next = lookup(0);
      for (int it = 0; it < nst; ++it) {
        const int page = next, slot = it % kStages, tok = t_begin + it * KEYS + pg * bp;
        next = lookup(it + 1);
        if (it >= kStages && !__all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, (it / kStages - 1) & 1))) break;
        const uint32_t dst = sbase + slot * kStageBytes + kv * TILEB + col * HALFB + pg * bp * 128;
        const bool live = mine && tok < t_end, copy = live && page >= 0 && page < a.kv.num_pages;
        if (live && !copy) {   // a page id outside the pool: zeros
          for (int i = 0; i < bp * 8; ++i)
            *reinterpret_cast<uint4*>(smem + (dst - sbase) + 16 * i) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
        }
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, copy)) * bp * 128;
        __syncwarp();
        if (lane == 0) mbar_expect_tx(full + 8 * slot, bytes);
        __syncwarp();
        if (copy) tma_load_4d(dst, map, 64 * col, a.div.slot(tok, a.div.page(tok)), kvh, page, full + 8 * slot);
      }
    } else {
      // lane l owns the addresses of key rows l, l + 32, ...; 8 lanes copy the 128 bytes of a row's column
      for (int it = 0; it < nst; ++it) {
        const int slot = it % kStages;
        if (it >= kStages && !__all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, (it / kStages - 1) & 1))) break;
        for (int r0 = 0; r0 < KEYS; r0 += 32) {
          const int tok = t_begin + it * KEYS + r0 + lane;
          int64_t ko = -1, vo = -1;
          if (tok < t_end) {
            const int pi = a.div.page(tok);
            const int page = __ldg((PREFIX || tok >= a.prefix_len ? table : a.prefix_table) + pi);
            if (page >= 0 && page < a.kv.num_pages) {
              const int64_t sl = a.div.slot(tok, pi);
              ko = page * a.kv.sk_p + kvh * a.kv.sk_h + sl * a.kv.sk_s;
              vo = page * a.kv.sv_p + kvh * a.kv.sv_h + sl * a.kv.sv_s;
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rr = 4 * i + lane / 8, r = r0 + rr, c = lane & 7;
            const int64_t k0 = __shfl_sync(0xffffffffu, ko, rr), v0 = __shfl_sync(0xffffffffu, vo, rr);
            const T* ks = static_cast<const T*>(a.kv.k) + (k0 < 0 ? 0 : k0 + c * 8);
            const T* vs = static_cast<const T*>(a.kv.v) + (k0 < 0 ? 0 : v0 + c * 8);
            const uint32_t dst = sbase + slot * kStageBytes + r * 128 + ((c ^ (r & 7)) << 4);
#pragma unroll
            for (int col = 0; col < HALVES; ++col) {
              cp_async16_zfill(dst + col * HALFB, ks + (k0 < 0 ? 0 : 64 * col), k0 >= 0);
              cp_async16_zfill(dst + TILEB + col * HALFB, vs + (k0 < 0 ? 0 : 64 * col), k0 >= 0);
            }
          }
        }
        mbar_arrive_cp_async(full + 8 * slot);
      }
      cp_async_wait<0>();
    }
  } else {
    // ---- consumers
    const int rw = warp % RW, kw = warp / RW;
    const int g = lane >> 2, tq = lane & 3, mi = lane >> 3, ri = lane & 7;
    int lim[2] = {a.shared, a.shared};   // keys that this thread's two rows see
    uint32_t qa[KSTEPS][4];              // Q fragments of the warp's 16 rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = row0 + 16 * rw + g + 8 * h;
      const bool live = row < rows;
      const int qb = PREFIX ? row / a.rows : b, qr = PREFIX ? row - qb * a.rows : row;
      const int t = qr / a.G, head = kvh * a.G + qr - t * a.G;
      if (!PREFIX) lim[h] = len - a.T + 1 + min(row, row_end - 1) / a.G;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + qb * a.sq_b + t * a.sq_t +
                                                              static_cast<int64_t>(head) * a.sq_h);
#pragma unroll
      for (int j = 0; j < KSTEPS; ++j) {
        qa[j][h] = live ? src[8 * j + tq] : 0u;           // d = 16j + 2tq, +1
        qa[j][2 + h] = live ? src[8 * j + 4 + tq] : 0u;   // d = 16j + 8 + 2tq, +1
      }
    }
    float o[NTILES][4];
#pragma unroll
    for (int n = 0; n < NTILES; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY};   // log2 domain
    float l_run[2] = {0.f, 0.f};               // this thread's keys only
    bool landed = true;

    for (int it = 0; it < nst; ++it) {
      const int slot = it % kStages;
      landed = landed && mbar_wait(full + 8 * slot, (it / kStages) & 1);
      const int stage0 = t_begin + it * KEYS;
      const uint32_t kbuf = sbase + slot * kStageBytes, vbuf = kbuf + TILEB;

      // The stage at the end: value rows past it become zeros. And keys that some rows of the tile see and
      // others do not (the newest T - 1): a zero weight times an infinite or NaN value would reach the rows
      // that must not see it, so such value rows (rare) are taken out of the stage and added to the rows
      // that do see them one by one below. At most two stages hold any.
      bool any_bad = false;
      const bool check = !PREFIX && a.T > 1 && min(stage0 + KEYS, t_end) > lim_min;
      if (check || stage0 + KEYS > t_end) {
#pragma unroll 4
        for (int ci = tid; ci < KEYS * CH; ci += kConsumers) {
          const int r = ci / CH, c = ci % CH;
          uint4* x = reinterpret_cast<uint4*>(smem + (vbuf - sbase) + (c >> 3) * HALFB + r * 128 + (((c & 7) ^ (r & 7)) << 4));
          if (stage0 + r >= t_end) *x = make_uint4(0, 0, 0, 0);
          else if (check && stage0 + r >= lim_min && nonfinite8<T>(*x)) atomicOr(&s_bad[it & 1][r >> 5], 1u << (r & 31));
        }
        named_sync<1, kConsumers>();
        if (check) {
#pragma unroll
          for (int i = 0; i < KEYS / 32; ++i) any_bad |= s_bad[it & 1][i] != 0;
          if (any_bad) {
            for (int ci = tid; ci < KEYS * CH; ci += kConsumers) {
              const int r = ci / CH, c = ci % CH;
              if (s_bad[it & 1][r >> 5] >> (r & 31) & 1)
                *reinterpret_cast<uint4*>(smem + (vbuf - sbase) + (c >> 3) * HALFB + r * 128 + ((c & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
            named_sync<1, kConsumers>();
          }
        }
      }
#pragma unroll
      for (int blk = 0; blk < WK / WB; ++blk) {
        const int first = kw * WK + blk * WB, key0 = stage0 + first;   // this warp's keys
        if (key0 >= t_end) break;
        const bool masked = key0 + WB > min(lim_min, t_end);
        float s[WB / 8][4];
        float tmax[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < WB / 8; ++n) {
          s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
          const int r = first + 8 * n + ri;
#pragma unroll
          for (int j = 0; j < KSTEPS; j += 2) {
            const int c = 2 * j + mi;
            uint32_t b0, b1, b2, b3;
            ldsm_x4(kbuf + (c >> 3) * HALFB + r * 128 + (((c & 7) ^ (r & 7)) << 4), b0, b1, b2, b3);
            Mma<T>::run(s[n], qa[j][0], qa[j][1], qa[j][2], qa[j][3], b0, b1);
            Mma<T>::run(s[n], qa[j + 1][0], qa[j + 1][1], qa[j + 1][2], qa[j + 1][3], b2, b3);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int tok = key0 + 8 * n + 2 * tq + (c & 1);
            s[n][c] *= a.scale_log2;
            if (masked && (tok >= lim[c >> 1] || tok >= t_end)) s[n][c] = -INFINITY;
            tmax[c >> 1] = fmaxf(tmax[c >> 1], s[n][c]);
          }
        }
        float alpha[2], msafe[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          tmax[r] = fmaxf(tmax[r], __shfl_xor_sync(0xffffffffu, tmax[r], 1));
          tmax[r] = fmaxf(tmax[r], __shfl_xor_sync(0xffffffffu, tmax[r], 2));
          const float m_new = fmaxf(m_run[r], tmax[r]);
          msafe[r] = m_new == -INFINITY ? 0.f : m_new;
          alpha[r] = exp2_fast(m_run[r] - msafe[r]);
          m_run[r] = m_new;
          l_run[r] *= alpha[r];
        }
#pragma unroll
        for (int n = 0; n < NTILES; ++n) {
          o[n][0] *= alpha[0]; o[n][1] *= alpha[0];
          o[n][2] *= alpha[1]; o[n][3] *= alpha[1];
        }
#pragma unroll
        for (int u = 0; u < WB / 16; ++u) {   // 16 keys at a time
          uint32_t pa[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float(&p)[4] = s[2 * u + h];
#pragma unroll
            for (int c = 0; c < 4; ++c) p[c] = exp2_fast(p[c] - msafe[c >> 1]);
            l_run[0] += p[0] + p[1];
            l_run[1] += p[2] + p[3];
            pa[2 * h] = Dt<T>::pack2(p[0], p[1]);
            pa[2 * h + 1] = Dt<T>::pack2(p[2], p[3]);
          }
#pragma unroll
          for (int np = 0; np < NTILES; np += 2) {
            const int r = first + 16 * u + 8 * (mi & 1) + ri, c = np + (mi >> 1);
            uint32_t v0, v1, v2, v3;
            ldsm_x4_t(vbuf + (c >> 3) * HALFB + r * 128 + (((c & 7) ^ (r & 7)) << 4), v0, v1, v2, v3);
            Mma<T>::run(o[np], pa[0], pa[1], pa[2], pa[3], v0, v1);
            Mma<T>::run(o[np + 1], pa[0], pa[1], pa[2], pa[3], v2, v3);
          }
        }
        if (!PREFIX && any_bad) {   // the value rows taken out above, for the rows that see them
#pragma unroll
          for (int n = 0; n < WB / 8; ++n) {
            for (int col = 0; col < 8; ++col) {
              const int r = first + 8 * n + col;
              if (!(s_bad[it & 1][r >> 5] >> (r & 31) & 1)) continue;
              const int src = (lane & ~3) | (col >> 1);
              const float p0 = __shfl_sync(0xffffffffu, (col & 1) ? s[n][1] : s[n][0], src);
              const float p1 = __shfl_sync(0xffffffffu, (col & 1) ? s[n][3] : s[n][2], src);
              const int tok = stage0 + r, pi = a.div.page(tok);
              const int page = (tok >= a.prefix_len ? table : a.prefix_table)[pi];
              const T* v = static_cast<const T*>(a.kv.v) + page * a.kv.sv_p + kvh * a.kv.sv_h +
                           a.div.slot(tok, pi) * a.kv.sv_s + 2 * tq;
#pragma unroll
              for (int d = 0; d < NTILES; ++d)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const float x = Dt<T>::to_f32(v[8 * d + e]);
                  if (tok < lim[0]) o[d][e] += p0 * x;
                  if (tok < lim[1]) o[d][2 + e] += p1 * x;
                }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * slot);
    }
    if (!landed) l_run[0] = l_run[1] = NAN;
    named_sync<1, kConsumers>();   // the ring becomes the merge buffer

    float* s_o = reinterpret_cast<float*>(smem);   // [kWarps][16][OPAD]
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
      const int row = g + 8 * r;
      if (tq == 0) {
        s_m[warp][row] = m_run[r];
        s_l[warp][row] = l_run[r];
      }
      float* dst = s_o + (warp * 16 + row) * OPAD + 2 * tq;
#pragma unroll
      for (int n = 0; n < NTILES; ++n)
        *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
    }
  }
  __syncthreads();

  // ---- the key warps meet: s_o[row] unnormalised, s_ml[row] = (m, l)
  float* s_o = reinterpret_cast<float*>(smem);   // [kWarps][16][OPAD]
  const int nrows = row_end - row0;
  if (tid < nrows) {
    const int w0 = tid / 16, rr = tid % 16;
    float mx = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) mx = fmaxf(mx, s_m[k * RW + w0][rr]);
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const int w = k * RW + w0;
      const float e = s_m[w][rr] == -INFINITY ? 0.f : exp2_fast(s_m[w][rr] - mx);
      l += e * s_l[w][rr];
      s_m[w][rr] = e;   // the warp's factor
    }
    s_ml[tid] = make_float2(mx, l);
  }
  __syncthreads();
  if constexpr (KW > 1) {
    for (int idx = tid; idx < nrows * D; idx += kThreads) {
      const int row = idx / D, d = idx - row * D, w0 = row / 16, rr = row % 16;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < KW; ++k) v += s_m[k * RW + w0][rr] * s_o[((k * RW + w0) * 16 + rr) * OPAD + d];
      s_o[row * OPAD + d] = v;   // (w0, rr) of key warp 0: this thread's own element
    }
  }
  if (a.cs > 1) cluster_sync();
  else __syncthreads();
  if constexpr (!PREFIX) {
    if (a.after_prefix) pdl_wait();   // the prefix launch's partials
  }

  // ---- the cluster meets (and, in the last stop, the prefix's partials): entries e < cs are the cluster's
  // CTAs, the others workspace partials; s_w[e][row] = (m, l), then the entry's factor
  const bool last = !PREFIX && a.ncl == 1;
  const int np = last && shares ? a.nparts : 0, ne = a.cs + np;
  const int64_t all_rows = static_cast<int64_t>(a.B) * a.T * a.H;
  float2* s_w = reinterpret_cast<float2*>(smem + kWarps * 16 * OPAD * 4);
  auto out_row = [&](int row) -> int64_t {   // (b T + t) H + h
    const int r = row0 + row, rb = PREFIX ? r / a.rows : b, rr = PREFIX ? r - rb * a.rows : r, t = rr / a.G;
    return (static_cast<int64_t>(rb) * a.T + t) * a.H + kvh * a.G + rr - t * a.G;
  };
  for (int idx = tid; idx < ne * nrows; idx += kThreads) {
    const int e = idx / nrows, row = idx - e * nrows;
    float2 v;
    if (e < a.cs) v = a.cs > 1 ? ld_cluster_f32x2(map_cluster(smem_u32(&s_ml[row]), e)) : s_ml[row];
    else v = *reinterpret_cast<const float2*>(a.ml + ((e - a.cs) * all_rows + out_row(row)) * 2);
    s_w[e * ROWS + row] = v;
  }
  __syncthreads();
  if (tid < nrows) {
    float mx = -INFINITY, l = 0.f;
    for (int e = 0; e < ne; ++e) mx = fmaxf(mx, s_w[e * ROWS + tid].x);
    for (int e = 0; e < ne; ++e) {
      const float2 v = s_w[e * ROWS + tid];
      const float f = v.x == -INFINITY ? 0.f : exp2_fast(v.x - mx);
      l += f * v.y;
      s_w[e * ROWS + tid].x = f;
    }
    // a row that sees no key: zeros (l is NaN, not 0, where a visible score is)
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int e = 0; e < ne; ++e) s_w[e * ROWS + tid].y = s_w[e * ROWS + tid].x * inv;
    if (!last && rank == 0) {
      const int64_t part = PREFIX ? split / a.cs : a.nparts + split / a.cs;
      *reinterpret_cast<float2*>(a.ml + (part * all_rows + out_row(tid)) * 2) = make_float2(mx, l);
    }
  }
  __syncthreads();
  for (int idx = rank * kThreads + tid; idx < nrows * D; idx += a.cs * kThreads) {
    const int row = idx / D, d = idx - row * D;
    const int64_t orow = out_row(row);
    float v = 0.f;
    const uint32_t local = smem_u32(s_o + row * OPAD + d);
    for (int e = 0; e < a.cs; ++e) {
      const float x = a.cs > 1 ? ld_cluster_f32(map_cluster(local, e)) : s_o[row * OPAD + d];
      v += (last ? s_w[e * ROWS + row].y : s_w[e * ROWS + row].x) * x;
    }
    if (last) {
      for (int e = 0; e < np; ++e) v += s_w[(a.cs + e) * ROWS + row].y * a.acc[(e * all_rows + orow) * D + d];
      const int t = (row0 + row) / a.G, head = kvh * a.G + row0 + row - t * a.G;
      store_out<T>(a, b * a.so_b + t * a.so_t + static_cast<int64_t>(head) * a.so_h + d, v);
    } else {
      const int64_t part = PREFIX ? split / a.cs : a.nparts + split / a.cs;
      a.acc[(part * all_rows + orow) * D + d] = v;
    }
  }
  if (a.cs > 1) cluster_sync_relaxed();   // this CTA's shared memory stays until the others have read it
}

// Merges the workspace's partials of a row: one warp per (b, t, h).
template <typename T, int D>
__global__ void __launch_bounds__(kConsumers) paged_combine_kernel(const PagedAttnArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t all_rows = static_cast<int64_t>(a.B) * a.T * a.H;
  const int64_t row = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= all_rows) return;
  const int h = static_cast<int>(row % a.H);
  const int64_t bt = row / a.H;
  const int t = static_cast<int>(bt % a.T), b = static_cast<int>(bt / a.T);
  int first = 0;   // a sequence that does not share the prefix takes its own partials only
  if (a.nparts > 0) {
    const int64_t reach = static_cast<int64_t>(a.pages_per_seq) * a.kv.page_size;
    int len = max(a.seqlens[b], 0);
    if (len > reach) len = max(static_cast<int>(reach), a.prefix_len);
    first = len - a.T + 1 >= a.shared && len > 0 ? 0 : a.nparts;
  }
  float mx = -INFINITY;
  for (int e = first + lane; e < a.parts; e += 32) mx = fmaxf(mx, a.ml[(e * all_rows + row) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  constexpr int PER = D / 32;
  float v[PER] = {}, l = 0.f;
  for (int e = first; e < a.parts; ++e) {
    const float2 p = *reinterpret_cast<const float2*>(a.ml + (e * all_rows + row) * 2);
    const float f = p.x == -INFINITY ? 0.f : exp2_fast(p.x - mx);
    l += f * p.y;
    const float* src = a.acc + (e * all_rows + row) * D + lane * PER;
    if constexpr (PER == 4) {
      const float4 x = *reinterpret_cast<const float4*>(src);
      v[0] += f * x.x; v[1] += f * x.y; v[2] += f * x.z; v[3] += f * x.w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(src);
      v[0] += f * x.x; v[1] += f * x.y;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t off = b * a.so_b + t * a.so_t + static_cast<int64_t>(h) * a.so_h + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; ++i) store_out<T>(a, off + i, v[i] * inv);
}

// ------------------------------------------------------------------ host
template <typename... KArgs, typename... Args>
int launch_cluster(void (*kern)(KArgs...), dim3 grid, size_t smem, int cs, bool pdl, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cs > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cs;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return B2D_ERR_LAUNCH;
  }
  return launch_status();
}

template <typename T, int D, int RW, bool PREFIX>
int launch(const PoolMaps& maps, const PagedAttnArgs& a, bool pdl, cudaStream_t s) {
  auto kern = paged_attention_kernel<T, D, RW, PREFIX>;
  constexpr size_t bytes = kRingBytes + 1024;   // and room to align it
  static_assert(kWarps * 16 * (D + 8) * 4 + (kMaxParts + kMaxCluster) * 16 * RW * 8 <= kRingBytes, "merge buffers fit the ring");
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
  const dim3 grid(a.tiles * a.cs * a.ncl, a.kv.KVH, PREFIX ? 1 : a.B);
  return launch_cluster(kern, grid, bytes, a.cs, pdl, s, maps, a);
}
template <typename T, int D, bool PREFIX>
int launch_rows(const PoolMaps& maps, const PagedAttnArgs& a, int rw, bool pdl, cudaStream_t s) {
  if (rw == 1) return launch<T, D, 1, PREFIX>(maps, a, pdl, s);
  if (rw == 2) return launch<T, D, 2, PREFIX>(maps, a, pdl, s);
  return launch<T, D, 4, PREFIX>(maps, a, pdl, s);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    else
      cudaGetLastError();
  });
  return fn;
}

bool encode_pool(CUtensorMap* m, const b2d_paged_kv& kv, void* base, int64_t sp, int64_t sh, int64_t ss, int rows) {
  const auto fn = encode_fn();
  if (!fn || sp <= 0 || sh <= 0 || ss <= 0) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(kv.D), static_cast<cuuint64_t>(kv.page_size),
                              static_cast<cuuint64_t>(kv.KVH), static_cast<cuuint64_t>(kv.num_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(ss) * 2, static_cast<cuuint64_t>(sh) * 2,
                                 static_cast<cuuint64_t>(sp) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1}, es[4] = {1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, base, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// Key rows of a tensor copy: a page, or 64 rows of a larger one; every copy starts on a multiple of 8 rows
// and ends inside its page, and the prefix ends between two copies. 0: the pages do not allow it.
int box_rows(const b2d_paged_kv& kv, int prefix_len) {
  const int ps = kv.page_size;
  if (kv.num_pages < 1 || ps < 8 || (64 % ps != 0 && ps % 64 != 0)) return 0;
  const int rows = ps < 64 ? ps : 64;
  return prefix_len % rows == 0 ? rows : 0;
}

// How a call is cut: the prefix launch's splits and the per-sequence kernel's clusters.
struct Plan {
  int shared, tc5, rw_p, tiles_p, cs_p, ncl_p, nparts, rw, tiles, cs, ncl, parts;
  size_t bytes;
};

int row_warps(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

// Splits over the keys for `groups` independent row tiles: about two CTAs per SM in all, at least 128 keys
// each; up to 8 form a cluster.
void split_keys(int64_t groups, int64_t keys, int sm, int most, int* cs, int* ncl) {
  int64_t want = 2 * sm / groups;
  const int64_t room = (keys + 127) / 128;
  if (want > room) want = room;
  if (want < 1) want = 1;
  *cs = 1;
  while (*cs < kMaxCluster && *cs * 2 <= want) *cs *= 2;
  int64_t n = *cs == kMaxCluster ? want / kMaxCluster : 1;
  if (n > most) n = most;
  *ncl = static_cast<int>(n < 1 ? 1 : n);
}

Plan make_plan(const b2d_paged_kv* kv, int B, int T, int H, int pages_per_seq, int prefix_len, int max_len, int sm) {
  Plan p{};
  const int64_t reach = static_cast<int64_t>(pages_per_seq) * kv->page_size;
  const int64_t rows = static_cast<int64_t>(T) * (H / kv->KVH);
  p.shared = B > 1 ? prefix_len / 64 * 64 : 0;   // one sequence has nothing to share; the rest of 64 is read per sequence
  p.rw = row_warps(rows);
  p.tiles = static_cast<int>((rows + 16 * p.rw - 1) / (16 * p.rw));
  int64_t keys = max_len > 0 && max_len < reach ? max_len : reach;
  if (keys < prefix_len) keys = prefix_len;
  split_keys(static_cast<int64_t>(B) * kv->KVH * p.tiles, keys - p.shared, sm, kMaxParts, &p.cs, &p.ncl);
  p.rw_p = row_warps(B * rows);
  p.tiles_p = static_cast<int>((B * rows + 16 * p.rw_p - 1) / (16 * p.rw_p));
  p.tc5 = p.shared >= 128 && B * rows > 64 && box_rows(*kv, prefix_len) > 0;
  if (p.tc5) {
    // one CTA per SM, at least two tiles of 128 keys each
    const int64_t groups = kv->KVH * ((B * rows + 255) / 256), tiles = (p.shared + 127) / 128;
    const int per = B * rows > 128 ? 1 : 2;   // partials of a CTA
    int64_t n = sm / groups;
    if (n > tiles / 2) n = tiles / 2;
    if (n > kMaxParts / per) n = kMaxParts / per;
    p.cs_p = 1;
    p.ncl_p = static_cast<int>(n < 1 ? 1 : n);
    p.nparts = p.ncl_p * per;
  } else if (p.shared > 0) {
    split_keys(static_cast<int64_t>(kv->KVH) * p.tiles_p, p.shared, sm, kMaxParts, &p.cs_p, &p.ncl_p);
    p.nparts = p.ncl_p;
  }
  p.parts = p.nparts + (p.ncl > 1 ? p.ncl : 0);
  p.bytes = static_cast<size_t>(p.parts) * B * T * H * (kv->D + 2) * 4;
  return p;
}

template <typename T, int D>
int run(PagedAttnArgs& a, const Plan& p, bool pdl, cudaStream_t s) {
  int st;
  PoolMaps maps;
  if (a.box_rows && (!encode_pool(&maps.k, a.kv, a.kv.k, a.kv.sk_p, a.kv.sk_h, a.kv.sk_s, a.box_rows) ||
                     !encode_pool(&maps.v, a.kv, a.kv.v, a.kv.sv_p, a.kv.sv_h, a.kv.sv_s, a.box_rows)))
    a.box_rows = 0;
  if (p.shared > 0) {
    PagedAttnArgs ap = a;
    ap.tiles = p.tiles_p; ap.cs = p.cs_p; ap.ncl = p.ncl_p;
    if (p.tc5 && a.box_rows) {
      st = launch_prefix_tc5(maps, ap, pdl, s);
    } else {
      if (p.tc5) ap.ncl = p.nparts;   // tensor maps refused: as many partials from the other kernel
      st = launch_rows<T, D, true>(maps, ap, p.rw_p, pdl, s);
    }
    if (st != B2D_OK) return st;
    a.after_prefix = 1;
  }
  if ((st = launch_rows<T, D, false>(maps, a, p.rw, pdl || a.after_prefix, s)) != B2D_OK) return st;
  if (p.ncl > 1) {
    const int64_t rows = static_cast<int64_t>(a.B) * a.T * a.H;
    st = launch_kernel(paged_combine_kernel<T, D>, dim3(static_cast<unsigned>((rows + kWarps - 1) / kWarps)),
                       dim3(kConsumers), 0, s, true, a);
  }
  return st;
}

int check_shapes(const b2d_paged_kv* kv, int B, int T, int H, int pages_per_seq, int prefix_len, int max_len) {
  const int st = check_paged_kv(kv);
  if (st != B2D_OK) return st;
  if (B < 0 || T < 0 || H < 0 || pages_per_seq < 0 || prefix_len < 0 || max_len < 0) return B2D_ERR_ARG;
  if ((kv->D != 64 && kv->D != 128) || H % kv->KVH != 0 || H / kv->KVH > kMaxG || T > kMaxT) return B2D_ERR_SHAPE;
  if (static_cast<int64_t>(pages_per_seq) * kv->page_size >= (int64_t(1) << 31) || B > 65535 || kv->KVH > 65535)
    return B2D_ERR_SHAPE;
  return B2D_OK;
}

}  // namespace
}  // namespace b2d

using namespace b2d;

extern "C" size_t b2d_paged_attention_workspace_bytes(const b2d_paged_kv* kv, int B, int T, int H, int pages_per_seq,
                                                      int prefix_len, int max_len) {
  if (check_shapes(kv, B, T, H, pages_per_seq, prefix_len, max_len) != B2D_OK || B == 0 || T == 0 || H == 0) return 0;
  DeviceInfo di;
  if (device_info(&di) != B2D_OK) return 0;
  return make_plan(kv, B, T, H, pages_per_seq, prefix_len, max_len, di.sm_count).bytes;
}

extern "C" int b2d_paged_attention(const b2d_paged_kv* kv, const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                                   const int32_t* page_table, int64_t ld_table, int pages_per_seq,
                                   const int32_t* seqlens, const int32_t* prefix_table, int prefix_len, int max_len,
                                   int B, int T, int H, float scale, void* out, int64_t so_b, int64_t so_t,
                                   int64_t so_h, int out_dtype, void* workspace, size_t workspace_bytes, int flags,
                                   void* stream) {
  int st;
  if ((st = check_shapes(kv, B, T, H, pages_per_seq, prefix_len, max_len)) != B2D_OK) return st;
  if (out_dtype != kv->dtype && out_dtype != B2D_F32) return B2D_ERR_DTYPE;
  if (B == 0 || T == 0 || H == 0) return B2D_OK;
  if (ld_table < 0) return B2D_ERR_SHAPE;
  if (!q || !seqlens || !out || (!page_table && pages_per_seq > 0) || (prefix_len > 0 && !prefix_table))
    return B2D_ERR_ARG;
  if (!aligned(q, 16) || (sq_b | sq_t | sq_h) % 8 || !aligned(page_table, 4) || !aligned(seqlens, 4) ||
      !aligned(prefix_table, 4) || !aligned(out, out_dtype == B2D_F32 ? 4 : 2))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  if ((st = device_info(&di)) != B2D_OK) return st;
  const Plan p = make_plan(kv, B, T, H, pages_per_seq, prefix_len, max_len, di.sm_count);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return B2D_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return B2D_ERR_ALIGN;
  if (static_cast<int64_t>(B) * T * H >= (int64_t(1) << 31) || static_cast<int64_t>(p.tiles_p) * p.cs_p * p.ncl_p >= (int64_t(1) << 31))
    return B2D_ERR_SHAPE;
  PagedAttnArgs a{};
  a.q = q; a.sq_b = sq_b; a.sq_t = sq_t; a.sq_h = sq_h;
  a.table = page_table; a.ld_table = ld_table; a.seqlens = seqlens; a.prefix_table = prefix_table;
  a.out = out; a.so_b = so_b; a.so_t = so_t; a.so_h = so_h;
  a.kv = *kv; a.div = page_div(kv->page_size);
  a.pages_per_seq = pages_per_seq; a.prefix_len = prefix_len;
  a.B = B; a.T = T; a.H = H; a.G = H / kv->KVH; a.rows = T * a.G;
  a.scale_log2 = scale * kLog2e;
  a.shared = p.shared; a.cs = p.cs; a.ncl = p.ncl; a.tiles = p.tiles; a.nparts = p.nparts; a.parts = p.parts;
  a.out_f32 = out_dtype == B2D_F32;
  a.box_rows = box_rows(*kv, prefix_len);
  a.acc = static_cast<float*>(workspace);
  a.ml = a.acc ? a.acc + static_cast<int64_t>(p.parts) * B * T * H * kv->D : nullptr;
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kv->dtype == B2D_F16) return kv->D == 64 ? run<__half, 64>(a, p, pdl, s) : run<__half, 128>(a, p, pdl, s);
  return kv->D == 64 ? run<__nv_bfloat16, 64>(a, p, pdl, s) : run<__nv_bfloat16, 128>(a, p, pdl, s);
}
