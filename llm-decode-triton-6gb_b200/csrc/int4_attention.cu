// Attention of the newest tokens of every sequence over the paged cache in 4 bits, causal among themselves (sm_100a). The
// layout is in int4_kv.cuh, the 16-bit counterpart in paged_attention.cu.
//
//   k = m + s c, so q.k = sum over runs (s sum q c + m sum q): the products are with the codes, and a key's two factors per run
//   enter its score in fp32 behind them. o = sum_j p_j v_j = sum_j (p_j s_j) c_j + sum_j p_j m_j: a value's s goes into its
//   weight (per run of elements), the second sum is fp32 and has one term per key, row and run.
//
// Codes become operands by masks (fp16 subnormals, see int4_kv.cuh): 5 instructions for 8 elements. Products are transposed as
// in the 16-bit kernel: keys (elements) as M, rows as N tiles of 8, where a row is one of the T x G query vectors that read a
// KV head.
//  * A query row is scaled by a power of two into [2^14, 2^15) so that it and its part for the high nibbles (2^-4) are as
//    exact in fp16 as in its own type.
//  * A weight p_j s_j is rounded to fp16 (2^-11) in a unit of its row: unit p s lies below 2^15, and was above 2^5 for the largest
//    p s that the row has met, so that all 11 bits are kept down to 2^-19 of that. What counts is what a key adds to the row: one with a
//    huge s and next to no weight, or one that the row does not see, takes nothing from the others. The unit and the running
//    maximum move rarely (a maximum only when a score exceeds it by 2^8), on one vote, and each row's by its own scores alone.
//  * Every warp is on its own: it copies its tiles of 16 keys (2.3 KB, keys, values and factors in one asynchronous bulk copy)
//    through a private ring of shared memory, waits on its own mbarriers, and meets the block's other warps only at the end
//    of a unit. Codes are finite whatever a page holds; factors of keys that a row does not see are taken out by selection.
//
// Units of work are (sequence, KV head, tile of up to 32 rows). As in the 16-bit kernel the units' stages (64 keys, a
// tile a warp) form one line of which every block takes an equal share, found from the lengths on the device; parts of a unit
// that several blocks share meet in a combine launch. No atomics: results are the same bits every run.
//
// Measured on B200 (GPU time of a call, graph replays over rotated inputs; each key and value once at the copy rate of 6.55 TB/s
// in brackets): 8 sequences of 16001..32768 keys, 32 / 8 heads of 128, fp16: 52 us (34); 64 of 100..4609, groups of 32: 55.7 us (30);
// 8 of 512..2048: 11.3 us (1.8); 16 x 5 drafts, up to 4099 keys: 33 us (6.0); one of 300 keys: 7.0 us. The 16-bit kernel takes 13.9,
// 38 and 7.5 us for the last three. A unit of a row's own costs 1 to 6 % of that (one for all of a warp's rows: 51.7, 54.4, 10.9, 31.0,
// 6.7), with 32 rows of a KV head 12 % (16 x 8 drafts 53.3 and 47.8). Long: the loop reads at 5.4 TB/s, 41 us of the call (300
// instructions a tile, 63 % of the slots issue, the logic pipe 51 % busy); 6 us pass before the first tiles land, 2 go to the
// combine. Groups of 32: 370 instructions a tile, 4.85 TB/s, 40 us of the call. Short: dependent steps of one warp -- lengths 0.7,
// segment and pages 1.4, queries 0.4, a tile 1.0, merge 0.9, combine 1.4 us. More row tiles: eight warps an SM (their
// accumulators take the registers) issue in 41 % of the slots. Spills (bytes stored, heads of 128, 1 to 4 row tiles): groups of 64 0, 12,
// 0, 192; of 32 24, 76, 0, 752; heads of 64 none. Not kept: a producer warp for one block of 15 consumers an SM (a
// lane's bulk copies serialise, all warps meet at a unit's end: 56 and 94 us for the first two); clusters in place of the combine (0.5 us
// more for 300 keys); five blocks an SM (63 us for the first); whole bytes as operands (fewer masks, more products: the same).
#include <type_traits>

#include "int4_kv.cuh"
#include "pipeline.cuh"

namespace b2d {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStage = kWarps * kTileKeys;      // keys of a position of the line
constexpr int kMaxT = 16, kMaxG = 16;
constexpr int kMaxBatch = 256;                  // sequences of a launch (larger batches take several)
constexpr int kMaxCtas = 640;
// Up to so many keys a unit is one CTA's, and there is no combine launch (8 sequences of up to 256 keys, 8 KV heads: 8.2 -> 7.5 us in a
// graph when the rule was made, 7.3 now; one of 300: 7.2 -> 7.7); with two units an SM or more up to 512 keys (64 sequences: 16.5 -> 13.7).
constexpr int kWholeKeys = 256, kWholeKeysMany = 512;
constexpr float kLazy = 8.f;                    // log2 of the largest weight before the running maximum moves
constexpr float kNone = -1.7e38f;               // running maximum before the first score
constexpr float kMost = 0x1p15f;                // largest weight times s in its row's unit (fp16 ends at 65504)
constexpr float kUnitMost = 0x1p115f;           // largest unit, and that before the first p s
constexpr float kLog2e = 1.4426950408889634f;

// Blocks of an SM, by registers (accumulators: 32 a row tile), and tiles of a warp's ring, by shared memory.
template <int NT>
constexpr int kBlocks = NT == 1 ? 4 : NT == 2 ? 3 : 2;
template <int D, int RUNS, int NT>
struct Smem {
  static constexpr int TILE = int4_tile_bytes(D, RUNS);
  static constexpr int MERGE = kWarps * 8 * (D + 4) * 4;
  static constexpr int Q = NT * (D / 16) * 32 * 8;              // prepared fragments
  static constexpr int FIXED = MERGE + Q + 2048;                // and the static arrays
  static constexpr int ROOM = 224 * 1024 / kBlocks<NT> - FIXED;
  static constexpr int SLOTS = ROOM / (kWarps * TILE) < 8 ? ROOM / (kWarps * TILE) : 8;
  static constexpr int RING = kWarps * SLOTS * TILE;
  static constexpr int BYTES = RING + MERGE + Q;
};

struct Int4AttnArgs {
  const void* q; int64_t sq_b, sq_t, sq_h;
  const int32_t* table; int64_t ld_table;
  const int32_t* seqlens;
  void* out; int64_t so_b, so_t, so_h;
  b2d_int4_kv kv;
  PageDiv div;
  int pages_per_seq, B, T, H, G, rows;   // rows = T G: query vectors of a sequence and KV head
  int inv_g;        // 2^16 / G, rounded up
  float scale_log2;
  int ctas, whole, out_f32, out_vec;
  // Workspace: [ctas][2][row tile] entries of D unnormalised fp32 sums, and (m in the log2 domain, l)
  float* acc;
  float* ml;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar) : "memory");
}

__device__ __align__(16) uint8_t g_zero_tile[int4_tile_bytes(128, 4)];   // never written

// N neighbouring words of shared memory, aligned to their size
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    static_assert(N == 1, "1, 2 or 4 words");
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// codes at 2^(-20 - SHIFT) -> themselves less 8
template <int SHIFT>
__device__ __forceinline__ uint32_t minus_8(uint32_t x) {
  const uint32_t eight = 0x00800080u >> SHIFT;
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&eight));
  return *reinterpret_cast<const uint32_t*>(&y);
}

template <typename T>
__device__ __forceinline__ void store_out(const Int4AttnArgs& a, int64_t off, float v) {
  if (a.out_f32) static_cast<float*>(a.out)[off] = v;
  else static_cast<T*>(a.out)[off] = Dt<T>::from_f32(v);
}
// two neighbouring outputs; `out_vec`: every row starts on a boundary of their size
template <typename T>
__device__ __forceinline__ void store_out2(const Int4AttnArgs& a, int64_t off, float x, float y) {
  if (!a.out_vec) {
    store_out<T>(a, off, x);
    store_out<T>(a, off + 1, y);
  } else if (a.out_f32) {
    *reinterpret_cast<float2*>(static_cast<float*>(a.out) + off) = make_float2(x, y);
  } else {
    *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + off) = Dt<T>::pack2(x, y);
  }
}

// The line of all units' work: the sequences in order, KV head by KV head and row tile by row tile. A unit takes LEAD
// positions, what its start and end cost in stages, and one for each stage; one without keys takes none. CTA c takes the
// positions [share(c), share(c + 1)); the host has checked that they fit 31 bits. In whole mode a unit is one position.
template <int NT>
struct Line {
  static constexpr int ROWS = 8 * NT, LEAD = 5;
  int tiles, units, ctas, quota, extra;
  __device__ __forceinline__ Line(const Int4AttnArgs& a) {
    tiles = (a.rows + ROWS - 1) / ROWS;
    units = a.kv.KVH * tiles;
  }
  static __device__ __forceinline__ int cost_of(const Int4AttnArgs& a, int len) {
    return a.whole ? 1 : len > 0 ? (len + kStage - 1) / kStage + LEAD : 0;
  }
  __device__ __forceinline__ void close(const Int4AttnArgs& a, int cost) {   // of all sequences
    const int total = cost * units;
    ctas = min(total, a.ctas);   // the CTAs with a share, none of them empty
    quota = ctas > 0 ? total / ctas : 0;
    extra = total - quota * ctas;   // so many CTAs take one position more
  }
  __device__ __forceinline__ int share(int c) const { return c < ctas ? c * quota + min(c, extra) : ctas * quota + extra; }
  __device__ __forceinline__ int owner(int x) const {
    const int cut = extra * (quota + 1);
    return x < cut ? x / (quota + 1) : extra + (x - cut) / quota;
  }
};

// The sequences' lengths, cut to the page table, into s_len and the exclusive running sums of their units' cost into
// s_sum[0 .. B] (all THREADS of the block take part). The lengths come from L2: the combine reads them ahead of its wait.
template <int NT, int THREADS>
__device__ __forceinline__ void scan_costs(const Int4AttnArgs& a, int* s_sum, int* s_len, int* s_warp) {
  constexpr int W = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int reach = a.pages_per_seq * a.kv.page_size;
  int run = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + tid;
    const int len = b < a.B ? min(max(load_l2(a.seqlens + b), 0), reach) : 0;
    const int own = b < a.B ? Line<NT>::cost_of(a, len) : 0;
    int v = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    if (lane == 31) s_warp[warp] = v;
    __syncthreads();
    int before = run;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += s_warp[w];
      run += s_warp[w];
    }
    if (b < a.B) {
      s_sum[b] = before + v - own;
      s_len[b] = len;
    }
    __syncthreads();
  }
  if (tid == 0) s_sum[a.B] = run;
  __syncthreads();
}

// A CTA's stretch of one unit: keys [t_begin, t_end).
struct Segment {
  int b, kvh, row0, nrows;
  int t_begin, t_end, limit;     // query t sees the keys before limit + t
  int kind;                      // 0: the whole unit, 1 / 2: the end (or middle) / the start of a shared one, < 0: none
  int next;                      // position behind it
};
// The segment at position pos of a share that ends at `end`; none where only a unit's lead lies in the share.
template <int NT>
__device__ __forceinline__ Segment segment_at(const Int4AttnArgs& a, const Line<NT>& line, const int* s_sum,
                                              const int* s_len, int pos, int end) {
  constexpr int ROWS = 8 * NT, LEAD = Line<NT>::LEAD;
  Segment g;
  int lo = 0, hi = a.B - 1;   // the last sequence that starts at or before pos
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_sum[mid] * line.units <= pos) lo = mid;
    else hi = mid - 1;
  }
  g.b = lo;
  const int len = s_len[lo], cost = s_sum[lo + 1] - s_sum[lo];
  int start = s_sum[lo] * line.units;
  const int u = (pos - start) / cost;
  start += u * cost;
  g.limit = len - a.T + 1;
  g.kvh = line.tiles == 1 ? u : u / line.tiles;
  g.row0 = (u - g.kvh * line.tiles) * ROWS;
  g.nrows = min(a.rows - g.row0, ROWS);
  g.next = min(end, start + cost);
  if (a.whole) {
    g.t_begin = 0;
    g.t_end = len;
    g.kind = 0;
  } else {
    const int s0 = max(pos - start - LEAD, 0), s1 = g.next - start - LEAD;
    g.t_begin = s0 * kStage;
    g.t_end = min(len, s1 * kStage);
    g.kind = s1 <= s0 ? -1 : s0 > 0 ? 1 : s1 < cost - LEAD ? 2 : 0;
  }
  return g;
}

__device__ __forceinline__ int div_g(const Int4AttnArgs& a, int r) { return r * a.inv_g >> 16; }   // r < 256, G <= 16: exact

template <typename T, int D, int RUNS, int NT>
__global__ void __launch_bounds__(kThreads, kBlocks<NT>) int4_attention_kernel(const __grid_constant__ Int4AttnArgs a) {
  using S = Smem<D, RUNS, NT>;
  constexpr int ROWS = 8 * NT, STEPS = D / 16, RSTEPS = STEPS / RUNS;   // products of a tile, and of a run of elements
  constexpr int TILE = S::TILE, SLOTS = S::SLOTS, KW = D / 32;          // KW: key words of a lane and key
  static_assert(SLOTS >= 2, "a ring of at least two tiles");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
  __shared__ __align__(8) float s_rowf[ROWS], s_qs[RUNS][ROWS];
  __shared__ __align__(8) uint64_t s_bar[kWarps * SLOTS];
  __shared__ int s_sum[kMaxBatch + 1], s_len[kMaxBatch], s_warp[kWarps];
  __shared__ int64_t s_at[ROWS];        // per row: offset in the output, or workspace entry

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g8 = lane >> 2, tq = lane & 3;
  uint8_t* const ring = smem + warp * (SLOTS * TILE);
  float* const s_o = reinterpret_cast<float*>(smem + S::RING);
  uint2* const s_q = reinterpret_cast<uint2*>(smem + S::RING + S::MERGE);   // [row tile][step][lane]
  const uint32_t ring_s = smem_u32(ring), full = smem_u32(s_bar + warp * SLOTS);
  if (lane < SLOTS) mbar_init(full + 8 * lane, 1);
  fence_mbar_init();
  pdl_wait();
  pdl_launch_dependents();
  const Line<NT> line = [&] {
    Line<NT> l(a);
    scan_costs<NT, kThreads>(a, s_sum, s_len, s_warp);
    l.close(a, s_sum[a.B]);
    return l;
  }();
  const int first = line.share(blockIdx.x), end = line.share(blockIdx.x + 1);

  // ---- the warp's copies, ahead of its products: tile `ft` of the warp's `fn` in segment `fg` next. The sources of tiles up
  // to `fc` are at hand: lane l has that of tile l (modulo 32).
  bool landed = true;   // until a wait runs out: no copies are sent after that
  int fpos = first, ft = 0, fn = 0, fc = 0, fslot = 0, ahead = 0;   // ahead: copies under way
  Segment fg{};
  const uint8_t* src = nullptr;
  auto lookup = [&] {
    fc = min(fn, ft + 32);
    const int key = fg.t_begin + ((ft + ((lane - ft) & 31)) * kWarps + warp) * kTileKeys;
    src = g_zero_tile;   // of a page id outside the pool: keys and values of zeros
    if (key < fg.t_end) {
      const int pi = a.div.page(key), page = a.table[fg.b * a.ld_table + pi];   // (not the read-only path: see int4_append.cu)
      if (page >= 0 && page < a.kv.num_pages)
        src = a.kv.pages + page * a.kv.sp_p + fg.kvh * a.kv.sp_h + static_cast<int64_t>(a.div.slot(key, pi) / kTileKeys) * TILE;
    }
  };
  auto issue = [&] {   // the next tile into the next slot, which is free
    if (landed && lane == (ft & 31)) {
      mbar_expect_tx(full + 8 * fslot, TILE);
      bulk_load(ring_s + fslot * TILE, src, TILE, full + 8 * fslot);
    }
    ++ft;
    fslot = fslot + 1 == SLOTS ? 0 : fslot + 1;
  };
  auto refill = [&] {   // every free slot, from the next segments if need be
    while (landed && ahead < SLOTS) {
      if (ft == fc) {
        while (ft == fn) {
          if (fpos >= end) return;
          fg = segment_at<NT>(a, line, s_sum, s_len, fpos, end);
          fpos = fg.next;
          const int tiles = fg.kind < 0 ? 0 : (fg.t_end - fg.t_begin + kTileKeys - 1) / kTileKeys;
          fn = tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0;
          ft = 0;
        }
        lookup();
      }
      issue();
      ++ahead;
    }
  };
  refill();

  int slot = 0, parity = 0;   // of the warp's next tile
  for (int pos = first; pos < end;) {
    const Segment g = segment_at<NT>(a, line, s_sum, s_len, pos, end);
    pos = g.next;
    if (g.kind < 0) continue;
    // ---- Q: D / 8 threads a row, 8 elements each (every thread is behind the last unit's barriers)
    constexpr int QL = D / 8, QROWS = kThreads / QL, QN = (ROWS + QROWS - 1) / QROWS;   // threads a row, rows at a time, times
    uint4 q_raw[QN];
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const int r = i * QROWS + tid / QL, rr = g.row0 + r, t = div_g(a, rr);
      q_raw[i] = make_uint4(0, 0, 0, 0);
      if (r < g.nrows)
        q_raw[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + g.b * a.sq_b + t * a.sq_t +
                                                   static_cast<int64_t>(g.kvh * a.G + rr - t * a.G) * a.sq_h + 8 * (tid % QL));
    }
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const int r = i * QROWS + tid / QL, l = tid % QL;
      const T* raw = reinterpret_cast<const T*>(&q_raw[i]);
      float q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = Dt<T>::to_f32(raw[e]);
      float big = fmaxf(fmaxf(fmaxf(fabsf(q[0]), fabsf(q[1])), fmaxf(fabsf(q[2]), fabsf(q[3]))),
                        fmaxf(fmaxf(fabsf(q[4]), fabsf(q[5])), fmaxf(fabsf(q[6]), fabsf(q[7]))));
#pragma unroll
      for (int x = 1; x < QL; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
      // up = 2^x with 2^x big in [2^14, 2^15); |x| <= 100
      const int ex = static_cast<int>(__float_as_uint(big) >> 23);
      const int x = big > 0.f && ex < 255 ? min(max(14 + 127 - ex, -100), 100) : 0;
      const float up = __uint_as_float((127 + x) << 23), down = __uint_as_float((127 - x) << 23);
      const bool on = ROWS % QROWS == 0 || r < ROWS;
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {   // elements 16 (l / 2) + 8 (l & 1) + 4 h ..: step l / 2, lane 4 (r & 7) + 2 (l & 1) + h
        const float q0 = q[4 * h] * up, q1 = q[4 * h + 1] * up, q2 = q[4 * h + 2] * up, q3 = q[4 * h + 3] * up;
        const __half2 lo = __floats2half2_rn(q0, q1), hi = __floats2half2_rn(q2, q3);
        sum += (__low2float(lo) + __high2float(lo)) + (__low2float(hi) + __high2float(hi));
        if (on)
          s_q[((r >> 3) * STEPS + l / 2) * 32 + 4 * (r & 7) + 2 * (l & 1) + h] =
              make_uint2(Dt<__half>::pack2(q0, q1), Dt<__half>::pack2(q2 * 0.0625f, q3 * 0.0625f));
      }
#pragma unroll
      for (int x = 1; x < QL / RUNS; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      if (on && l % (QL / RUNS) == 0) s_qs[l / (QL / RUNS)][r] = sum * 0x1p-24f;
      if (on && l == 0) s_rowf[r] = down * 0x1p24f * a.scale_log2;
    }
    if (tid < g.nrows) {
      const int rr = g.row0 + tid, t = div_g(a, rr), head = g.kvh * a.G + rr - t * a.G;
      s_at[tid] = g.kind == 0 ? g.b * a.so_b + t * a.so_t + head * a.so_h
                              : (static_cast<int64_t>(blockIdx.x) * 2 + (g.kind - 1)) * ROWS + tid;
    }
    __syncthreads();
    // The rows' factors, of rows 8 n + 2 tq (+ 1): in registers for a unit, but in each tile from shared memory where they would
    // spill (16 x 8 drafts of up to 4000 keys, groups of 64: 53 us against 67; 16 x 3, groups of 32: 34.6, 39.4; but 16 x 5, groups of 64: 37.0,
    // 35.9)
    constexpr bool FAR = D == 128 && NT * RUNS >= 8;
    float rowf[NT][2], qs[RUNS][NT][2];
    auto pair = [&](float (&to)[2], const float* row, int n) {
      const float2 x = *reinterpret_cast<const float2*>(row + 8 * n + 2 * tq);
      to[0] = x.x;
      to[1] = x.y;
    };
    if constexpr (!FAR) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        pair(rowf[n], s_rowf, n);
#pragma unroll
        for (int u = 0; u < RUNS; ++u) pair(qs[u][n], s_qs[u], n);
      }
    }
    // keys that this thread's rows see; below lim_min no row is masked
    const bool causal = a.T > 1;
    const int lim_min = causal ? g.limit + div_g(a, g.row0) : g.limit;
    auto lim = [&](int n, int e) { return causal ? g.limit + div_g(a, g.row0 + min(8 * n + 2 * tq + e, g.nrows - 1)) : g.limit; };

    float o[STEPS][NT][4];   // element 16 m + g8 (+ 8), row 8 n + 2 tq (+ 1), times the row's unit and 2^-24 (2^-20)
    float om[RUNS][NT][2];   // sum of p (m + 8 s) over this thread's keys
    float m_run[NT][2], l_run[NT][2];   // log2 domain; the sum over this thread's keys only
    float unit[NT][2];       // a weight enters the second product as p s unit
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int m = 0; m < STEPS; ++m) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
#pragma unroll
      for (int u = 0; u < RUNS; ++u) om[u][n][0] = om[u][n][1] = 0.f;
      m_run[n][0] = m_run[n][1] = kNone;
      l_run[n][0] = l_run[n][1] = 0.f;
      unit[n][0] = unit[n][1] = kUnitMost;
    }

    // One tile: its scores, its weights, its part of o. MASKED: some row does not see some key of it.
    auto tile = [&](auto masked_, int key0) {
      constexpr bool MASKED = decltype(masked_)::value;
      landed = landed && mbar_wait(full + 8 * slot, parity);
      const uint8_t* const buf = ring + slot * TILE;
      float acc[RUNS][NT][4];   // key g8 (+ 8), row 8 n + 2 tq (+ 1)
      {
        uint32_t kw[2][KW];
#pragma unroll
        for (int h = 0; h < 2; ++h) load_words(buf + (g8 + 8 * h) * (D / 2) + tq * (D / 8), kw[h]);
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
          const int sh = 8 * (j & 1), u = j / RSTEPS;
          const uint32_t x = kw[0][j / 2] >> sh, y = kw[1][j / 2] >> sh;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 q = s_q[(n * STEPS + j) * 32 + lane];
            if (j % RSTEPS == 0) Mma<__half>::run0(acc[u][n], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q.x, q.y);
            else Mma<__half>::run(acc[u][n], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q.x, q.y);
          }
        }
      }
      // scores: acc[0] becomes them over rowf, d what they are past the running maximum
      float d[NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t f[RUNS];
        load_words(buf + int4_ks_off(D) + (g8 + 8 * h) * (4 * RUNS), f);
#pragma unroll
        for (int u = 0; u < RUNS; ++u) {
          const float2 sm = unpack_sm<T>(f[u]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (FAR) pair(qs[u][n], s_qs[u], n);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = acc[u][n][2 * h + e];
              acc[0][n][2 * h + e] = fmaf(sm.y, qs[u][n][e], u == 0 ? sm.x * x : fmaf(sm.x, x, acc[0][n][2 * h + e]));
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (FAR) pair(rowf[n], s_rowf, n);
#pragma unroll
          for (int e = 0; e < 2; ++e) d[n][2 * h + e] = fmaf(acc[0][n][2 * h + e], rowf[n][e], -m_run[n][e]);
        }
      }
      float2 vf[2][RUNS];   // the values' factors of keys g8 (+ 8)
      float s_top[2] = {0.f, 0.f}, d_top = -INFINITY;   // the largest s of keys g8 (+ 8)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t f[RUNS];
        load_words(buf + int4_vs_off(D, RUNS) + (g8 + 8 * h) * (4 * RUNS), f);
#pragma unroll
        for (int u = 0; u < RUNS; ++u) vf[h][u] = unpack_sm<T>(f[u]);
      }
      auto hidden = [&](int n, int h, int e) {
        const int key = key0 + g8 + 8 * h;
        return MASKED && (key >= lim(n, e) || key >= g.t_end);
      };
      if constexpr (MASKED) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = key0 + g8 + 8 * h;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (hidden(n, h, e)) d[n][2 * h + e] = -INFINITY;
          if (key >= g.t_end) {   // what lies behind the last key is not the cache's
#pragma unroll
            for (int u = 0; u < RUNS; ++u) vf[h][u] = make_float2(0.f, 0.f);
          }
        }
      }
      float w[NT][4], w_top[2] = {0.f, 0.f};   // the weights in their rows' units
      auto weigh = [&](int n, int c) {
        d[n][c] = exp2_fast(d[n][c]);
        w[n][c] = d[n][c] * unit[n][c & 1];
      };
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int u = 0; u < RUNS; ++u) s_top[h] = fmaxf(s_top[h], vf[h][u].x);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          d_top = fmaxf(d_top, fmaxf(d[n][2 * h], d[n][2 * h + 1]));
          weigh(n, 2 * h);
          weigh(n, 2 * h + 1);
          w_top[h] = fmaxf(w_top[h], fmaxf(w[n][2 * h], w[n][2 * h + 1]));
        }
      }
      if (__any_sync(0xffffffffu, fmaxf(w_top[0] * s_top[0], w_top[1] * s_top[1]) > kMost || d_top > kLazy)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if constexpr (FAR) pair(rowf[n], s_rowf, n);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = -INFINITY, most = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) top = fmaxf(top, hidden(n, h, e) ? -INFINITY : __fmul_rn(acc[0][n][2 * h + e], rowf[n][e]));
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
            const bool up = top > m_run[n][e] + kLazy;
            const float alpha = up ? exp2_fast(m_run[n][e] - top) : 1.f;   // m_run = kNone: 0
            if (up) m_run[n][e] = top;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              // behind a new maximum by the rounded scores, as it is one: at sizes whose rounding is above one its key keeps its weight
              const float a0 = acc[0][n][2 * h + e], by_score = __fmul_rn(a0, rowf[n][e]) - m_run[n][e];
              const float by_product = fmaf(a0, rowf[n][e], -m_run[n][e]);   // as without the vote
              d[n][2 * h + e] = hidden(n, h, e) ? -INFINITY : up || by_product > kLazy ? by_score : by_product;
              most = fmaxf(most, exp2_fast(d[n][2 * h + e]) * s_top[h]);
            }
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, i));
            // what alpha takes from the sums the unit may give back; then the tile's largest p s goes to [2^5, 2^6)
            float now = up ? fminf(__fdividef(unit[n][e], alpha), kUnitMost) : unit[n][e];
            if (most * now > kMost) {
              const int ex = min(static_cast<int>(__float_as_uint(most) >> 23) - 127, 108);
              now = __uint_as_float((127 + 5 - ex) << 23);
            }
            const float keep = __fdividef(alpha * now, unit[n][e]);
            unit[n][e] = now;
            l_run[n][e] *= alpha;
#pragma unroll
            for (int u = 0; u < RUNS; ++u) om[u][n][e] *= alpha;
#pragma unroll
            for (int m = 0; m < STEPS; ++m) {
              o[m][n][e] *= keep;
              o[m][n][2 + e] *= keep;
            }
            weigh(n, e);
            weigh(n, 2 + e);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) l_run[n][c & 1] += d[n][c];
      uint32_t pb[RUNS][NT][2];   // P s as the B operand: row 8 n + g8, keys 2 tq .. (+ 8)
#pragma unroll
      for (int u = 0; u < RUNS; ++u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float su = vf[h][u].x, center = fmaf(8.f, su, vf[h][u].y);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float w0 = w[n][2 * h] * su, w1 = w[n][2 * h + 1] * su;
            if constexpr (MASKED) {   // factors that are infinite or NaN reach the rows that see their key, and no other
              const int key = key0 + g8 + 8 * h;
              if (key < lim(n, 0)) om[u][n][0] = fmaf(d[n][2 * h], center, om[u][n][0]);
              else w0 = 0.f;
              if (key < lim(n, 1)) om[u][n][1] = fmaf(d[n][2 * h + 1], center, om[u][n][1]);
              else w1 = 0.f;
            } else {
              om[u][n][0] = fmaf(d[n][2 * h], center, om[u][n][0]);
              om[u][n][1] = fmaf(d[n][2 * h + 1], center, om[u][n][1]);
            }
            pb[u][n][h] = transpose8(Dt<__half>::pack2(w0, w1));
          }
        }
      }
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        uint32_t vw[4];
        load_words(buf + int4_v_off(D) + c * 512 + lane * 16, vw);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int m = 4 * c + i, u = m / RSTEPS;
          const uint32_t y = vw[i] >> 8;
          // around their middle: weights times codes from 0 to 15 would grow with the number of keys where their values cancel, and
          // the tensor cores' sums cut what does not fit below
          const uint32_t a0 = minus_8<4>(vw[i] & 0x000F000Fu), a1 = minus_8<0>(vw[i] & 0x00F000F0u);
          const uint32_t a2 = minus_8<4>(y & 0x000F000Fu), a3 = minus_8<0>(y & 0x00F000F0u);
#pragma unroll
          for (int n = 0; n < NT; ++n) Mma<__half>::run(o[m][n], a0, a1, a2, a3, pb[u][n][0], pb[u][n][1]);
        }
      }
      __syncwarp();   // the warp is done with the slot
      slot += landed;
      if (slot == SLOTS) {
        slot = 0;
        parity ^= 1;
      }
    };
    const int tiles = (g.t_end - g.t_begin + kTileKeys - 1) / kTileKeys, seen = min(lim_min, g.t_end) / kTileKeys - g.t_begin / kTileKeys;
    int left = tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0;     // the warp's tiles
    int clear = seen > warp ? (seen - warp + kWarps - 1) / kWarps : 0;      // of which the first are seen whole by all rows
    int key0 = g.t_begin + warp * kTileKeys;
    // While the segment has further tiles to fetch: one follows each tile into its slot. Nothing but this in the loop: the
    // search for pages and segments, or the masks, would cost every tile 50 to 80 register moves and tests.
    while (clear > 0 && fg.next == g.next && ft < fn) {
      if (ft == fc) lookup();
      const int n = min(clear, fc - ft);
#pragma unroll 1
      for (int i = 0; i < n; ++i, key0 += kStage) {
        tile(std::false_type{}, key0);
        issue();
      }
      clear -= n;
      left -= n;
    }
#pragma unroll 1
    for (; left > 0; --left, key0 += kStage) {
      tile(std::true_type{}, key0);
      ahead -= landed;
      refill();
    }

    // ---- the unit's (or this CTA's part of it) result: the warps meet in shared memory
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l_run[n][e] += __shfl_xor_sync(0xffffffffu, l_run[n][e], x);
#pragma unroll
          for (int u = 0; u < RUNS; ++u) om[u][n][e] += __shfl_xor_sync(0xffffffffu, om[u][n][e], x);
        }
        if (g8 == 0) {
          s_m[warp][8 * n + 2 * tq + e] = m_run[n][e];
          s_l[warp][8 * n + 2 * tq + e] = landed ? l_run[n][e] : NAN;
        }
      }
    __syncthreads();
    if (tid < g.nrows) {   // (m, l) of a row, and the warps' factors in the place of their maxima
      float mx = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_m[w][tid]);
      float f[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        f[w] = exp2_fast(s_m[w][tid] - mx);   // (without a key: no weights, and their factor is of no account)
        l += f[w] * s_l[w][tid];
      }
      // a row that sees no key: zeros (l is NaN, not 0, where a visible score is)
      const float inv = g.kind == 0 ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
      if (g.kind != 0) *reinterpret_cast<float2*>(a.ml + s_at[tid] * 2) = make_float2(mx, l);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) s_m[w][tid] = f[w] * inv;
    }
    __syncthreads();
    constexpr int PAD = D + 4;   // the rows 2 tq of the accumulators' columns fall into different banks
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (8 * n >= g.nrows) break;
      if (n > 0) __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float factor = s_m[warp][8 * n + 2 * tq + e], to_lo = 0x1p24f / unit[n][e], to_hi = 0.0625f * to_lo;
        float* dst = s_o + (warp * 8 + 2 * tq + e) * PAD + g8;
#pragma unroll
        for (int m = 0; m < STEPS; ++m) {
          const float b = om[m / RSTEPS][n][e];
          dst[16 * m] = fmaf(o[m][n][e], to_lo, b) * factor;
          dst[16 * m + 8] = fmaf(o[m][n][2 + e], to_hi, b) * factor;
        }
      }
      __syncthreads();
      const int live = min(g.nrows - 8 * n, 8);
      for (int idx = tid; idx < live * (D / 4); idx += kThreads) {
        const int row = idx / (D / 4), d = 4 * (idx % (D / 4));
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(s_o + (w * 8 + row) * PAD + d);
          v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        const int64_t at = s_at[8 * n + row];
        if (g.kind == 0) {
          store_out2<T>(a, at + d, v.x, v.y);
          store_out2<T>(a, at + d + 2, v.z, v.w);
        } else {
          *reinterpret_cast<float4*>(a.acc + at * D + d) = v;
        }
      }
    }
    __syncthreads();   // s_at, s_m and s_o are free again
  }
  // Nothing is under way into this block's memory when it ends: every tile that was sent has been waited for, unless a wait ran out
  if (!landed) {
    for (; ahead > 0; --ahead) {
      landed = mbar_wait(full + 8 * slot, parity);
      if (++slot == SLOTS) {
        slot = 0;
        parity ^= 1;
      }
    }
  }
}

// Merges the entries of units that several CTAs share: a block of 128 threads for 512 / D rows of a (sequence, KV head), four
// elements a thread, with a running maximum, so that one round trip to memory follows the first kernel's end. GROUPS > 1: so
// many groups of 128 threads share the entries of a unit that many CTAs have cut.
template <typename T, int D, int NT, int GROUPS>
__global__ void __launch_bounds__(128 * GROUPS) int4_combine_kernel(const __grid_constant__ Int4AttnArgs a) {
  constexpr int ROWS = 8 * NT, QUADS = D / 4, BLOCK_ROWS = 128 / QUADS;
  __shared__ int s_sum[kMaxBatch + 1], s_len[kMaxBatch], s_warp[4 * GROUPS];
  __shared__ float4 s_v[GROUPS > 1 ? 128 * GROUPS : 1];   // the groups' sums and (m, l)
  __shared__ float2 s_ml[GROUPS > 1 ? 128 * GROUPS : 1];
  const int tid = threadIdx.x, group = tid / 128;
  pdl_launch_dependents();
  // the lengths are inputs of the whole call, complete before its first kernel began
  Line<NT> line(a);
  scan_costs<NT, 128 * GROUPS>(a, s_sum, s_len, s_warp);
  line.close(a, s_sum[a.B]);
  const int b = blockIdx.x / a.kv.KVH, kvh = blockIdx.x - b * a.kv.KVH, cost = s_sum[b + 1] - s_sum[b];
  const int row = blockIdx.y * BLOCK_ROWS + tid % 128 / QUADS, d = (tid % QUADS) * 4;
  const bool on = row < a.rows;
  // the CTAs that share the row's unit: entry (c, started there) of each
  int c0 = 0, c1 = -1, p0 = 0;
  if (on && cost > 0) {
    const int start = s_sum[b] * line.units + (kvh * line.tiles + row / ROWS) * cost;
    p0 = start + Line<NT>::LEAD;
    c0 = line.owner(p0);
    c1 = line.owner(start + cost - 1);
    if (c0 == c1) c1 = -2;   // written by the first kernel
  }
  pdl_wait();
  float m = -INFINITY, l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c = c0 + 8 * group; c <= c1; c += 8 * GROUPS) {   // eight entries in flight
    float4 x[8];
    float2 ml[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c + k <= c1) {
        const int64_t at = (static_cast<int64_t>(c + k) * 2 + (line.share(c + k) <= p0 ? 1 : 0)) * ROWS + row % ROWS;
        ml[k] = *reinterpret_cast<const float2*>(a.ml + at * 2);
        x[k] = *reinterpret_cast<const float4*>(a.acc + at * D + d);
      }
    }
    float mx = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) mx = fmaxf(mx, ml[k].x);
    const float keep = m == -INFINITY ? 0.f : exp2_fast(m - mx);
    m = mx;
    l *= keep;
    v.x *= keep; v.y *= keep; v.z *= keep; v.w *= keep;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = ml[k].x == -INFINITY ? 0.f : exp2_fast(ml[k].x - mx);
      l = fmaf(f, ml[k].y, l);
      v.x = fmaf(f, x[k].x, v.x); v.y = fmaf(f, x[k].y, v.y);
      v.z = fmaf(f, x[k].z, v.z); v.w = fmaf(f, x[k].w, v.w);
    }
  }
  if constexpr (GROUPS > 1) {
    s_v[tid] = v;
    s_ml[tid] = make_float2(m, l);
    __syncthreads();
    if (group > 0) return;
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) mx = fmaxf(mx, s_ml[tid + 128 * k].x);
    l = 0.f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      const float2 ml = s_ml[tid + 128 * k];
      const float4 x = s_v[tid + 128 * k];
      const float f = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - mx);
      l = fmaf(f, ml.y, l);
      v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y);
      v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
    }
  }
  if (!on || c1 == -2) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;   // a row that sees no key, or a sequence without keys: zeros
  const int t = div_g(a, row), head = kvh * a.G + row - t * a.G;
  const int64_t at = b * a.so_b + t * a.so_t + static_cast<int64_t>(head) * a.so_h + d;
  store_out2<T>(a, at, v.x * inv, v.y * inv);
  store_out2<T>(a, at + 2, v.z * inv, v.w * inv);
}

// ------------------------------------------------------------------ host
// Row tiles of 8 in a unit, at most 4: as few units as possible, of equal size (40 rows: two of 24)
int row_tiles(int rows) {
  const int units = (rows + 31) / 32, per = (rows + units - 1) / units;
  return (per + 7) / 8;
}

struct Plan {
  int nt, ctas, whole, groups, fits;
  int64_t entries;
  size_t bytes;
};

Plan make_plan(const b2d_int4_kv* kv, int B, int T, int H, int pages_per_seq, int max_len, int sm) {
  Plan p{};
  const int64_t reach = static_cast<int64_t>(pages_per_seq) * kv->page_size;
  const int rows = T * (H / kv->KVH);
  p.nt = row_tiles(rows);
  const int tile = 8 * p.nt;
  const int64_t keys = max_len > 0 && max_len < reach ? max_len : reach;
  const int64_t units = static_cast<int64_t>(B) * kv->KVH * ((rows + tile - 1) / tile);
  p.fits = units * ((reach + kStage - 1) / kStage + Line<1>::LEAD) < (int64_t(1) << 31);
  p.whole = keys <= kWholeKeys || (keys <= kWholeKeysMany && units >= 2 * sm);
  int64_t ctas = p.whole ? units : units * ((keys + kStage - 1) / kStage + Line<1>::LEAD);
  const int per_sm = p.nt == 1 ? kBlocks<1> : p.nt == 2 ? kBlocks<2> : kBlocks<3>;
  if (ctas > static_cast<int64_t>(per_sm) * sm) ctas = per_sm * sm;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  p.ctas = static_cast<int>(ctas < 1 ? 1 : ctas);
  // a unit's parts, eight in flight a group of the combine's threads: 9 of them take 10.8 us a call in two groups (8 x 512..2048 keys)
  // against 12.0 in one; 74 of them (one sequence of 30000 keys, 8 KV heads) 18.7 in four against 20.6 in eight
  p.groups = p.ctas > 16 * units ? 4 : p.ctas > 4 * units ? 2 : 1;
  if (!p.whole) {
    p.entries = static_cast<int64_t>(p.ctas) * 2 * tile;
    p.bytes = static_cast<size_t>(p.entries) * (kv->D + 2) * 4;
  }
  return p;
}

template <typename T, int D, int RUNS, int NT>
int launch_attention(const Int4AttnArgs& a, int groups, bool pdl, cudaStream_t s) {
  auto kern = int4_attention_kernel<T, D, RUNS, NT>;
  constexpr int bytes = Smem<D, RUNS, NT>::BYTES;
  static bool configured[64] = {};   // per device; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) {
      set_cuda_error(e);
      return B2D_ERR_LAUNCH;
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  const int st = launch_kernel(kern, dim3(a.ctas), dim3(kThreads), bytes, s, pdl, a);
  if (st != B2D_OK || a.whole) return st;
  const dim3 grid(a.B * a.kv.KVH, (a.rows + 512 / D - 1) / (512 / D));
  if (groups == 4) return launch_kernel(int4_combine_kernel<T, D, NT, 4>, grid, dim3(512), 0, s, true, a);
  if (groups == 2) return launch_kernel(int4_combine_kernel<T, D, NT, 2>, grid, dim3(256), 0, s, true, a);
  return launch_kernel(int4_combine_kernel<T, D, NT, 1>, grid, dim3(128), 0, s, true, a);
}

template <typename T, int D, int RUNS>
int run(const Int4AttnArgs& a, const Plan& p, bool pdl, cudaStream_t s) {
  switch (p.nt) {
    case 1: return launch_attention<T, D, RUNS, 1>(a, p.groups, pdl, s);
    case 2: return launch_attention<T, D, RUNS, 2>(a, p.groups, pdl, s);
    case 3: return launch_attention<T, D, RUNS, 3>(a, p.groups, pdl, s);
    default: return launch_attention<T, D, RUNS, 4>(a, p.groups, pdl, s);
  }
}
template <typename T>
int run(const Int4AttnArgs& a, const Plan& p, bool pdl, cudaStream_t s) {
  if (a.kv.D == 64) return a.kv.group == 64 ? run<T, 64, 1>(a, p, pdl, s) : run<T, 64, 2>(a, p, pdl, s);
  return a.kv.group == 64 ? run<T, 128, 2>(a, p, pdl, s) : run<T, 128, 4>(a, p, pdl, s);
}

int check_shapes(const b2d_int4_kv* kv, int B, int T, int H, int pages_per_seq, int max_len) {
  const int st = check_int4_kv(kv);
  if (st != B2D_OK) return st;
  if (B < 0 || T < 0 || H < 0 || pages_per_seq < 0 || max_len < 0) return B2D_ERR_ARG;
  if (H % kv->KVH != 0 || H / kv->KVH > kMaxG || T > kMaxT) return B2D_ERR_SHAPE;
  // positions fit 31 bits, and so do those up to 32 stages past the end
  if (static_cast<int64_t>(pages_per_seq) * kv->page_size > (int64_t(1) << 31) - 4096) return B2D_ERR_SHAPE;
  return B2D_OK;
}

}  // namespace
}  // namespace b2d

using namespace b2d;

extern "C" size_t b2d_int4_attention_workspace_bytes(const b2d_int4_kv* kv, int B, int T, int H, int pages_per_seq,
                                                     int max_len) {
  if (check_shapes(kv, B, T, H, pages_per_seq, max_len) != B2D_OK || B == 0 || T == 0 || H == 0) return 0;
  DeviceInfo di;
  if (device_info(&di) != B2D_OK) return 0;
  // the launches of a large batch: full ones and a rest
  const size_t full = B >= kMaxBatch ? make_plan(kv, kMaxBatch, T, H, pages_per_seq, max_len, di.sm_count).bytes : 0;
  const size_t rest = B % kMaxBatch ? make_plan(kv, B % kMaxBatch, T, H, pages_per_seq, max_len, di.sm_count).bytes : 0;
  return full > rest ? full : rest;
}

extern "C" int b2d_int4_attention(const b2d_int4_kv* kv, const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                                  const int32_t* page_table, int64_t ld_table, int pages_per_seq, const int32_t* seqlens,
                                  int max_len, int B, int T, int H, float scale, void* out, int64_t so_b, int64_t so_t,
                                  int64_t so_h, int out_dtype, void* workspace, size_t workspace_bytes, int flags,
                                  void* stream) {
  int st;
  if ((st = check_shapes(kv, B, T, H, pages_per_seq, max_len)) != B2D_OK) return st;
  if (out_dtype != kv->dtype && out_dtype != B2D_F32) return B2D_ERR_DTYPE;
  if (B == 0 || T == 0 || H == 0) return B2D_OK;
  if (ld_table < 0) return B2D_ERR_SHAPE;
  if (!q || !seqlens || !out || (!page_table && pages_per_seq > 0)) return B2D_ERR_ARG;
  if (!aligned(q, 16) || (sq_b | sq_t | sq_h) % 8 || !aligned(page_table, 4) || !aligned(seqlens, 4) ||
      !aligned(out, out_dtype == B2D_F32 ? 4 : 2) || !aligned(workspace, 16))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  if ((st = device_info(&di)) != B2D_OK) return st;
  const int size = out_dtype == B2D_F32 ? 4 : 2;
  // full launches of a large batch and its rest, which may need scratch where a full one runs its units whole: all is
  // checked before the first one, so that a refused call has written nothing (out may be q)
  Plan plans[2] = {};
  for (int i = 0; i < 2; ++i) {
    const int n = i == 0 ? (B < kMaxBatch ? B : kMaxBatch) : B % kMaxBatch;
    if (n == 0) continue;
    const Plan p = plans[i] = make_plan(kv, n, T, H, pages_per_seq, max_len, di.sm_count);
    if (!p.fits) return B2D_ERR_SHAPE;
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return B2D_ERR_WORKSPACE;
  }
  for (int b0 = 0; b0 < B; b0 += kMaxBatch) {
    const int n = B - b0 < kMaxBatch ? B - b0 : kMaxBatch;
    const Plan& p = plans[n == kMaxBatch || B < kMaxBatch ? 0 : 1];
    Int4AttnArgs a{};
    a.q = static_cast<const uint8_t*>(q) + b0 * sq_b * 2;
    a.sq_b = sq_b; a.sq_t = sq_t; a.sq_h = sq_h;
    a.table = page_table ? page_table + b0 * ld_table : nullptr;
    a.ld_table = ld_table; a.seqlens = seqlens + b0;
    a.out = static_cast<uint8_t*>(out) + b0 * so_b * size;
    a.so_b = so_b; a.so_t = so_t; a.so_h = so_h;
    a.kv = *kv; a.div = page_div(kv->page_size);
    a.pages_per_seq = pages_per_seq;
    a.B = n; a.T = T; a.H = H; a.G = H / kv->KVH; a.rows = T * a.G; a.inv_g = (65536 + a.G - 1) / a.G;
    a.scale_log2 = scale * kLog2e;
    a.ctas = p.ctas; a.whole = p.whole;
    a.out_f32 = out_dtype == B2D_F32;
    a.out_vec = aligned(a.out, 2 * size) && (so_b | so_t | so_h) % 2 == 0;
    a.acc = static_cast<float*>(workspace);
    a.ml = a.acc ? a.acc + p.entries * kv->D : nullptr;
    const bool pdl = (flags & B2D_LAUNCH_PDL) != 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    st = kv->dtype == B2D_F16 ? run<__half>(a, p, pdl, s) : run<__nv_bfloat16>(a, p, pdl, s);
    if (st != B2D_OK) return st;
  }
  return B2D_OK;
}
