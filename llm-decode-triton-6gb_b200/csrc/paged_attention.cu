// Attention of the newest tokens of every sequence over a paged KV cache, causal among themselves, with an
// optional prefix shared by the whole batch (sm_100a). The contiguous one-token counterpart is
// csrc/gqa_decode.cu (reference: profiling/kernels/decode_attention.py:18-91).
//
// o[b, t, h] = sum_{j < limit} softmax_j(scale q.k_j) v_j, limit = seqlens[b] - T + 1 + t. Key j lies in
// prefix_table's pages for j < prefix_len and in page_table[b]'s behind.
//
// Streaming kernel. A unit of work is (sequence, KV head, tile of up to 32 rows): rows are the T x G query vectors
// that read this KV head (row = t G + g), so K and V are read once for all of them. The units' stages (64 keys
// of 128, 128 keys of 64) form one line, of which every CTA (two per SM) takes an equal share: a ragged batch
// is balanced from its lengths on the device, and a CTA's ring never drains between two units.
//  * A producer warp copies Q rows, then K and V through a ring of five 16 KB slots: its lanes look the pages
//    up one stage ahead and issue one tensor copy per (page, 64 elements), 128-byte swizzled, so that the
//    ldmatrix reads hit 8 distinct bank groups; completion on mbarriers. Pages that tensor copies do not fit
//    (sizes that neither divide nor are divided by 64, ...) take 16-byte cp.async from the same warp.
//  * Each of four consumer warps takes a quarter of a stage's keys, transposed so that few rows waste little of
//    the products: S^T = K Q^T and O^T += V^T P^T by mma.sync m16n8k16 (fp32 accumulate) with 16 keys (16
//    elements) as M and 8 rows as N. Online softmax in the log2 domain; the warps meet in shared memory at a
//    unit's end. P is rounded to the cache's dtype for the second product, as its V operand is; the sum of the
//    weights is taken before that rounding, in fp32. The running maximum moves only when a score exceeds it
//    by 2^8 (weights up to 256 are as exact), so O is rarely rescaled. Value rows at or past the length are
//    set to zero before they are multiplied (a zero weight times a stale NaN would not be zero).
//  * A unit that one CTA finishes is written out; the parts of a unit that several CTAs share go to the
//    workspace as (O, m, l), and the combine kernel (a programmatic dependent) merges them in CTA order.
// Short calls give whole units to CTAs and need no combine.
//
// Shared prefix: all sequences' rows form one row axis, [0, B T G), over the prefix's pages -- up to 32 rows as
// further units of the streaming kernel, more on tcgen05 (csrc/paged_prefix.cu, a launch of its own); the
// sequences' units start behind the prefix, and the combine merges both. A sequence with a query that does not
// see the whole shared part is computed from position 0 by its own units.
//
// Measured on B200 (GPU time of a call, graph replays over rotated inputs; bytes: each key and value once;
// copy rate 6.52 TB/s): 8 sequences of 16001..32768 keys, 8 KV heads of 64, fp16: 66 us, 6.0 TB/s. 8 of
// 512..2048 keys, 32 / 8 heads of 128: 13.9 us, 3.0 TB/s. 16 x 5 drafts over up to 4099 keys: 38 us, 3.6 TB/s; the
// warps issue in 25 % of the slots and HMMA is 16 % busy at 9.4 warps per SM, so latency bounds it. One sequence
// of 300 keys: 7.5 us, latency. Earlier forms, first case and second: splits in thread-block clusters with cp.async by
// every thread 168 and 23.6 us (about 690 instructions per warp and stage, most of them addresses); tensor copies
// from a producer warp 67.5 and 15.2; equal shares of one line of stages with transposed products 66 and 14.5.
// Three CTAs per SM with three slots each (one row tile) took 14.9 us for the second case against 13.6, and 35.1
// against 37.1 for 64 sequences on a shared 4096 prefix: not kept.
#include <mutex>
#include <type_traits>

#include "paged_attention.cuh"
#include "pipeline.cuh"

namespace b2d {
namespace {

constexpr int kWarps = 4;                       // consumer warps
constexpr int kConsumers = kWarps * 32;
constexpr int kThreads = kConsumers + 32;       // and the producer warp
constexpr int kSlotBytes = 16 * 1024;           // K or V of a stage
constexpr int kSlots = 5;
constexpr int kMaxT = 16, kMaxG = 16;
constexpr int kMaxBatch = 256;                  // sequences of a launch (larger batches take several)
constexpr int kMaxCtas = 320;
constexpr float kLazy = 8.f;                    // log2 of the largest weight before the running maximum moves
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
__host__ __device__ constexpr int stage_keys() { return kSlotBytes / (D * 2); }
template <int D, int NT>
__host__ __device__ constexpr uint32_t smem_bytes() {
  return kSlots * kSlotBytes + 8 * NT * D * 2 /* Q */ + kWarps * 8 * (D + 4) * 4 /* merge */ + 1024;
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
// two neighbouring outputs; `out_vec`: every row starts on a boundary of their size
template <typename T>
__device__ __forceinline__ void store_out2(const PagedAttnArgs& a, int64_t off, float x, float y) {
  if (!a.out_vec) {
    store_out<T>(a, off, x);
    store_out<T>(a, off + 1, y);
  } else if (a.out_f32) {
    *reinterpret_cast<float2*>(static_cast<float*>(a.out) + off) = make_float2(x, y);
  } else {
    *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + off) = Dt<T>::pack2(x, y);
  }
}

// The keys that sequence b computes itself: [begin, len), cut to what the page table and the prefix reach.
struct Span {
  int len, begin;
  bool shares;      // takes the shared prefix's part in
};
__device__ __forceinline__ int length_of(const PagedAttnArgs& a, int b) {
  const int64_t reach = static_cast<int64_t>(a.pages_per_seq) * a.kv.page_size;
  return min(max(a.seqlens[b], 0), max(static_cast<int>(reach), a.prefix_len));
}
__device__ __forceinline__ Span span_of(const PagedAttnArgs& a, int len) {
  Span s;
  s.len = len;
  s.shares = a.shared > 0 && s.len - a.T + 1 >= a.shared;
  s.begin = s.shares ? a.shared : 0;
  return s;
}

// The line of all units' work: the prefix's units first (where the streaming kernel takes them), then the
// sequences' in order, KV head by KV head and row tile by row tile. A unit takes `lead` positions, what its start
// and end cost in stages, and one for each of its stages; one without keys takes none. CTA c takes the
// positions [share(c), share(c + 1)); the host has checked that they fit 31 bits. In whole mode a unit is one
// position.
template <int D, int NT>
struct Line {
  static constexpr int KEYS = stage_keys<D>(), ROWS = 8 * NT;
  // from time stamps in the kernel, which lengthen what they measure: a unit's start and end cost 1.3 us with one row
  // tile and 4 us with more, a stage 1 us (1.6 with three row tiles). Four row tiles have the value of three, without a
  // measurement of their own.
  static constexpr int LEAD = NT == 1 ? 2 : NT == 2 ? 4 : 3;
  int tiles, units, tiles_p, cost_p, base, ctas, quota, extra;
  __device__ __forceinline__ Line(const PagedAttnArgs& a) {
    tiles = (a.rows + ROWS - 1) / ROWS;
    units = a.kv.KVH * tiles;
    const bool streams = a.shared > 0 && a.nparts == 0;
    tiles_p = streams ? (a.B * a.rows + ROWS - 1) / ROWS : 0;
    cost_p = streams ? (a.shared + KEYS - 1) / KEYS + LEAD : 0;
    base = a.kv.KVH * tiles_p * cost_p;
  }
  static __device__ __forceinline__ int cost_of(const PagedAttnArgs& a, int len) {
    const Span s = span_of(a, len);
    return a.whole ? 1 : s.len > s.begin ? (s.len - s.begin + KEYS - 1) / KEYS + LEAD : 0;
  }
  __device__ __forceinline__ void close(const PagedAttnArgs& a, int cost) {   // of all sequences
    const int total = base + cost * units;
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

// The sequences' lengths into s_len and the exclusive running sums of their units' cost into s_sum[0 .. B] (all
// THREADS of the block take part).
template <int D, int NT, int THREADS>
__device__ __forceinline__ void scan_costs(const PagedAttnArgs& a, int* s_sum, int* s_len, int* s_warp) {
  constexpr int W = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int run = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + tid;
    const int len = b < a.B ? length_of(a, b) : 0;
    const int own = b < a.B ? Line<D, NT>::cost_of(a, len) : 0;
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

// A CTA's stretch of one unit: keys [t_begin, t_end). The producer finds it and hands it to the consumers.
struct Segment {
  int b, kvh, row0, nrows;       // b < 0: the prefix
  int t_begin, t_end, limit;     // query t sees the keys before limit + t (the prefix: before t_end)
  int kind;                      // 0: the final output, 1: a whole part, 2 / 3: the end (or middle) / the start of
                                 // a unit shared with other CTAs, < 0: none
  int next;                      // position behind it
};
// The segment at position pos of a share that ends at `end`; none where only a unit's lead lies in the share.
template <int D, int NT>
__device__ __forceinline__ Segment segment_at(const PagedAttnArgs& a, const Line<D, NT>& line, const int* s_sum,
                                              const int* s_len, int pos, int end) {
  constexpr int KEYS = stage_keys<D>(), ROWS = 8 * NT;
  Segment g;
  int u, cost, tile, start, first = 0, last;   // start: the unit's first position
  bool shares = true;
  if (pos < line.base) {
    cost = line.cost_p;
    u = pos / cost;
    start = u * cost;
    g.b = -1;
    g.kvh = u / line.tiles_p;
    tile = u - g.kvh * line.tiles_p;
    last = a.shared;
    g.limit = a.shared;
    g.nrows = min(a.B * a.rows - tile * ROWS, ROWS);
  } else {
    int lo = 0, hi = a.B - 1;   // the last sequence that starts at or before pos
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (line.base + s_sum[mid] * line.units <= pos) lo = mid;
      else hi = mid - 1;
    }
    g.b = lo;
    const Span s = span_of(a, s_len[lo]);
    first = s.begin;
    last = s.len;
    shares = s.shares;
    g.limit = s.len - a.T + 1;
    cost = s_sum[lo + 1] - s_sum[lo];
    start = line.base + s_sum[lo] * line.units;
    u = (pos - start) / cost;
    start += u * cost;
    g.kvh = line.tiles == 1 ? u : u / line.tiles;
    tile = u - g.kvh * line.tiles;
    g.nrows = min(a.rows - tile * ROWS, ROWS);
  }
  g.row0 = tile * ROWS;
  g.next = min(end, start + cost);
  if (a.whole) {
    g.t_begin = first;
    g.t_end = last;
    g.kind = 0;
  } else {
    const int stages = cost - Line<D, NT>::LEAD, s0 = max(pos - start - Line<D, NT>::LEAD, 0);
    const int s1 = g.next - start - Line<D, NT>::LEAD;
    g.t_begin = first + s0 * KEYS;
    g.t_end = min(last, first + s1 * KEYS);
    g.kind = s1 <= s0 ? -1 : s0 > 0 ? 2 : s1 < stages ? 3 : shares ? 1 : 0;
  }
  return g;
}

// r / G for a sequence's rows (r < 256, G <= 16: exact)
__device__ __forceinline__ int div_g(const PagedAttnArgs& a, int r) { return r * a.inv_g >> 16; }
// Row r of a unit -> its (b, t, head).
struct Row {
  int b, t, head;
};
__device__ __forceinline__ Row row_of(const PagedAttnArgs& a, int b, int kvh, int r) {
  const int rb = b < 0 ? r / a.rows : b, rr = b < 0 ? r - rb * a.rows : r, t = div_g(a, rr);
  return Row{rb, t, kvh * a.G + rr - t * a.G};
}
__device__ __forceinline__ int64_t all_rows(const PagedAttnArgs& a) { return static_cast<int64_t>(a.B) * a.T * a.H; }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, 2) paged_stream_kernel(const __grid_constant__ PoolMaps maps,
                                                                   const __grid_constant__ PagedAttnArgs a) {
  constexpr int KEYS = stage_keys<D>();
  constexpr int WK = KEYS / kWarps, MT = WK / 16;   // keys of a stage that a warp takes, in tiles of 16
  constexpr int ROWS = 8 * NT;
  constexpr int KSTEPS = D / 16, DT = D / 16, CH = D / 8, HALVES = D / 64;
  constexpr bool Q_REGS = NT * KSTEPS <= 16;        // Q stays in registers (else it is read per stage)
  constexpr uint32_t HALFB = KEYS * 128;   // a slot's 64-element column
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ float s_m[kWarps][ROWS], s_l[kWarps][ROWS];
  __shared__ __align__(8) uint64_t s_bar[2 * kSlots + 2];
  __shared__ int s_sum[kMaxBatch + 1], s_len[kMaxBatch], s_warp[kThreads / 32];
  __shared__ Segment s_seg;
  __shared__ int64_t s_at[ROWS];        // per row: offset in the output, or workspace entry

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* const smem = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  const uint32_t ring = smem_u32(smem), q_s = ring + kSlots * kSlotBytes;
  float* const s_o = reinterpret_cast<float*>(smem + kSlots * kSlotBytes + ROWS * D * 2);   // the key warps' merge buffer
  const uint32_t full = smem_u32(s_bar), empty = full + 8 * kSlots, q_full = empty + 8 * kSlots, q_empty = q_full + 8;
  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(full + 8 * i, a.box_rows ? 1 : 32);
      mbar_init(empty + 8 * i, kWarps);
    }
    mbar_init(q_full, 33);
    mbar_init(q_empty, kWarps);
    fence_mbar_init();
  }
  if (a.box_rows && tid == kConsumers) {
    prefetch_tensormap(&maps.k);
    prefetch_tensormap(&maps.v);
  }
  if (!a.after_prefix) pdl_wait();   // behind the prefix launch the inputs are complete
  pdl_launch_dependents();
  Line<D, NT> line(a);
  scan_costs<D, NT, kThreads>(a, s_sum, s_len, s_warp);   // (its barriers also publish the mbarriers)
  line.close(a, s_sum[a.B]);
  const int first = line.share(blockIdx.x), end = line.share(blockIdx.x + 1);

  if (warp == kWarps) {
    // ---- producer
    int it = 0, seg = 0, sent = 0;   // stages, segments and slots filled so far
    bool ok = true;
    // lane -> (K or V, 64-element column, page of the stage): 32 lanes are enough from boxes of 8 rows on
    const int bp = a.box_rows, boxes = bp ? KEYS / bp : 1, per = HALVES * boxes;
    const int kv = lane / per, rest = lane - kv * per, col = rest / boxes, pg = rest - col * boxes;
    // page of this lane's box in stage i of a segment; -1: nothing to copy
    auto lookup = [&](const Segment& g, int i) {
      const int tok = g.t_begin + i * KEYS + pg * bp;
      if (kv > 1 || tok >= g.t_end) return -1;
      return __ldg((g.b >= 0 && tok >= a.prefix_len ? a.table + g.b * a.ld_table : a.prefix_table) + a.div.page(tok));
    };
    // the next segment, found while this one's first copies are under way, and the pages of its first stage
    Segment ahead;
    int ahead_page = -1;
    auto find = [&](int pos) {
      ahead.kind = -1;
      while (pos < end) {
        ahead = segment_at(a, line, s_sum, s_len, pos, end);
        if (ahead.kind >= 0) break;
        pos = ahead.next;
      }
      if (bp && ahead.kind >= 0) ahead_page = lookup(ahead, 0);
    };
    find(first);
    int behind = first;   // position behind the last segment
    while (ahead.kind >= 0 && ok) {
      const Segment g = ahead;
      int next = ahead_page;
      behind = g.next;
      const int t_begin = g.t_begin, t_end = g.t_end;
      const int32_t* table = g.b < 0 ? a.prefix_table : a.table + g.b * a.ld_table;
      const int split_at = g.b < 0 ? 0 : a.prefix_len;   // positions before it lie in prefix_table's pages
      const int nst = (t_end - t_begin + KEYS - 1) / KEYS;
      // Q rows of the tile, behind the first stage's copies: [64-element column][row][128 bytes] swizzled; rows
      // past the end are zeros. Lane l owns the address of row l.
      auto send_q = [&]() {
        if (seg > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait(q_empty, (seg - 1) & 1));
        if (!ok) {
          ahead.kind = -1;
          return;
        }
        int64_t off = -1;
        if (lane < g.nrows) {
          const Row x = row_of(a, g.b, g.kvh, g.row0 + lane);
          off = x.b * a.sq_b + x.t * a.sq_t + static_cast<int64_t>(x.head) * a.sq_h;
        }
#pragma unroll
        for (int i = 0; i < ROWS / 4; ++i) {
          const int r = 4 * i + lane / 8, c = lane & 7;
          const int64_t o = __shfl_sync(0xffffffffu, off, r);
          const T* src = static_cast<const T*>(a.q) + (o < 0 ? 0 : o + c * 8);
#pragma unroll
          for (int col = 0; col < HALVES; ++col)
            cp_async16_zfill(q_s + col * (ROWS * 128) + r * 128 + ((c ^ (r & 7)) << 4), src + (o < 0 ? 0 : 64 * col), o >= 0);
        }
        if (lane == 0) {
          s_seg = g;
          mbar_arrive(q_full);
        }
        mbar_arrive_cp_async(q_full);
        find(g.next);
      };
      if (nst == 0) send_q();
      if (a.box_rows) {
        for (int i = 0; i < nst && ok; ++i, ++it) {
          const int page = next, tok = t_begin + i * KEYS + pg * bp;
          next = lookup(g, i + 1);
#pragma unroll
          for (int x = 0; x < 2; ++x) {   // K, then V
            const int u = 2 * it + x, slot = u % kSlots;
            if (u >= kSlots) ok = ok && __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, (u / kSlots - 1) & 1));
            if (!ok) break;
            const uint32_t dst = ring + slot * kSlotBytes + col * HALFB + pg * bp * 128;
            const bool live = kv == x && tok < t_end, copy = live && page >= 0 && page < a.kv.num_pages;
            if (live && !copy) {   // a page id outside the pool: zeros
              for (int j = 0; j < bp * 8; ++j)
                *reinterpret_cast<uint4*>(smem + (dst - ring) + 16 * j) = make_uint4(0, 0, 0, 0);
              fence_proxy_async();
            }
            const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, copy)) * bp * 128;
            __syncwarp();
            if (lane == 0) mbar_expect_tx(full + 8 * slot, bytes);
            __syncwarp();
            sent = u + 1;
            if (copy) tma_load_4d(dst, x ? &maps.v : &maps.k, 64 * col, a.div.slot(tok, a.div.page(tok)), g.kvh, page, full + 8 * slot);
          }
          if (i == 0) send_q();
        }
      } else {
        // lane l owns the addresses of key rows l, l + 32, ...; 8 lanes copy the 128 bytes of a row's column
        for (int i = 0; i < nst && ok; ++i, ++it) {
#pragma unroll 1
          for (int x = 0; x < 2; ++x) {
            const int u = 2 * it + x, slot = u % kSlots;
            if (u >= kSlots) ok = ok && __all_sync(0xffffffffu, mbar_wait(empty + 8 * slot, (u / kSlots - 1) & 1));
            if (!ok) break;
            const T* pool = static_cast<const T*>(x ? a.kv.v : a.kv.k);
            const int64_t sp = x ? a.kv.sv_p : a.kv.sk_p, sh = x ? a.kv.sv_h : a.kv.sk_h, ss = x ? a.kv.sv_s : a.kv.sk_s;
#pragma unroll 1
            for (int r0 = 0; r0 < KEYS; r0 += 32) {
              const int tok = t_begin + i * KEYS + r0 + lane;
              int64_t off = -1;
              if (tok < t_end) {
                const int pi = a.div.page(tok);
                const int page = __ldg((tok >= split_at ? table : a.prefix_table) + pi);
                if (page >= 0 && page < a.kv.num_pages) off = page * sp + g.kvh * sh + a.div.slot(tok, pi) * ss;
              }
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int rr = 4 * j + lane / 8, r = r0 + rr, c = lane & 7;
                const int64_t o = __shfl_sync(0xffffffffu, off, rr);
                const T* src = o < 0 ? pool : pool + o + c * 8;
                const uint32_t dst = ring + slot * kSlotBytes + r * 128 + ((c ^ (r & 7)) << 4);
#pragma unroll
                for (int col = 0; col < HALVES; ++col) cp_async16_zfill(dst + col * HALFB, src + (o < 0 ? 0 : 64 * col), o >= 0);
              }
            }
            mbar_arrive_cp_async(full + 8 * slot);
          }
          if (i == 0) send_q();
        }
      }
      ++seg;
    }
    if (ok && behind < end) {   // only a unit's lead is left: the consumers stop
      if (seg > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait(q_empty, (seg - 1) & 1));
      if (ok && lane == 0) {
        ahead.kind = -1;
        ahead.next = end;
        s_seg = ahead;
        mbar_arrive(q_full);
      }
      if (ok) mbar_arrive(q_full);
    }
    cp_async_wait<0>();
    // Nothing is under way into this block's memory when it ends (the consumers wait for every copy as well, unless one
    // of their waits ran out)
    bool landed = true;
    for (int u = max(sent - kSlots, 0); u < sent; ++u) landed = landed && mbar_wait(full + 8 * (u % kSlots), (u / kSlots) & 1);
  } else {
    // ---- consumers: keys are the products' M axis (16 of a warp's keys), rows their N axis (8 per tile)
    const int g8 = lane >> 2, tq = lane & 3, mi = lane >> 3, ri = lane & 7;
    const int lead = warp * WK;   // this warp's keys of a stage
    int it = 0, seg = 0;
    bool landed = true;
    for (int pos = first; pos < end; ++seg) {
      // (the last unit's readers are done with s_at, s_m, s_o behind this barrier)
      landed = named_all<1, kConsumers>(landed && mbar_wait(q_full, seg & 1));
      Segment g = s_seg;
      if (!landed) g = segment_at(a, line, s_sum, s_len, pos, end);   // a wait ran out: NaN for what is left
      pos = g.next;
      if (g.kind < 0) {
        if (landed) break;
        continue;
      }
      uint32_t qb[NT][KSTEPS][2];   // Q as the B operand: row 8 n + g8, elements 16 j + 2 tq ..
      auto load_q = [&](int n, int j) {   // two k-steps at a time
        const int r = 8 * n + ri, c = 2 * j + mi;
        ldsm_x4(q_s + (c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4), qb[n][j][0], qb[n][j][1],
                qb[n][j + 1][0], qb[n][j + 1][1]);
      };
      if constexpr (Q_REGS) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < KSTEPS; j += 2) load_q(n, j);
        __syncwarp();
        if (lane == 0) mbar_arrive(q_empty);
      }
      const int t_begin = g.t_begin, t_end = g.t_end, nst = (t_end - t_begin + KEYS - 1) / KEYS;
      if (tid < g.nrows) {
        const Row x = row_of(a, g.b, g.kvh, g.row0 + tid);
        const int64_t index = (static_cast<int64_t>(x.b) * a.T + x.t) * a.H + x.head;
        s_at[tid] = g.kind == 0   ? x.b * a.so_b + x.t * a.so_t + static_cast<int64_t>(x.head) * a.so_h
                    : g.kind == 1 ? (a.nparts + (g.b < 0 ? 1 : 0)) * all_rows(a) + index
                                  : a.slot0 + (static_cast<int64_t>(blockIdx.x) * 2 + (g.kind - 2)) * ROWS + tid;
      }
      // keys that this thread's rows 8 n + 2 tq + e see; below lim_min no row is masked
      const bool causal = g.b >= 0 && a.T > 1;
      const int lim_min = causal ? g.limit + div_g(a, g.row0) : g.limit;
      auto lim = [&](int n, int e) { return causal ? g.limit + div_g(a, g.row0 + min(8 * n + 2 * tq + e, g.nrows - 1)) : g.limit; };

      float o[DT][NT][4];   // element 16 m + g8 (+ 8), row 8 n + 2 tq (+ 1)
#pragma unroll
      for (int m = 0; m < DT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.f;
      float m_run[NT][2], l_run[NT][2];   // log2 domain; the sum over this thread's keys only
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        m_run[n][0] = m_run[n][1] = -INFINITY;
        l_run[n][0] = l_run[n][1] = 0.f;
      }

      for (int i = 0; i < nst; ++i, ++it) {
        const int ks = (2 * it) % kSlots, vs = (2 * it + 1) % kSlots;
        const uint32_t kbuf = ring + ks * kSlotBytes, vbuf = ring + vs * kSlotBytes;
        const int key0 = t_begin + i * KEYS + lead;   // this warp's first key
        const bool idle = key0 >= t_end;
        float s[MT][NT][4];   // key 16 mt + g8 (+ 8), row 8 n + 2 tq (+ 1)
        landed = landed && mbar_wait(full + 8 * ks, (2 * it / kSlots) & 1);
        if (!idle) {
          // with one row tile, even and odd k-steps in sums of their own: short chains of dependent products
          constexpr int SETS = NT == 1 ? 2 : 1;
          float sum[SETS][MT][NT][4];
#pragma unroll
          for (int x = 0; x < SETS; ++x)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int n = 0; n < NT; ++n) sum[x][mt][n][0] = sum[x][mt][n][1] = sum[x][mt][n][2] = sum[x][mt][n][3] = 0.f;
#pragma unroll
          for (int j = 0; j < KSTEPS; ++j) {
            if (!Q_REGS && j % 2 == 0) {
#pragma unroll
              for (int n = 0; n < NT; ++n) load_q(n, j);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              const int r = lead + 16 * mt + (mi & 1) * 8 + ri, c = 2 * j + (mi >> 1);
              uint32_t k0, k1, k2, k3;
              ldsm_x4(kbuf + (c >> 3) * HALFB + r * 128 + (((c & 7) ^ (r & 7)) << 4), k0, k1, k2, k3);
#pragma unroll
              for (int n = 0; n < NT; ++n) Mma<T>::run(sum[j % SETS][mt][n], k0, k1, k2, k3, qb[n][j][0], qb[n][j][1]);
            }
          }
          const bool masked = key0 + WK > min(lim_min, t_end);
          float tmax[NT][2];
          bool move = false;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            tmax[n][0] = tmax[n][1] = -INFINITY;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                float x = sum[0][mt][n][c];
                if constexpr (SETS == 2) x += sum[SETS - 1][mt][n][c];
                x *= a.scale_log2;
                if (masked) {
                  const int tok = key0 + 16 * mt + g8 + 8 * (c >> 1);
                  if (tok >= lim(n, c & 1) || tok >= t_end) x = -INFINITY;
                }
                s[mt][n][c] = x;
                tmax[n][c & 1] = fmaxf(tmax[n][c & 1], x);
              }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) tmax[n][e] = fmaxf(tmax[n][e], __shfl_xor_sync(0xffffffffu, tmax[n][e], x));
              move |= tmax[n][e] > m_run[n][e] + kLazy;
            }
          }
          // the running maximum moves only when a score passes it by kLazy (or is the first)
          if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const bool up = tmax[n][e] > m_run[n][e] + kLazy;
                const float alpha = up ? exp2_fast(m_run[n][e] - tmax[n][e]) : 1.f;   // m_run = -inf: 0
                if (up) m_run[n][e] = tmax[n][e];
                l_run[n][e] *= alpha;
#pragma unroll
                for (int m = 0; m < DT; ++m) {
                  o[m][n][e] *= alpha;
                  o[m][n][2 + e] *= alpha;
                }
              }
          }
        }
        __syncwarp();   // the warp is done with K (and, after the last stage, with Q)
        if (lane == 0) {
          mbar_arrive(empty + 8 * ks);
          if (!Q_REGS && i == nst - 1) mbar_arrive(q_empty);
        }
        landed = landed && mbar_wait(full + 8 * vs, ((2 * it + 1) / kSlots) & 1);
        // The keys at the end: value rows past it become zeros. And keys that some rows of the tile see and
        // others do not (the newest T - 1): a zero weight times an infinite or NaN value would reach the rows
        // that must not see it, so such value rows (rare) are taken out of the stage (`bad`) and added to the
        // rows that do see them one by one below. A warp alone reads its keys' rows.
        uint32_t bad = 0;
        const bool check = causal && min(key0 + WK, t_end) > lim_min;
        if (!idle && (check || key0 + WK > t_end)) {
          constexpr int PASS = 32 / CH;   // rows per pass of the warp
          const int c = lane % CH;
#pragma unroll
          for (int p = 0; p < WK / PASS; ++p) {
            const int y = p * PASS + lane / CH, r = lead + y, tok = key0 + y;
            uint4* const x = reinterpret_cast<uint4*>(smem + (vbuf - ring) + (c >> 3) * HALFB + r * 128 + (((c & 7) ^ (r & 7)) << 4));
            const uint32_t hit = __ballot_sync(0xffffffffu, check && tok >= lim_min && tok < t_end && nonfinite8<T>(*x));
#pragma unroll
            for (int z = 0; z < PASS; ++z)
              if (hit >> (z * CH) & (CH == 8 ? 0xFFu : 0xFFFFu)) bad |= 1u << (p * PASS + z);
            if (tok >= t_end || (bad >> y & 1)) *x = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();   // the slot's next tensor copy comes after these writes
          __syncwarp();
        }
        if (!idle) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t pb[NT][2];   // P as the B operand: row 8 n + g8, keys 2 tq .. (+ 8)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float mr = m_run[n][c & 1];
                s[mt][n][c] = exp2_fast(s[mt][n][c] - (mr == -INFINITY ? 0.f : mr));
                l_run[n][c & 1] += s[mt][n][c];
              }
              pb[n][0] = transpose8(Dt<T>::pack2(s[mt][n][0], s[mt][n][1]));
              pb[n][1] = transpose8(Dt<T>::pack2(s[mt][n][2], s[mt][n][3]));
            }
#pragma unroll
            for (int m = 0; m < DT; ++m) {
              const int r = lead + 16 * mt + (mi >> 1) * 8 + ri, c = 2 * m + (mi & 1);
              uint32_t v0, v1, v2, v3;
              ldsm_x4_t(vbuf + (c >> 3) * HALFB + r * 128 + (((c & 7) ^ (r & 7)) << 4), v0, v1, v2, v3);
#pragma unroll
              for (int n = 0; n < NT; ++n) Mma<T>::run(o[m][n], v0, v1, v2, v3, pb[n][0], pb[n][1]);
            }
            if (bad >> (16 * mt) & 0xFFFFu) {   // the value rows taken out above, for the rows that see them
              for (int y = 0; y < 16; ++y) {
                if (!(bad >> (16 * mt + y) & 1)) continue;
                const int tok = key0 + 16 * mt + y, pi = a.div.page(tok);
                const int page = (tok >= a.prefix_len ? a.table + g.b * a.ld_table : a.prefix_table)[pi];
                const T* v = static_cast<const T*>(a.kv.v) + page * a.kv.sv_p + g.kvh * a.kv.sv_h + a.div.slot(tok, pi) * a.kv.sv_s + g8;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const float w = __shfl_sync(0xffffffffu, y < 8 ? s[mt][n][e] : s[mt][n][2 + e], (y & 7) * 4 + tq);
                    if (tok >= lim(n, e)) continue;
#pragma unroll
                    for (int m = 0; m < DT; ++m) {
                      o[m][n][e] += w * Dt<T>::to_f32(v[16 * m]);
                      o[m][n][2 + e] += w * Dt<T>::to_f32(v[16 * m + 8]);
                    }
                  }
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * vs);
      }
      if (!Q_REGS && nst == 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(q_empty);
      }

      // ---- the unit's (or this CTA's part of it) result: the key warps meet in shared memory
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) l_run[n][e] += __shfl_xor_sync(0xffffffffu, l_run[n][e], x);
          if (g8 == 0) {
            s_m[warp][8 * n + 2 * tq + e] = m_run[n][e];
            s_l[warp][8 * n + 2 * tq + e] = landed ? l_run[n][e] : NAN;
          }
        }
      landed = named_all<1, kConsumers>(landed);
      if (tid < g.nrows) {   // (m, l) of a row, and the warps' factors in the place of their maxima
        float mx = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_m[w][tid]);
        float f[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          f[w] = s_m[w][tid] == -INFINITY ? 0.f : exp2_fast(s_m[w][tid] - mx);
          l += f[w] * s_l[w][tid];
        }
        if (!landed) l = NAN;
        // a row that sees no key: zeros (l is NaN, not 0, where a visible score is)
        const float inv = g.kind == 0 ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        if (g.kind != 0) *reinterpret_cast<float2*>(a.ml + s_at[tid] * 2) = make_float2(mx, l);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) s_m[w][tid] = f[w] * inv;
      }
      named_sync<1, kConsumers>();
      constexpr int PAD = D + 4;   // the rows 2 tq of the accumulators' columns fall into different banks
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (8 * n >= g.nrows) break;
        if (n > 0) named_sync<1, kConsumers>();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float factor = s_m[warp][8 * n + 2 * tq + e];
          float* dst = s_o + (warp * 8 + 2 * tq + e) * PAD + g8;
#pragma unroll
          for (int m = 0; m < DT; ++m) {
            dst[16 * m] = o[m][n][e] * factor;
            dst[16 * m + 8] = o[m][n][2 + e] * factor;
          }
        }
        named_sync<1, kConsumers>();
        const int live = min(g.nrows - 8 * n, 8);
        for (int idx = tid; idx < live * (D / 4); idx += kConsumers) {
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
    }
  }
  if (a.after_prefix) pdl_wait();   // this launch completes after the prefix's, so the combine sees both
}

// Merges rows' entries: a block of 128 threads for 512 / D rows of a (sequence, KV head), four elements a thread.
// A thread reads its row's (m, l) along with the sums and keeps a running maximum, so that one round trip to
// memory follows the streaming kernel's end; the rest is done while that kernel still runs (its shared memory
// is sized to leave room for these blocks). GROUPS > 1: so many groups of 128 threads share the entries of a
// unit that many CTAs have cut.
template <typename T, int D, int NT, int GROUPS>
__global__ void __launch_bounds__(128 * GROUPS, GROUPS == 1 ? 6 : 1) paged_combine_kernel(const __grid_constant__ PagedAttnArgs a) {
  constexpr int ROWS = 8 * NT, QUADS = D / 4, BLOCK_ROWS = 128 / QUADS;
  constexpr int MOST = kMaxParts + kMaxCtas + 2;   // a prefix unit's and an own unit's CTAs have at most one in common
  __shared__ int s_sum[kMaxBatch + 1], s_len[kMaxBatch], s_warp[4 * GROUPS];
  __shared__ float4 s_v[GROUPS > 1 ? 128 * GROUPS : 1];   // the groups' sums and (m, l)
  __shared__ float2 s_ml[GROUPS > 1 ? 128 * GROUPS : 1];
  __shared__ int64_t s_entry[MOST];   // entry of the first row, or -1 - (its block of R rows in the output's order)
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  // the lengths are inputs of the whole call, complete before its first kernel began
  Line<D, NT> line(a);
  scan_costs<D, NT, 128 * GROUPS>(a, s_sum, s_len, s_warp);
  line.close(a, s_sum[a.B]);
  const int64_t R = all_rows(a);
  const int b = blockIdx.x / a.kv.KVH, kvh = blockIdx.x - b * a.kv.KVH;
  const Span sp = span_of(a, s_len[b]);
  const int cost = s_sum[b + 1] - s_sum[b];
  auto put = [&](int b, int t, int head, int d, const float4& v, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;   // a row that sees no key: zeros
    const int64_t at = b * a.so_b + t * a.so_t + static_cast<int64_t>(head) * a.so_h + d;
    store_out2<T>(a, at, v.x * inv, v.y * inv);
    store_out2<T>(a, at + 2, v.z * inv, v.w * inv);
  };
  bool waited = false;
  const int stop = min(a.rows, (static_cast<int>(blockIdx.y) + 1) * BLOCK_ROWS);
  for (int row0 = blockIdx.y * BLOCK_ROWS, n; row0 < stop; row0 += n) {
    // n rows of one unit (and of one unit of the prefix)
    const int pr = b * a.rows + row0;
    n = stop - row0;
    if (sp.shares && line.tiles_p > 0) n = min(n, ROWS - pr % ROWS);
    int ne = 0;
    bool written = false;   // by the streaming kernel
    // a unit's entries: one whole part, or a slot of every CTA that shares it
    auto unit = [&](int start, int cost, int r, int block, bool direct) {
      if (cost == 0) return;
      const int p0 = start + Line<D, NT>::LEAD, c0 = line.owner(p0), c1 = line.owner(start + cost - 1);
      if (c0 == c1) {
        if (direct) written = true;
        else if (tid == 0) s_entry[ne] = -1 - block;
        ne += !direct;
      } else {
        for (int c = c0 + tid; c <= c1; c += 128 * GROUPS)
          s_entry[ne + c - c0] = a.slot0 + (static_cast<int64_t>(c) * 2 + (line.share(c) <= p0 ? 1 : 0)) * ROWS + r;
        ne += c1 - c0 + 1;
      }
    };
    if (sp.shares) {
      if (a.nparts > 0) {
        if (tid < a.nparts) s_entry[tid] = -1 - tid;
        ne = a.nparts;
      } else {
        unit((kvh * line.tiles_p + pr / ROWS) * line.cost_p, line.cost_p, pr % ROWS, a.nparts + 1, false);
      }
    }
    unit(line.base + s_sum[b] * line.units + (kvh * line.tiles + row0 / ROWS) * cost, cost, row0 % ROWS, a.nparts,
         !sp.shares);
    if (!waited) pdl_wait();
    waited = true;
    if (written) continue;
    __syncthreads();
    const int group = tid / 128, r = tid % 128 / QUADS, d = (tid % 128 - r * QUADS) * 4;
    if (r < n) {
      const int t = div_g(a, row0 + r), head = kvh * a.G + row0 + r - t * a.G;
      const int64_t index = (static_cast<int64_t>(b) * a.T + t) * a.H + head;
      float m = -INFINITY, l = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int e = 8 * group; e < ne; e += 8 * GROUPS) {   // eight entries in flight
        float4 x[8];
        float2 ml[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          ml[k] = make_float2(-INFINITY, 0.f);
          x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (e + k < ne) {
            const int64_t s = s_entry[e + k], at = s >= 0 ? s + r : (-1 - s) * R + index;
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
      }
      if constexpr (GROUPS == 1) put(b, t, head, d, v, l);
    }
    if constexpr (GROUPS > 1) {
      __syncthreads();
      if (group == 0 && r < n) {
        const int t = div_g(a, row0 + r), head = kvh * a.G + row0 + r - t * a.G;
        float mx = -INFINITY, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) mx = fmaxf(mx, s_ml[tid + 128 * k].x);
#pragma unroll
        for (int k = 0; k < GROUPS; ++k) {
          const float2 ml = s_ml[tid + 128 * k];
          const float4 x = s_v[tid + 128 * k];
          const float f = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - mx);
          l = fmaf(f, ml.y, l);
          v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y);
          v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w);
        }
        put(b, t, head, d, v, l);
      }
    }
    __syncthreads();   // the next rows reuse the table
  }
  if (!waited) pdl_wait();
}

// ------------------------------------------------------------------ host
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
// and ends inside its page, and the prefix ends between two copies. 0: the pages do not allow it, and the whole call
// takes cp.async and keeps its prefix on the streaming kernel (64 sequences on 4096 shared keys, pages of 16, bf16: 37 us;
// on 4100: 137).
int box_rows(const b2d_paged_kv& kv, int prefix_len) {
  const int ps = kv.page_size;
  if (kv.num_pages < 1 || ps < 8 || (64 % ps != 0 && ps % 64 != 0)) return 0;
  const int rows = ps < 64 ? ps : 64;
  return prefix_len % rows == 0 ? rows : 0;
}

// Row tiles of 8 in a unit, at most 4: as few units as possible, of equal size (40 rows: two of 24)
int row_tiles(int64_t rows) {
  const int64_t units = (rows + 31) / 32, per = (rows + units - 1) / units;
  return static_cast<int>((per + 7) / 8);
}

// How a call is cut.
struct Plan {
  int shared, tc5, splits, nparts, nt, ctas, whole, combine, many, fits;
  int64_t slot0, entries;
  size_t bytes;
};

Plan make_plan(const b2d_paged_kv* kv, int B, int T, int H, int pages_per_seq, int prefix_len, int max_len, int sm) {
  Plan p{};
  const int64_t reach = static_cast<int64_t>(pages_per_seq) * kv->page_size;
  const int64_t rows = static_cast<int64_t>(T) * (H / kv->KVH), all = B * rows;
  p.shared = B > 1 ? prefix_len / 64 * 64 : 0;   // one sequence has nothing to share; the rest of 64 is read per sequence
  p.tc5 = p.shared >= 128 && all > 32 && box_rows(*kv, prefix_len) > 0;
  if (p.tc5) {
    // one CTA per SM, at least two tiles of 128 keys each
    const int64_t groups = kv->KVH * ((all + 255) / 256), tiles = (p.shared + 127) / 128;
    const int per = all > 128 ? 1 : 2;   // partials of a CTA
    int64_t n = sm / groups;
    if (n > tiles / 2) n = tiles / 2;
    if (n > kMaxParts / per) n = kMaxParts / per;
    p.splits = static_cast<int>(n < 1 ? 1 : n);
    p.nparts = p.splits * per;
  }
  const bool streams_prefix = p.shared > 0 && !p.tc5;
  p.nt = row_tiles(streams_prefix ? all : rows);
  const int tile = 8 * p.nt, keys_per_stage = kSlotBytes / (kv->D * 2);
  int64_t keys = max_len > 0 && max_len < reach ? max_len : reach;
  if (keys < prefix_len) keys = prefix_len;
  // the most stages that there can be
  const int64_t units = B * static_cast<int64_t>(kv->KVH) * ((rows + tile - 1) / tile);
  const int64_t units_p = streams_prefix ? kv->KVH * ((all + tile - 1) / tile) : 0;
  const int64_t most = units * ((keys - p.shared + keys_per_stage - 1) / keys_per_stage) +
                       units_p * ((p.shared + keys_per_stage - 1) / keys_per_stage);
  const int64_t longest = reach > prefix_len ? reach : prefix_len;
  p.fits = (units + units_p) * ((longest + keys_per_stage - 1) / keys_per_stage + 4) < (int64_t(1) << 31);
  p.whole = keys <= keys_per_stage && p.shared == 0;
  int64_t ctas = p.whole ? units : most + 4 * (units + units_p);
  if (ctas > 2 * sm) ctas = 2 * sm;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  p.ctas = static_cast<int>(ctas < 1 ? 1 : ctas);
  p.combine = !p.whole;
  // a unit's parts: with fewer units than CTAs they are many (75 of them: 7 us in one group of threads)
  p.many = p.ctas > 16 * (units_p > 0 ? units_p : units);
  if (p.combine) {
    const int64_t R = static_cast<int64_t>(B) * T * H;
    p.slot0 = (p.nparts + (p.shared > 0 ? 2 : 0)) * R;
    p.entries = p.slot0 + static_cast<int64_t>(p.ctas) * 2 * tile;
    p.bytes = static_cast<size_t>(p.entries) * (kv->D + 2) * 4;
  }
  return p;
}

template <typename T, int D, int NT>
int launch_stream(const PoolMaps& maps, const PagedAttnArgs& a, bool combine, bool many, bool pdl, cudaStream_t s) {
  auto kern = paged_stream_kernel<T, D, NT>;
  constexpr uint32_t bytes = smem_bytes<D, NT>();
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
  int st = launch_kernel(kern, dim3(a.ctas), dim3(kThreads), bytes, s, pdl || a.after_prefix, maps, a);
  if (st != B2D_OK || !combine) return st;
  const dim3 grid(a.B * a.kv.KVH, (a.rows + 512 / D - 1) / (512 / D));
  if (many) return launch_kernel(paged_combine_kernel<T, D, NT, 4>, grid, dim3(512), 0, s, true, a);
  return launch_kernel(paged_combine_kernel<T, D, NT, 1>, grid, dim3(128), 0, s, true, a);
}

template <typename T, int D>
int run(PagedAttnArgs& a, const Plan& p, bool pdl, cudaStream_t s) {
  PoolMaps maps;
  if (a.box_rows && (!encode_pool(&maps.k, a.kv, a.kv.k, a.kv.sk_p, a.kv.sk_h, a.kv.sk_s, a.box_rows) ||
                     !encode_pool(&maps.v, a.kv, a.kv.v, a.kv.sv_p, a.kv.sv_h, a.kv.sv_s, a.box_rows)))
    a.box_rows = 0;
  if (p.tc5 && a.box_rows) {
    const int st = launch_prefix_tc5(maps, a, pdl, s);
    if (st != B2D_OK) return st;
    a.after_prefix = 1;
  } else if (p.tc5) {   // tensor maps refused: every sequence reads the prefix itself
    a.shared = 0;
  }
  switch (p.nt) {
    case 1: return launch_stream<T, D, 1>(maps, a, p.combine, p.many, pdl, s);
    case 2: return launch_stream<T, D, 2>(maps, a, p.combine, p.many, pdl, s);
    case 3: return launch_stream<T, D, 3>(maps, a, p.combine, p.many, pdl, s);
    default: return launch_stream<T, D, 4>(maps, a, p.combine, p.many, pdl, s);
  }
}

int check_shapes(const b2d_paged_kv* kv, int B, int T, int H, int pages_per_seq, int prefix_len, int max_len) {
  const int st = check_paged_kv(kv);
  if (st != B2D_OK) return st;
  if (B < 0 || T < 0 || H < 0 || pages_per_seq < 0 || prefix_len < 0 || max_len < 0) return B2D_ERR_ARG;
  if ((kv->D != 64 && kv->D != 128) || H % kv->KVH != 0 || H / kv->KVH > kMaxG || T > kMaxT) return B2D_ERR_SHAPE;
  // positions and their sums with a stage's keys fit 31 bits
  constexpr int64_t most = (int64_t(1) << 31) - 1024;
  if (static_cast<int64_t>(pages_per_seq) * kv->page_size > most || prefix_len > most || kv->KVH > 65535) return B2D_ERR_SHAPE;
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
  // the launches of a large batch: full ones and a rest
  const size_t full = B >= kMaxBatch ? make_plan(kv, kMaxBatch, T, H, pages_per_seq, prefix_len, max_len, di.sm_count).bytes : 0;
  const size_t rest = B % kMaxBatch ? make_plan(kv, B % kMaxBatch, T, H, pages_per_seq, prefix_len, max_len, di.sm_count).bytes : 0;
  return full > rest ? full : rest;
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
      !aligned(prefix_table, 4) || !aligned(out, out_dtype == B2D_F32 ? 4 : 2) || !aligned(workspace, 16))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  if ((st = device_info(&di)) != B2D_OK) return st;
  const int size = out_dtype == B2D_F32 ? 4 : 2;
  for (int b0 = 0; b0 < B; b0 += kMaxBatch) {
    const int n = B - b0 < kMaxBatch ? B - b0 : kMaxBatch;
    const Plan p = make_plan(kv, n, T, H, pages_per_seq, prefix_len, max_len, di.sm_count);
    if (!p.fits) return B2D_ERR_SHAPE;
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes)) return B2D_ERR_WORKSPACE;
    PagedAttnArgs a{};
    a.q = static_cast<const uint8_t*>(q) + b0 * sq_b * 2;
    a.sq_b = sq_b; a.sq_t = sq_t; a.sq_h = sq_h;
    a.table = page_table ? page_table + b0 * ld_table : nullptr;
    a.ld_table = ld_table; a.seqlens = seqlens + b0; a.prefix_table = prefix_table;
    a.out = static_cast<uint8_t*>(out) + b0 * so_b * size;
    a.so_b = so_b; a.so_t = so_t; a.so_h = so_h;
    a.kv = *kv; a.div = page_div(kv->page_size);
    a.pages_per_seq = pages_per_seq; a.prefix_len = prefix_len;
    a.B = n; a.T = T; a.H = H; a.G = H / kv->KVH; a.rows = T * a.G; a.inv_g = (65536 + a.G - 1) / a.G;
    a.scale_log2 = scale * kLog2e;
    a.shared = p.shared; a.nparts = p.nparts; a.splits = p.splits; a.ctas = p.ctas; a.whole = p.whole; a.slot0 = p.slot0;
    a.out_f32 = out_dtype == B2D_F32;
    a.out_vec = aligned(a.out, 2 * size) && (so_b | so_t | so_h) % 2 == 0;
    a.box_rows = box_rows(*kv, prefix_len);
    a.acc = static_cast<float*>(workspace);
    a.ml = a.acc ? a.acc + p.entries * kv->D : nullptr;
    const bool pdl = (flags & B2D_LAUNCH_PDL) != 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kv->dtype == B2D_F16) st = kv->D == 64 ? run<__half, 64>(a, p, pdl, s) : run<__half, 128>(a, p, pdl, s);
    else st = kv->D == 64 ? run<__nv_bfloat16, 64>(a, p, pdl, s) : run<__nv_bfloat16, 128>(a, p, pdl, s);
    if (st != B2D_OK) return st;
  }
  return B2D_OK;
}
