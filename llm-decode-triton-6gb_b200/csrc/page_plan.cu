// Page tables, positions and slots of a step's new tokens from the requests' lengths (b2d_page_plan, sm_100a).
//
// Two running sums over the sequences decide: pages and tokens asked for say who is refused, pages taken, pages given back
// and tokens of the others say where each one's lie. Every block of one cluster forms them for itself (a block scan in 32 bits
// that saturate; the state is read by all and written behind a cluster barrier) and keeps what the rest needs of a sequence
// in shared memory. Tokens and moved pages are then shared out by their number: a thread finds the sequence of its first one
// by bisection. A token's page comes from the ring itself where the step took it, so nothing waits for the table's new entries.
// Bound by latency: dependent rounds of loads and the scans between them. Measured on B200, a step that takes pages and one that
// gives them back by turns: 3.9 us for 8 requests of one token, 4.8 for 8 x 256 tokens, 9.8 for 1024 x 64 (one block alone: 61).
#include "common.cuh"
#include "paged.cuh"

namespace b2d {
namespace {

constexpr int kMaxSeqs = 8192;
constexpr int kClusterSize = 16;   // 1024 x 64 tokens: 9.8 us, with 8 blocks 12.9

struct PlanArgs {
  int32_t* table; int64_t ld_table;
  int32_t* held;
  int32_t* free_pages;
  int32_t* ring;
  const int32_t* cached;
  const int32_t* fresh;
  int64_t* positions;
  int32_t* seq_ids;
  int64_t* slots;
  int32_t* seqlens;
  int32_t* starts;
  int32_t* granted;
  PageDiv div;
  int pages_per_seq, num_pages, B, max_tokens, wide;   // wide: the tokens' rows take 16-byte stores
};

struct Seq {
  int cached, held;
  int64_t fresh, target;
  bool fits;
};
__device__ __forceinline__ Seq load_seq(const PlanArgs& a, int b) {
  Seq s;
  s.cached = max(a.cached[b], 0);
  s.fresh = max(a.fresh[b], 0);
  s.held = min(max(a.held[b], 0), a.pages_per_seq);
  s.target = (s.cached + s.fresh + a.div.size - 1) / a.div.size;
  s.fits = s.target <= a.pages_per_seq;
  return s;
}

__device__ __forceinline__ uint32_t sat_add(uint32_t x, uint32_t y) { return min(x + y, 0x7FFFFFFFu); }   // of such sums

// Exclusive running sums over the block's threads of K values each, on top of `run`, which moves on by their totals.
template <int K, int WARPS>
__device__ __forceinline__ void block_scan(uint32_t (&v)[K], uint32_t (&run)[K], uint32_t (*s_warp)[WARPS]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t before[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, v[k], o);
      if (lane >= o) v[k] = sat_add(v[k], up);
    }
    if (lane == 31) s_warp[k][warp] = v[k];
    const uint32_t up = __shfl_up_sync(0xffffffffu, v[k], 1);
    before[k] = lane > 0 ? up : 0;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    uint32_t w = lane < WARPS ? s_warp[k][lane] : 0;
#pragma unroll
    for (int o = 1; o < WARPS; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w = sat_add(w, up);
    }
    const uint32_t upto = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0), total = __shfl_sync(0xffffffffu, w, WARPS - 1);
    v[k] = sat_add(run[k], sat_add(warp > 0 ? upto : 0, before[k]));
    run[k] = sat_add(run[k], total);
  }
  __syncthreads();
}

// The last of n sequences whose sum lies at or before x
__device__ __forceinline__ int sequence_at(const int32_t* sums, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sums[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int CLUSTER, int THREADS>
__global__ void __launch_bounds__(THREADS) page_plan_kernel(const __grid_constant__ PlanArgs a) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ int32_t s_mem[];
  int32_t* const s_start = s_mem;              // [B + 1] tokens before the sequence
  int32_t* const s_take = s_start + a.B + 1;   // [B + 1] pages taken before it
  int32_t* const s_give = s_take + a.B + 1;    // [B + 1] pages given back before it
  int32_t* const s_held = s_give + a.B + 1;    // [B] pages held before the step; of a refused one -1
  int32_t* const s_cached = s_held + a.B;      // [B]
  __shared__ uint32_t s_warp[3][WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, rank = CLUSTER > 1 ? cluster_rank() : 0;
  const int P = a.num_pages;
  const int first0 = a.ring[0], count = min(max(a.ring[1], 0), P);

  uint32_t asked[2] = {0, 0}, run[3] = {0, 0, 0};
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + tid;
    const bool on = b < a.B;
    Seq s{};
    if (on) s = load_seq(a, b);
    const uint32_t need = on && s.fits && s.target > s.held ? static_cast<uint32_t>(s.target - s.held) : 0;
    const uint32_t tokens = on && s.fits ? static_cast<uint32_t>(s.fresh) : 0;
    uint32_t want[2] = {need, tokens};
    block_scan<2, WARPS>(want, asked, s_warp);
    const bool ok = on && s.fits && (need == 0 || sat_add(want[0], need) <= static_cast<uint32_t>(count)) &&
                    (tokens == 0 || sat_add(want[1], tokens) <= static_cast<uint32_t>(a.max_tokens));
    uint32_t got[3] = {ok ? need : 0, ok && s.held > s.target ? static_cast<uint32_t>(s.held - s.target) : 0, ok ? tokens : 0};
    block_scan<3, WARPS>(got, run, s_warp);
    if (on) {
      s_start[b] = static_cast<int>(got[2]);
      s_take[b] = static_cast<int>(got[0]);
      s_give[b] = static_cast<int>(got[1]);
      s_held[b] = ok ? s.held : -1;
      s_cached[b] = s.cached;
      if (rank == 0) {
        a.starts[b] = static_cast<int>(got[2]);
        a.granted[b] = ok ? static_cast<int>(tokens) : -1;
        a.seqlens[b] = s.cached + (ok ? static_cast<int>(tokens) : 0);
      }
    }
  }
  const int total = static_cast<int>(run[2]), taken = static_cast<int>(run[0]), given = static_cast<int>(run[1]);
  if (tid == 0) {
    s_start[a.B] = total;
    s_take[a.B] = taken;
    s_give[a.B] = given;
    if (rank == 0) a.starts[a.B] = total;
  }
  __syncthreads();

  int first = P > 0 ? first0 % P : 0;
  if (first < 0) first += P;
  auto ring_at = [&](int i) {   // the ring's i-th page from its first, 0 <= i <= P
    const int64_t at = static_cast<int64_t>(first) + i;
    return static_cast<int>(at < P ? at : at - P);
  };
  // tokens, four a thread
  constexpr int64_t kAll = static_cast<int64_t>(CLUSTER) * THREADS;
  const int64_t self = static_cast<int64_t>(rank) * THREADS + tid;
  for (int64_t n0 = self * 4; n0 < a.max_tokens; n0 += kAll * 4) {
    int64_t pos[4], slot[4];
    int id[4];
    int b = n0 < total ? sequence_at(s_start, a.B, static_cast<int>(n0)) : 0, end = n0 < total ? s_start[b + 1] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = n0 + i;
      pos[i] = slot[i] = -1;
      id[i] = -1;
      if (n < total) {
        while (n >= end) end = s_start[++b + 1];
        const int at = s_cached[b] + (static_cast<int>(n) - s_start[b]), pi = a.div.page(at), held = s_held[b];
        const int page = pi < held ? a.table[b * a.ld_table + pi] : a.free_pages[ring_at(s_take[b] + (pi - held))];
        pos[i] = at;
        id[i] = b;
        if (page >= 0 && page < P) slot[i] = static_cast<int64_t>(page) * a.div.size + a.div.slot(at, pi);
      }
    }
    if (a.wide && n0 + 4 <= a.max_tokens) {
      reinterpret_cast<longlong2*>(a.positions + n0)[0] = make_longlong2(pos[0], pos[1]);
      reinterpret_cast<longlong2*>(a.positions + n0)[1] = make_longlong2(pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.seq_ids + n0) = make_int4(id[0], id[1], id[2], id[3]);
      reinterpret_cast<longlong2*>(a.slots + n0)[0] = make_longlong2(slot[0], slot[1]);
      reinterpret_cast<longlong2*>(a.slots + n0)[1] = make_longlong2(slot[2], slot[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (n0 + i >= a.max_tokens) break;
        a.positions[n0 + i] = pos[i];
        a.seq_ids[n0 + i] = id[i];
        a.slots[n0 + i] = slot[i];
      }
    }
  }
  // pages, one a thread
  for (int64_t i = self; i < taken; i += kAll) {
    const int b = sequence_at(s_take, a.B, static_cast<int>(i));
    a.table[b * a.ld_table + s_held[b] + (static_cast<int>(i) - s_take[b])] = a.free_pages[ring_at(static_cast<int>(i))];
  }
  for (int64_t i = self; i < given; i += kAll) {   // a sequence's last ones: [target, held)
    const int b = sequence_at(s_give, a.B, static_cast<int>(i));
    int32_t* const entry = a.table + b * a.ld_table + s_held[b] - (s_give[b + 1] - static_cast<int>(i));
    const int64_t place = count + i;
    if (place < P) a.free_pages[ring_at(static_cast<int>(place))] = *entry;   // always, unless the state counts a page twice
    *entry = -1;
  }
  // nobody reads the old state any more
  if constexpr (CLUSTER > 1) cluster_sync();
  else __syncthreads();
  for (int64_t b = self; b < a.B; b += kAll)
    if (s_held[b] >= 0) {
      const int64_t want = static_cast<int64_t>(s_cached[b]) + max(a.fresh[b], 0);
      a.held[b] = static_cast<int>((want + a.div.size - 1) / a.div.size);
    }
  if (rank == 0 && tid == 0) {
    a.ring[0] = P > 0 ? (taken < P ? ring_at(taken) : first) : 0;
    a.ring[1] = static_cast<int>(min(static_cast<int64_t>(count) - taken + given, static_cast<int64_t>(P)));
  }
}

template <int CLUSTER, int THREADS>
int launch_plan(const PlanArgs& a, bool pdl, cudaStream_t s) {
  auto kern = page_plan_kernel<CLUSTER, THREADS>;
  static bool configured[64] = {};   // per device; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    constexpr int most = (5 * kMaxSeqs + 3) * 4;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (CLUSTER > 8 && e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) {
      set_cuda_error(e);
      return B2D_ERR_LAUNCH;
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CLUSTER);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = (5 * static_cast<size_t>(a.B) + 3) * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CLUSTER;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return B2D_ERR_LAUNCH;
  }
  return launch_status();
}

}  // namespace
}  // namespace b2d

using namespace b2d;

extern "C" int b2d_page_plan(int32_t* page_table, int64_t ld_table, int pages_per_seq, int32_t* held, int32_t* free_pages,
                             int num_pages, int32_t* ring, const int32_t* cached, const int32_t* new_tokens, int B,
                             int page_size, int max_tokens, int64_t* positions, int32_t* seq_ids, int64_t* slots,
                             int32_t* seqlens, int32_t* starts, int32_t* granted, int flags, void* stream) {
  constexpr int64_t most = (int64_t(1) << 31) - 1024;
  if (B < 0 || pages_per_seq < 0 || num_pages < 0 || max_tokens < 0) return B2D_ERR_ARG;
  if (page_size < 1 || page_size > kMaxPageSize || B > kMaxSeqs || num_pages > most || max_tokens > most ||
      static_cast<int64_t>(pages_per_seq) * page_size > most || ld_table < 0)
    return B2D_ERR_SHAPE;
  if (!ring || !starts || (B > 0 && (!held || !cached || !new_tokens || !seqlens || !granted)) ||
      (B > 0 && pages_per_seq > 0 && !page_table) || (num_pages > 0 && !free_pages) ||
      (max_tokens > 0 && (!positions || !seq_ids || !slots)))
    return B2D_ERR_ARG;
  if (!aligned(page_table, 4) || !aligned(held, 4) || !aligned(free_pages, 4) || !aligned(ring, 4) || !aligned(cached, 4) ||
      !aligned(new_tokens, 4) || !aligned(positions, 8) || !aligned(seq_ids, 4) || !aligned(slots, 8) || !aligned(seqlens, 4) ||
      !aligned(starts, 4) || !aligned(granted, 4))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  int st;
  if ((st = device_info(&di)) != B2D_OK) return st;
  const PlanArgs a{page_table, ld_table, held, free_pages, ring, cached, new_tokens, positions, seq_ids, slots, seqlens, starts,
                   granted, page_div(page_size), pages_per_seq, num_pages, B, max_tokens,
                   aligned(positions, 16) && aligned(seq_ids, 16) && aligned(slots, 16)};
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // us a step, half of the steps taking pages and half giving them back; one block against a cluster, which starts and ends
  // later. The host knows the sequences and the most tokens, not how many pages will move. Up to 1024 tokens, four a thread, the block
  // takes 4.5 against 5.0 for 8 x 128 and 4.8 against 5.8 for 512 x 2; above, 5.5 against 4.8 for 8 x 256. Above 512 sequences
  // the cluster loses little without pages to move (1024 x 1 token 7.1 against 6.8) and wins much with them (1024 move four each 7.1
  // against 11.3). The rule is on the wrong side for 512 sequences that move four pages each with few tokens (block, 6.6 against 5.3)
  // and for 512 x 4 tokens (cluster, 6.2 against 5.5). The scans go over the sequences in rounds of a block, where more warps cost more in
  // each: 256 threads and 512 take 3.9 and 4.1 for 8 x 1, 5.6 and 4.9 for 512 x 1; in a cluster 4.8 and 5.9 for 8 x 256,
  // 12.4 and 9.8 for 1024 x 64.
  const bool few = B <= 256;
  if (max_tokens <= 1024 && B <= 512) return few ? launch_plan<1, 256>(a, pdl, s) : launch_plan<1, 512>(a, pdl, s);
  return few ? launch_plan<kClusterSize, 256>(a, pdl, s) : launch_plan<kClusterSize, 512>(a, pdl, s);
}
