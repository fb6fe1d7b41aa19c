// Page tables, positions and slots of a step's new tokens from the requests' lengths (b2d_page_plan, sm_100a).
//
// Two running sums over the sequences decide: pages and tokens asked for say who is refused, pages taken, pages given back
// and tokens of the others say where each one's lie. Every block of one cluster forms them for itself (a block
// scan, 1024 sequences a trip; the state is read by all and written behind a cluster barrier), keeps them in shared memory,
// and takes its share of the tokens (four neighbouring ones a thread, whose first finds its sequence by bisection) and of the
// sequences' pages (a warp each). A token's page comes from the ring itself where the step took it, so nothing waits for the
// table's new entries. Bound by latency: two dependent rounds of loads and the scans between them.
#include "common.cuh"
#include "paged.cuh"

namespace b2d {
namespace {

constexpr int kMaxSeqs = 8192;
constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kClusterSize = 8;

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
  int pages_per_seq, num_pages, B, max_tokens;
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

// Exclusive running sums over the block's threads of K values each, on top of `run`, which moves on by their totals.
template <int K, typename V>
__device__ __forceinline__ void block_scan(V (&v)[K], V (&run)[K], V (*s_warp)[kWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V own[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    own[k] = v[k];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V up = __shfl_up_sync(0xffffffffu, v[k], o);
      if (lane >= o) v[k] += up;
    }
    if (lane == 31) s_warp[k][warp] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    V w = s_warp[k][lane];   // kWarps = 32
    const V mine = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V up = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += up;
    }
    const V before = __shfl_sync(0xffffffffu, w - mine, warp), total = __shfl_sync(0xffffffffu, w, 31);
    v[k] += run[k] + before - own[k];
    run[k] += total;
  }
  __syncthreads();
}

template <int CLUSTER>
__global__ void __launch_bounds__(kThreads) page_plan_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int32_t s_mem[];
  int32_t* const s_start = s_mem;              // [B + 1] tokens before the sequence
  int32_t* const s_take = s_start + a.B + 1;   // [B] pages taken before it; -1: refused
  int32_t* const s_give = s_take + a.B;        // [B] pages given back before it
  __shared__ int64_t s_warp2[2][kWarps];
  __shared__ int64_t s_warp3[3][kWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, rank = CLUSTER > 1 ? cluster_rank() : 0;
  const int P = a.num_pages;
  const int count = min(max(a.ring[1], 0), P);
  int first = P > 0 ? a.ring[0] % P : 0;
  if (first < 0) first += P;

  int64_t asked[2] = {0, 0};
  int64_t run[3] = {0, 0, 0};
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + tid;
    const bool on = b < a.B;
    Seq s{};
    if (on) s = load_seq(a, b);
    int64_t want[2] = {on && s.fits && s.target > s.held ? s.target - s.held : 0, on && s.fits ? s.fresh : 0};
    const int64_t need = want[0], tokens = want[1];
    block_scan<2, int64_t>(want, asked, s_warp2);
    const bool ok = on && s.fits && (need == 0 || want[0] + need <= count) && (tokens == 0 || want[1] + tokens <= a.max_tokens);
    int64_t got[3] = {ok ? need : 0, ok && s.held > s.target ? s.held - s.target : 0, ok ? tokens : 0};
    block_scan<3, int64_t>(got, run, s_warp3);
    if (on) {
      s_start[b] = static_cast<int>(got[2]);
      s_take[b] = ok ? static_cast<int>(got[0]) : -1;
      s_give[b] = static_cast<int>(min(got[1], static_cast<int64_t>(P)));   // past P: a state that counts pages twice
      if (rank == 0) {
        a.starts[b] = static_cast<int>(got[2]);
        a.granted[b] = ok ? static_cast<int>(tokens) : -1;
        a.seqlens[b] = s.cached + (ok ? static_cast<int>(tokens) : 0);
      }
    }
  }
  if (tid == 0) {
    s_start[a.B] = static_cast<int>(run[2]);
    if (rank == 0) a.starts[a.B] = static_cast<int>(run[2]);
  }
  __syncthreads();

  // the ring's i-th page from its first, i < 2 P
  auto ring_at = [&](int64_t i) {
    i += first;
    while (i >= P) i -= P;
    return static_cast<int>(i);
  };
  // tokens
  const int total = static_cast<int>(run[2]), threads = CLUSTER * kThreads;
  for (int64_t n0 = (static_cast<int64_t>(rank) * kThreads + tid) * 4; n0 < a.max_tokens; n0 += static_cast<int64_t>(threads) * 4) {
    int b = 0, end = 0;
    if (n0 < total) {
      int lo = 0, hi = a.B - 1;   // the last sequence that starts at or before n0
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_start[mid] <= n0) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
      end = s_start[b + 1];
    }
    int cached = 0, held = 0, of = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = n0 + i;
      if (n >= a.max_tokens) break;
      int64_t pos = -1, slot = -1;
      int id = -1;
      if (n < total) {
        while (n >= end) end = s_start[++b + 1];
        if (of != b) {
          cached = max(a.cached[b], 0);
          held = min(max(a.held[b], 0), a.pages_per_seq);
          of = b;
        }
        const int at = cached + (static_cast<int>(n) - s_start[b]), pi = a.div.page(at);
        const int page = pi < held ? a.table[b * a.ld_table + pi] : a.free_pages[ring_at(s_take[b] + pi - held)];
        pos = at;
        id = b;
        if (page >= 0 && page < P) slot = static_cast<int64_t>(page) * a.div.size + a.div.slot(at, pi);
      }
      a.positions[n] = pos;
      a.seq_ids[n] = id;
      a.slots[n] = slot;
    }
  }
  // pages: a warp a sequence
  for (int b = rank * kWarps + (tid >> 5); b < a.B; b += CLUSTER * kWarps) {
    if (s_take[b] < 0) continue;
    const Seq s = load_seq(a, b);
    int32_t* const row = a.table + b * a.ld_table;
    const int target = static_cast<int>(s.target);
    for (int i = s.held + lane; i < target; i += 32) row[i] = a.free_pages[ring_at(s_take[b] + i - s.held)];
    for (int i = target + lane; i < s.held; i += 32) {
      const int64_t place = static_cast<int64_t>(count) + s_give[b] + i - target;
      if (place < P) a.free_pages[ring_at(place)] = row[i];
      row[i] = -1;
    }
  }
  // nobody reads the old state any more
  if constexpr (CLUSTER > 1) cluster_sync();
  else __syncthreads();
  for (int b = rank * kThreads + tid; b < a.B; b += threads)
    if (s_take[b] >= 0) {
      const int64_t want = static_cast<int64_t>(max(a.cached[b], 0)) + max(a.fresh[b], 0);
      a.held[b] = static_cast<int>((want + a.div.size - 1) / a.div.size);
    }
  if (rank == 0 && tid == 0) {
    a.ring[0] = P > 0 ? ring_at(run[0]) : 0;
    a.ring[1] = static_cast<int>(min(count - run[0] + run[1], static_cast<int64_t>(P)));
  }
}

template <int CLUSTER>
int launch_plan(const PlanArgs& a, size_t smem, bool pdl, cudaStream_t s) {
  auto kern = page_plan_kernel<CLUSTER>;
  static bool configured[64] = {};   // per device; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    constexpr int most = (3 * kMaxSeqs + 1) * 4;
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) {
      set_cuda_error(e);
      return B2D_ERR_LAUNCH;
    }
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CLUSTER);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
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
                   granted, page_div(page_size), pages_per_seq, num_pages, B, max_tokens};
  const size_t smem = (3 * static_cast<size_t>(B) + 1) * 4;
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (B <= 256 && max_tokens <= 4096) return launch_plan<1>(a, smem, pdl, s);
  return launch_plan<kClusterSize>(a, smem, pdl, s);
}
