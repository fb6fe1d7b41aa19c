// Verification of drafted tokens by speculative sampling (sm_100a): accept the leading drafts with
// u_i q_i(x_i) < p_i(x_i), then draw one token from max(p - q, 0) of the first refused position, or from p
// behind the last draft, by inverting its running sum at a given random number. No counterpart in the
// reference, which decodes greedily.
//
// Only the row that the draw needs is read (V values of p, and of q after a refusal), not all K + 1.
// Every product, sum and comparison is in 64 bits: with fp32 running sums over 10^5 weights the border
// between two tokens moves by more than a small token's own weight.
// A sequence takes a thread-block cluster of up to 8 CTAs:
//  1. thread i < n tests draft i (in every CTA: the few loads are cheaper than an exchange); the first refusal
//     is the lowest clear bit of a ballot;
//  2. every warp sums its contiguous piece of the row (loads of 8 steps in flight), and the pieces' sums meet
//     through distributed shared memory;
//  3. a warp of each CTA scans them; the CTA that holds the target sums the piece again in 256 chunks (from
//     L2), scans those, and the thread that holds the target walks its chunk.
// Measured on B200 (fp32 probabilities; copy rate 6.52 TB/s): 128 sequences x 131071 tokens 34 us (3.9 TB/s of the
// rows that are read; 25 warps per SM issue in 48 % of the slots: latency and the phases that wait for one
// another), 64 x 32768 without draft probabilities 6.8 us, one x 32000 5.4 us (launch and dependent reads).
// One CTA per sequence took 93, 16.0 and 12.6; clusters with widening by conversions in part 43, 9.4 and 5.7.
#include <type_traits>

#include "common.cuh"

namespace b2d {
namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCluster = 8;
constexpr int kMaxDrafts = 31;

struct VerifyArgs {
  const int64_t* draft; int64_t ld_tokens;
  const int32_t* draft_lens;
  const void* target; int64_t st_b, st_k;
  const void* probs; int64_t sd_b, sd_k;
  const float* u; int64_t ld_u;
  int64_t* tokens; int64_t ld_out;
  int32_t* accepted;
  int K, V;
};

template <typename P> __device__ __forceinline__ double to_f64(P v) { return static_cast<double>(Dt<P>::to_f32(v)); }
template <> __device__ __forceinline__ double to_f64<float>(float v) { return static_cast<double>(v); }
// The weights of a row are summed times 2^30: exact, and no fp32 value is subnormal then, so that a positive one
// widens by moving its exponent and mantissa into place -- the conversion instruction has a small share of the
// SM's rate and bounded the kernel. (An infinity counts as 2^128.)
constexpr float kWeightScale = 1073741824.f;
__device__ __forceinline__ double widen(float x) {   // x > 0 and normal
  const uint32_t u = __float_as_uint(x);
  return __hiloint2double(static_cast<int>((u >> 3) + 0x38000000u), static_cast<int>(u << 29));
}
// 2^30 (p - q) for a negative q (no probability; out of line, so that its conversions stay off the usual path)
__device__ __noinline__ double weight_of_negative(float p, float q) {
  return (static_cast<double>(p) - static_cast<double>(q)) * static_cast<double>(kWeightScale);
}
// sum += 2^30 max(p - q, 0); NaN counts as zero. HAS_Q false: q is zero.
template <bool HAS_Q>
__device__ __forceinline__ void add_weight(float p, float q, double& sum) {
  if constexpr (HAS_Q) {
    if (p > q) {
      if (q >= 0.f) {
        const double wide = widen(q * kWeightScale);
        sum += widen(p * kWeightScale) - (q == 0.f ? 0.0 : wide);
      } else {
        sum += weight_of_negative(p, q);
      }
    }
  } else {
    if (p > 0.f) sum += widen(p * kWeightScale);
  }
}
// The same weight for token v of a row: max(p - q, 0), or p with the drafted token x left out (q null).
template <typename P>
__device__ __forceinline__ double weight(const P* p, const P* q, int64_t x, int v) {
  double w = 0.0;
  if (q) add_weight<true>(Dt<P>::to_f32(p[v]), Dt<P>::to_f32(q[v]), w);
  else if (v != x) add_weight<false>(Dt<P>::to_f32(p[v]), 0.f, w);
  return w;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_scan(double v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
__device__ __forceinline__ double ld_dsmem_f64(uint32_t local_addr, int rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(local_addr), "r"(rank));
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];\n" : "=d"(v) : "r"(remote) : "memory");
  return v;
}

template <typename P>
__global__ void __launch_bounds__(kVerifyThreads, 4) verify_drafts_kernel(const VerifyArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int s_accepted, s_owner, s_place[kVerifyWarps];
  __shared__ double s_sum[kVerifyWarps];   // read by the cluster
  __shared__ double s_start, s_total, s_scan[kVerifyWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ranks = cluster_size(), rank = cluster_rank(), b = static_cast<int>(blockIdx.x) / ranks;
  const int n = a.draft_lens ? max(0, min(a.K, a.draft_lens[b])) : a.K;
  const P* target = static_cast<const P*>(a.target) + b * a.st_b;
  const P* probs = a.probs ? static_cast<const P*>(a.probs) + b * a.sd_b : nullptr;
  const double u_draw = static_cast<double>(a.u[b * a.ld_u + a.K]);
  if (warp == 0) {
    bool ok = false;
    if (lane < n) {
      const int64_t x = a.draft[b * a.ld_tokens + lane];
      if (x >= 0 && x < a.V) {
        const double q = probs ? to_f64<P>(probs[lane * a.sd_k + x]) : 1.0;
        ok = static_cast<double>(a.u[b * a.ld_u + lane]) * q < to_f64<P>(target[lane * a.st_k + x]);
      }
    }
    const uint32_t refused = ~__ballot_sync(0xffffffffu, ok);   // lanes >= n count as refused (n <= 31)
    if (lane == 0) s_accepted = __ffs(refused) - 1;
  }
  __syncthreads();
  const int acc = s_accepted;
  const P* p = target + acc * a.st_k;
  const P* q = acc < n && probs ? probs + acc * a.sd_k : nullptr;
  int64_t x = acc < n && !probs ? a.draft[b * a.ld_tokens + acc] : -1;
  const int pieces = ranks * kVerifyWarps, piece = (a.V + pieces - 1) / pieces;
  const int v0 = min(a.V, (rank * kVerifyWarps + warp) * piece), v1 = min(a.V, v0 + piece);
  for (int pass = 0;; ++pass) {
    double sum = 0.0;
    auto add_piece = [&](auto has_q) {
      constexpr bool HAS_Q = decltype(has_q)::value;
      P pv[2][8], qv[2][8];   // 8 steps of 32 values are added while the next 8 are under way
      auto load = [&](int set, int base) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int v = base + 32 * i;
          pv[set][i] = v < v1 ? p[v] : P(0.f);
          if constexpr (HAS_Q) qv[set][i] = v < v1 ? q[v] : P(0.f);
        }
      };
      auto add = [&](int set, int base) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (HAS_Q) add_weight<true>(Dt<P>::to_f32(pv[set][i]), Dt<P>::to_f32(qv[set][i]), sum);
          else add_weight<false>(base + 32 * i == x ? 0.f : Dt<P>::to_f32(pv[set][i]), 0.f, sum);
        }
      };
      load(0, v0 + lane);
      for (int base = v0 + lane; base - lane < v1; base += 512) {
        load(1, base + 256);
        add(0, base);
        load(0, base + 512);
        add(1, base + 256);
      }
    };
    if (q) add_piece(std::true_type{});
    else add_piece(std::false_type{});
    sum = warp_sum(sum);
    if (lane == 0) s_sum[warp] = sum;
    if (ranks > 1) cluster_sync();
    else __syncthreads();
    if (warp == 0) {   // up to 64 pieces, two a lane
      double w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = 2 * lane + i;
        w[i] = e >= pieces ? 0.0
               : ranks > 1 ? ld_dsmem_f64(static_cast<uint32_t>(__cvta_generic_to_shared(&s_sum[e % kVerifyWarps])), e / kVerifyWarps)
                           : s_sum[e];
      }
      const double incl = warp_scan(w[0] + w[1], lane), start = incl - (w[0] + w[1]);
      const double total = __shfl_sync(0xffffffffu, incl, 31), goal = u_draw * total;
      const uint32_t above0 = __ballot_sync(0xffffffffu, w[0] > 0.0 && start + w[0] > goal);
      const uint32_t above1 = __ballot_sync(0xffffffffu, w[1] > 0.0 && incl > goal);
      const uint32_t some0 = __ballot_sync(0xffffffffu, w[0] > 0.0), some1 = __ballot_sync(0xffffffffu, w[1] > 0.0);
      int owner = -1;   // the first piece whose end is above the goal, else the last one with any weight
      if (above0 | above1) {
        const int l = __ffs(above0 | above1) - 1;
        owner = 2 * l + ((above0 >> l & 1) ? 0 : 1);
      } else if (some0 | some1) {
        const int l = 31 - __clz(some0 | some1);
        owner = 2 * l + ((some1 >> l & 1) ? 1 : 0);
      }
      const double begin0 = __shfl_sync(0xffffffffu, start, max(owner, 0) >> 1);
      const double first = __shfl_sync(0xffffffffu, w[0], max(owner, 0) >> 1);
      if (lane == 0) {
        s_owner = owner;
        s_total = total;
        s_start = (owner & 1) ? begin0 + first : begin0;
      }
    }
    if (ranks > 1) cluster_sync();   // the sums are read; also a barrier of this CTA
    else __syncthreads();
    if (s_total > 0.0 || pass == 1 || acc == n) break;
    q = nullptr;   // max(p - q, 0) is zero everywhere: draw from p
    x = -1;
  }
  const int owner = s_owner;
  if (rank == 0) {
    if (tid < a.K + 1 && tid != acc) a.tokens[b * a.ld_out + tid] = tid < acc ? a.draft[b * a.ld_tokens + tid] : -1;
    if (tid == 0 && a.accepted) a.accepted[b] = acc;
    if (owner < 0 && tid == 0) a.tokens[b * a.ld_out + acc] = -1;
  }
  if (owner < 0 || owner / kVerifyWarps != rank) return;
  // ---- the owner's piece in 256 chunks, one a thread
  const double goal = u_draw * s_total;
  const int o0 = min(a.V, owner * piece), o1 = min(a.V, o0 + piece), chunk = (piece + kVerifyThreads - 1) / kVerifyThreads;
  const int c0 = min(o1, o0 + tid * chunk), c1 = min(o1, c0 + chunk);
  double sum = 0.0;
#pragma unroll 4
  for (int v = c0; v < c1; ++v) sum += weight<P>(p, q, x, v);
  const double incl = warp_scan(sum, lane);
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  double run = s_start;
#pragma unroll
  for (int w = 0; w < kVerifyWarps; ++w)
    if (w < warp) run += s_scan[w];
  const uint32_t above = __ballot_sync(0xffffffffu, sum > 0.0 && run + incl > goal);
  const uint32_t some = __ballot_sync(0xffffffffu, sum > 0.0);
  // the first thread whose end is above the goal, else the last one with any weight (as 2 T - thread)
  constexpr int T2 = 2 * kVerifyThreads;
  if (lane == 0)
    s_place[warp] = above ? 32 * warp + __ffs(above) - 1 : some ? T2 - (32 * warp + 31 - __clz(some)) : T2 + 1;
  __syncthreads();
  int place = s_place[0];
#pragma unroll
  for (int w = 1; w < kVerifyWarps; ++w) place = min(place, s_place[w]);
  if (place > T2 || tid != (place < kVerifyThreads ? place : T2 - place)) return;
  run += incl - sum;
  int found = -1, last = -1;
  for (int v = c0; v < c1; ++v) {
    const double w = weight<P>(p, q, x, v);
    if (w > 0.0) {
      last = v;
      run += w;
      if (run > goal) {
        found = v;
        break;
      }
    }
  }
  a.tokens[b * a.ld_out + acc] = found >= 0 ? found : last;
}

template <typename P>
int launch_verify(const VerifyArgs& a, int B, int ranks, bool pdl, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B) * ranks);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_drafts_kernel<P>, a);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return B2D_ERR_LAUNCH;
  }
  return launch_status();
}

}  // namespace
}  // namespace b2d

using namespace b2d;

extern "C" int b2d_verify_drafts(const int64_t* draft_tokens, int64_t ld_tokens, const int32_t* draft_lens,
                                 const void* target_probs, int64_t st_b, int64_t st_k, const void* draft_probs,
                                 int64_t sd_b, int64_t sd_k, int probs_dtype, const float* uniforms, int64_t ld_u,
                                 int64_t* tokens, int64_t ld_out, int32_t* accepted, int B, int K, int V, int flags,
                                 void* stream) {
  if (B < 0 || K < 0 || V < 0) return B2D_ERR_ARG;
  if (probs_dtype != B2D_F32 && probs_dtype != B2D_F16 && probs_dtype != B2D_BF16) return B2D_ERR_DTYPE;
  if (K > kMaxDrafts || V == 0 || V > (1 << 30) || ld_tokens < 0 || ld_u < 0 || ld_out < K + 1) return B2D_ERR_SHAPE;
  if (B == 0) return B2D_OK;
  if ((!draft_tokens && K > 0) || !target_probs || !uniforms || !tokens) return B2D_ERR_ARG;
  const int size = probs_dtype == B2D_F32 ? 4 : 2;
  if (!aligned(draft_tokens, 8) || !aligned(draft_lens, 4) || !aligned(target_probs, size) ||
      !aligned(draft_probs, size) || !aligned(uniforms, 4) || !aligned(tokens, 8) || !aligned(accepted, 4))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  int st;
  if ((st = device_info(&di)) != B2D_OK) return st;
  const VerifyArgs a{draft_tokens, ld_tokens, draft_lens, target_probs, st_b, st_k, draft_probs, sd_b, sd_k,
                     uniforms, ld_u, tokens, ld_out, accepted, K, V};
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // CTAs of a sequence: as many as fit the SMs at once (four each), with at least 1024 tokens
  int ranks = 1;
  while (ranks < kVerifyCluster && static_cast<int64_t>(B) * ranks * 2 <= 4 * di.sm_count && V / (ranks * 2) >= 1024) ranks *= 2;
  if (static_cast<int64_t>(B) * ranks > (int64_t(1) << 31) - 1) return B2D_ERR_SHAPE;
  if (probs_dtype == B2D_F32) return launch_verify<float>(a, B, ranks, pdl, s);
  if (probs_dtype == B2D_F16) return launch_verify<__half>(a, B, ranks, pdl, s);
  return launch_verify<__nv_bfloat16>(a, B, ranks, pdl, s);
}
