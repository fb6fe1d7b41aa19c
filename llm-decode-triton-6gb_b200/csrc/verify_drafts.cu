// Verification of drafted tokens by speculative sampling (sm_100a): accept the leading drafts with
// u_i q_i(x_i) < p_i(x_i), then draw one token from max(p - q, 0) of the first refused position, or from p
// behind the last draft, by inverting its running sum at a given random number. No counterpart in the
// reference, which decodes greedily.
//
// Only the row that the draw needs is read (V values of p, and of q after a refusal), not all K + 1.
// Every product, sum and comparison is in 64 bits: with fp32 running sums over 10^5 weights the border
// between two tokens moves by more than a small token's own weight.
//  1. thread i < n tests draft i; the first refusal is the lowest clear bit of a ballot;
//  2. every warp sums its contiguous piece of the row;
//  3. the pieces are scanned in order; the warp whose piece holds the target walks it 32 values at a time.
#include "common.cuh"

namespace b2d {
namespace {

constexpr int kVerifyThreads = 1024;
constexpr int kVerifyWarps = kVerifyThreads / 32;
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

// The weight of token v: p (q null and x < 0), max(p - q, 0), or p with the drafted token x left out.
// NaN and negative weights count as zero.
template <typename P>
__device__ __forceinline__ double weight(const P* p, const P* q, int64_t x, int v) {
  double w = to_f64<P>(p[v]);
  if (q) w -= to_f64<P>(q[v]);
  else if (v == x) w = 0.0;
  return w > 0.0 ? w : 0.0;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename P>
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ int s_accepted;
  __shared__ double s_sum[kVerifyWarps], s_start[kVerifyWarps];
  __shared__ double s_total;
  __shared__ int s_owner, s_last;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = a.draft_lens ? max(0, min(a.K, a.draft_lens[b])) : a.K;
  const P* target = static_cast<const P*>(a.target) + b * a.st_b;
  const P* probs = a.probs ? static_cast<const P*>(a.probs) + b * a.sd_b : nullptr;
  if (warp == 0) {
    bool ok = false;
    if (lane < n) {
      const int64_t x = a.draft[b * a.ld_tokens + lane];
      if (x >= 0 && x < a.V) {
        const double q = probs ? to_f64<P>(probs[lane * a.sd_k + x]) : 1.0;
        ok = static_cast<double>(a.u[b * a.ld_u + lane]) * q < to_f64<P>(target[lane * a.st_k + x]);
      }
    }
    const uint32_t refused = ~__ballot_sync(0xffffffffu, ok);   // lanes >= n count as refused
    if (lane == 0) {
      const int acc = min(n, __ffs(refused) - 1);
      s_accepted = refused ? acc : n;
    }
  }
  __syncthreads();
  const int acc = s_accepted;
  const P* p = target + acc * a.st_k;
  const P* q = acc < n && probs ? probs + acc * a.sd_k : nullptr;
  int64_t x = acc < n && !probs ? a.draft[b * a.ld_tokens + acc] : -1;
  const int piece = ((a.V + kVerifyWarps - 1) / kVerifyWarps + 31) / 32 * 32;
  const int v0 = min(a.V, warp * piece), v1 = min(a.V, v0 + piece);
  for (int pass = 0;; ++pass) {
    double sum = 0.0;
    for (int v = v0 + lane; v < v1; v += 32) sum += weight<P>(p, q, x, v);
    sum = warp_sum(sum);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      double run = 0.0;
      for (int w = 0; w < kVerifyWarps; ++w) {
        s_start[w] = run;
        run += s_sum[w];
      }
      s_total = run;
      const double goal = static_cast<double>(a.u[b * a.ld_u + a.K]) * run;
      int owner = -1, last = -1;
      for (int w = 0; w < kVerifyWarps; ++w) {
        if (s_sum[w] > 0.0) last = w;
        if (owner < 0 && s_start[w] + s_sum[w] > goal) owner = w;
      }
      s_owner = owner < 0 ? last : owner;   // no piece reaches the goal: the last one with any weight
      s_last = last;
    }
    __syncthreads();
    if (s_total > 0.0 || pass == 1 || acc == n) break;
    q = nullptr;   // max(p - q, 0) is zero everywhere: draw from p
    x = -1;
    __syncthreads();
  }
  const int owner = s_owner;
  if (tid < a.K + 1 && tid != acc) a.tokens[b * a.ld_out + tid] = tid < acc ? a.draft[b * a.ld_tokens + tid] : -1;
  if (tid == 0 && a.accepted) a.accepted[b] = acc;
  if (owner < 0) {
    if (tid == 0) a.tokens[b * a.ld_out + acc] = -1;
    return;
  }
  if (warp != owner) return;
  const double goal = static_cast<double>(a.u[b * a.ld_u + a.K]) * s_total;
  double run = s_start[warp];
  int found = -1, last = -1;
  for (int base = v0; base < v1; base += 32) {
    const int v = base + lane;
    const double w = v < v1 ? weight<P>(p, q, x, v) : 0.0;
    double scan = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    const uint32_t some = __ballot_sync(0xffffffffu, w > 0.0);
    if (some) last = base + 31 - __clz(some);
    const uint32_t above = __ballot_sync(0xffffffffu, w > 0.0 && run + scan > goal);
    if (above) {
      found = base + __ffs(above) - 1;
      break;
    }
    run += __shfl_sync(0xffffffffu, scan, 31);
  }
  if (lane == 0) a.tokens[b * a.ld_out + acc] = found >= 0 ? found : last;
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
  if (K > kMaxDrafts || V == 0 || ld_tokens < 0 || ld_u < 0 || ld_out < K + 1) return B2D_ERR_SHAPE;
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
  const dim3 grid(static_cast<unsigned>(B)), block(kVerifyThreads);
  if (probs_dtype == B2D_F32) return launch_kernel(verify_drafts_kernel<float>, grid, block, 0, s, pdl, a);
  if (probs_dtype == B2D_F16) return launch_kernel(verify_drafts_kernel<__half>, grid, block, 0, s, pdl, a);
  return launch_kernel(verify_drafts_kernel<__nv_bfloat16>, grid, block, 0, s, pdl, a);
}
