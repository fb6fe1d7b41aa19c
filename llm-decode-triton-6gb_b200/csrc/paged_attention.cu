// Attention of the newest tokens of every sequence over a paged KV cache, causal among themselves, with an
// optional prefix shared by the whole batch (sm_100a). The contiguous one-token counterpart is
// csrc/gqa_decode.cu (reference: profiling/kernels/decode_attention.py:18-91).
//
// o[b, t, h] = sum_{j < limit} softmax_j(scale q.k_j) v_j, limit = seqlens[b] - T + 1 + t. Key j lies in
// prefix_table's pages for j < prefix_len and in page_table[b]'s behind.
//
// A CTA owns one (sequence, KV head, tile of 16 RW rows): rows are the T x G query vectors that read this KV
// head (row = t G + g), so K and V are read once for all of them. Stages of 64 keys pass through a 3-stage
// shared-memory ring filled by 16-byte cp.async (each thread looks the page of its key rows up, keys at or
// past the length are zero-filled without a read, so what a page holds behind its last key never enters).
// 16-byte chunk c of key row r sits at chunk c ^ (r & 7), so ldmatrix reads hit 8 distinct bank groups.
// S = Q K^T and O += P V by mma.sync m16n8k16 (fp32 accumulate): warp (rw, kw) takes rows [16 rw, 16 rw + 16)
// and keys [kw 16 RW, ...) of each stage; online softmax in the log2 domain; the key warps meet in shared
// memory. P is rounded to the cache's dtype for the second product, as its V operand is; the sum of the
// weights is taken before that rounding, in fp32.
#include "paged.cuh"

namespace b2d {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 64;      // keys of a stage
constexpr int kStages = 3;
constexpr int kMaxT = 16, kMaxG = 16;
constexpr float kLog2e = 1.4426950408889634f;

struct PagedAttnArgs {
  const void* q; int64_t sq_b, sq_t, sq_h;
  const int32_t* table; int64_t ld_table;
  const int32_t* seqlens;
  const int32_t* prefix_table;
  void* out; int64_t so_b, so_t, so_h;
  b2d_paged_kv kv;
  PageDiv div;
  int pages_per_seq, prefix_len, B, T, H, G, rows;   // rows = T G
  float scale_log2;
};

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

template <int D>
constexpr size_t ring_bytes() { return static_cast<size_t>(kStages) * 2 * kKeys * D * 2; }

template <typename T, typename OT, int D, int RW>
__global__ void __launch_bounds__(kThreads, 2) paged_attention_kernel(const PagedAttnArgs a) {
  constexpr int KW = kWarps / RW;       // warps that share a row tile and split a stage's keys
  constexpr int WK = kKeys / KW;        // keys of a stage that a warp takes
  constexpr int KSTEPS = D / 16, NTILES = D / 8, CH = D / 8;
  constexpr uint32_t ROWB = D * 2, TILEB = kKeys * ROWB;
  constexpr int OPAD = D + 8;
  constexpr int LOADS = kKeys * CH / kThreads;   // key rows of a stage that a thread copies a chunk of
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][16], s_l[kWarps][16];

  pdl_launch_dependents();
  pdl_wait();
  const int row0 = blockIdx.x * 16 * RW, kvh = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rw = warp % RW, kw = warp / RW;
  const int g = lane >> 2, tq = lane & 3, mi = lane >> 3, ri = lane & 7;
  const uint32_t sbase = smem_u32(smem);
  const T* kpool = static_cast<const T*>(a.kv.k) + kvh * a.kv.sk_h;
  const T* vpool = static_cast<const T*>(a.kv.v) + kvh * a.kv.sv_h;
  const int32_t* table = a.table + b * a.ld_table;

  const int64_t reach = static_cast<int64_t>(a.pages_per_seq) * a.kv.page_size;
  int len = max(a.seqlens[b], 0);
  if (len > reach) len = max(static_cast<int>(reach), a.prefix_len);
  const int row_end = min(a.rows, row0 + 16 * RW);
  // keys that any row of the tile sees; limits of this thread's two rows
  const int t_last = (row_end - 1) / a.G;
  const int t_end = max(0, len - a.T + 1 + t_last);
  int lim[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) lim[h] = len - a.T + 1 + min(row0 + 16 * rw + g + 8 * h, row_end - 1) / a.G;
  const int lim_min = len - a.T + 1 + row0 / a.G;   // below it no row is masked

  auto issue = [&](int it) {
    const uint32_t kdst = sbase + static_cast<uint32_t>(it % kStages) * 2 * TILEB, vdst = kdst + TILEB;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int ci = tid + i * kThreads, r = ci / CH, c = ci % CH;
      const int tok = it * kKeys + r;
      const T* ks = kpool;
      const T* vs = vpool;
      bool ok = tok < t_end;
      if (ok) {
        const int pi = a.div.page(tok);
        const int page = tok < a.prefix_len ? a.prefix_table[pi] : table[pi];
        ok = page >= 0 && page < a.kv.num_pages;
        if (ok) {
          const int64_t slot = a.div.slot(tok, pi);
          ks += page * a.kv.sk_p + slot * a.kv.sk_s + c * 8;
          vs += page * a.kv.sv_p + slot * a.kv.sv_s + c * 8;
        }
      }
      const uint32_t off = static_cast<uint32_t>(r) * ROWB + static_cast<uint32_t>((c ^ (r & 7)) * 16);
      cp_async16_zfill(kdst + off, ks, ok);
      cp_async16_zfill(vdst + off, vs, ok);
    }
  };

  const int nst = (t_end + kKeys - 1) / kKeys;
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < nst) issue(i);
    cp_async_commit();
  }

  // Q fragments of this warp's 16 rows
  uint32_t qa[KSTEPS][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = row0 + 16 * rw + g + 8 * h;
    const bool live = row < a.rows;
    const int t = row / a.G, head = kvh * a.G + row - t * a.G;
    const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + b * a.sq_b + t * a.sq_t +
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

  for (int it = 0; it < nst; ++it) {
    cp_async_wait<kStages - 2>();
    __syncthreads();
    if (it + kStages - 1 < nst) issue(it + kStages - 1);
    cp_async_commit();
    const int key0 = it * kKeys + kw * WK;
    if (key0 >= t_end) continue;
    const uint32_t kbuf = sbase + static_cast<uint32_t>(it % kStages) * 2 * TILEB, vbuf = kbuf + TILEB;
    const bool masked = key0 + WK > lim_min;

    float s[WK / 8][4];
    float tmax[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < WK / 8; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      const int r = kw * WK + 8 * n + ri;
#pragma unroll
      for (int j = 0; j < KSTEPS; j += 2) {
        const int c = 2 * j + mi;
        uint32_t b0, b1, b2, b3;
        ldsm_x4(kbuf + static_cast<uint32_t>(r) * ROWB + static_cast<uint32_t>((c ^ (r & 7)) * 16), b0, b1, b2, b3);
        Mma<T>::run(s[n], qa[j][0], qa[j][1], qa[j][2], qa[j][3], b0, b1);
        Mma<T>::run(s[n], qa[j + 1][0], qa[j + 1][1], qa[j + 1][2], qa[j + 1][3], b2, b3);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int tok = key0 + 8 * n + 2 * tq + (c & 1);
        s[n][c] *= a.scale_log2;
        if (masked && tok >= lim[c >> 1]) s[n][c] = -INFINITY;
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
    for (int u = 0; u < WK / 16; ++u) {   // 16 keys at a time
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
        const int r = kw * WK + 16 * u + 8 * (mi & 1) + ri, c = np + (mi >> 1);
        uint32_t v0, v1, v2, v3;
        ldsm_x4_t(vbuf + static_cast<uint32_t>(r) * ROWB + static_cast<uint32_t>((c ^ (r & 7)) * 16), v0, v1, v2, v3);
        Mma<T>::run(o[np], pa[0], pa[1], pa[2], pa[3], v0, v1);
        Mma<T>::run(o[np + 1], pa[0], pa[1], pa[2], pa[3], v2, v3);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();   // the ring becomes the merge buffer

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
  __syncthreads();

  for (int idx = tid; idx < (row_end - row0) * D; idx += kThreads) {
    const int row = idx / D, d = idx - row * D;
    const int w0 = row / 16, rr = row % 16;
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < KW; ++k) mx = fmaxf(mx, s_m[k * RW + w0][rr]);
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const int w = k * RW + w0;
      const float e = s_m[w][rr] == -INFINITY ? 0.f : exp2_fast(s_m[w][rr] - mx);
      num += e * s_o[(w * 16 + rr) * OPAD + d];
      den += e * s_l[w][rr];
    }
    const int t = (row0 + row) / a.G, head = kvh * a.G + row0 + row - t * a.G;
    // a row that sees no key: zeros (den is NaN, not 0, where a visible score is)
    static_cast<OT*>(a.out)[b * a.so_b + t * a.so_t + static_cast<int64_t>(head) * a.so_h + d] =
        Dt<OT>::from_f32(den == 0.f ? 0.f : num / den);
  }
}

template <typename T, typename OT, int D, int RW>
int launch(const PagedAttnArgs& a, bool pdl, cudaStream_t s) {
  auto kern = paged_attention_kernel<T, OT, D, RW>;
  constexpr size_t bytes = ring_bytes<D>();
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return B2D_ERR_LAUNCH;
  }
  const dim3 grid((a.rows + 16 * RW - 1) / (16 * RW), a.kv.KVH, a.B);
  return launch_kernel(kern, grid, dim3(kThreads), bytes, s, pdl, a);
}
template <typename T, typename OT>
int launch_shape(const PagedAttnArgs& a, bool pdl, cudaStream_t s) {
  const int rw = a.rows <= 16 ? 1 : a.rows <= 32 ? 2 : 4;
  if (a.kv.D == 64)
    return rw == 1 ? launch<T, OT, 64, 1>(a, pdl, s) : rw == 2 ? launch<T, OT, 64, 2>(a, pdl, s)
                                                               : launch<T, OT, 64, 4>(a, pdl, s);
  return rw == 1 ? launch<T, OT, 128, 1>(a, pdl, s) : rw == 2 ? launch<T, OT, 128, 2>(a, pdl, s)
                                                              : launch<T, OT, 128, 4>(a, pdl, s);
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
  if (check_shapes(kv, B, T, H, pages_per_seq, prefix_len, max_len) != B2D_OK) return 0;
  return 0;
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
  PagedAttnArgs a{};
  a.q = q; a.sq_b = sq_b; a.sq_t = sq_t; a.sq_h = sq_h;
  a.table = page_table; a.ld_table = ld_table; a.seqlens = seqlens; a.prefix_table = prefix_table;
  a.out = out; a.so_b = so_b; a.so_t = so_t; a.so_h = so_h;
  a.kv = *kv; a.div = page_div(kv->page_size);
  a.pages_per_seq = pages_per_seq; a.prefix_len = prefix_len;
  a.B = B; a.T = T; a.H = H; a.G = H / kv->KVH; a.rows = T * a.G;
  a.scale_log2 = scale * kLog2e;
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (kv->dtype == B2D_F16)
    return out_dtype == B2D_F32 ? launch_shape<__half, float>(a, pdl, s) : launch_shape<__half, __half>(a, pdl, s);
  return out_dtype == B2D_F32 ? launch_shape<__nv_bfloat16, float>(a, pdl, s)
                              : launch_shape<__nv_bfloat16, __nv_bfloat16>(a, pdl, s);
}
