// Append to the 4-bit paged cache (norm, rotation, quantisation) and the read back of its values (sm_100a); the layout is in
// int4_kv.cuh, the 16-bit counterpart in paged_append.cu.
//
// D / 16 neighbouring lanes own a head, 16 elements each as two chunks of 8 that hold whole rotation pairs: [8 j, 8 j + 8) and
// [R / 2 + 8 j, ...) for the half layout's turning elements, 16 neighbouring ones otherwise. A warp takes a token's query heads,
// or its key and value heads, four (D = 128) or eight at a time; few tokens are cut over more warps. The next heads' loads are
// under way while the present ones are worked on.
//  * q: fp32, one rounding; the weights' products with cos and sin are formed once per warp.
//  * k: the mean in 64 bits and every product and sum rounded as the definition says (no contraction), so that a code is the
//    formula's and not its neighbour; the row passes through shared memory to the order of the runs, 16 neighbouring
//    elements a lane, where a run's extrema are one or two shuffles and the codes of a lane are a step of the fragment order.
//  * v: loaded in that order at once. A position's codes lie in single bytes (the other bytes of a word are other
//    positions'), so that no store reads what another token writes.
//
// Measured on B200: 8168 tokens of 32 + 8 + 8 heads of 128 with norms, bf16: 49 us, 3.6 TB/s of the bytes that it cannot do
// without (177 MB; copy rate 6.55); 320 tokens 4.1 us; one token 2.6 us (launch and a chain of three loads). Bound by issued
// instructions and latency: 3400 warp instructions a token, 56 % of the slots, 21 warps per SM (six blocks; their 80 registers a
// thread spill 32 to 48 bytes in every form). Earlier forms: one warp for all heads of
// a token with a division per code 87 us; packed fp32 instructions and corrected quotients 50; queries apart from keys 48. Reading
// 8 x 4001 tokens: 35.7 us, 4.8 TB/s, with 16-byte stores 38.5; 8 x 1021 tokens 12.0 and 14.6 (a warp a token without the
// shared words and with stores of 16 bytes: 44).
#include <type_traits>

#include "int4_kv.cuh"

namespace b2d {
namespace {

struct Int4AppendArgs {
  const void* q; int64_t sq_n, sq_h;
  const void* k; int64_t sk_n, sk_h;
  const void* v; int64_t sv_n, sv_h;
  const int64_t* positions;
  const int32_t* seq_ids;
  const int32_t* table; int64_t ld_table;
  const void* cos; const void* sin; int64_t ld_cs;
  const void* q_weight; const void* k_weight;
  float eps;
  void* q_out; int64_t sqo_n, sqo_h;
  b2d_int4_kv kv;
  PageDiv div;
  int N, H, B, per_seq, pages_per_seq, rotary, q_parts;
  uint32_t per_inv;
  int64_t limit;   // positions from here on are padding
};

constexpr int kWarps = 4;

// Sequence of token n where every one has `per` tokens; inv = 2^32 / per, rounded down: the quotient or one less
__device__ __forceinline__ int sequence_of(int n, int per, uint32_t inv) {
  const int q = static_cast<int>(__umulhi(static_cast<uint32_t>(n), inv));
  return n - q * per >= per ? q + 1 : q;
}
uint32_t inverse_of(int per) { return per < 2 ? 0xFFFFFFFFu : static_cast<uint32_t>((uint64_t(1) << 32) / per); }

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float* f) {
  const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = Dt<T>::to_f32(h[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(Dt<T>::pack2(f[0], f[1]), Dt<T>::pack2(f[2], f[3]), Dt<T>::pack2(f[4], f[5]), Dt<T>::pack2(f[6], f[7]));
}
// (ordinary loads: read-only ones may be moved above the wait for the kernel before)
template <typename C>
__device__ __forceinline__ void load8(const C* p, float* f) {
  if constexpr (sizeof(C) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    unpack8<C>(*reinterpret_cast<const uint4*>(p), f);
  }
}

struct Chunks {
  uint4 a, b;
};

// Two fp32 operations an instruction (the kernels are bound by issued instructions, not by arithmetic).
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 pack(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack(const F2& a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(a.v)); }
__device__ __forceinline__ F2 add2(const F2& a, const F2& b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(const F2& a, const F2& b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(const F2& a, const F2& b, const F2& c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// 8 values as four pairs of neighbours
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, F2 (&f)[4]) {
  float x[8];
  unpack8<T>(u, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = pack(x[2 * i], x[2 * i + 1]);
}

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The smallest normal number of the 16-bit types
template <typename T> __device__ constexpr float kNormal = 0x1p-14f;
template <> constexpr float kNormal<__nv_bfloat16> = 0x1p-126f;

// 16 neighbouring elements of a run's lanes -> {s, m} and the codes, each in the low bits of a word whose others are
// 0x4B400000.
// The quotients (x - m) / s share their divisor: each is the product with 1 / s corrected by its exact remainder, which rounds as
// the division does (P. Markstein, Computation of elementary functions on the IBM RISC System/6000, 1990), and a sum with
// 2^23 + 2^22 rounds it to a whole number, ties to even. They lie in 0..15 by themselves where s is a normal number (its rounding
// moves 15 by less than a half) and m, where it was rounded up past elements, passed them by less than half a step; other
// runs, and divisors whose reciprocal could overflow, take the division and the clamps.
template <typename T>
__device__ __forceinline__ uint32_t quantise(const float (&x)[16], int run_lanes, uint32_t (&code)[16]) {
  float lo = min3(x[0], x[1], x[2]), hi = max3_nan(x[0], x[1], x[2]);
#pragma unroll
  for (int e = 3; e < 15; e += 2) {
    lo = min3(lo, x[e], x[e + 1]);
    hi = max3_nan(hi, x[e], x[e + 1]);
  }
  lo = fminf(lo, x[15]);
  hi = max_nan(hi, x[15]);
  for (int o = 1; o < run_lanes; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const float m = Dt<T>::to_f32(Dt<T>::from_f32(lo));
  // the product with the fp32 number next to 1 / 15, which is also what torch's division by 15 on a GPU does: another last bit of fp32
  // now and then lies across a 16-bit step, and the run's codes move with its scale
  const float s = Dt<T>::to_f32(Dt<T>::from_f32(fmaxf(__fmul_rn(__fsub_rn(hi, m), 1.f / 15.f), 0.f)));
  const bool sound = fabsf(hi) < INFINITY && fabsf(m) < INFINITY && s < INFINITY;
  constexpr float kEven = 12582912.f;   // 2^23 + 2^22
  if (sound && s >= kNormal<T> && s >= 0x1p-100f && fabsf(m) < 256.f * s) {
    const float r = __fdiv_rn(1.f, s);
    const F2 r2 = pack(r, r), s2 = pack(-s, -s), m2 = pack(-m, -m), even2 = pack(kEven, kEven);
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const F2 d = add2(pack(x[e], x[e + 1]), m2), q = mul2(d, r2);
      float c0, c1;
      unpack(add2(fma2(fma2(q, s2, d), r2, q), even2), c0, c1);
      code[e] = __float_as_uint(c0);
      code[e + 1] = __float_as_uint(c1);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float c = sound && s > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[e], m), s)) : 0.f;
      code[e] = __float_as_uint(fminf(fmaxf(c, 0.f), 15.f) + kEven);
    }
  }
  return sound ? Dt<T>::pack2(s, m) : Dt<T>::pack2(NAN, NAN);
}

// What both parts of the append know of a lane: head `sub` of its warp's, elements [o1, o1 + 8) and [o2, o2 + 8) of it.
template <int D>
struct Place {
  static constexpr int LANES = D / 16, HPW = 32 / LANES;   // lanes of a head, heads of a warp
  int j, sub, o1, o2;
  bool turns;
  __device__ __forceinline__ Place(int rotary, bool near) {
    const int lane = threadIdx.x & 31;
    j = lane % LANES;
    sub = lane / LANES;
    turns = 16 * j < rotary;
    o1 = turns && !near ? 8 * j : 16 * j;
    o2 = turns && !near ? rotary / 2 + 8 * j : 16 * j + 8;
  }
};

// The query heads of token n: items part, part + parts, ... of HPW heads each; the next one is under way behind the present one.
template <typename T, typename C, int D, bool NEAR>
__device__ __forceinline__ void append_queries(const Int4AppendArgs& a, int64_t n, int64_t pos, int part, int parts) {
  const Place<D> at(a.rotary, NEAR);
  constexpr int LANES = Place<D>::LANES, HPW = Place<D>::HPW;
  const int64_t q_step = static_cast<int64_t>(parts) * HPW * a.sq_h, o_step = static_cast<int64_t>(parts) * HPW * a.sqo_h;
  const T* q1 = static_cast<const T*>(a.q) + n * a.sq_n + (part * HPW + at.sub) * a.sq_h + at.o1;
  const T* q2 = q1 + (at.o2 - at.o1);
  int qh = part * HPW + at.sub, h = qh;   // the head that is loaded next, and the one that is stored next
  auto load = [&](Chunks& x) {
    if (qh < a.H) {
      x.a = *reinterpret_cast<const uint4*>(q1);
      x.b = *reinterpret_cast<const uint4*>(q2);
    }
    q1 += q_step;
    q2 += q_step;
    qh += parts * HPW;
  };
  Chunks c0{}, c1{};
  load(c0);
  // y1 = r (x1 f11 + x2 f12), y2 = r (x2 f22 + x1 f21), r the norm's factor: the weights' products with cos and sin. Pairs
  // 2 i and 2 i + 1 share an instruction (neighbours: the two chunks' i-th pairs).
  F2 f11[4], f12[4], f22[4], f21[4];
  {
    float c[8], sn[8], w[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c[e] = 1.f;
      sn[e] = 0.f;
      w[e] = w[8 + e] = 1.f;
    }
    if (at.turns) {
      load8(static_cast<const C*>(a.cos) + pos * a.ld_cs + 8 * at.j, c);
      load8(static_cast<const C*>(a.sin) + pos * a.ld_cs + 8 * at.j, sn);
    }
    if (a.q_weight) {
      load8(static_cast<const T*>(a.q_weight) + at.o1, w);
      load8(static_cast<const T*>(a.q_weight) + at.o2, w + 8);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e0 = NEAR ? i : 2 * i, e1 = NEAR ? i + 4 : 2 * i + 1;   // the pairs
      const float u0 = w[NEAR ? 2 * e0 : e0], v0 = w[NEAR ? 2 * e0 + 1 : 8 + e0], u1 = w[NEAR ? 2 * e1 : e1], v1 = w[NEAR ? 2 * e1 + 1 : 8 + e1];
      f11[i] = pack(c[e0] * u0, c[e1] * u1);
      f12[i] = pack(-sn[e0] * v0, -sn[e1] * v1);
      f22[i] = pack(c[e0] * v0, c[e1] * v1);
      f21[i] = pack(sn[e0] * u0, sn[e1] * u1);
    }
  }
  T* p1 = static_cast<T*>(a.q_out) + n * a.sqo_n + h * a.sqo_h + at.o1;
  T* p2 = p1 + (at.o2 - at.o1);
  auto step = [&](const Chunks& now) {
    F2 x1[4], x2[4];
    if constexpr (NEAR) {
      float xa[8], xb[8];
      unpack8<T>(now.a, xa);
      unpack8<T>(now.b, xb);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x1[i] = pack(xa[2 * i], xb[2 * i]);
        x2[i] = pack(xa[2 * i + 1], xb[2 * i + 1]);
      }
    } else {
      unpack8<T>(now.a, x1);
      unpack8<T>(now.b, x2);
    }
    float r = 1.f;
    if (a.q_weight) {
      auto squares = [&] {
        F2 s1 = mul2(x1[0], x1[0]), s2 = mul2(x2[0], x2[0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) {
          s1 = fma2(x1[i], x1[i], s1);
          s2 = fma2(x2[i], x2[i], s2);
        }
        float ss, st;
        unpack(add2(s1, s2), ss, st);
        ss += st;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        return ss;
      };
      float ss = squares(), eps = a.eps;
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        // squares that leave fp32 (elements of 2^60 and more, or none above 2^-40 and no eps to speak of): the head times 2^-70 or 2^80
        const float f = h >= a.H ? 1.f : ss > 0x1p120f ? 0x1p-70f : ss < 0x1p-80f && eps < 0x1p-60f ? 0x1p80f : 1.f;
        if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x1[i] = mul2(x1[i], pack(f, f));
            x2[i] = mul2(x2[i], pack(f, f));
          }
          ss = squares();
          eps = eps * f * f;
        }
      }
      r = rsqrtf(fmaf(ss, 1.f / D, eps));
    }
    const F2 r2 = pack(r, r);
    float y[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      F2 y1 = mul2(x1[i], f11[i]), y2 = mul2(x2[i], f22[i]);
      if (at.turns) {   // (else f12 and f21 are zeros, which an infinity would make NaN)
        y1 = fma2(x2[i], f12[i], y1);
        y2 = fma2(x1[i], f21[i], y2);
      }
      y1 = mul2(y1, r2);
      y2 = mul2(y2, r2);
      if constexpr (NEAR) {
        unpack(y1, y[2 * i], y[8 + 2 * i]);
        unpack(y2, y[2 * i + 1], y[8 + 2 * i + 1]);
      } else {
        unpack(y1, y[2 * i], y[2 * i + 1]);
        unpack(y2, y[8 + 2 * i], y[8 + 2 * i + 1]);
      }
    }
    if (h < a.H) {
      *reinterpret_cast<uint4*>(p1) = pack8<T>(y);
      *reinterpret_cast<uint4*>(p2) = pack8<T>(y + 8);
    }
    p1 += o_step;
    p2 += o_step;
    h += parts * HPW;
  };
  int left = ((a.H + HPW - 1) / HPW - part + parts - 1) / parts;
  while (left > 0) {   // two buffers in turn, neither of them moved
    load(c1);
    step(c0);
    if (--left == 0) break;
    load(c0);
    step(c1);
    --left;
  }
}

// The key and value heads of token n: items part, part + parts, ... of the keys', then the values'.
template <typename T, typename C, int D, bool NEAR>
__device__ __forceinline__ void append_keys_values(const Int4AppendArgs& a, int64_t n, int64_t pos, int seq, int part, int parts,
                                                   float (*s_row)[D]) {
  const Place<D> at(a.rotary, NEAR);
  constexpr int LANES = Place<D>::LANES, HPW = Place<D>::HPW;
  const int KVH = a.kv.KVH, run_lanes = a.kv.group / 16, runs = D / a.kv.group, items = (KVH + HPW - 1) / HPW, j = at.j;
  auto load = [&](int item) {
    Chunks x{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    const bool key = item < items;
    const int h = (key ? item : item - items) * HPW + at.sub;
    if (item < 2 * items && h < KVH) {
      const T* p = key ? static_cast<const T*>(a.k) + n * a.sk_n + h * a.sk_h : static_cast<const T*>(a.v) + n * a.sv_n + h * a.sv_h;
      x.a = *reinterpret_cast<const uint4*>(p + (key ? at.o1 : 16 * j));
      x.b = *reinterpret_cast<const uint4*>(p + (key ? at.o2 : 16 * j + 8));
    }
    return x;
  };
  Chunks next = load(part);
  if (pos >= static_cast<int64_t>(a.pages_per_seq) * a.kv.page_size) return;
  const int p = static_cast<int>(pos), pi = a.div.page(p), slot = a.div.slot(p, pi), tile_row = slot % kTileKeys;
  const int page = a.table[static_cast<int64_t>(seq) * a.ld_table + pi];
  if (page < 0 || page >= a.kv.num_pages) return;   // the whole warp
  uint8_t* const head0 = a.kv.pages + page * a.kv.sp_p + static_cast<int64_t>(slot / kTileKeys) * int4_tile_bytes(D, runs) + at.sub * a.kv.sp_h;
#pragma unroll 1
  for (int item = part; item < 2 * items; item += parts) {
    const Chunks now = next;
    next = load(item + parts);
    const bool key = item < items;
    const int h0 = (key ? item : item - items) * HPW;
    const bool on = h0 + at.sub < KVH;
    uint8_t* const tile = head0 + h0 * a.kv.sp_h;
    float x[16];
    uint32_t code[16];
    unpack8<T>(now.a, x);
    unpack8<T>(now.b, x + 8);
    if (key) {
      if (a.k_weight) {
        float w[16];
        load8(static_cast<const T*>(a.k_weight) + at.o1, w);
        load8(static_cast<const T*>(a.k_weight) + at.o2, w + 8);
        double ss = 0.0, st = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss = fma(static_cast<double>(x[e]), static_cast<double>(x[e]), ss);
          st = fma(static_cast<double>(x[8 + e]), static_cast<double>(x[8 + e]), st);
        }
        ss += st;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = static_cast<float>(rsqrt(ss / D + static_cast<double>(a.eps)));
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = __fmul_rn(__fmul_rn(x[e], r), w[e]);
      }
      if (at.turns) {
        float c[8], s[8];
        load8(static_cast<const C*>(a.cos) + pos * a.ld_cs + 8 * j, c);
        load8(static_cast<const C*>(a.sin) + pos * a.ld_cs + 8 * j, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) {   // (a, b) -> (a c - b s, b c + a s), every product and sum rounded by itself
          float &x1 = x[NEAR ? 2 * e : e], &x2 = x[NEAR ? 2 * e + 1 : 8 + e];
          const float y1 = __fsub_rn(__fmul_rn(x1, c[e]), __fmul_rn(x2, s[e]));
          x2 = __fadd_rn(__fmul_rn(x2, c[e]), __fmul_rn(x1, s[e]));
          x1 = y1;
        }
      }
      if (!NEAR && a.rotary > 0) {   // into neighbouring elements
        float* row = s_row[at.sub];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          *reinterpret_cast<float4*>(row + at.o1 + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
          *reinterpret_cast<float4*>(row + at.o2 + e) = make_float4(x[8 + e], x[9 + e], x[10 + e], x[11 + e]);
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 y = *reinterpret_cast<const float4*>(row + 16 * j + e);
          x[e] = y.x; x[e + 1] = y.y; x[e + 2] = y.z; x[e + 3] = y.w;
        }
        __syncwarp();
      }
    }
    const uint32_t sm = quantise<T>(x, run_lanes, code);
    if (key) {
      // lane j has step j: one byte of each half of the words (t', j / 2), t' = 0..3; the pair of lanes joins them
      uint32_t v[4];
      constexpr uint32_t kAbove = 0x4B400000u * (1u + (1u << 4) + (1u << 16) + (1u << 20));   // what lies above the codes
#pragma unroll
      for (int u = 0; u < 4; ++u)
        v[u] = code[4 * u] + (code[4 * u + 2] << 4) + (code[4 * u + 1] << 16) + (code[4 * u + 3] << 20) - kAbove;
      const bool upper = j & 1;
      const uint32_t r0 = __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[2], 1);
      const uint32_t r1 = __shfl_xor_sync(0xffffffffu, upper ? v[1] : v[3], 1);
      if (on) {
        uint8_t* row = tile + tile_row * (D / 2) + (upper ? 2 : 0) * (D / 8) + 4 * (j / 2);
        *reinterpret_cast<uint32_t*>(row) = upper ? r0 | v[2] << 8 : v[0] | r0 << 8;
        *reinterpret_cast<uint32_t*>(row + D / 8) = upper ? r1 | v[3] << 8 : v[1] | r1 << 8;
        if (j % run_lanes == 0)
          *reinterpret_cast<uint32_t*>(tile + int4_ks_off(D) + (tile_row * runs + j / run_lanes) * 4) = sm;
      }
    } else if (on) {
      uint8_t* b = tile + int4_v_off(D) + (j / 4) * 512 + ((tile_row % 8) / 2) * 16 + (j % 4) * 4 + (tile_row & 1) * 2 + tile_row / 8;
#pragma unroll
      for (int g = 0; g < 8; ++g) b[g * 64] = static_cast<uint8_t>(code[g] + (code[g + 8] << 4));
      if (j % run_lanes == 0)
        *reinterpret_cast<uint32_t*>(tile + int4_vs_off(D, runs) + (tile_row * runs + j / run_lanes) * 4) = sm;
    }
  }
}

// T: cache and activation dtype, C: the tables' type, NEAR: pairs of neighbouring elements. Of a token's gridDim.y warps (in
// blocks of their own) the first q_parts take the queries.
template <typename T, typename C, int D, bool NEAR>
__global__ void __launch_bounds__(kWarps * 32, 6) int4_append_kernel(const __grid_constant__ Int4AppendArgs a) {
  __shared__ __align__(16) float s_row[kWarps][Place<D>::HPW][D];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, part = blockIdx.y;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (n >= a.N) return;
  const int64_t pos = a.positions[n];
  const int seq = a.seq_ids ? a.seq_ids[n] : sequence_of(static_cast<int>(n), a.per_seq, a.per_inv);
  if (seq < 0 || seq >= a.B || pos < 0 || pos >= a.limit) return;   // padding
  if (part < a.q_parts) append_queries<T, C, D, NEAR>(a, n, pos, part, a.q_parts);
  else append_keys_values<T, C, D, NEAR>(a, n, pos, seq, part - a.q_parts, gridDim.y - a.q_parts, s_row[warp]);
}

struct Int4ReadArgs {
  const int64_t* positions;
  const int32_t* seq_ids;
  const int32_t* table; int64_t ld_table;
  void* k; int64_t sk_n, sk_h;
  void* v; int64_t sv_n, sv_h;
  b2d_int4_kv kv;
  PageDiv div;
  int N, B, per_seq, pages_per_seq;
  uint32_t per_inv;
};

// Ordinary loads for what an earlier kernel of the stream may have written: this one may be resident, behind other dependent
// launches, before that kernel begins, and the read-only path does not promise to see what is written meanwhile.
__device__ __forceinline__ uint32_t load32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }

// The inverse, lane for lane: 16 neighbouring elements of a head from the step's bytes. O: output type, WIDE: stores of 32 bytes. A warp has a token. A value
// word holds four positions' bytes; where the 16 tokens of a tile lie together in the call (their 16 warps see that alike),
// each of these warps takes four positions of the keys or of the values, and a quarter of the loads is left.
template <typename T, typename O, bool WIDE>
__device__ __forceinline__ void put_values(O* o, uint32_t sm, const uint32_t (&code)[16]) {   // codes in the words' low bits
  const float2 f = unpack_sm<T>(sm);
  const F2 s2 = pack(f.x, f.x), m2 = pack(f.y, f.y), base2 = pack(-8388608.f, -8388608.f);
  float x[16];
#pragma unroll
  for (int e = 0; e < 16; e += 2) {   // a code behind 2^23 in a float's bits
    const F2 c = pack(__uint_as_float((code[e] & 15u) | 0x4B000000u), __uint_as_float((code[e + 1] & 15u) | 0x4B000000u));
    unpack(fma2(s2, add2(c, base2), m2), x[e], x[e + 1]);
  }
  uint32_t w[sizeof(O) * 4];
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(x[e]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = Dt<O>::pack2(x[2 * i], x[2 * i + 1]);
  }
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(O)) * 4; i += 8) {
    uint32_t* const to = reinterpret_cast<uint32_t*>(o) + i;
    if constexpr (WIDE) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(to), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]),
                   "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7]) : "memory");
    } else {
      reinterpret_cast<uint4*>(to)[0] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      reinterpret_cast<uint4*>(to)[1] = make_uint4(w[i + 4], w[i + 5], w[i + 6], w[i + 7]);
    }
  }
}
template <typename T, typename O, bool WIDE>
__device__ __forceinline__ void put_key(O* o, uint32_t sm, const uint32_t (&w)[4], int j) {
  uint32_t code[16];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint32_t x = w[u] >> 8 * (j & 1);
    code[4 * u] = x;
    code[4 * u + 1] = x >> 16;
    code[4 * u + 2] = x >> 4;
    code[4 * u + 3] = x >> 20;
  }
  put_values<T, O, WIDE>(o, sm, code);
}
template <typename T, typename O, bool WIDE>
__device__ __forceinline__ void put_value(O* o, uint32_t sm, const uint32_t (&w)[8], int shift) {
  uint32_t code[16];
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    code[g] = w[g] >> shift;
    code[g + 8] = w[g] >> (shift + 4);
  }
  put_values<T, O, WIDE>(o, sm, code);
}

template <typename T, typename O, int D, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32) int4_read_kernel(const __grid_constant__ Int4ReadArgs a) {
  constexpr int LANES = D / 16, HPW = 32 / LANES;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = lane % LANES, sub = lane / LANES;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (n >= a.N) return;
  const int64_t pos = a.positions[n];
  const int seq = a.seq_ids ? a.seq_ids[n] : sequence_of(static_cast<int>(n), a.per_seq, a.per_inv);
  if (seq < 0 || seq >= a.B || pos < 0 || pos >= static_cast<int64_t>(a.pages_per_seq) * a.kv.page_size) return;
  const int KVH = a.kv.KVH, run_lanes = a.kv.group / 16, runs = D / a.kv.group;
  const int items = (KVH + HPW - 1) / HPW;
  const int p = static_cast<int>(pos), pi = a.div.page(p), slot = a.div.slot(p, pi), row = slot % kTileKeys;
  const int page = a.table[static_cast<int64_t>(seq) * a.ld_table + pi];
  const bool there = page >= 0 && page < a.kv.num_pages;
  const uint8_t* const tile0 = a.kv.pages + (there ? page * a.kv.sp_p + static_cast<int64_t>(slot / kTileKeys) * int4_tile_bytes(D, runs) : 0);
  bool whole = gridDim.y == 1 && n >= row && n - row + kTileKeys <= a.N;
  if (whole) {
    const int64_t other = n - row + (lane & 15);
    whole = a.positions[other] == pos - row + (lane & 15) &&
            (a.seq_ids ? a.seq_ids[other] : sequence_of(static_cast<int>(other), a.per_seq, a.per_inv)) == seq;
    whole = __all_sync(0xffffffffu, whole);
  }
  if (whole) {
    const bool values = row & 4;
    const int quarter = row & 3;
    if (!(values ? a.v : a.k)) return;
    const int64_t sn = values ? a.sv_n : a.sk_n, sh = values ? a.sv_h : a.sk_h;
    O* const out0 = static_cast<O*>(values ? a.v : a.k) + (n - row) * sn + 16 * j;
    for (int item = row >> 3; item < items; item += 2) {
      const int h = item * HPW + sub;
      if (h >= KVH) continue;
      const uint8_t* const tile = tile0 + h * a.kv.sp_h;
      O* const out = out0 + h * sh;
      uint32_t sm[4] = {0, 0, 0, 0};
      if (values) {   // the bytes of a word: rows 2 t, 2 t + 8, 2 t + 1, 2 t + 9
        uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const int row0 = 2 * quarter;
        if (there) {
#pragma unroll
          for (int g = 0; g < 8; ++g)
            w[g] = load32(tile + int4_v_off(D) + (j / 4) * 512 + (g * 4 + quarter) * 16 + (j % 4) * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sm[i] = load32(tile + int4_vs_off(D, runs) + ((row0 + (i >> 1) + 8 * (i & 1)) * runs + j / run_lanes) * 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) put_value<T, O, WIDE>(out + (row0 + (i >> 1) + 8 * (i & 1)) * sn, sm[i], w, 8 * i);
      } else {
        uint32_t w[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) w[i][u] = 0;
        if (there) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sm[i] = load32(tile + int4_ks_off(D) + ((4 * quarter + i) * runs + j / run_lanes) * 4);
#pragma unroll
            for (int u = 0; u < 4; ++u)
              w[i][u] = load32(tile + (4 * quarter + i) * (D / 2) + 4 * (j / 2) + u * (D / 8));
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) put_key<T, O, WIDE>(out + (4 * quarter + i) * sn, sm[i], w[i], j);
      }
    }
    return;
  }
  for (int item = blockIdx.y; item < items; item += gridDim.y) {
    const int h = item * HPW + sub;
    if (h >= KVH) continue;
    const uint8_t* const tile = tile0 + h * a.kv.sp_h;
    uint32_t kw[4], vw[8], ksm = 0, vsm = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) kw[u] = vw[u] = vw[4 + u] = 0;
    if (there) {   // every load under way before the first is used
      if (a.k) {
        ksm = load32(tile + int4_ks_off(D) + (row * runs + j / run_lanes) * 4);
        const uint8_t* b = tile + row * (D / 2) + 4 * (j / 2);
#pragma unroll
        for (int u = 0; u < 4; ++u) kw[u] = load32(b + u * (D / 8));
      }
      if (a.v) {
        vsm = load32(tile + int4_vs_off(D, runs) + (row * runs + j / run_lanes) * 4);
        const uint8_t* b = tile + int4_v_off(D) + (j / 4) * 512 + ((row % 8) / 2) * 16 + (j % 4) * 4 + (row & 1) * 2 + row / 8;
#pragma unroll
        for (int g = 0; g < 8; ++g) vw[g] = b[g * 64];
      }
    }
    if (a.k) put_key<T, O, WIDE>(static_cast<O*>(a.k) + n * a.sk_n + h * a.sk_h + 16 * j, ksm, kw, j);
    if (a.v) put_value<T, O, WIDE>(static_cast<O*>(a.v) + n * a.sv_n + h * a.sv_h + 16 * j, vsm, vw, 0);
  }
}

// Warps a token of a share of the work, at most one per item, so that eight of an SM have some: 64 x 5 tokens 4.2 us (one warp a token
// 5.6, 24 an SM 5.2), 8 x 100 7.0 (8.2, 7.9), one token 2.7 (4.6, 2.6), 8 x 1021 48.9 (49.0, 48.9); reading 300 tokens 2.7 (3.3, 2.7).
int warps_per_token(int64_t N, int items, int sm) {
  const int64_t parts = (static_cast<int64_t>(sm) * 8 + N - 1) / N;
  return static_cast<int>(parts < items ? parts : items);
}

template <typename T, typename C, int D>
int launch_append(Int4AppendArgs& a, bool near, int sm, bool pdl, cudaStream_t s) {
  constexpr int HPW = Place<D>::HPW;
  a.q_parts = a.q && a.H > 0 ? warps_per_token(a.N, (a.H + HPW - 1) / HPW, sm) : 0;
  const dim3 grid((a.N + kWarps - 1) / kWarps, a.q_parts + warps_per_token(a.N, 2 * ((a.kv.KVH + HPW - 1) / HPW), sm));
  if (grid.y > 65535) return B2D_ERR_SHAPE;
  if (near) return launch_kernel(int4_append_kernel<T, C, D, true>, grid, dim3(kWarps * 32), 0, s, pdl, a);
  return launch_kernel(int4_append_kernel<T, C, D, false>, grid, dim3(kWarps * 32), 0, s, pdl, a);
}
template <typename T, typename O, int D>
int launch_read(const Int4ReadArgs& a, int sm, bool pdl, cudaStream_t s) {
  constexpr int HPW = 512 / D;
  const int items = (a.kv.KVH + HPW - 1) / HPW;
  const dim3 grid((a.N + kWarps - 1) / kWarps, warps_per_token(a.N, items, sm));
  // 32 bytes a store where all rows begin at multiples of 32 (8 x 4001 tokens 35.7 us, in halves 38.5)
  const bool wide = aligned(a.k, 32) && aligned(a.v, 32) && (a.sk_n | a.sk_h | a.sv_n | a.sv_h) * sizeof(O) % 32 == 0;
  if (wide) return launch_kernel(int4_read_kernel<T, O, D, true>, grid, dim3(kWarps * 32), 0, s, pdl, a);
  return launch_kernel(int4_read_kernel<T, O, D, false>, grid, dim3(kWarps * 32), 0, s, pdl, a);
}

int check_tokens(const b2d_int4_kv* kv, const int32_t* seq_ids, int N, int B, int64_t ld_table, int pages_per_seq) {
  if (B == 0 || (!seq_ids && N % B != 0) || ld_table < 0) return B2D_ERR_SHAPE;
  if (static_cast<int64_t>(pages_per_seq) * kv->page_size > (int64_t(1) << 31) - 1024) return B2D_ERR_SHAPE;
  return B2D_OK;
}

}  // namespace
}  // namespace b2d

using namespace b2d;

extern "C" size_t b2d_int4_page_bytes(int page_size, int D, int group) {
  return int4_sizes(page_size, D, group) ? static_cast<size_t>(page_size / kTileKeys) * int4_tile_bytes(D, D / group) : 0;
}

extern "C" int b2d_int4_append(const b2d_int4_kv* kv, const void* q, int64_t sq_n, int64_t sq_h, const void* k, int64_t sk_n,
                               int64_t sk_h, const void* v, int64_t sv_n, int64_t sv_h, const int64_t* positions,
                               const int32_t* seq_ids, const int32_t* page_table, int64_t ld_table, int pages_per_seq, int B,
                               const void* cos, const void* sin, int64_t ld_cs, int S_max, int cs_dtype, int rotary_dim,
                               int interleaved, const void* q_weight, const void* k_weight, float eps, void* q_out,
                               int64_t sqo_n, int64_t sqo_h, int N, int H, int flags, void* stream) {
  int st;
  if ((st = check_int4_kv(kv)) != B2D_OK) return st;
  if (N < 0 || H < 0 || B < 0 || pages_per_seq < 0 || (cos && (S_max < 0 || rotary_dim < 0))) return B2D_ERR_ARG;
  if (cos && cs_dtype != kv->dtype && cs_dtype != B2D_F32) return B2D_ERR_DTYPE;
  if (q && (H % kv->KVH != 0 || H > 65535)) return B2D_ERR_SHAPE;
  if (cos && (rotary_dim % 16 != 0 || rotary_dim < 16 || rotary_dim > kv->D)) return B2D_ERR_SHAPE;
  if (N == 0) return B2D_OK;
  if ((st = check_tokens(kv, seq_ids, N, B, ld_table, pages_per_seq)) != B2D_OK) return st;
  if (!k || !v || !positions || (!page_table && pages_per_seq > 0) || !cos != !sin || (q && !q_out) || (cos && ld_cs < 0)) return B2D_ERR_ARG;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) || !aligned(cos, 16) || !aligned(sin, 16) ||
      !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(positions, 8) || !aligned(page_table, 4) ||
      !aligned(seq_ids, 4) || (sk_n | sk_h | sv_n | sv_h) % 8 || (q && (sq_n | sq_h | sqo_n | sqo_h) % 8) ||
      (cos && ld_cs % (cs_dtype == B2D_F32 ? 4 : 8)))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  if ((st = device_info(&di)) != B2D_OK) return st;
  Int4AppendArgs a{q, sq_n, sq_h, k, sk_n, sk_h, v, sv_n, sv_h, positions, seq_ids, page_table, ld_table, cos, sin, ld_cs,
                   q_weight, k_weight, eps, q_out, sqo_n, sqo_h, *kv, page_div(kv->page_size), N, H, B, seq_ids ? 1 : N / B,
                   pages_per_seq, cos ? rotary_dim : 0, 0, inverse_of(seq_ids ? 1 : N / B), cos ? S_max : INT64_MAX};
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0, f32 = cos && cs_dtype == B2D_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sm = di.sm_count;
  const bool near = cos && interleaved;
  if (kv->dtype == B2D_F16) {
    if (kv->D == 64) return f32 ? launch_append<__half, float, 64>(a, near, sm, pdl, s) : launch_append<__half, __half, 64>(a, near, sm, pdl, s);
    return f32 ? launch_append<__half, float, 128>(a, near, sm, pdl, s) : launch_append<__half, __half, 128>(a, near, sm, pdl, s);
  }
  if (kv->D == 64)
    return f32 ? launch_append<__nv_bfloat16, float, 64>(a, near, sm, pdl, s) : launch_append<__nv_bfloat16, __nv_bfloat16, 64>(a, near, sm, pdl, s);
  return f32 ? launch_append<__nv_bfloat16, float, 128>(a, near, sm, pdl, s) : launch_append<__nv_bfloat16, __nv_bfloat16, 128>(a, near, sm, pdl, s);
}

extern "C" int b2d_int4_read(const b2d_int4_kv* kv, const int64_t* positions, const int32_t* seq_ids, const int32_t* page_table,
                             int64_t ld_table, int pages_per_seq, int B, void* k_out, int64_t sk_n, int64_t sk_h, void* v_out,
                             int64_t sv_n, int64_t sv_h, int out_dtype, int N, int flags, void* stream) {
  int st;
  if ((st = check_int4_kv(kv)) != B2D_OK) return st;
  if (N < 0 || B < 0 || pages_per_seq < 0) return B2D_ERR_ARG;
  if (out_dtype != kv->dtype && out_dtype != B2D_F32) return B2D_ERR_DTYPE;
  if (N == 0 || (!k_out && !v_out)) return B2D_OK;
  if ((st = check_tokens(kv, seq_ids, N, B, ld_table, pages_per_seq)) != B2D_OK) return st;
  if (!positions || (!page_table && pages_per_seq > 0)) return B2D_ERR_ARG;
  if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(positions, 8) || !aligned(page_table, 4) || !aligned(seq_ids, 4) ||
      (k_out && (sk_n | sk_h) % 8) || (v_out && (sv_n | sv_h) % 8))
    return B2D_ERR_ALIGN;
  DeviceInfo di;
  if ((st = device_info(&di)) != B2D_OK) return st;
  Int4ReadArgs a{positions, seq_ids, page_table, ld_table, k_out, sk_n, sk_h, v_out, sv_n, sv_h, *kv,
                 page_div(kv->page_size), N, B, seq_ids ? 1 : N / B, pages_per_seq, inverse_of(seq_ids ? 1 : N / B)};
  const bool pdl = (flags & B2D_LAUNCH_PDL) != 0, f32 = out_dtype == B2D_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sm = di.sm_count;
  if (kv->dtype == B2D_F16) {
    if (kv->D == 64) return f32 ? launch_read<__half, float, 64>(a, sm, pdl, s) : launch_read<__half, __half, 64>(a, sm, pdl, s);
    return f32 ? launch_read<__half, float, 128>(a, sm, pdl, s) : launch_read<__half, __half, 128>(a, sm, pdl, s);
  }
  if (kv->D == 64) return f32 ? launch_read<__nv_bfloat16, float, 64>(a, sm, pdl, s) : launch_read<__nv_bfloat16, __nv_bfloat16, 64>(a, sm, pdl, s);
  return f32 ? launch_read<__nv_bfloat16, float, 128>(a, sm, pdl, s) : launch_read<__nv_bfloat16, __nv_bfloat16, 128>(a, sm, pdl, s);
}
