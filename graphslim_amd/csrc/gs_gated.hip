// Gated feed-forward block:  g = x Wg^T, u = x Wu^T, h = act(g) u,  and its backward pass
//   du = dh act(g), dg = dh u act'(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x.
// Every product C(m, n) = sum_k A(m, k) B(n, k) runs on the 16-bit matrix pipe with fp32 accumulation; an operand may have k contiguous
// in memory (x and the weights in the forward pass) or its other index (the weights in dx, both operands of dW): tiles of the
// latter are transposed on their way from LDS to the registers.  16-bit operands enter as they are; an fp32 operand is the exact sum of three bf16 parts
// (x = h + m + l, 8 + 8 + 8 significant bits), and six products of parts make one product: what they leave out is below 2^-23 of it.
// (Parts have bf16's smallest step, 2^-133: a value is represented to 2^-134 or to 24 bits, whichever is coarser.)
// dg and du of 16-bit operands are computed in fp32 and enter as two bf16 parts (17 bits and fp32's range).  Rounded to the operands'
// type they would cost the gradients a second rounding as large as that of the result, and in fp16 dh u act'(g) can lie outside of the
// type though the gradients do not.  The parts lie one behind the other along k, against the same weights or x a second time:
//   bf16:  dg W = lo W + hi W;      fp16:  W = V + R, bf16 parts that hold all of its 11 bits, dg W = lo V + hi R + hi V
// A rounded bf16 leaves at most 2^-8 of a value, the second part's rounding 2^-9 of that: dg is held to 2^-17.  lo R, at most 2^-8 2^-8 of the
// product, is left out, so fp16's products are off by up to 2^-16 + 2^-17 of their terms; the result's own rounding is 2^-11.
// The parts of fp32 operands, and [dg | du], are laid out in the caller's scratch first, rows padded with zeros to a multiple of 64;
// so are 16-bit operands whose rows do not consist of whole, aligned chunks of 16 bytes, unless it is cheaper to read them as they are.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gs_types.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* gbl_ptr;

constexpr int GF_PAD = 64;   // rows of laid-out operands are multiples of this many elements

constexpr long GF_MAX_THREADS = 0xffffffffL;   // of a launch
constexpr long GF_MAX_BLOCKS = 0xffffffL;      // of 256 threads

inline long gf_up(long n) { return (n + GF_PAD - 1) / GF_PAD * GF_PAD; }

// ---- activations: the value and its derivative ---------------------------------------------------------------------------------
// Both tails keep their digits: Phi(g) = erfc(-g / sqrt 2) / 2 (1 + erf(g / sqrt 2) has none left below -5), and the sigmoid and what it
// leaves of 1 come from e^-|g|, neither by a difference.  16-bit types take the short exponential, off by 2^-23 |g| of itself (8192 x 2048 x
// 8192 bf16, silu: 470 us where the other one takes 493).
template <int T, int ACT>
__device__ __forceinline__ void gf_act(float g, float& a, float& da) {
  if constexpr (ACT == GS_ACT_RELU) {
    a = g > 0.f ? g : (g == g ? 0.f : g);
    da = g > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == GS_ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * g), x = -0.5f * g * g;
    a = g * cdf;
    da = cdf + g * (T == GS_TYPE_F32 ? expf(x) : __expf(x)) * 0.39894228040143268f;
  } else {
    const float x = -fabsf(g), e = T == GS_TYPE_F32 ? expf(x) : __expf(x), one = 1.f / (1.f + e), zero = e * one;
    const float sig = g >= 0.f ? one : zero, rest = g >= 0.f ? zero : one;
    a = ACT == GS_ACT_SILU ? g * sig : sig;
    da = ACT == GS_ACT_SILU ? sig * (1.f + g * rest) : sig * rest;
  }
}

// f(activation as a constant); act is the same for a whole launch, and the choice is made once, outside of all loops
template <typename Fn>
__device__ __forceinline__ void gf_with_act(int act, Fn f) {
  switch (act) {
    case GS_ACT_SILU: f(std::integral_constant<int, GS_ACT_SILU>{}); break;
    case GS_ACT_GELU: f(std::integral_constant<int, GS_ACT_GELU>{}); break;
    case GS_ACT_RELU: f(std::integral_constant<int, GS_ACT_RELU>{}); break;
    default: f(std::integral_constant<int, GS_ACT_SIGMOID>{}); break;
  }
}

// ---- the three bf16 parts of an fp32, each the rounded remainder of those before ------------------------------------------------
__device__ __forceinline__ void gf_split(float w, __bf16& h, __bf16& m, __bf16& l) {
  h = (__bf16)w;
  float hf = (float)h;
  if (!(fabsf(hf) < INFINITY)) {   // not finite (nothing is left over), or finite and rounded up beyond the largest bf16: cut instead
    hf = fabsf(w) < INFINITY ? __uint_as_float(__float_as_uint(w) & 0xffff0000u) : w;
    h = (__bf16)hf;
    if (!(fabsf(w) < INFINITY)) {
      m = (__bf16)0.f;
      l = (__bf16)0.f;
      return;
    }
  }
  const float r = w - hf;
  m = (__bf16)r;
  l = (__bf16)(r - (float)m);
}

template <int T, int PL>
struct GfPlane;   // the 16-bit type the operand is multiplied in
template <>
struct GfPlane<GS_TYPE_F16, 1> {
  typedef _Float16 type;
};
template <>
struct GfPlane<GS_TYPE_BF16, 1> {
  typedef __bf16 type;
};
template <>
struct GfPlane<GS_TYPE_F32, 3> {
  typedef __bf16 type;
};
template <>
struct GfPlane<GS_TYPE_F16, 2> {   // 2: dg, du of 16-bit types
  typedef __bf16 type;
};
template <>
struct GfPlane<GS_TYPE_BF16, 2> {
  typedef __bf16 type;
};

// stretches of k that a product of such parts has
constexpr int gf_stretches(int type, int pl) { return pl != 2 ? 1 : (type == GS_TYPE_F16 ? 3 : 2); }

template <int T, int PL, typename P>
__device__ __forceinline__ void gf_put8(const float* v, P* __restrict__ o, long plane) {
  typedef P V __attribute__((ext_vector_type(8)));
  if constexpr (PL == 1) {
    V r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (P)v[j];
    *(V*)o = r;
  } else {
    V h, m, l;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      __bf16 a, b, c;
      gf_split(v[j], a, b, c);
      h[j] = a;
      m[j] = b;
      l[j] = c;
    }
    *(V*)o = h;
    *(V*)(o + plane) = m;
    if constexpr (PL == 3) *(V*)(o + 2 * plane) = l;
  }
}

// ---- operand layout -------------------------------------------------------------------------------------------------------------
// Three matrices [R][C] as [PL][Rp][Cp], zeros behind the columns and rows
struct GatedPack {
  const void* in[3];
  void* out[3];
  long ld[3], R[3], Rp[3], first[3];   // first: the matrix's first block
  long C, Cp;
};

template <int T, int PL>
__global__ __launch_bounds__(256) void gs_gated_pack_kernel(GatedPack a) {
  typedef typename GsElt<T>::type E;
  typedef typename GfPlane<T, PL>::type P;
  const int w = (long)blockIdx.x >= a.first[2] ? 2 : ((long)blockIdx.x >= a.first[1] ? 1 : 0);
  const unsigned per = (unsigned)(a.Cp / 8), i = (blockIdx.x - (unsigned)a.first[w]) * 256u + threadIdx.x, q = i / per;
  const long r = q, c = (long)(i - q * per) * 8;
  if (r >= a.Rp[w]) return;
  float v[8];
  if (c < a.C && r < a.R[w]) {
    gs_load<E, 8>((const E*)a.in[w] + r * a.ld[w] + c, a.C - c, 0.f, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
  }
  gf_put8<T, PL>(v, (P*)a.out[w] + r * a.Cp + c, a.Rp[w] * a.Cp);
}

// dg, du from dh and the saved g, u: [PL][Mp][2 Fp], columns [0, Fp) dg, [Fp, 2 Fp) du, zeros in the padding of both.  Bound by HBM
// (8192 x 8192 bf16: 134 + 537 MB read, 537 MB written), so `saved`, which nobody reads again, passes the caches by.
template <int T, int PL>
__global__ __launch_bounds__(256) void gs_gated_slopes_kernel(int act, const typename GsElt<T>::type* __restrict__ dh, long lddh,
                                                              const float* __restrict__ saved, long M, long F,
                                                              typename GfPlane<T, PL>::type* __restrict__ out, long Mp, long Fp, long plane) {
  typedef typename GfPlane<T, PL>::type P;
  const unsigned per = (unsigned)(Fp / 8), i = blockIdx.x * 256u + threadIdx.x, q = i / per;
  const long m = q, f = (long)(i - q * per) * 8;
  if (m >= Mp) return;
  float dg[8], du[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) dg[j] = du[j] = 0.f;
  if (m < M && f < F) {
    float d[8], g[8], u[8];
    gs_load<typename GsElt<T>::type, 8>(dh + m * lddh + f, F - f, 0.f, d);
    if (f + 8 <= F) {
      const auto x = gs_load_past<float, 8>(saved + m * F + f), y = gs_load_past<float, 8>(saved + (M + m) * F + f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] = x[j];
        u[j] = y[j];
      }
    } else {
      gs_load<float, 8>(saved + m * F + f, F - f, 0.f, g);
      gs_load<float, 8>(saved + (M + m) * F + f, F - f, 0.f, u);
    }
    gf_with_act(act, [&](auto ac) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float a, da;
        gf_act<T, decltype(ac)::value>(g[j], a, da);
        du[j] = d[j] * a;
        dg[j] = d[j] * u[j] * da;
      }
    });
  }
  P* o = out + m * 2 * Fp + f;
  gf_put8<T, PL>(dg, o, plane);
  gf_put8<T, PL>(du, o + Fp, plane);
}

// ---- few rows -------------------------------------------------------------------------------------------------------------------
// For a few rows (eight at a time) the weights are all there is to read, and the vector units keep up: a wave takes RF rows of both weights,
// its lanes 16 bytes each of a stretch of k, and adds across the lanes at the end.  Exact fp32 products for every type.  Bound by the
// reading of the weights: one row, 2048 x 8192 bf16, 67 MB, 11.6 us = 5.8 TB/s (from the 256 MB cache when repeated, as here).
struct GatedRows {
  const void *x, *wg, *wu;
  long ldx, ldw, M, D, F, ldh;
  void* h;
  float* saved;
  int act;
};

template <int T, int MB, int RF>
__global__ __launch_bounds__(256) void gs_gated_rows_kernel(GatedRows q) {
  typedef typename GsElt<T>::type E;
  constexpr int N = 16 / sizeof(E);
  typedef typename GsVec<E, N>::type V;
  const int lane = threadIdx.x & 63;
  const long f0 = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * RF, m0 = (long)blockIdx.y * MB;
  if (f0 >= q.F) return;
  const E* w[2 * RF];
#pragma unroll
  for (int r = 0; r < RF; ++r) {
    const long f = min(f0 + r, q.F - 1);
    w[r] = (const E*)q.wg + f * q.ldw;
    w[RF + r] = (const E*)q.wu + f * q.ldw;
  }
  const E* x[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) x[m] = (const E*)q.x + min(m0 + m, q.M - 1) * q.ldx;
  float acc[MB][2 * RF];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int r = 0; r < 2 * RF; ++r) acc[m][r] = 0.f;
  long k = (long)lane * N;
#pragma unroll 2
  for (; k + N <= q.D; k += 64 * N) {
    V v[2 * RF], y[MB];
#pragma unroll
    for (int r = 0; r < 2 * RF; ++r) v[r] = *(const V*)(w[r] + k);
#pragma unroll
    for (int m = 0; m < MB; ++m) y[m] = *(const V*)(x[m] + k);
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float xe = (float)y[m][e];
#pragma unroll
        for (int r = 0; r < 2 * RF; ++r) acc[m][r] = fmaf((float)v[r][e], xe, acc[m][r]);
      }
  }
  if (k < q.D) {             // one lane has the end of a row whose length is no multiple of N
    for (long e = k; e < q.D; ++e)
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int r = 0; r < 2 * RF; ++r) acc[m][r] = fmaf((float)w[r][e], (float)x[m][e], acc[m][r]);
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int r = 0; r < 2 * RF; ++r) acc[m][r] = gs_wave_sum(acc[m][r]);
  float g = 0.f, u = 0.f;    // a lane finishes one result
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int r = 0; r < RF; ++r)
      if (lane == m * RF + r) {
        g = acc[m][r];
        u = acc[m][RF + r];
      }
  const long m = m0 + lane / RF, f = f0 + lane % RF;
  if (lane >= MB * RF || m >= q.M || f >= q.F) return;
  gf_with_act(q.act, [&](auto ac) {
    float a, da;
    gf_act<T, decltype(ac)::value>(g, a, da);
    ((E*)q.h)[m * q.ldh + f] = (E)(a * u);
  });
  if (q.saved) {
    q.saved[m * q.F + f] = g;
    q.saved[(q.M + m) * q.F + f] = u;
  }
}

// ---- the product ----------------------------------------------------------------------------------------------------------------
struct GatedGemm {
  const void* A;        // [PL] planes; k contiguous: rows of m, else rows of k
  long lda, plane_a;
  const void* B[2];     // gated: gate and up projection; n contiguous: rows of k below `kb` in the first, the others in the second
  long ldb, plane_b;
  long M, N, K;         // K a multiple of 64, all stretches together
  long stretch;         // of k; a multiple of 64
  long k_end;           // k contiguous in both: elements that a row of k has (K or less; RAW: 8 or more)
  long bcols;           // n contiguous: columns that rows of B have (a multiple of 8, N or more)
  long kb, brows;       // n contiguous: rows that B[0] stands for (a multiple of 64), and rows that each of B has; behind them A is 0
  void* C[2];           // plain form: rows [0, rows) go to C[0], rows [rows1, rows1 + rows) to C[1], others nowhere
  long ldc, rows, rows1;
  float* saved;         // gated form: g [M][N] and u [M][N], or null
  int act;
  float* part;          // k cut into slices: slice z writes its sums to part + z * slice ([M][N]; gated: two of them), nothing to C
  long slice;
  int gx;               // tiles of m
  long kslice;          // of k per slice, a multiple of BK
};

// row m of a plain product, or null if it is kept nowhere
template <typename E>
__device__ __forceinline__ E* gf_row(const GatedGemm& q, long m) {
  if (m < q.rows) return (E*)q.C[0] + m * q.ldc;
  return m >= q.rows1 && m < q.rows1 + q.rows ? (E*)q.C[1] + (m - q.rows1) * q.ldc : nullptr;
}

__device__ __forceinline__ f32x4 gf_mfma(h16x8 a, h16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 gf_mfma(b16x8 a, b16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Eight fp16 as bf16: what a bf16 holds of them, or the 3 bits that are left.  In pairs, since one instruction rounds two; what is left is
// exact, so a byte permutation packs it.
template <bool REST>
__device__ __forceinline__ b16x8 gf_part(b16x8 bits) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
  const h16x8 w = __builtin_bit_cast(h16x8, bits);
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const f32x2 v = {(float)w[e], (float)w[e + 1]};
    const unsigned first = __builtin_bit_cast(unsigned, __builtin_convertvector(v, b16x2));
    if (REST) {
      const float lo = v[0] - __uint_as_float(first << 16), hi = v[1] - __uint_as_float(first & 0xffff0000u);
      r[e / 2] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
    } else {
      r[e / 2] = first;
    }
    asm volatile("" : "+v"(r[e / 2]));   // (pair after pair: all at once would take more registers than there are)
  }
  return __builtin_bit_cast(b16x8, r);
}

template <int N, typename Fn>
__device__ __forceinline__ void gf_static_for(Fn f) {
  if constexpr (N > 0) {
    gf_static_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

template <typename P>
struct GfFrag;
template <>
struct GfFrag<_Float16> {
  typedef h16x8 type;
};
template <>
struct GfFrag<__bf16> {
  typedef b16x8 type;
};

// An operand's tile in LDS, in 16-byte chunks; chunk c of row r lies at place c ^ s(r) of its row.  The permutation is made on the
// global side, since the direct-to-LDS load writes 64 consecutive chunks.
//   k contiguous: rows of BK elements; the eight lanes that a 16-byte LDS read serves at once (eight rows, one chunk) fall on all banks.
//   else:         BK rows of W elements; ds_read_b64_tr_b16 reads four rows by 16 elements per 16 lanes and hands lane i the four
//                 values of element i; rows that one read serves at once (r & 3, and the next group's r >> 3) fall on different banks.
template <bool TALL, int BK>
__device__ __forceinline__ int gf_swz(int r) {
  if (TALL) return ((r & 3) | ((r >> 3) & 1) << 2) << 1;
  return BK == 64 ? (r & 7) : ((r >> 1) & 3);
}

template <typename Frag, int BK, typename P>
__device__ __forceinline__ Frag gf_frag(const P* tile, int row0, int ks, int lane) {
  const int r = row0 + (lane & 15), c = ks * 4 + (lane >> 4);
  return *(const Frag*)(tile + (r * (BK / 8) + (c ^ gf_swz<false, BK>(r))) * 8);
}

// LDS byte address of a lane's first four values of fragment 0 of a tile whose rows are k; fragment i lies at that ^ (i << 5) (the
// permutation flips the same bits), four rows of k further at + 8 W, 32 at + 64 W.
template <int W, int BK, typename P>
__device__ __forceinline__ unsigned gf_tr_addr(const P* tile, int row0, int lane) {
  const int k = (lane >> 4) * 8 + ((lane >> 2) & 3), c = row0 / 8 + ((lane & 3) >> 1);
  return (unsigned)(size_t)(lds_ptr)(tile + (k * (W / 8) + (c ^ gf_swz<true, BK>(k))) * 8 + (lane & 1) * 4);
}

// N (2 or 4) fragments from `first` on.  In assembly, with its own wait: the compiler lets no transposing read of its own pass a
// direct-to-LDS load that is under way, though the two are on different buffers here.
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <int OFF, int W, typename Frag>
__device__ __forceinline__ void gf_tr_read4(unsigned addr, int first, Frag* x) {
  const unsigned a0 = addr ^ (first << 5), a1 = addr ^ ((first + 1) << 5), a2 = addr ^ ((first + 2) << 5), a3 = addr ^ ((first + 3) << 5);
  i32x2 l0, h0, l1, h1, l2, h2, l3, h3;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
      "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(l0), "=&v"(h0), "=&v"(l1), "=&v"(h1), "=&v"(l2), "=&v"(h2), "=&v"(l3), "=&v"(h3)
      : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(OFF), "n"(OFF + 8 * W)
      : "memory");
  x[0] = __builtin_bit_cast(Frag, __builtin_shufflevector(l0, h0, 0, 1, 2, 3));
  x[1] = __builtin_bit_cast(Frag, __builtin_shufflevector(l1, h1, 0, 1, 2, 3));
  x[2] = __builtin_bit_cast(Frag, __builtin_shufflevector(l2, h2, 0, 1, 2, 3));
  x[3] = __builtin_bit_cast(Frag, __builtin_shufflevector(l3, h3, 0, 1, 2, 3));
}

__device__ const int gf_zeros[4] __attribute__((aligned(16))) = {};   // a chunk behind the end of a row

// T: type of the outputs (and of 16-bit operands), PL: parts (3: side by side; 2: those of A one behind the other along k), WM x WN waves
// of (16 FM) x (16 FN) results.  TA, TB: the operand's other index is contiguous, not k.  RAW: x and the weights are read where they are
// though their rows begin or end inside a 16-byte chunk: through registers, with zeros behind a row's end.  GATED: rows of B alternate
// between gate and up every 16, so that a lane holds both sums of its outputs and the activation is applied in registers.
// Bound by the matrix pipe where tiles are many: 16 FM x 16 FN results of a wave need FM + FN fragments from LDS a step for FM FN
// instructions, so that 8 x 4 fragments (256 x 256 by eight waves) keep LDS reads below the pipe's time, and 4 x 4 do not quite.
// 8192 x 2048 x 8192 bf16: forward 470 us = 1.17 PFLOP/s (a library's product of 8192^3 reaches 1.32), 528 with `saved` (537 MB more),
// backward 2040 us with the pass that makes [dg | du] = 1.08 PFLOP/s of the two parts' products (dg and du rounded to bf16: 1055 us); fp16
// backward, three products and x and the weights split in registers, 3600 us.  fp32, six products of bf16 parts, 2708 x 500 x 1024: 152 us
// for both passes = 109 TFLOP/s (the library: 153): the forward product has 176 large tiles for 256 compute units.
template <int T, int PL, int WM, int WN, int FM, int FN, int BK, bool TA, bool TB, bool RAW, bool GATED>
__device__ __forceinline__ void gf_product(const GatedGemm& q, unsigned block, unsigned slice, char* smem) {
  typedef typename GfPlane<T, PL>::type P;
  typedef typename GfFrag<P>::type Frag;
  typedef typename GsElt<T>::type E;
  constexpr int NP = PL == 3 ? 3 : 1;   // parts that are in LDS at a time
  constexpr int STRETCHES = gf_stretches(T, PL);
  static_assert(PL != 2 || (TB && !RAW && !GATED), "the backward products");
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16, NT = WM * WN * 64;
  constexpr int CA = (TA ? BM : BK) / 8, CB = (TB ? BN : BK) / 8;   // 16-byte chunks of a row
  constexpr int TILE_A = BM * BK, TILE_B = BN * BK, STAGE = NP * (TILE_A + TILE_B);
  constexpr int ITA = TILE_A / 8 / NT, ITB = TILE_B / 8 / NT;
  static_assert(TILE_A / 8 % NT == 0 && TILE_B / 8 % NT == 0, "whole waves load a tile");
  constexpr bool PHASES = WM * WN == 8 && BK == 64 && !RAW;       // eight waves that take turns, see below
  P* lds = (P*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WN, wn = wave % WN;
  // Tiles of m first: what runs at a time on an XCD (every eighth workgroup) shares four rows of tiles and their columns in its L2.
  // (8192 x 2048 x 8192: giving each XCD a run of consecutive tiles instead changes nothing without `saved`, and with it costs 100 us
  // of 560, since neighbouring pieces of its rows are then written far apart in time.)
  const long m0 = (long)(block % q.gx) * BM;
  const long n0 = (long)(block / q.gx) * (GATED ? BN / 2 : BN);
  const long k_begin = slice * q.kslice, k_end = min(k_begin + q.kslice, q.K);
  const P* A = (const P*)q.A;

  const P* srcA[ITA];
  int colA[ITA];
  int colB[ITB];        // of a chunk in its row
  long srcB[ITB];       // offsets from B's base
#pragma unroll
  for (int i = 0; i < ITA; ++i) {
    const int s = i * NT + tid, r = s / CA, c = (s % CA) ^ gf_swz<TA, BK>(r);
    colA[i] = c * 8;
    srcA[i] = TA ? A + r * q.lda + min(m0 + c * 8, q.M - 8) : A + min(m0 + r, q.M - 1) * q.lda + (RAW ? 0 : c * 8);
  }
#pragma unroll
  for (int i = 0; i < ITB; ++i) {
    const int s = i * NT + tid, r = s / CB, c = (s % CB) ^ gf_swz<TB, BK>(r);
    const long n = GATED ? n0 + (r >> 5) * 16 + (r & 15) : n0 + r;
    const P* base = (const P*)q.B[GATED ? (r >> 4) & 1 : 0];
    const long in_row = TB ? min(n0 + c * 8, q.bcols - 8) : (RAW ? 0 : c * 8);   // (RAW, k contiguous: the column comes with the step)
    colB[i] = c * 8;
    srcB[i] = (TB ? r * q.ldb : (long)(base + min(n, q.N - 1) * q.ldb - (const P*)q.B[0])) + in_row;
  }
  static_assert(!RAW || (!TA && !TB), "rows of k");
  // RAW: the chunks of the next tile on their way through registers.  A chunk that reaches behind its row's end is loaded from the
  // row's last 8 elements and shifted down when it goes to LDS, zeros behind.
  typedef typename GsVec<P, 8>::type Chunk;
  Chunk ra[RAW ? ITA : 1], rb[RAW ? ITB : 1];
  long k_raw = 0;                                                  // the step that is on its way
  auto raw_shift = [&](Chunk v, long at) {
    if (at <= q.k_end - 8) return v;
    const int by = (int)(at - (q.k_end - 8));
    unsigned __int128 x = __builtin_bit_cast(unsigned __int128, v);
    x = by >= 8 ? (unsigned __int128)0 : x >> (16 * by);
    return __builtin_bit_cast(Chunk, x);
  };
  auto stage = [&](int buf, long k0) {
    P* base = lds + buf * STAGE;
    long a_at = 0;                                                 // of the stretch's part of A
    if constexpr (STRETCHES > 1) {                                 // the low part of A first, then the high one (fp16: twice)
      if (k0 < q.stretch) a_at = q.plane_a;
      k0 -= k0 >= q.stretch ? q.stretch : 0;
      if constexpr (STRETCHES > 2) k0 -= k0 >= q.stretch ? q.stretch : 0;
    }
    const P* b0 = (const P*)q.B[0] + k0;
    bool end = false;
    if constexpr (TB) {
      // A is zero behind B's rows: a step that lies there altogether takes B's last ones
      const long kk = min(k0 < q.kb ? k0 : k0 - q.kb, (q.brows - 1) / BK * BK);
      b0 = (const P*)q.B[k0 < q.kb ? 0 : 1] + kk * q.ldb;
      end = kk + BK > q.brows;
    }
    k_raw = k0;
    if constexpr (RAW) {
      const long last = q.k_end - 8 - k0;                          // (of the step's elements, where its last chunks would pass the end)
#pragma unroll
      for (int i = 0; i < ITA; ++i) ra[i] = *(const Chunk*)(srcA[i] + (k0 + min((long)colA[i], last)));
#pragma unroll
      for (int i = 0; i < ITB; ++i) rb[i] = *(const Chunk*)((const P*)q.B[0] + srcB[i] + (k0 + min((long)colB[i], last)));
      return;
    }
    if constexpr (PL == 1 && !TA && !TB) {
      if (k0 + BK > q.k_end) {
        // The last step: from chunks behind the end of a row zeros are read.  (The assembly keeps this a branch; selected address by
        // address in every step it costs a tenth of the whole, 8192 x 2048 x 8192 bf16 500 us against 454.)
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < ITA; ++i)
          if (k0 + colA[i] >= q.k_end) srcA[i] = (const P*)gf_zeros - k0;
#pragma unroll
        for (int i = 0; i < ITB; ++i)
          if (k0 + colB[i] >= q.k_end) srcB[i] = (const P*)gf_zeros - b0;
      }
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
      for (int i = 0; i < ITA; ++i) {
        const P* at = srcA[i] + p * q.plane_a + (a_at + (TA ? k0 * q.lda : k0));
        __builtin_amdgcn_global_load_lds((gbl_ptr)at, (lds_ptr)(base + p * TILE_A + (i * NT + wave * 64) * 8), 16, 0, 0);
      }
      auto load_b = [&](auto beyond) {
#pragma unroll
        for (int i = 0; i < ITB; ++i) {
          const P* at = b0 + p * q.plane_b + srcB[i] - beyond(i);
          __builtin_amdgcn_global_load_lds((gbl_ptr)at, (lds_ptr)(base + NP * TILE_A + p * TILE_B + (i * NT + wave * 64) * 8), 16, 0, 0);
        }
      };
      // (the step with B's last rows, where they are fewer than BK: the last one again for those that there are not)
      if (TB && end) load_b([&](int i) { return max((i * NT + tid) / CB - (q.brows - 1) % BK, 0L) * q.ldb; });
      else load_b([](int) { return 0; });
    }
  };
  auto land = [&](int buf) {
    typedef P Whole __attribute__((ext_vector_type(8)));
    P* base = lds + buf * STAGE;
    if constexpr (RAW) {
      const bool ends = k_raw + BK > q.k_end;                      // (the whole workgroup's)
#pragma unroll
      for (int i = 0; i < ITA; ++i) *(Whole*)(base + (i * NT + tid) * 8) = ends ? raw_shift(ra[i], k_raw + colA[i]) : ra[i];
#pragma unroll
      for (int i = 0; i < ITB; ++i) *(Whole*)(base + TILE_A + (i * NT + tid) * 8) = ends ? raw_shift(rb[i], k_raw + colB[i]) : rb[i];
    }
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  const unsigned tra = TA ? gf_tr_addr<BM, BK>(lds, wm * FM * 16, lane) : 0u;
  const unsigned trb = TB ? gf_tr_addr<BN, BK>(lds + NP * TILE_A, wn * FN * 16, lane) : 0u;
  stage(0, k_begin);
  land(0);
  int buf = 0;
  Frag a[NP][FM], b[NP][FN];
  const P* ta = lds;
  const P* tb = lds;
  // the fragments of 32 of k; those of a transposed A are read four rows of tiles at a time, before their products
  auto read = [&](auto ks_, int at, long k0) {
    constexpr int ks = decltype(ks_)::value;
    gf_static_for<NP>([&](auto p_) {
      constexpr int p = decltype(p_)::value;
      if constexpr (TB) {
        gf_static_for<FN / 4>([&](auto j_) {
          constexpr int j = decltype(j_)::value * 4;
          gf_tr_read4<p * TILE_B * 2 + ks * 64 * BN, BN>(trb + at * STAGE * 2, j, &b[p][j]);
        });
      } else {
#pragma unroll
        for (int j = 0; j < FN; ++j) b[p][j] = gf_frag<Frag, BK>(tb + p * TILE_B, (wn * FN + j) * 16, ks, lane);
      }
      if constexpr (TA) {
        gf_static_for<FM / 4>([&](auto i_) {
          constexpr int i0 = decltype(i_)::value * 4;
          gf_tr_read4<p * TILE_A * 2 + ks * 64 * BM, BM>(tra + at * STAGE * 2, i0, &a[p][i0]);
        });
      } else {
#pragma unroll
        for (int i = 0; i < FM; ++i) a[p][i] = gf_frag<Frag, BK>(ta + p * TILE_A, (wm * FM + i) * 16, ks, lane);
      }
    });
    if constexpr (STRETCHES == 3) {
      auto part = [&](auto rest) {
#pragma unroll
        for (int j = 0; j < FN; ++j) b[0][j] = gf_part<decltype(rest)::value>(b[0][j]);
      };
      if (k0 >= q.stretch && k0 < 2 * q.stretch) part(std::true_type{});
      else part(std::false_type{});
    }
  };
  auto multiply = [&] {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if constexpr (PL == 3) {   // small terms first
          acc[i][j] = gf_mfma(b[2][j], a[0][i], acc[i][j]);
          acc[i][j] = gf_mfma(b[0][j], a[2][i], acc[i][j]);
          acc[i][j] = gf_mfma(b[1][j], a[1][i], acc[i][j]);
          acc[i][j] = gf_mfma(b[1][j], a[0][i], acc[i][j]);
          acc[i][j] = gf_mfma(b[0][j], a[1][i], acc[i][j]);
        }
        acc[i][j] = gf_mfma(b[0][j], a[0][i], acc[i][j]);
      }
    __builtin_amdgcn_s_setprio(0);
  };
  if constexpr (PHASES) {
    // Two waves share a SIMD, one of each group.  A step of k is four phases with a barrier behind each: read 32 of k, multiply, read the
    // other 32, multiply; the second group is one phase behind, so that one group's reads run beside the other's products.  In phases
    // of the first group, P0 .. P3 of step n: the next tile is asked for at P0 (P1 by the second group), when the buffer's last reader,
    // the second group's second read, was done at the P3 before; it has to be there at the next P0, so the first group waits for its
    // part at the end of P3 and the second at the end of its second read, which is P3 too.  Every wave passes the same number of
    // barriers: one more at the beginning for the second group, one more at the end for the first.
    const bool second = __builtin_amdgcn_readfirstlane(wave) >= WM * WN / 2;   // (a scalar: a wave branches around a barrier, or not)
    auto phase_end = [&](bool landed) {
      // (a fence would wait for the tile that is on its way, too: what has to be waited for is this wave's reads)
      if (landed) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("" ::: "memory");
    };
    __syncthreads();                                      // the first tile has landed
    if (second) phase_end(false);
    for (long k0 = k_begin; k0 < k_end; k0 += BK, buf ^= 1) {
      ta = lds + buf * STAGE;
      tb = ta + NP * TILE_A;
      if (k0 + BK < k_end) stage(buf ^ 1, k0 + BK);
      read(std::integral_constant<int, 0>{}, buf, k0);
      phase_end(false);
      multiply();
      phase_end(false);
      read(std::integral_constant<int, 1>{}, buf, k0);
      phase_end(second);
      multiply();
      phase_end(!second);
    }
    if (!second) phase_end(false);
  } else {
    for (long k0 = k_begin; k0 < k_end; k0 += BK, buf ^= 1) {
      __syncthreads();   // this step's tile has landed; the other buffer has been read by all
      ta = lds + buf * STAGE;
      tb = ta + NP * TILE_A;
      if (k0 + BK < k_end) stage(buf ^ 1, k0 + BK);
      gf_static_for<BK / 32>([&](auto ks) {
        read(ks, buf, k0);
        multiply();
      });
      if (k0 + BK < k_end) land(buf ^ 1);
    }
  }

  // B is the first operand, so a lane holds four consecutive n of one m
  const int lr = lane & 15, lc = lane >> 4;
  auto finish = [&](auto ac) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const long m = m0 + (wm * FM + i) * 16 + lr;
      if (m >= q.M) continue;
      if constexpr (GATED) {
#pragma unroll
        for (int j = 0; j < FN; j += 2) {
          const long n = n0 + (wn * FN + j) * 8 + lc * 4;
          if (n >= q.N) continue;
          float g[4], u[4], h[4], da;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            g[e] = acc[i][j][e];
            u[e] = acc[i][j + 1][e];
          }
          if constexpr (decltype(ac)::value < 0) {
            float* o = q.part + slice * q.slice + m * q.N + n;
            gs_store<float, 4>(o, q.N - n, g);
            gs_store<float, 4>(o + q.M * q.N, q.N - n, u);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              gf_act<T, decltype(ac)::value>(g[e], h[e], da);
              h[e] *= u[e];
            }
            gs_store<E, 4>((E*)q.C[0] + m * q.ldc + n, q.N - n, h);
            if (q.saved) {
              gs_store_past<float, 4>(q.saved + m * q.N + n, q.N - n, g);
              gs_store_past<float, 4>(q.saved + (q.M + m) * q.N + n, q.N - n, u);
            }
          }
        }
      } else {
        E* row = gf_row<E>(q, m);
        if (!row) continue;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const long n = n0 + (wn * FN + j) * 16 + lc * 4;
          if (n >= q.N) continue;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e];
          if (q.part) gs_store<float, 4>(q.part + slice * q.slice + m * q.N + n, q.N - n, v);
          else gs_store<E, 4>(row + n, q.N - n, v);
        }
      }
    }
  };
  if constexpr (GATED) {
    if (q.part) finish(std::integral_constant<int, -1>{});
    else gf_with_act(q.act, finish);
  } else {
    finish(std::integral_constant<int, -1>{});
  }
}

template <int T, int PL, int WM, int WN, int FM, int FN, int BK, bool TA, bool TB, bool RAW, bool GATED>
__global__ __launch_bounds__(WM * WN * 64) void gs_gated_gemm_kernel(GatedGemm q) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  gf_product<T, PL, WM, WN, FM, FN, BK, TA, TB, RAW, GATED>(q, blockIdx.x, blockIdx.y, smem);
}

// dx and dW in one launch, where neither fills the chip alone: blocks [0, a_blocks) are dx's tiles and slices, the others dW's.
template <int T, int PL, int WM, int WN, int FM, int FN, int BK>
__global__ __launch_bounds__(WM * WN * 64) void gs_gated_pair_kernel(GatedGemm a, unsigned a_tiles, unsigned a_blocks, GatedGemm b, unsigned b_tiles) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  if (blockIdx.x < a_blocks) {
    gf_product<T, PL, WM, WN, FM, FN, BK, false, true, false, false>(a, blockIdx.x % a_tiles, blockIdx.x / a_tiles, smem);
  } else {
    const unsigned i = blockIdx.x - a_blocks;
    gf_product<T, PL, WM, WN, FM, FN, BK, true, true, false, false>(b, i % b_tiles, i / b_tiles, smem);
  }
}

// Sums the slices of k in their order and finishes what the product's epilogue does.  A thread takes four columns of a row.
template <int T, bool GATED>
__device__ __forceinline__ void gf_join(const GatedGemm& q, int slices, unsigned block) {
  typedef typename GsElt<T>::type E;
  const unsigned per = (unsigned)((q.N + 3) / 4), i = block * 256u + threadIdx.x, r = i / per;
  const long m = r, n = (long)(i - r * per) * 4;
  if (m >= q.M) return;
  E* row = GATED ? (E*)q.C[0] + m * q.ldc : gf_row<E>(q, m);
  if (!row) return;
  float g[4] = {}, u[4] = {};
  const float* at = q.part + m * q.N + n;
  for (int z = 0; z < slices; ++z) {
    float v[4];
    gs_load<float, 4>(at + z * q.slice, q.N - n, 0.f, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] += v[e];
    if constexpr (GATED) {
      gs_load<float, 4>(at + z * q.slice + q.M * q.N, q.N - n, 0.f, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] += v[e];
    }
  }
  if constexpr (GATED) {
    if (q.saved) {
      gs_store<float, 4>(q.saved + m * q.N + n, q.N - n, g);
      gs_store<float, 4>(q.saved + (q.M + m) * q.N + n, q.N - n, u);
    }
    gf_with_act(q.act, [&](auto ac) {
      float da;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        gf_act<T, decltype(ac)::value>(g[e], g[e], da);
        g[e] *= u[e];
      }
    });
  }
  gs_store<E, 4>(row + n, q.N - n, g);
}

template <int T, bool GATED>
__global__ __launch_bounds__(256) void gs_gated_join_kernel(GatedGemm q, int slices) {
  gf_join<T, GATED>(q, slices, blockIdx.x);
}

template <int T>
__global__ __launch_bounds__(256) void gs_gated_join_pair_kernel(GatedGemm a, int a_slices, unsigned a_blocks, GatedGemm b, int b_slices) {
  if (blockIdx.x < a_blocks) gf_join<T, false>(a, a_slices, blockIdx.x);
  else gf_join<T, false>(b, b_slices, blockIdx.x - a_blocks);
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
// What a product costs, in units of one workgroup's 64 of k in the small tile, and the scratch that its slices take.
struct GatedSplit {
  bool big;
  int slices;
  long kslice;        // in elements
  size_t part;        // floats
  double cost;
};

// 16-bit operands: 128 x 128 (two workgroups on a compute unit) or 256 x 256 (one), which takes 1.75 times as long a step of 64 for twice
// the products of the two.  fp32: 128 x 128 or 256 x 128, one workgroup each, 1.4 times as long a step of 32 for twice the products.  A
// product that does not fill the 256 compute units is cut along k; its slices are summed by a second launch, which costs about 4 steps
// and the traffic of the partial sums.
GatedSplit gf_split_of(long M, long N, long K, bool gated, int pl) {
  GatedSplit best = {};
  double least = 1e300;
  const long cols = gated ? 2 * N : N;
  for (int big = 0; big < 2; ++big) {
    const long bm = big ? 256 : 128, bn = big && pl != 3 ? 256 : 128, bk = pl == 3 ? 32 : 64;
    const long tiles = ((M + bm - 1) / bm) * ((cols + bn - 1) / bn), slots = big || pl == 3 ? 256 : 512, steps = K / bk;
    const double step = big ? (pl == 3 ? 1.4 : 1.75) : 1.0;
    for (long want = 1; want <= 64 && want <= steps; ++want) {
      const long per = (steps + want - 1) / want, slices = (steps + per - 1) / per;
      if (want > 1 && tiles * slices > 2 * slots) break;
      double cost = (double)((tiles * slices + slots - 1) / slots) * step * (per + 2);
      if (slices > 1) cost += 4 + (double)slices * M * cols * 8 / 4e6;
      if (cost < least) {
        least = cost;
        best = {big != 0, (int)slices, per * bk, slices > 1 ? (size_t)slices * M * cols : 0, cost};
      }
    }
  }
  return best;
}

// dx (M x D, k over 2 Fp) and dW (2 Fp x D, k over Mp), each in so many stretches: one launch of both, cut into pieces of about equal
// length, where that costs less than one after the other (the same units, a launch about 3).
struct GatedPair {
  bool together;
  GatedSplit dx, dw;
};

GatedPair gf_pair_of(long M, long D, long Fp, long Mp, int pl, int stretches) {
  GatedPair best = {false, gf_split_of(M, D, 2 * Fp * stretches, false, pl), gf_split_of(2 * Fp, D, Mp * stretches, false, pl)};
  double least = best.dx.cost + best.dw.cost + 3;
  for (int big = 0; big < 2; ++big) {
    const long bm = big ? 256 : 128, bn = big && pl != 3 ? 256 : 128, bk = pl == 3 ? 32 : 64, gy = (D + bn - 1) / bn;
    const long tx = (M + bm - 1) / bm * gy, tw = (2 * Fp + bm - 1) / bm * gy, slots = big || pl == 3 ? 256 : 512;
    const long sx = 2 * Fp * stretches / bk, sw = Mp * stretches / bk, most = std::max(sx, sw);
    const double step = big ? (pl == 3 ? 1.4 : 1.75) : 1.0;
    for (long len = most;; len = (len * 3 + 3) / 4) {
      const long nx = std::min(64L, (sx + len - 1) / len), nw = std::min(64L, (sw + len - 1) / len);
      const long px = (sx + nx - 1) / nx, pw = (sw + nw - 1) / nw, cx = (sx + px - 1) / px, cw = (sw + pw - 1) / pw;
      const double all = (double)(tx * cx * (px + 2) + tw * cw * (pw + 2)) / slots, one = (double)std::max(px, pw) + 2;
      double cost = step * (tx * cx + tw * cw <= slots ? one : std::max(all + 0.35 * one, one));
      if (cx > 1 || cw > 1) cost += 4 + (double)((cx > 1 ? cx * M : 0) + (cw > 1 ? cw * 2 * Fp : 0)) * D * 8 / 4e6;
      if (cost < least) {
        least = cost;
        best = {true, {big != 0, (int)cx, px * bk, cx > 1 ? (size_t)cx * M * D : 0, 0}, {big != 0, (int)cw, pw * bk, cw > 1 ? (size_t)cw * 2 * Fp * D : 0, 0}};
      }
      if (len <= 4 || tx * cx + tw * cw > 2 * slots) break;
    }
  }
  return best;
}

// Where the laid-out operands lie in the scratch (elements of 2 bytes).  The sizes go by the shapes and the type alone.
struct GatedPlan {
  int pl, slopes;                     // parts of x and the weights, of dg and du
  bool pack;                          // x, Wg and Wu are laid out in the scratch (both passes)
  long Dp, Fp, Mp;
  size_t x, wg, wu, fwd;              // their places, with padded rows
  size_t dgu, bwd;                    // backward: [dg | du]
  size_t part_fwd, part_bwd;          // partial sums of products that are cut along k, behind the operands
  GatedSplit split;                   // of the forward product
  GatedPair pair;                     // of the backward ones
};

// Whether a forward call lays out 16-bit operands whose rows do not consist of whole, aligned chunks, as every backward call does, rather
// than read them through registers: laying out takes a launch and its traffic, reading so 1.6 ns more for a million products (fp16:
// 300 x 2047 x 8192 read 54 us, laid out 81; 8000 x 301 x 500 21.5 and 24.7; 2000 x 1433 x 4096 72 and 66; 4000 x 2047 x 8192 377 and 307).
inline bool gf_lay_out(long M, long D, long F) {
  return D < 8 || 1.6e-9 * M * D * F > 4 + 0.9e-6 * (M + 2 * F) * D;
}

GatedPlan gf_plan(long M, long D, long F, int type, bool plain, bool bwd) {
  GatedPlan p = {};
  p.pl = type == GS_TYPE_F32 ? 3 : 1;
  p.slopes = type == GS_TYPE_F32 ? 3 : 2;
  p.Dp = gf_up(D);
  p.Fp = gf_up(F);
  p.Mp = gf_up(M);
  size_t o = 0;
  auto take = [&](size_t n, int parts) { size_t at = o; o += n * parts; return at; };
  p.pack = p.pl > 1 || (!plain && (bwd || gf_lay_out(M, D, F)));
  if (p.pack) {
    p.x = take((size_t)p.Mp * p.Dp, p.pl);
    p.wg = take((size_t)p.Fp * p.Dp, p.pl);
    p.wu = take((size_t)p.Fp * p.Dp, p.pl);
  }
  p.part_fwd = o;
  if (!bwd) {
    p.split = gf_split_of(M, F, p.Dp, true, p.pl);
    p.fwd = o + 2 * p.split.part;
  }
  p.dgu = take((size_t)p.Mp * 2 * p.Fp, p.slopes);
  p.part_bwd = o;
  if (bwd) {
    p.pair = gf_pair_of(M, D, p.Fp, p.Mp, p.slopes, gf_stretches(type, p.slopes));
    const size_t dx = p.pair.dx.part, dw = p.pair.dw.part;
    p.bwd = o + 2 * (p.pair.together ? dx + dw : std::max(dx, dw));
  }
  return p;
}

// dynamic LDS beyond 64 KB is asked for once for each kernel and device
template <typename Kernel>
int gf_lds(Kernel kern, int bytes, std::atomic<unsigned long long>& known) {
  if (bytes <= 65536) return GS_OK;
  int dev = 0;
  GS_HIP(hipGetDevice(&dev));
  if (dev <= 63 && (known.load(std::memory_order_relaxed) >> dev & 1)) return GS_OK;
  GS_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev <= 63) known.fetch_or(1ull << dev, std::memory_order_relaxed);
  return GS_OK;
}

// Sets a product's slices; its tiles of BM x BN, or an error
int gf_prepare(GatedGemm& q, const GatedSplit& sp, int BM, int BN, int threads, bool gated, float* part, long* tiles) {
  const long gx = (q.M + BM - 1) / BM, gy = (q.N + BN - 1) / BN;
  if (gx * gy * sp.slices * threads > GF_MAX_THREADS) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated: %ld x %ld is beyond one launch", q.M, q.N);
  q.gx = (int)gx;
  q.kslice = sp.kslice;
  if (sp.slices > 1) {
    q.part = part;
    q.slice = q.M * q.N * (gated ? 2 : 1);
  }
  *tiles = gx * gy;
  return GS_OK;
}

inline long gf_join_blocks(const GatedGemm& q) { return (q.M * ((q.N + 3) / 4) + 255) / 256; }   // (a product that is cut has few tiles)

template <int T, int PL, int WM, int WN, int FM, int FN, int BK, bool TA, bool TB, bool RAW, bool GATED>
int gf_tile(GatedGemm q, const GatedSplit& sp, float* part, hipStream_t s) {
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16 / (GATED ? 2 : 1), LDS = 2 * (PL == 3 ? 3 : 1) * (WM * FM + WN * FN) * 16 * BK * 2;
  auto kern = gs_gated_gemm_kernel<T, PL, WM, WN, FM, FN, BK, TA, TB, RAW, GATED>;
  static std::atomic<unsigned long long> known{0};
  GS_TRY(gf_lds(kern, LDS, known));
  long tiles;
  GS_TRY(gf_prepare(q, sp, BM, BN, WM * WN * 64, GATED, part, &tiles));
  kern<<<dim3((unsigned)tiles, (unsigned)sp.slices), dim3(WM * WN * 64), LDS, s>>>(q);
  GS_LAUNCH_CHECK();
  if (sp.slices > 1) {
    if (gf_join_blocks(q) > GF_MAX_BLOCKS) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated: %ld x %ld is beyond one launch", q.M, q.N);
    gs_gated_join_kernel<T, GATED><<<dim3((unsigned)gf_join_blocks(q)), dim3(256), 0, s>>>(q, sp.slices);
    GS_LAUNCH_CHECK();
  }
  return GS_OK;
}

template <int T, int PL, bool TA, bool TB, bool GATED>
int gf_gemm(const GatedGemm& q, const GatedSplit& sp, bool raw, float* part, hipStream_t s) {
  if constexpr (PL == 3) {
    if (sp.big) return gf_tile<T, PL, 4, 2, 4, 4, 32, TA, TB, false, GATED>(q, sp, part, s);
    return gf_tile<T, PL, 2, 2, 4, 4, 32, TA, TB, false, GATED>(q, sp, part, s);
  } else {
    if constexpr (!TA && !TB) {
      if (raw) return sp.big ? gf_tile<T, PL, 2, 4, 8, 4, 64, TA, TB, true, GATED>(q, sp, part, s)
                             : gf_tile<T, PL, 2, 2, 4, 4, 64, TA, TB, true, GATED>(q, sp, part, s);
    }
    if (sp.big) return gf_tile<T, PL, 2, 4, 8, 4, 64, TA, TB, false, GATED>(q, sp, part, s);
    return gf_tile<T, PL, 2, 2, 4, 4, 64, TA, TB, false, GATED>(q, sp, part, s);
  }
}

template <int T, int PL, int WM, int WN, int FM, int FN, int BK>
int gf_pair_tile(GatedGemm a, GatedGemm b, const GatedPair& p, float* part, hipStream_t s) {
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16, LDS = 2 * (PL == 3 ? 3 : 1) * (WM * FM + WN * FN) * 16 * BK * 2;
  auto kern = gs_gated_pair_kernel<T, PL, WM, WN, FM, FN, BK>;
  static std::atomic<unsigned long long> known{0};
  GS_TRY(gf_lds(kern, LDS, known));
  long ta, tb;
  GS_TRY(gf_prepare(a, p.dx, BM, BN, WM * WN * 64, false, part, &ta));
  GS_TRY(gf_prepare(b, p.dw, BM, BN, WM * WN * 64, false, part + p.dx.part, &tb));
  if ((ta * p.dx.slices + tb * p.dw.slices) * WM * WN * 64 > GF_MAX_THREADS) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated: %ld x %ld is beyond one launch", b.M, b.N);
  kern<<<dim3((unsigned)(ta * p.dx.slices + tb * p.dw.slices)), dim3(WM * WN * 64), LDS, s>>>(a, (unsigned)ta, (unsigned)(ta * p.dx.slices), b, (unsigned)tb);
  GS_LAUNCH_CHECK();
  const long ja = p.dx.slices > 1 ? gf_join_blocks(a) : 0, jb = p.dw.slices > 1 ? gf_join_blocks(b) : 0;
  if (ja + jb > GF_MAX_BLOCKS) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated: %ld x %ld is beyond one launch", b.M, b.N);
  if (ja + jb) {
    gs_gated_join_pair_kernel<T><<<dim3((unsigned)(ja + jb)), dim3(256), 0, s>>>(a, p.dx.slices, (unsigned)ja, b, p.dw.slices);
    GS_LAUNCH_CHECK();
  }
  return GS_OK;
}

template <int T, int PL>
int gf_pair(const GatedGemm& a, const GatedGemm& b, const GatedPair& p, float* part, hipStream_t s) {
  if constexpr (PL == 3) {
    if (p.dx.big) return gf_pair_tile<T, PL, 4, 2, 4, 4, 32>(a, b, p, part, s);
    return gf_pair_tile<T, PL, 2, 2, 4, 4, 32>(a, b, p, part, s);
  } else {
    if (p.dx.big) return gf_pair_tile<T, PL, 2, 4, 8, 4, 64>(a, b, p, part, s);
    return gf_pair_tile<T, PL, 2, 2, 4, 4, 64>(a, b, p, part, s);
  }
}

// whether rows of `n` 16-bit elements with stride ld consist of whole, aligned chunks of 16 bytes
inline bool gf_plain(const void* p, long ld, long n) { return n % 8 == 0 && ld % 8 == 0 && ((size_t)p & 15) == 0; }

// whether x and the weights can be read as they are
inline bool gf_plain(const void* x, long ldx, const void* wg, const void* wu, long ldw, long D) {
  return gf_plain(x, ldx, D) && gf_plain(wg, ldw, D) && gf_plain(wu, ldw, D);
}

struct GatedCall {
  const void *x, *wg, *wu, *dh;
  long ldx, ldw, lddh;
  long M, D, F;
  int act;
  void *h, *dx, *dwg, *dwu;
  long ldh, lddx, lddw;
  float* saved;
  char* scratch;
};

// x, Wg and Wu as operands: as they are, or laid out (fp32: split) in the scratch
struct GatedOperands {
  const void *x, *w[2];
  long ldx, ldw, plane_x, plane_w;
};

template <int T, int PL>
int gf_operands(const GatedCall& c, const GatedPlan& p, GatedOperands* o, hipStream_t s) {
  typedef typename GfPlane<T, PL>::type P;
  *o = {c.x, {c.wg, c.wu}, c.ldx, c.ldw, 0, 0};
  if (p.pack) {
    P* sc = (P*)c.scratch;
    *o = {sc + p.x, {sc + p.wg, sc + p.wu}, p.Dp, p.Dp, p.Mp * p.Dp, p.Fp * p.Dp};
    const long bx = (p.Mp * (p.Dp / 8) + 255) / 256, bw = (p.Fp * (p.Dp / 8) + 255) / 256;
    if (bx + 2 * bw > GF_MAX_BLOCKS) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated: operands of width %ld are beyond one launch", c.D);
    const GatedPack a = {{c.x, c.wg, c.wu}, {sc + p.x, sc + p.wg, sc + p.wu}, {c.ldx, c.ldw, c.ldw}, {c.M, c.F, c.F}, {p.Mp, p.Fp, p.Fp},
                         {0, bx, bx + bw}, c.D, p.Dp};
    gs_gated_pack_kernel<T, PL><<<dim3((unsigned)(bx + 2 * bw)), dim3(256), 0, s>>>(a);
    GS_LAUNCH_CHECK();
  }
  return GS_OK;
}

// Rows up to which the weights are read by gs_gated_rows_kernel.  2048 x 8192: bf16, 4 rows 14 us (8 rows took 25), by the matrix pipe 5 to 8
// rows 16; fp32, 24 rows 92 us and 25 by the matrix pipe 113, of which laying out the split weights is most.
inline bool gf_few(long M, int type) { return M <= (type == GS_TYPE_F32 ? 24 : 4); }

template <int T, int MB>
int gf_rows(const GatedCall& c, hipStream_t s) {
  constexpr int RF = 2;
  if ((c.F + 4 * RF - 1) / (4 * RF) > GF_MAX_BLOCKS) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated_fwd: weights of %ld rows are beyond one launch", c.F);
  GatedRows q = {c.x, c.wg, c.wu, c.ldx, c.ldw, c.M, c.D, c.F, c.ldh, c.h, c.saved, c.act};
  gs_gated_rows_kernel<T, MB, RF><<<dim3((unsigned)((c.F + 4 * RF - 1) / (4 * RF)), (unsigned)((c.M + MB - 1) / MB)), dim3(256), 0, s>>>(q);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

template <int T, int PL>
int gf_fwd(const GatedCall& c, hipStream_t s) {
  typedef typename GfPlane<T, PL>::type P;
  if (gf_few(c.M, T)) {
    if (c.M == 1) return gf_rows<T, 1>(c, s);
    if (c.M == 2) return gf_rows<T, 2>(c, s);
    if constexpr (T == GS_TYPE_F32) {
      if (c.M > 4) return gf_rows<T, 8>(c, s);
    }
    return gf_rows<T, 4>(c, s);
  }
  const bool plain = gf_plain(c.x, c.ldx, c.wg, c.wu, c.ldw, c.D);
  const GatedPlan p = gf_plan(c.M, c.D, c.F, T, plain, false);
  GatedOperands o;
  GS_TRY((gf_operands<T, PL>(c, p, &o, s)));
  const bool raw = !p.pack && !plain;
  GatedGemm q = {};
  q.A = o.x; q.lda = o.ldx; q.plane_a = o.plane_x;
  q.B[0] = o.w[0]; q.B[1] = o.w[1]; q.ldb = o.ldw; q.plane_b = o.plane_w;
  q.M = c.M; q.N = c.F; q.K = q.stretch = p.Dp;
  q.C[0] = c.h; q.ldc = c.ldh;
  q.saved = c.saved; q.act = c.act;
  q.k_end = p.pack ? p.Dp : c.D;
  return gf_gemm<T, PL, false, false, true>(q, p.split, raw, (float*)((P*)c.scratch + p.part_fwd), s);
}

template <int T, int PL>
int gf_bwd(const GatedCall& c, hipStream_t s) {
  constexpr int SL = PL == 3 ? 3 : 2, STRETCHES = gf_stretches(T, SL);
  typedef typename GsElt<T>::type E;
  typedef typename GfPlane<T, SL>::type P;
  const GatedPlan p = gf_plan(c.M, c.D, c.F, T, gf_plain(c.x, c.ldx, c.wg, c.wu, c.ldw, c.D), true);
  P* dgu = (P*)c.scratch + p.dgu;
  const long plane = p.Mp * 2 * p.Fp, blocks = (p.Mp * (p.Fp / 8) + 255) / 256;
  if (blocks > GF_MAX_BLOCKS) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated_bwd: %ld x %ld is beyond one launch", c.M, c.F);
  GatedOperands o;
  GS_TRY((gf_operands<T, PL>(c, p, &o, s)));
  gs_gated_slopes_kernel<T, SL><<<dim3((unsigned)blocks), dim3(256), 0, s>>>(c.act, (const E*)c.dh, c.lddh, c.saved, c.M, c.F, dgu, p.Mp, p.Fp, plane);
  GS_LAUNCH_CHECK();
  // dx: k runs over the columns of dg, then of du, and over the rows of Wg, then of Wu
  GatedGemm q = {};
  q.A = dgu; q.lda = 2 * p.Fp; q.plane_a = plane;
  q.B[0] = o.w[0]; q.B[1] = o.w[1]; q.ldb = o.ldw; q.plane_b = o.plane_w;
  q.M = c.M; q.K = 2 * p.Fp * STRETCHES; q.stretch = 2 * p.Fp; q.kb = p.Fp; q.brows = p.pack ? p.Fp : c.F;
  q.N = c.D; q.bcols = p.pack ? p.Dp : c.D;
  q.C[0] = c.dx; q.ldc = c.lddx; q.rows = q.rows1 = c.M;
  float* part = (float*)((P*)c.scratch + p.part_bwd);
  // dWg, dWu: k runs over the tokens
  GatedGemm w = q;
  w.B[0] = o.x; w.ldb = o.ldx; w.plane_b = o.plane_x;
  w.M = 2 * p.Fp; w.K = p.Mp * STRETCHES; w.stretch = p.Mp; w.kb = p.Mp; w.brows = p.pack ? p.Mp : c.M;
  w.bcols = p.pack ? p.Dp : c.D;
  w.C[0] = c.dwg; w.C[1] = c.dwu; w.ldc = c.lddw; w.rows = c.F; w.rows1 = p.Fp;
  if (p.pair.together) return gf_pair<T, SL>(q, w, p.pair, part, s);
  GS_TRY((gf_gemm<T, SL, false, true, false>(q, p.pair.dx, false, part, s)));
  return gf_gemm<T, SL, true, true, false>(w, p.pair.dw, false, part, s);
}

// dW = 0 where there are no tokens
template <typename E>
__global__ void gs_gated_zero_kernel(E* a, E* b, long R, long C, long ld) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < R * C; i += (long)gridDim.x * 256) {
    a[i / C * ld + i % C] = (E)0.f;
    b[i / C * ld + i % C] = (E)0.f;
  }
}

template <int T>
int gf_empty(const GatedCall& c, hipStream_t s) {
  typedef typename GsElt<T>::type E;
  gs_gated_zero_kernel<E><<<dim3((unsigned)std::min((c.F * c.D + 255) / 256, 65536L)), dim3(256), 0, s>>>((E*)c.dwg, (E*)c.dwu, c.F, c.D, c.lddw);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

template <int T, int PL>
int gf_dispatch(const GatedCall& c, bool bwd, hipStream_t s) {
  if (bwd && c.M == 0) return gf_empty<T>(c, s);
  return bwd ? gf_bwd<T, PL>(c, s) : gf_fwd<T, PL>(c, s);
}

int gf_check(const char* who, const GatedCall& c, int type) {
  if (!gs_type_bytes(type)) GS_FAIL(GS_ERR_ARG, "%s: unknown element type %d", who, type);
  if (c.act < GS_ACT_SILU || c.act > GS_ACT_SIGMOID) GS_FAIL(GS_ERR_ARG, "%s: unknown activation %d", who, c.act);
  if (c.M < 0 || c.D < 1 || c.F < 1) GS_FAIL(GS_ERR_ARG, "%s: %ld rows, widths %ld and %ld", who, c.M, c.D, c.F);
  if (c.M > 0x7fffffffL || c.D > 0x3fffffffL || c.F > 0x3fffffffL) GS_FAIL(GS_ERR_UNSUPPORTED, "%s: sizes are counted in 32 bits", who);
  if (c.ldx < c.D || c.ldw < c.D) GS_FAIL(GS_ERR_ARG, "%s: a row stride is below the width %ld", who, c.D);
  return GS_OK;
}

// Whether an output lies on another operand
bool gf_clash(const GatedCall& c, int type) {
  const int e = gs_type_bytes(type);
  const GsSpan in[] = {gs_span(c.x, c.M, c.ldx, c.D, e), gs_span(c.wg, c.F, c.ldw, c.D, e), gs_span(c.wu, c.F, c.ldw, c.D, e),
                       gs_span(c.dh, c.M, c.lddh, c.F, e)};
  const GsSpan saved = gs_span(c.saved, 2 * c.M * c.F, 4);
  const GsSpan out[] = {gs_span(c.h, c.M, c.ldh, c.F, e), gs_span(c.dx, c.M, c.lddx, c.D, e), gs_span(c.dwg, c.F, c.lddw, c.D, e),
                        gs_span(c.dwu, c.F, c.lddw, c.D, e)};
  bool clash = false;
  for (int o = 0; o < 4; ++o) {
    clash |= gs_overlap(out[o], saved);
    for (const GsSpan& i : in) clash |= gs_overlap(out[o], i) || (c.h && gs_overlap(saved, i));
    for (int q = 0; q < o; ++q) clash |= gs_overlap(out[o], out[q]);
  }
  return clash;
}

int gf_run(const GatedCall& c, int type, bool bwd, hipStream_t s) {
  if (type == GS_TYPE_F32) return gf_dispatch<GS_TYPE_F32, 3>(c, bwd, s);
  if (type == GS_TYPE_F16) return gf_dispatch<GS_TYPE_F16, 1>(c, bwd, s);
  return gf_dispatch<GS_TYPE_BF16, 1>(c, bwd, s);
}

}  // namespace

extern "C" size_t gs_gated_fwd_scratch_bytes(long M, long D, long F, int type, int plain) {
  if (M < 1 || D < 1 || F < 1 || !gs_type_bytes(type)) return 0;
  return gf_few(M, type) ? 0 : gf_plan(M, D, F, type, plain != 0, false).fwd * 2;
}

extern "C" size_t gs_gated_bwd_scratch_bytes(long M, long D, long F, int type, int plain) {
  if (M < 1 || D < 1 || F < 1 || !gs_type_bytes(type)) return 0;
  return gf_plan(M, D, F, type, plain != 0, true).bwd * 2;
}

extern "C" int gs_gated_fwd(const void* x, long ldx, const void* w_gate, const void* w_up, long ldw, int type, long M, long D, long F, int act,
                            void* h, long ldh, float* saved, void* scratch, gs_stream_t stream) {
  GatedCall c = {};
  c.x = x; c.wg = w_gate; c.wu = w_up; c.ldx = ldx; c.ldw = ldw; c.M = M; c.D = D; c.F = F; c.act = act;
  c.h = h; c.ldh = ldh; c.saved = saved; c.scratch = (char*)scratch;
  GS_TRY(gf_check("gs_gated_fwd", c, type));
  if (ldh < F) GS_FAIL(GS_ERR_ARG, "gs_gated_fwd: a row stride is below the width %ld", F);
  if (M == 0) return GS_OK;
  if (!x || !w_gate || !w_up || !h || (!scratch && gs_gated_fwd_scratch_bytes(M, D, F, type, gf_plain(x, ldx, w_gate, w_up, ldw, D)) > 0))
    GS_FAIL(GS_ERR_ARG, "gs_gated_fwd: null pointer");
  if (gf_clash(c, type)) GS_FAIL(GS_ERR_ARG, "gs_gated_fwd: an output lies on another operand");
  if ((size_t)scratch & 15) GS_FAIL(GS_ERR_ARG, "gs_gated_fwd: the scratch is not 16-byte aligned");
  return gf_run(c, type, false, (hipStream_t)stream);
}

extern "C" int gs_gated_bwd(const void* dh, long lddh, const void* x, long ldx, const void* w_gate, const void* w_up, long ldw,
                            const float* saved, int type, long M, long D, long F, int act, void* dx, long lddx, void* dw_gate,
                            void* dw_up, long lddw, void* scratch, gs_stream_t stream) {
  GatedCall c = {};
  c.x = x; c.wg = w_gate; c.wu = w_up; c.dh = dh; c.ldx = ldx; c.ldw = ldw; c.lddh = lddh; c.M = M; c.D = D; c.F = F; c.act = act;
  c.dx = dx; c.lddx = lddx; c.dwg = dw_gate; c.dwu = dw_up; c.lddw = lddw; c.saved = (float*)saved; c.scratch = (char*)scratch;
  GS_TRY(gf_check("gs_gated_bwd", c, type));
  if (lddh < F || lddx < D || lddw < D) GS_FAIL(GS_ERR_ARG, "gs_gated_bwd: a row stride is below the width");
  if (!dw_gate || !dw_up || (M > 0 && (!dh || !x || !w_gate || !w_up || !saved || !dx || !scratch)))
    GS_FAIL(GS_ERR_ARG, "gs_gated_bwd: null pointer");
  if (gf_clash(c, type)) GS_FAIL(GS_ERR_ARG, "gs_gated_bwd: an output lies on another operand");
  if ((size_t)scratch & 15) GS_FAIL(GS_ERR_ARG, "gs_gated_bwd: the scratch is not 16-byte aligned");
  return gf_run(c, type, true, (hipStream_t)stream);
}
