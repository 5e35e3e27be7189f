// Gated feed-forward block:  g = x Wg^T, u = x Wu^T, h = act(g) u,  and its backward pass
//   du = dh act(g), dg = dh u act'(g), dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x.
// Every product is brought to the form C(m, n) = sum_k A(m, k) B(n, k) with k contiguous in both operands, and runs on the 16-bit
// matrix pipe with fp32 accumulation.  16-bit operands enter as they are; an fp32 operand is the exact sum of three bf16 parts
// (x = h + m + l, 8 + 8 + 8 significant bits), and six products of parts make one product: what they leave out is below 2^-23 of it.
// (Parts have bf16's smallest step, 2^-133: a value is represented to 2^-134 or to 24 bits, whichever is coarser.)
// Operands whose rows are no multiple of 64 elements, or not 16-byte aligned, that have to be split or transposed, are laid out in
// the caller's scratch first, rows padded with zeros to a multiple of 64.
#include "gs_types.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* gbl_ptr;

constexpr int GF_PAD = 64;   // rows of laid-out operands are multiples of this many elements

inline long gf_up(long n) { return (n + GF_PAD - 1) / GF_PAD * GF_PAD; }

// ---- activations: the value and its derivative ---------------------------------------------------------------------------------
template <int ACT>
__device__ __forceinline__ void gf_act(float g, float& a, float& da) {
  if constexpr (ACT == GS_ACT_RELU) {
    a = g > 0.f ? g : (g == g ? 0.f : g);
    da = g > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == GS_ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * cdf;
    da = cdf + g * __expf(-0.5f * g * g) * 0.39894228040143268f;
  } else {
    const float sig = 1.f / (1.f + __expf(-g));
    if constexpr (ACT == GS_ACT_SILU) {
      a = g * sig;
      da = sig * (1.f + g * (1.f - sig));
    } else {
      a = sig;
      da = sig * (1.f - sig);
    }
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

template <int T, int PL, typename P>
__device__ __forceinline__ void gf_put(float v, P* __restrict__ o, long plane) {
  if constexpr (PL == 1) {
    o[0] = (P)v;
  } else {
    __bf16 h, m, l;
    gf_split(v, h, m, l);
    o[0] = h;
    o[plane] = m;
    o[2 * plane] = l;
  }
}

// ---- operand layout -------------------------------------------------------------------------------------------------------------
// out [PL][R][ldo] = in [R][C], zeros behind column C up to `cols`
template <int T, int PL>
__global__ __launch_bounds__(256) void gs_gated_pack_kernel(const typename GsElt<T>::type* __restrict__ in, long ldi, long R, long C,
                                                            typename GfPlane<T, PL>::type* __restrict__ out, long ldo, long cols, long plane) {
  const long per = cols / 8;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const long r = i / per, c = (i - r * per) * 8;
  if (r >= R) return;
  float v[8];
  if (c < C) {
    gs_load<typename GsElt<T>::type, 8>(in + r * ldi + c, C - c, 0.f, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) gf_put<T, PL>(v[j], out + r * ldo + c + j, plane);
}

// out [PL][C][ldo] = in [R][C] transposed, zeros behind column R up to the next multiple of 64
template <int T, int PL>
__global__ __launch_bounds__(256) void gs_gated_pack_t_kernel(const typename GsElt<T>::type* __restrict__ in, long ldi, long R, long C,
                                                              typename GfPlane<T, PL>::type* __restrict__ out, long ldo, long plane) {
  __shared__ float tile[64][65];
  const long r0 = (long)blockIdx.x * 64, c0 = (long)blockIdx.y * 64;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  for (int i = y; i < 64; i += 4) tile[i][x] = r0 + i < R && c0 + x < C ? (float)in[(r0 + i) * ldi + c0 + x] : 0.f;
  __syncthreads();
  for (int i = y; i < 64; i += 4)
    if (c0 + i < C) gf_put<T, PL>(tile[x][i], out + (c0 + i) * ldo + r0 + x, plane);
}

// dg, du from dh and the saved g, u: row-major [PL][M][2 Fp] (columns [0, Fp) dg, [Fp, 2 Fp) du) and transposed [PL][2 F][Mp]
template <int T, int PL, int ACT>
__global__ __launch_bounds__(256) void gs_gated_slopes_kernel(const typename GsElt<T>::type* __restrict__ dh, long lddh,
                                                              const float* __restrict__ saved, long M, long F,
                                                              typename GfPlane<T, PL>::type* __restrict__ rows, long Fp, long plane_r,
                                                              typename GfPlane<T, PL>::type* __restrict__ cols, long Mp, long plane_c) {
  __shared__ float tg[64][65], tu[64][65];
  const long m0 = (long)blockIdx.x * 64, f0 = (long)blockIdx.y * 64;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  for (int i = y; i < 64; i += 4) {
    float dg = 0.f, du = 0.f;
    const long m = m0 + i, f = f0 + x;
    if (m < M && f < F) {
      const float d = (float)dh[m * lddh + f], g = saved[m * F + f], u = saved[(M + m) * F + f];
      float a, da;
      gf_act<ACT>(g, a, da);
      du = d * a;
      dg = d * u * da;
    }
    tg[i][x] = dg;
    tu[i][x] = du;
    if (m < M) {
      gf_put<T, PL>(dg, rows + m * 2 * Fp + f, plane_r);
      gf_put<T, PL>(du, rows + m * 2 * Fp + Fp + f, plane_r);
    }
  }
  __syncthreads();
  for (int i = y; i < 64; i += 4)
    if (f0 + i < F) {
      gf_put<T, PL>(tg[x][i], cols + (f0 + i) * Mp + m0 + x, plane_c);
      gf_put<T, PL>(tu[x][i], cols + (F + f0 + i) * Mp + m0 + x, plane_c);
    }
}

// ---- the product ----------------------------------------------------------------------------------------------------------------
struct GatedGemm {
  const void* A;        // [PL][M][lda]
  long lda, plane_a;
  const void* B[2];     // [PL][N][ldb]; the gated form: gate and up projection, N rows each
  long ldb, plane_b;
  long M, N, K;         // K a multiple of 64
  void* C[2];           // plain form: rows below `rows0` go to C[0], the others to C[1] (from its row 0 on)
  long ldc, rows0;
  float* saved;         // gated form: g [M][N] and u [M][N], or null
};

__device__ __forceinline__ f32x4 gf_mfma(h16x8 a, h16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 gf_mfma(b16x8 a, b16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

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

// One operand's tile in LDS: rows of BK elements as 16-byte chunks, chunk c of row r at place c ^ s(r), so that the eight lanes that a
// 16-byte LDS read serves at once (eight rows, one chunk) fall on all banks; the permutation is made on the global side, since the
// direct-to-LDS load writes 64 consecutive chunks.
template <int BK>
__device__ __forceinline__ int gf_swz(int r) {
  return BK == 64 ? (r & 7) : ((r >> 1) & 3);
}

// T: type of the outputs (and of 16-bit operands), PL: parts, WM x WN waves of (16 FM) x (16 FN) results, GATED: rows of B alternate
// between gate and up every 16, so that a lane holds both sums of its outputs and the activation is applied in registers.
template <int T, int PL, int WM, int WN, int FM, int FN, int BK, bool GATED, int ACT>
__global__ __launch_bounds__(WM * WN * 64) void gs_gated_gemm_kernel(GatedGemm q) {
  typedef typename GfPlane<T, PL>::type P;
  typedef typename GfFrag<P>::type Frag;
  typedef typename GsElt<T>::type E;
  constexpr int BM = WM * FM * 16, BN = WN * FN * 16, NT = WM * WN * 64;
  constexpr int CH = BK / 8;                                  // 16-byte chunks of a row
  constexpr int TILE_A = BM * BK, TILE_B = BN * BK, STAGE = PL * (TILE_A + TILE_B);
  constexpr int ITA = BM * CH / NT, ITB = BN * CH / NT;
  static_assert(BM * CH % NT == 0 && BN * CH % NT == 0, "whole waves load a tile");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  P* lds = (P*)smem;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const long m0 = (long)blockIdx.x * BM;
  const long n0 = (long)blockIdx.y * (GATED ? BN / 2 : BN);
  const P* A = (const P*)q.A;

  const P* srcA[ITA];
  const P* srcB[ITB];
#pragma unroll
  for (int i = 0; i < ITA; ++i) {
    const int s = i * NT + tid, r = s / CH, c = (s % CH) ^ gf_swz<BK>(r);
    srcA[i] = A + min(m0 + r, q.M - 1) * q.lda + c * 8;
  }
#pragma unroll
  for (int i = 0; i < ITB; ++i) {
    const int s = i * NT + tid, r = s / CH, c = (s % CH) ^ gf_swz<BK>(r);
    const long n = GATED ? n0 + (r >> 5) * 16 + (r & 15) : n0 + r;
    srcB[i] = (const P*)q.B[GATED ? (r >> 4) & 1 : 0] + min(n, q.N - 1) * q.ldb + c * 8;
  }
  auto stage = [&](int buf, long k0) {
    P* base = lds + buf * STAGE;
#pragma unroll
    for (int p = 0; p < PL; ++p) {
#pragma unroll
      for (int i = 0; i < ITA; ++i)
        __builtin_amdgcn_global_load_lds((gbl_ptr)(srcA[i] + p * q.plane_a + k0), (lds_ptr)(base + p * TILE_A + (i * NT + wave * 64) * 8), 16, 0, 0);
#pragma unroll
      for (int i = 0; i < ITB; ++i)
        __builtin_amdgcn_global_load_lds((gbl_ptr)(srcB[i] + p * q.plane_b + k0), (lds_ptr)(base + PL * TILE_A + p * TILE_B + (i * NT + wave * 64) * 8), 16, 0, 0);
    }
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  const int lr = lane & 15, lc = lane >> 4;
  stage(0, 0);
  int buf = 0;
  for (long k0 = 0; k0 < q.K; k0 += BK, buf ^= 1) {
    __syncthreads();   // this step's tile has landed; the other buffer has been read by all
    if (k0 + BK < q.K) stage(buf ^ 1, k0 + BK);
    const P* base = lds + buf * STAGE;
#pragma unroll
    for (int ks = 0; ks < BK / 32; ++ks) {
      Frag a[PL][FM], b[PL][FN];
#pragma unroll
      for (int p = 0; p < PL; ++p) {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const int r = (wm * FM + i) * 16 + lr;
          a[p][i] = *(const Frag*)(base + p * TILE_A + (r * CH + ((ks * 4 + lc) ^ gf_swz<BK>(r))) * 8);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int r = (wn * FN + j) * 16 + lr;
          b[p][j] = *(const Frag*)(base + PL * TILE_A + p * TILE_B + (r * CH + ((ks * 4 + lc) ^ gf_swz<BK>(r))) * 8);
        }
      }
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
    }
  }

  // B is the first operand, so a lane holds four consecutive n of one m
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
          gf_act<ACT>(g[e], h[e], da);
          h[e] *= u[e];
        }
        gs_store<E, 4>((E*)q.C[0] + m * q.ldc + n, q.N - n, h);
        if (q.saved) {
          gs_store<float, 4>(q.saved + m * q.N + n, q.N - n, g);
          gs_store<float, 4>(q.saved + (q.M + m) * q.N + n, q.N - n, u);
        }
      }
    } else {
      E* row = m < q.rows0 ? (E*)q.C[0] + m * q.ldc : (E*)q.C[1] + (m - q.rows0) * q.ldc;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const long n = n0 + (wn * FN + j) * 16 + lc * 4;
        if (n >= q.N) continue;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e];
        gs_store<E, 4>(row + n, q.N - n, v);
      }
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------
// Where the laid-out operands lie in the scratch (elements of 2 bytes).  The sizes go by the shapes and the type alone.
struct GatedPlan {
  int pl;
  long Dp, Fp, Mp;
  size_t x, wg, wu, fwd;                       // forward: x, Wg, Wu with padded rows
  size_t rows, cols, wt, xt, bwd;              // backward: [dg | du], its transpose, [Wg; Wu]^T, x^T
};

GatedPlan gf_plan(long M, long D, long F, int type) {
  GatedPlan p;
  p.pl = type == GS_TYPE_F32 ? 3 : 1;
  p.Dp = gf_up(D);
  p.Fp = gf_up(F);
  p.Mp = gf_up(M);
  size_t o = 0;
  auto take = [&](size_t n) { size_t at = o; o += n * p.pl; return at; };
  p.x = take((size_t)M * p.Dp);
  p.wg = take((size_t)F * p.Dp);
  p.wu = take((size_t)F * p.Dp);
  p.fwd = o;
  o = 0;
  p.rows = take((size_t)M * 2 * p.Fp);
  p.cols = take((size_t)2 * F * p.Mp);
  p.wt = take((size_t)D * 2 * p.Fp);
  p.xt = take((size_t)D * p.Mp);
  p.bwd = o;
  return p;
}

template <int T, int PL, bool GATED, int ACT>
int gf_gemm(const GatedGemm& q, hipStream_t s) {
  constexpr int BK = PL == 3 ? 32 : 64;
  constexpr int LDS = 2 * PL * (128 + 128) * BK * 2;
  auto kern = gs_gated_gemm_kernel<T, PL, 2, 2, 4, 4, BK, GATED, ACT>;
  GS_HIP(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
  const long gx = (q.M + 127) / 128, gy = (q.N + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
  if (gx > 0x7fffffffL || gy > 65535) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated: %ld x %ld is beyond one launch", q.M, q.N);
  kern<<<dim3((unsigned)gx, (unsigned)gy), dim3(256), LDS, s>>>(q);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

template <int T, int PL>
int gf_pack(const void* in, long ldi, long R, long C, void* out, long ldo, long plane, hipStream_t s) {
  typedef typename GsElt<T>::type E;
  typedef typename GfPlane<T, PL>::type P;
  const long cols = gf_up(C), blocks = (R * (cols / 8) + 255) / 256;
  if (blocks > 0x7fffffffL) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated: %ld x %ld is beyond one launch", R, C);
  gs_gated_pack_kernel<T, PL><<<dim3((unsigned)blocks), dim3(256), 0, s>>>((const E*)in, ldi, R, C, (P*)out, ldo, cols, plane);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

template <int T, int PL>
int gf_pack_t(const void* in, long ldi, long R, long C, void* out, long ldo, long plane, hipStream_t s) {
  typedef typename GsElt<T>::type E;
  typedef typename GfPlane<T, PL>::type P;
  const long gx = (R + 63) / 64, gy = (C + 63) / 64;
  if (gx > 0x7fffffffL || gy > 65535) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated: %ld x %ld is beyond one launch", R, C);
  gs_gated_pack_t_kernel<T, PL><<<dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, s>>>((const E*)in, ldi, R, C, (P*)out, ldo, plane);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

// whether rows of `n` elements with stride ld can be read as they are
inline bool gf_plain(const void* p, long ld, long n) { return n % GF_PAD == 0 && ld % 8 == 0 && ((size_t)p & 15) == 0; }

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

template <int T, int PL, int ACT>
int gf_fwd(const GatedCall& c, hipStream_t s) {
  typedef typename GfPlane<T, PL>::type P;
  const GatedPlan p = gf_plan(c.M, c.D, c.F, T);
  P* sc = (P*)c.scratch;
  GatedGemm q = {};
  q.M = c.M; q.N = c.F; q.K = p.Dp;
  q.C[0] = c.h; q.ldc = c.ldh; q.rows0 = c.M;
  q.saved = c.saved;
  if (PL == 1 && gf_plain(c.x, c.ldx, c.D)) {
    q.A = c.x; q.lda = c.ldx;
  } else {
    q.A = sc + p.x; q.lda = p.Dp; q.plane_a = c.M * p.Dp;
    GS_TRY((gf_pack<T, PL>(c.x, c.ldx, c.M, c.D, sc + p.x, p.Dp, q.plane_a, s)));
  }
  if (PL == 1 && gf_plain(c.wg, c.ldw, c.D) && gf_plain(c.wu, c.ldw, c.D)) {
    q.B[0] = c.wg; q.B[1] = c.wu; q.ldb = c.ldw;
  } else {
    q.B[0] = sc + p.wg; q.B[1] = sc + p.wu; q.ldb = p.Dp; q.plane_b = c.F * p.Dp;
    GS_TRY((gf_pack<T, PL>(c.wg, c.ldw, c.F, c.D, sc + p.wg, p.Dp, q.plane_b, s)));
    GS_TRY((gf_pack<T, PL>(c.wu, c.ldw, c.F, c.D, sc + p.wu, p.Dp, q.plane_b, s)));
  }
  return gf_gemm<T, PL, true, ACT>(q, s);
}

template <int T, int PL, int ACT>
int gf_bwd(const GatedCall& c, hipStream_t s) {
  typedef typename GsElt<T>::type E;
  typedef typename GfPlane<T, PL>::type P;
  const GatedPlan p = gf_plan(c.M, c.D, c.F, T);
  P* sc = (P*)c.scratch;
  const long plane_r = c.M * 2 * p.Fp, plane_c = 2 * c.F * p.Mp, plane_w = c.D * 2 * p.Fp, plane_x = c.D * p.Mp;
  const long gx = p.Mp / 64, gy = p.Fp / 64;
  if (gx > 0x7fffffffL || gy > 65535) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_gated_bwd: %ld x %ld is beyond one launch", c.M, c.F);
  gs_gated_slopes_kernel<T, PL, ACT><<<dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, s>>>(
      (const E*)c.dh, c.lddh, c.saved, c.M, c.F, sc + p.rows, p.Fp, plane_r, sc + p.cols, p.Mp, plane_c);
  GS_LAUNCH_CHECK();
  GS_TRY((gf_pack_t<T, PL>(c.wg, c.ldw, c.F, c.D, sc + p.wt, 2 * p.Fp, plane_w, s)));
  GS_TRY((gf_pack_t<T, PL>(c.wu, c.ldw, c.F, c.D, sc + p.wt + p.Fp, 2 * p.Fp, plane_w, s)));
  GS_TRY((gf_pack_t<T, PL>(c.x, c.ldx, c.M, c.D, sc + p.xt, p.Mp, plane_x, s)));
  GatedGemm q = {};
  q.A = sc + p.rows; q.lda = 2 * p.Fp; q.plane_a = plane_r;
  q.B[0] = sc + p.wt; q.ldb = 2 * p.Fp; q.plane_b = plane_w;
  q.M = c.M; q.N = c.D; q.K = 2 * p.Fp;
  q.C[0] = c.dx; q.ldc = c.lddx; q.rows0 = c.M;
  GS_TRY((gf_gemm<T, PL, false, GS_ACT_SILU>(q, s)));
  q.A = sc + p.cols; q.lda = p.Mp; q.plane_a = plane_c;
  q.B[0] = sc + p.xt; q.ldb = p.Mp; q.plane_b = plane_x;
  q.M = 2 * c.F; q.N = c.D; q.K = p.Mp;
  q.C[0] = c.dwg; q.C[1] = c.dwu; q.ldc = c.lddw; q.rows0 = c.F;
  return gf_gemm<T, PL, false, GS_ACT_SILU>(q, s);
}

// dW = 0 where there are no tokens
template <typename E>
__global__ void gs_gated_zero_kernel(E* a, E* b, long R, long C, long ld) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= R * C) return;
  a[i / C * ld + i % C] = (E)0.f;
  b[i / C * ld + i % C] = (E)0.f;
}

template <int T>
int gf_empty(const GatedCall& c, hipStream_t s) {
  typedef typename GsElt<T>::type E;
  gs_gated_zero_kernel<E><<<dim3((unsigned)((c.F * c.D + 255) / 256)), dim3(256), 0, s>>>((E*)c.dwg, (E*)c.dwu, c.F, c.D, c.lddw);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

template <int T, int PL>
int gf_dispatch(const GatedCall& c, bool bwd, hipStream_t s) {
  if (bwd && c.M == 0) return gf_empty<T>(c, s);
  switch (c.act) {
    case GS_ACT_SILU: return bwd ? gf_bwd<T, PL, GS_ACT_SILU>(c, s) : gf_fwd<T, PL, GS_ACT_SILU>(c, s);
    case GS_ACT_GELU: return bwd ? gf_bwd<T, PL, GS_ACT_GELU>(c, s) : gf_fwd<T, PL, GS_ACT_GELU>(c, s);
    case GS_ACT_RELU: return bwd ? gf_bwd<T, PL, GS_ACT_RELU>(c, s) : gf_fwd<T, PL, GS_ACT_RELU>(c, s);
    default: return bwd ? gf_bwd<T, PL, GS_ACT_SIGMOID>(c, s) : gf_fwd<T, PL, GS_ACT_SIGMOID>(c, s);
  }
}

int gf_check(const char* who, const GatedCall& c, int type) {
  if (!gs_type_bytes(type)) GS_FAIL(GS_ERR_ARG, "%s: unknown element type %d", who, type);
  if (c.act < GS_ACT_SILU || c.act > GS_ACT_SIGMOID) GS_FAIL(GS_ERR_ARG, "%s: unknown activation %d", who, c.act);
  if (c.M < 0 || c.D < 1 || c.F < 1) GS_FAIL(GS_ERR_ARG, "%s: %ld rows, widths %ld and %ld", who, c.M, c.D, c.F);
  if (c.M > 0x7fffffffL || c.D > 0x3fffffffL || c.F > 0x3fffffffL) GS_FAIL(GS_ERR_UNSUPPORTED, "%s: sizes are counted in 32 bits", who);
  if (c.ldx < c.D || c.ldw < c.D) GS_FAIL(GS_ERR_ARG, "%s: a row stride is below the width %ld", who, c.D);
  return GS_OK;
}

int gf_run(const GatedCall& c, int type, bool bwd, hipStream_t s) {
  if (type == GS_TYPE_F32) return gf_dispatch<GS_TYPE_F32, 3>(c, bwd, s);
  if (type == GS_TYPE_F16) return gf_dispatch<GS_TYPE_F16, 1>(c, bwd, s);
  return gf_dispatch<GS_TYPE_BF16, 1>(c, bwd, s);
}

}  // namespace

extern "C" size_t gs_gated_fwd_scratch_bytes(long M, long D, long F, int type) {
  if (M < 0 || D < 1 || F < 1 || !gs_type_bytes(type)) return 0;
  return gf_plan(M, D, F, type).fwd * 2;
}

extern "C" size_t gs_gated_bwd_scratch_bytes(long M, long D, long F, int type) {
  if (M < 0 || D < 1 || F < 1 || !gs_type_bytes(type)) return 0;
  return gf_plan(M, D, F, type).bwd * 2;
}

extern "C" int gs_gated_fwd(const void* x, long ldx, const void* w_gate, const void* w_up, long ldw, int type, long M, long D, long F, int act,
                            void* h, long ldh, float* saved, void* scratch, gs_stream_t stream) {
  GatedCall c = {};
  c.x = x; c.wg = w_gate; c.wu = w_up; c.ldx = ldx; c.ldw = ldw; c.M = M; c.D = D; c.F = F; c.act = act;
  c.h = h; c.ldh = ldh; c.saved = saved; c.scratch = (char*)scratch;
  GS_TRY(gf_check("gs_gated_fwd", c, type));
  if (ldh < F) GS_FAIL(GS_ERR_ARG, "gs_gated_fwd: a row stride is below the width %ld", F);
  if (M == 0) return GS_OK;
  if (!x || !w_gate || !w_up || !h || !scratch) GS_FAIL(GS_ERR_ARG, "gs_gated_fwd: null pointer");
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
  if ((size_t)scratch & 15) GS_FAIL(GS_ERR_ARG, "gs_gated_bwd: the scratch is not 16-byte aligned");
  return gf_run(c, type, true, (hipStream_t)stream);
}
