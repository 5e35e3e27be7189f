// Embedding lookup with scaling, and the gradient of its table:
//   out[t] = s W[id_t]              (0 where id_t is no row of the table: padding)
//   dW[v]  = s sum_{t : id_t = v} dOut[t], the tokens in ascending order, in fp32, rounded once.
#include "gs_types.h"

namespace {

// One thread takes 16 bytes of one output row.
template <int T>
__global__ __launch_bounds__(256) void gs_embedding_fwd_kernel(const typename GsElt<T>::type* __restrict__ W, long ldw, long V, int F,
                                                               const int* __restrict__ ids, long n, float scale,
                                                               typename GsElt<T>::type* __restrict__ out, long ldo, int pieces) {
  typedef typename GsElt<T>::type E;
  constexpr int N = 16 / sizeof(E);
  const long c = (long)blockIdx.x * 256 + threadIdx.x;
  const long t = c / pieces;
  if (t >= n) return;
  const int f = (int)(c - t * pieces) * N;
  const long id = ids[t];
  float v[N];
  if (id >= 0 && id < V) {
    gs_load<E, N>(W + id * ldw + f, F - f, 0.f, v);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= scale;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
  }
  gs_store<E, N>(out + t * ldo + f, F - f, v);
}

// One wave per (table row, 64 N columns): it walks all ids and adds the rows of its own, in order.
template <int T, int TO>
__global__ __launch_bounds__(256) void gs_embedding_bwd_kernel(const typename GsElt<T>::type* __restrict__ dout, long ldd,
                                                               const int* __restrict__ ids, long n, long V, int F, float scale,
                                                               int accumulate, typename GsElt<TO>::type* __restrict__ dW, long ldw) {
  typedef typename GsElt<T>::type E;
  typedef typename GsElt<TO>::type EO;
  constexpr int N = 16 / sizeof(E);
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= V) return;
  const int f = (blockIdx.y * 64 + lane) * N;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (long base = 0; base < n; base += 64) {
    unsigned long long hit = __ballot(base + lane < n && ids[min(base + lane, n - 1)] == row);
    while (hit) {
      const long t = base + __ffsll(hit) - 1;
      hit &= hit - 1;
      if (f < F) {
        float v[N];
        gs_load<E, N>(dout + t * ldd + f, F - f, 0.f, v);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += v[i];
      }
    }
  }
  if (f >= F) return;
  EO* o = dW + row * ldw + f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    acc[i] *= scale;
    if (accumulate && f + i < F) acc[i] += (float)o[i];
  }
  gs_store<EO, N>(o, F - f, acc);
}

template <int T>
int emb_fwd(const void* W, long ldw, long V, int F, const int* ids, long n, float scale, void* out, long ldo, hipStream_t s) {
  typedef typename GsElt<T>::type E;
  const int pieces = gs_cdiv(F, 16 / sizeof(E));
  const long blocks = (n * pieces + 255) / 256;
  if (blocks > 0x7fffffffL) GS_FAIL(GS_ERR_UNSUPPORTED, "gs_embedding_fwd: %ld x %d is beyond one launch", n, F);
  gs_embedding_fwd_kernel<T><<<dim3((unsigned)blocks), dim3(256), 0, s>>>((const E*)W, ldw, V, F, ids, n, scale, (E*)out, ldo, pieces);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

template <int T, int TO>
int emb_bwd(const void* dout, long ldd, const int* ids, long n, long V, int F, float scale, int accumulate, void* dW, long ldw,
            hipStream_t s) {
  typedef typename GsElt<T>::type E;
  const dim3 grid((unsigned)gs_cdiv(V, 4), (unsigned)gs_cdiv(F, 64 * 16 / sizeof(E)));
  gs_embedding_bwd_kernel<T, TO><<<grid, dim3(256), 0, s>>>((const E*)dout, ldd, ids, n, V, F, scale, accumulate,
                                                          (typename GsElt<TO>::type*)dW, ldw);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

int emb_check(const char* who, long n, long V, int F, int type, long ld0, long ld1) {
  if (!gs_type_bytes(type)) GS_FAIL(GS_ERR_ARG, "%s: unknown element type %d", who, type);
  if (n < 0 || V < 1 || F < 1) GS_FAIL(GS_ERR_ARG, "%s: %ld ids, a table of %ld x %d", who, n, V, F);
  if (V > 0x7fffffffL || n > 0x7fffffffL) GS_FAIL(GS_ERR_UNSUPPORTED, "%s: ids and rows are counted in 32 bits", who);
  if (ld0 < F || ld1 < F) GS_FAIL(GS_ERR_ARG, "%s: a row stride is below the width %d", who, F);
  return GS_OK;
}

}  // namespace

extern "C" int gs_embedding_fwd(const void* W, long ldw, long V, int F, int type, const int* ids, long n, float scale, void* out, long ldo,
                                gs_stream_t stream) {
  GS_TRY(emb_check("gs_embedding_fwd", n, V, F, type, ldw, ldo));
  if (n == 0) return GS_OK;
  if (!W || !ids || !out) GS_FAIL(GS_ERR_ARG, "gs_embedding_fwd: null pointer");
  hipStream_t s = (hipStream_t)stream;
  if (type == GS_TYPE_F32) return emb_fwd<GS_TYPE_F32>(W, ldw, V, F, ids, n, scale, out, ldo, s);
  if (type == GS_TYPE_F16) return emb_fwd<GS_TYPE_F16>(W, ldw, V, F, ids, n, scale, out, ldo, s);
  return emb_fwd<GS_TYPE_BF16>(W, ldw, V, F, ids, n, scale, out, ldo, s);
}

extern "C" size_t gs_embedding_bwd_scratch_bytes(long n, long V, int F) { return 0; }

extern "C" int gs_embedding_bwd(const void* dout, long ldd, int type, const int* ids, long n, long V, int F, float scale, int accumulate,
                                void* dW, long ldw, int type_dw, void* scratch, gs_stream_t stream) {
  GS_TRY(emb_check("gs_embedding_bwd", n, V, F, type, ldd, ldw));
  if (type_dw != type && type_dw != GS_TYPE_F32)
    GS_FAIL(GS_ERR_ARG, "gs_embedding_bwd: the gradient is held in the type of d_out or in fp32 (got %d for %d)", type_dw, type);
  if (!dW || (n > 0 && (!dout || !ids))) GS_FAIL(GS_ERR_ARG, "gs_embedding_bwd: null pointer");
  hipStream_t s = (hipStream_t)stream;
  if (type == GS_TYPE_F32) return emb_bwd<GS_TYPE_F32, GS_TYPE_F32>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, s);
  if (type == GS_TYPE_F16)
    return type_dw == GS_TYPE_F16 ? emb_bwd<GS_TYPE_F16, GS_TYPE_F16>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, s)
                                  : emb_bwd<GS_TYPE_F16, GS_TYPE_F32>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, s);
  return type_dw == GS_TYPE_BF16 ? emb_bwd<GS_TYPE_BF16, GS_TYPE_BF16>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, s)
                                 : emb_bwd<GS_TYPE_BF16, GS_TYPE_F32>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, s);
}
