// Distillation from a teacher's top logits.  A row has logits z over V classes and k entries (class c_j, teacher logit t_j); with
// p = softmax(t / tau) over the row's entries and q = softmax(z / tau) over all classes
//   loss = tau^2 sum_j p_j (log p_j - log q_{c_j}),      dz_i = w tau (q_i - sum_{j : c_j = i} p_j)      (w = d total / d loss).
// An entry whose class is none of the V, or whose logit is -inf, is not there; a row without entries (padding) has loss 0 and gradient 0.
// Everything is computed in fp32 and rounded once, on the gradient's store.
#include "gs_types.h"

namespace {

constexpr int DS_MAX_TOP = 1024;
constexpr float DS_LOG2E = 1.4426950408889634f;

struct DistillArgs {
  const void* Z;
  long ldz;
  int V, k;
  const void* tv;
  const int* ti;
  float tau, inv_hi, inv_lo;   // 1 / tau as a sum of two floats: z / tau enters differences with the log-sum, whose error is absolute
  const float* lse_in;
  const float* w;
  float* loss;
  float* lse;
  void* dZ;
  long ldd;
};

template <int OP>   // 0 sum, 1 max
__device__ __forceinline__ float ds_reduce(float v, float* sh) {
  v = OP ? gs_wave_max(v) : gs_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (int i = 1; i < (int)(blockDim.x >> 6); ++i) v = OP ? fmaxf(v, sh[i]) : v + sh[i];
  return v;
}

// log q = z / tau - lse; a masked class (-inf) stays at -inf whatever the log-sum is
__device__ __forceinline__ float ds_logq(const DistillArgs& a, float z, float lse) {
  return z == -INFINITY ? z : fmaf(z, a.inv_lo, fmaf(z, a.inv_hi, -lse));
}

__device__ __forceinline__ float ds_exp(float x) { return __builtin_amdgcn_exp2f(x * DS_LOG2E); }

// One workgroup per row.  STATS: the log-sum is taken from z (a running maximum and sum per thread, one pass), else it is given.
template <int T, bool STATS, bool LOSS, bool GRAD>
__global__ __launch_bounds__(256) void gs_distill_row_kernel(DistillArgs a) {
  typedef typename GsElt<T>::type E;
  constexpr int N = 16 / sizeof(E);
  extern __shared__ float sh_top[];   // p [k], class [k]
  __shared__ float red[4];
  float* sp = sh_top;
  int* si = (int*)(sh_top + a.k);
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  const E* z = (const E*)a.Z + row * a.ldz;
  // the teacher's softmax
  float tm = -INFINITY, any = 0.f;
  for (int j = tid; j < a.k; j += 256) {
    const int c = a.ti[row * a.k + j];
    const float v = (float)((const E*)a.tv)[row * a.k + j] / a.tau;
    const bool there = c >= 0 && c < a.V && v != -INFINITY;
    si[j] = there ? c : -1;
    sp[j] = there ? v : -INFINITY;
    if (there) { any = 1.f; tm = fmaxf(tm, v); }
  }
  tm = ds_reduce<1>(tm, red);
  any = ds_reduce<1>(any, red);
  float ts = 0.f;
  for (int j = tid; j < a.k; j += 256)
    if (si[j] >= 0) ts += ds_exp(sp[j] - tm);
  ts = ds_reduce<0>(ts, red);
  const float lts = logf(ts);
  float w = 0.f;
  if (GRAD) w = a.w[row] * a.tau;
  // the student's log-sum
  float m = -INFINITY, s = 0.f, lse = 0.f;
  if (STATS) {
    for (long f = (long)tid * N; f < a.V; f += 256 * N) {
      float v[N];
      gs_load<E, N>(z + f, a.V - f, -INFINITY, v);
      float mx = v[0];
#pragma unroll
      for (int i = 1; i < N; ++i) mx = fmaxf(mx, v[i]);
      mx = fmaxf(mx, m);
      const float ref = mx == -INFINITY ? 0.f : mx;
      s *= ds_exp((m - ref) * a.inv_hi);
#pragma unroll
      for (int i = 0; i < N; ++i) s += ds_exp((v[i] - ref) * a.inv_hi);
      m = mx;
    }
    const float all = ds_reduce<1>(m, red);
    const float ref = all == -INFINITY ? 0.f : all;
    s = ds_reduce<0>(s * ds_exp((m - ref) * a.inv_hi), red);
    lse = ref / a.tau + logf(s);
    m = ref;
  } else {
    lse = a.lse_in[row];
  }
  if (LOSS) {
    float sum = 0.f;
    for (int j = tid; j < a.k; j += 256)
      if (si[j] >= 0) {
        const float lp = sp[j] - tm - lts, p = ds_exp(sp[j] - tm) / ts;
        if (p != 0.f) sum += p * (lp - ds_logq(a, (float)z[si[j]], lse));
      }
    sum = ds_reduce<0>(sum, red);
    if (tid == 0) {
      a.loss[row] = any ? a.tau * a.tau * sum : 0.f;
      if (a.lse) a.lse[row] = lse;
    }
  }
  if (!GRAD) return;
  E* d = (E*)a.dZ + row * a.ldd;
  const bool zero = any == 0.f || w == 0.f;
  // the entries' gradients, before any of the row is written (dz may lie on z); of equal classes the first one holds the sum
  float mine[DS_MAX_TOP / 256];
  int at[DS_MAX_TOP / 256];
#pragma unroll
  for (int q = 0; q < DS_MAX_TOP / 256; ++q) {
    const int j = tid + q * 256;
    at[q] = -1;
    if (j < a.k && !zero && si[j] >= 0) {
      const int c = si[j];
      float p = 0.f;
      bool first = true;
      for (int o = 0; o < a.k; ++o)
        if (si[o] == c) {
          p += ds_exp(sp[o] - tm) / ts;
          first &= o >= j;
        }
      const float zc = (float)z[c];
      const float qc = lse == -INFINITY ? 0.f
                       : STATS          ? ds_exp((zc - m) * a.inv_hi) / s
                                        : ds_exp(ds_logq(a, zc, lse));
      mine[q] = w * (qc - p);
      if (first) at[q] = c;
    }
  }
  __syncthreads();
  const float ws = STATS ? (s == 0.f ? 0.f : w / s) : w;
  for (long f = (long)tid * N; f < a.V; f += 256 * N) {
    float v[N];
    gs_load<E, N>(z + f, a.V - f, 0.f, v);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (zero || lse == -INFINITY) v[i] = 0.f;
      else if (STATS) v[i] = ws * ds_exp((v[i] - m) * a.inv_hi);
      else v[i] = ws * ds_exp(ds_logq(a, v[i], lse));
    }
    gs_store<E, N>(d + f, a.V - f, v);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < DS_MAX_TOP / 256; ++q)
    if (at[q] >= 0) d[at[q]] = (E)mine[q];
}

template <int T>
int ds_launch(const DistillArgs& a, long n, hipStream_t s) {
  const dim3 grid((unsigned)n), block(256);
  const size_t lds = (size_t)a.k * 8;
  if (!a.dZ) gs_distill_row_kernel<T, true, true, false><<<grid, block, lds, s>>>(a);
  else if (a.loss) gs_distill_row_kernel<T, true, true, true><<<grid, block, lds, s>>>(a);
  else gs_distill_row_kernel<T, false, false, true><<<grid, block, lds, s>>>(a);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

int ds_run(const char* who, DistillArgs a, int type, long n, hipStream_t s) {
  if (!gs_type_bytes(type)) GS_FAIL(GS_ERR_ARG, "%s: unknown element type %d", who, type);
  if (n < 0 || a.V < 1 || a.k < 1) GS_FAIL(GS_ERR_ARG, "%s: %ld rows of %d classes, %d teacher entries", who, n, a.V, a.k);
  if (a.k > DS_MAX_TOP) GS_FAIL(GS_ERR_UNSUPPORTED, "%s: at most %d teacher entries a row (got %d)", who, DS_MAX_TOP, a.k);
  if (n > 0x7fffffffL) GS_FAIL(GS_ERR_UNSUPPORTED, "%s: rows are counted in 32 bits", who);
  if (!(a.tau > 0.f) || !(a.tau < INFINITY)) GS_FAIL(GS_ERR_ARG, "%s: temperature %g", who, (double)a.tau);
  if (a.ldz < a.V || (a.dZ && a.ldd < a.V)) GS_FAIL(GS_ERR_ARG, "%s: a row stride is below the %d classes", who, a.V);
  if (n == 0) return GS_OK;
  if (!a.Z || !a.tv || !a.ti) GS_FAIL(GS_ERR_ARG, "%s: null pointer", who);
  a.inv_hi = 1.f / a.tau;
  a.inv_lo = (float)(1.0 / (double)a.tau - (double)a.inv_hi);
  if (type == GS_TYPE_F32) return ds_launch<GS_TYPE_F32>(a, n, s);
  if (type == GS_TYPE_F16) return ds_launch<GS_TYPE_F16>(a, n, s);
  return ds_launch<GS_TYPE_BF16>(a, n, s);
}

}  // namespace

extern "C" int gs_distill_fwd(const void* Z, long ldz, int type, long n, int V, const void* top_val, const int* top_cls, int k, float tau,
                              float* loss, float* lse, gs_stream_t stream) {
  if (n > 0 && (!loss || !lse)) GS_FAIL(GS_ERR_ARG, "gs_distill_fwd: null pointer");
  DistillArgs a = {Z, ldz, V, k, top_val, top_cls, tau, 0.f, 0.f, nullptr, nullptr, loss, lse, nullptr, 0};
  return ds_run("gs_distill_fwd", a, type, n, (hipStream_t)stream);
}

extern "C" int gs_distill_bwd(const void* Z, long ldz, int type, long n, int V, const void* top_val, const int* top_cls, int k, float tau,
                              const float* lse, const float* d_loss, void* dZ, long ldd, gs_stream_t stream) {
  if (n > 0 && (!lse || !d_loss || !dZ)) GS_FAIL(GS_ERR_ARG, "gs_distill_bwd: null pointer");
  DistillArgs a = {Z, ldz, V, k, top_val, top_cls, tau, 0.f, 0.f, lse, d_loss, nullptr, nullptr, dZ, ldd};
  return ds_run("gs_distill_bwd", a, type, n, (hipStream_t)stream);
}

extern "C" int gs_distill_loss_grad(const void* Z, long ldz, int type, long n, int V, const void* top_val, const int* top_cls, int k,
                                    float tau, const float* d_loss, float* loss, void* dZ, long ldd, gs_stream_t stream) {
  if (n > 0 && (!d_loss || !loss || !dZ)) GS_FAIL(GS_ERR_ARG, "gs_distill_loss_grad: null pointer");
  DistillArgs a = {Z, ldz, V, k, top_val, top_cls, tau, 0.f, 0.f, nullptr, d_loss, loss, nullptr, dZ, ldd};
  return ds_run("gs_distill_loss_grad", a, type, n, (hipStream_t)stream);
}
