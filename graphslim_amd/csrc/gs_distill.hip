// Distillation from a teacher's top logits.  A row has logits z over V classes and k entries (class c_j, teacher logit t_j); with
// p = softmax(t / tau) over the row's entries and q = softmax(z / tau) over all classes
//   loss = tau^2 sum_j p_j (log p_j - log q_{c_j}),      dz_i = w tau (q_i - sum_{j : c_j = i} p_j)      (w = d total / d loss).
// An entry whose class is none of the V, or whose logit is -inf, is not there; a row without entries (padding) has loss 0 and gradient 0.
// Everything is computed in fp32 and rounded once, on the gradient's store.
#include <algorithm>

#include "gs_types.h"

namespace {

constexpr int DS_MAX_TOP = 1024;
constexpr float DS_LOG2E = 1.4426950408889634f, DS_LOG2E_REST = (float)(1.4426950408889634 - (double)DS_LOG2E), DS_LN2 = 0.69314718055994531f;

struct DistillArgs {
  const void* Z;
  long ldz, n;
  int V, k;
  const void* tv;
  const int* ti;
  float tau, inv_hi, inv_lo;   // 1 / tau as a sum of two floats: z / tau enters differences with the log-sum, whose error is absolute
  float c_hi, c_lo;            // log2(e) / tau, too
  const float* lse_in;
  const float* w;
  float* loss;
  float* lse;
  void* dZ;
  long ldd;
};

// 2^(d (hi + lo)) for d <= 0.  FULL: with what the product d hi rounds away, up to 2^-24 |d hi| of the result; fp32 gradients show it,
// 16-bit ones do not, and there the exponentials are half of the time.
template <bool FULL>
__device__ __forceinline__ float ds_pow(float d, float hi, float lo) {
  const float t = d * hi, r = __builtin_amdgcn_exp2f(t);
  if constexpr (!FULL) return r;
  const float rest = fmaf(d, lo, fmaf(d, hi, -t));
  return t < -160.f ? 0.f : fmaf(r, rest * DS_LN2, r);
}
template <typename E>
__device__ __forceinline__ float ds_exp(float x) {
  return ds_pow<sizeof(E) == 4>(x, DS_LOG2E, DS_LOG2E_REST);
}

// log q = z / tau - lse; a masked class (-inf) stays at -inf whatever the log-sum is
__device__ __forceinline__ float ds_logq(const DistillArgs& a, float z, float lse) {
  return z == -INFINITY ? z : fmaf(z, a.inv_lo, fmaf(z, a.inv_hi, -lse));
}

// A barrier for what lies in LDS: loads of the row stay under way across it.
__device__ __forceinline__ void ds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A row is worked on by G threads (a wave, or a workgroup).  Reductions over them: the wave's, then one value a wave through LDS, with
// a slot for each reduction, so that one barrier does.
template <int G, bool MAX>
__device__ __forceinline__ float ds_reduce(float v, float* slot) {
  v = MAX ? gs_wave_max(v) : gs_wave_sum(v);
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    ds_barrier();
    v = slot[0];
#pragma unroll
    for (int i = 1; i < G / 64; ++i) v = MAX ? fmaxf(v, slot[i]) : v + slot[i];
  }
  return v;
}

// One row's teacher.  Every wave of the row finds out by itself whether there are any entries; the first one also keeps them in LDS
// and works out the loss and the gradient at their classes, while the others are at the row.
template <typename E>
struct DistillTeacher {
  static constexpr int WORDS = 4;   // of LDS per entry
  int* c;       // [k rounded up to 4] class or -1
  float* v;     // [k] t, then log p
  float* r;     // [k] gradient at the entry's class, if the entry is the first of that class
  int* at;      // [k] that class, else -1
  int c0;       // the first 64 entries: their loads come before the row's, so that they need not wait for it
  float v0;
  bool any;

  __device__ __forceinline__ DistillTeacher(void* lds, int k) {
    const int k4 = (k + 3) & ~3;
    c = (int*)lds;
    v = (float*)(c + k4);
    r = v + k4;
    at = (int*)(r + k4);
  }

  __device__ __forceinline__ void entry(const DistillArgs& a, long row, int j, int& cj, float& vj) {
    cj = -1;
    vj = -INFINITY;
    if (j < a.k) {
      cj = a.ti[row * a.k + j];
      vj = (float)((const E*)a.tv)[row * a.k + j];
    }
  }

  __device__ __forceinline__ void look(const DistillArgs& a, long row, int lane, bool first) {
    const int k4 = (a.k + 3) & ~3;
    bool have = false;
    float top = -INFINITY;
    for (int base = 0; base < k4; base += 64) {
      const int j = base + lane;
      int cj = c0;
      float vj = v0;
      if (base) entry(a, row, j, cj, vj);
      const bool ok = cj >= 0 && cj < a.V && vj != -INFINITY;
      have |= ok;
      if (first && j < k4) {
        c[j] = ok ? cj : -1;
        v[j] = vj;
        if (ok) top = fmaxf(top, vj);
      }
    }
    any = __ballot(have) != 0;
    if (!first) return;
    top = gs_wave_max(top);
    float s = 0.f;
    for (int j = lane; j < a.k; j += 64) {
      v[j] = (v[j] - top) / a.tau;                        // (in this order: t / tau may lie beyond fp32)
      if (c[j] >= 0) s += ds_exp<E>(v[j]);
    }
    const float log_sum = logf(gs_wave_sum(s));
    for (int j = lane; j < a.k; j += 64) v[j] -= log_sum;
  }

  // sum of p (log p - log q) over the entries, with log q = (z - m) / tau - log_s from the row's maximum m and its sum: the log-sum m / tau
  // + log_s may lie beyond fp32, or hold nothing of log_s
  __device__ __forceinline__ float loss(const DistillArgs& a, const E* z, int lane, float m, float log_s) {
    float s = 0.f;
    for (int j = lane; j < a.k; j += 64)
      if (c[j] >= 0) {
        const float p = ds_exp<E>(v[j]);
        const float zc = (float)z[c[j]], d = zc - m;
        float logq = fmaf(d, a.inv_lo, fmaf(d, a.inv_hi, -log_s));
        if (d == -INFINITY) logq = zc == -INFINITY ? zc : d - log_s;   // a masked class; a difference beyond fp32
        if (p != 0.f) s += p * (v[j] - logq);
      }
    return gs_wave_sum(s);
  }

  // The gradient at the entries' classes, w (q - sum of p over the entries of that class); before any of the row is written, since dz
  // may lie on z.
  template <typename QOf>
  __device__ __forceinline__ void slopes(const DistillArgs& a, const E* z, int lane, float w, QOf q_of) {
    for (int j = lane; j < a.k; j += 64) {
      const int cj = c[j];
      bool first = cj >= 0;
      if (first) {
        const float zc = (float)z[cj];
        float p = 0.f;
        for (int o = 0; o < a.k; o += 4) {
          const int4 four = *(const int4*)(c + o);
          const int cs[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (cs[e] == cj) {
              p += ds_exp<E>(v[o + e]);
              first &= o + e >= j;
            }
        }
        r[j] = w * (q_of(zc) - p);
      }
      at[j] = first ? cj : -1;
    }
  }

  __device__ __forceinline__ void store(const DistillArgs& a, E* d, int lane) const {
    for (int j = lane; j < a.k; j += 64)
      if (at[j] >= 0) d[at[j]] = (E)r[j];
  }
};

// The row in registers, EP logits a thread: read once, written once.  Bound by HBM: 8192 x 32000 bf16, loss and gradient, 1.05 GB, 195 us
// = 5.4 TB/s (more than a copy's 4.9: the logits are read once and the gradient written once, both past the caches); 454 x 40 fp32 12.5 us, a launch and its host call.
template <int T, int G, int EP, bool LOSS, bool GRAD, bool PAST>
__global__ __launch_bounds__(G < 256 ? 256 : G) void gs_distill_regs_kernel(DistillArgs a) {
  typedef typename GsElt<T>::type E;
  constexpr int N = 16 / sizeof(E), NV = EP / N, ROWS = G < 256 ? 256 / G : 1, W = G / 64;
  typedef typename GsVec<E, N>::type V;
  extern __shared__ __attribute__((aligned(16))) char sh[];
  __shared__ float red[2][W];
  const int g = threadIdx.x % G, sub = threadIdx.x / G, lane = threadIdx.x & 63, full = a.V / N;
  const bool first = g < 64;
  const long mine = (long)blockIdx.x * ROWS + sub;
  const bool live = mine < a.n;
  const long row = live ? mine : a.n - 1;
  const E* z = (const E*)a.Z + row * a.ldz;
  DistillTeacher<E> t(sh + (size_t)sub * ((a.k + 3) & ~3) * 4 * DistillTeacher<E>::WORDS, a.k);
  t.entry(a, row, lane, t.c0, t.v0);
  float w = 0.f;
  if (GRAD) w = a.w[row] * a.tau;
  V raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < N; ++e) raw[i][e] = (E)-INFINITY;
    if (i * G + g < full) raw[i] = PAST ? gs_load_past<E, N>(z + (long)(i * G + g) * N) : *(const V*)(z + (long)(i * G + g) * N);
  }
  float end = -INFINITY;                                  // what is left behind whole vectors: one element of the first lanes
  const bool has_end = g < a.V - full * N;
  if (has_end) end = (float)z[full * N + g];
  t.look(a, row, lane, first);
  float m = end;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) m = fmaxf(m, (float)raw[i][e]);
  m = ds_reduce<G, true>(m, red[0]);
  if (m == -INFINITY) m = 0.f;
  constexpr bool KEEP = sizeof(E) == 4;
  auto e_of = [&](float v) { return ds_pow<KEEP>(v - m, a.c_hi, a.c_lo); };   // (x - m first: x c - m c would be off by an ulp of m c)
  // fp32 rows keep the exponentials in place; 16-bit rows stay packed, half the registers, and are converted and raised again in each
  // pass (opaque in between, or the compiler keeps what it has seen, in 32 bits)
  auto hide = [&] {
    if constexpr (!KEEP) {
#pragma unroll
      for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(raw[i]));
    }
  };
  hide();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float v = e_of((float)raw[i][e]);
      if constexpr (KEEP) raw[i][e] = v;
      s += v;
    }
  end = e_of(end);
  s += end;
  s = ds_reduce<G, false>(s, red[1]);
  if (first) {
    const float log_s = logf(s), lse = m / a.tau + log_s;
    const float sum = t.loss(a, z, lane, m, log_s);
    if (lane == 0 && live) {
      a.loss[row] = t.any ? a.tau * a.tau * sum : 0.f;
      if (a.lse) a.lse[row] = lse;
    }
    if (GRAD) t.slopes(a, z, lane, w, [&](float zc) { return s == 0.f ? 0.f : e_of(zc) / s; });
  }
  if (!GRAD) return;
  E* d = (E*)a.dZ + row * a.ldd;
  const bool zero = !t.any || w == 0.f;
  const float ws = s == 0.f ? 0.f : w / s;                // (all logits -inf: q = 0)
  if (a.dZ == a.Z) __syncthreads();                       // in place: z has been read at the entries' classes
  if (live) {
    hide();
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * G + g < full) {
        V r;
#pragma unroll
        for (int e = 0; e < N; ++e) r[e] = (E)(zero ? 0.f : (KEEP ? (float)raw[i][e] : e_of((float)raw[i][e])) * ws);
        if constexpr (PAST) __builtin_nontemporal_store(r, (V*)(d + (long)(i * G + g) * N));
        else *(V*)(d + (long)(i * G + g) * N) = r;
      }
    if (has_end) d[full * N + g] = (E)(zero ? 0.f : end * ws);
  }
  __syncthreads();
  if (first && live && !zero) t.store(a, d, lane);
}

// Rows of any length, a workgroup each.  STATS: the log-sum is taken from z (a running maximum and sum per thread, one pass), else it is
// given.  Bound by HBM: losses, 2047 x 100003 fp16, 410 MB, 89 us = 4.6 TB/s; the gradient alone, 1024 x 50001 fp32, 411 MB,
// 101 us = 4.1 TB/s (rows of odd length: three of four are read and written across cache lines).
template <int T, int G, bool STATS, bool LOSS, bool GRAD>
__global__ __launch_bounds__(G) void gs_distill_row_kernel(DistillArgs a) {
  typedef typename GsElt<T>::type E;
  constexpr int N = 16 / sizeof(E), U = 4;
  typedef typename GsVec<E, N>::type V;
  extern __shared__ __attribute__((aligned(16))) char sh[];
  __shared__ float red[2][G / 64];
  const long row = blockIdx.x;
  const int g = threadIdx.x, lane = g & 63, full = a.V / N;
  const bool first = g < 64, has_end = g < a.V - full * N;
  const E* z = (const E*)a.Z + row * a.ldz;
  DistillTeacher<E> t(sh, a.k);
  t.entry(a, row, lane, t.c0, t.v0);
  float w = 0.f, lse = 0.f;
  if (GRAD) w = a.w[row] * a.tau;
  if (!STATS) lse = a.lse_in[row];
  t.look(a, row, lane, first);
  const bool zero = GRAD && (!t.any || w == 0.f);
  constexpr bool FULL = sizeof(E) == 4;
  float m = 0.f, s = 0.f, log_s = 0.f;
  if (STATS) {
    m = -INFINITY;
    auto add = [&](float mx, auto each) {                 // values whose maximum is mx
      mx = fmaxf(mx, m);
      const float ref = mx == -INFINITY ? 0.f : mx;
      s *= ds_pow<FULL>(m - ref, a.c_hi, a.c_lo);
      each(ref);
      m = mx;
    };
    for (int base = 0; base < full; base += U * G) {
      V r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int e = 0; e < N; ++e) r[u][e] = (E)-INFINITY;
        if (base + u * G + g < full) r[u] = *(const V*)(z + (long)(base + u * G + g) * N);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) mx = fmaxf(mx, (float)r[u][e]);
      add(mx, [&](float ref) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < N; ++e) s += ds_pow<FULL>((float)r[u][e] - ref, a.c_hi, a.c_lo);
      });
    }
    if (has_end) {
      const float v = (float)z[full * N + g];
      add(v, [&](float ref) { s += ds_pow<FULL>(v - ref, a.c_hi, a.c_lo); });
    }
    float all = ds_reduce<G, true>(m, red[0]);
    if (all == -INFINITY) all = 0.f;
    s = ds_reduce<G, false>(s * ds_pow<FULL>(m - all, a.c_hi, a.c_lo), red[1]);
    m = all;
    log_s = logf(s);
    lse = m / a.tau + log_s;
  }
  auto q_of = [&](float v) {
    if (STATS) return ds_pow<FULL>(v - m, a.c_hi, a.c_lo);
    return ds_pow<FULL>(fminf(ds_logq(a, v, lse), 0.f), DS_LOG2E, DS_LOG2E_REST);        // (a log-sum of 1e38 in fp32 is off by more than any exponent)
  };
  const float over = STATS ? (s == 0.f ? 0.f : 1.f / s) : (lse == -INFINITY ? 0.f : (lse == lse ? 1.f : lse)), ws = w * over;
  if (first) {
    if (LOSS) {
      const float sum = t.loss(a, z, lane, m, log_s);
      if (lane == 0) {
        a.loss[row] = t.any ? a.tau * a.tau * sum : 0.f;
        if (a.lse) a.lse[row] = lse;
      }
    }
    if (GRAD) t.slopes(a, z, lane, w, [&](float zc) { return q_of(zc) * over; });
  }
  if (!GRAD) return;
  E* d = (E*)a.dZ + row * a.ldd;
  if (a.dZ == a.Z) __syncthreads();                       // in place: z has been read at the entries' classes
  for (int base = 0; base < full; base += U * G) {
    V r[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (!zero && base + u * G + g < full) r[u] = *(const V*)(z + (long)(base + u * G + g) * N);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (base + u * G + g < full) {
        V o;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = (E)(zero ? 0.f : q_of((float)r[u][e]) * ws);
        *(V*)(d + (long)(base + u * G + g) * N) = o;
      }
  }
  if (has_end) d[full * N + g] = (E)(zero ? 0.f : q_of((float)z[full * N + g]) * ws);
  __syncthreads();
  if (first && !zero) t.store(a, d, lane);
}

inline size_t ds_lds(int k) { return (size_t)((k + 3) & ~3) * 4 * DistillTeacher<float>::WORDS; }

template <int T, int G, int EP, bool LOSS, bool GRAD>
void ds_regs(const DistillArgs& a, hipStream_t s) {
  constexpr int ROWS = G < 256 ? 256 / G : 1;
  const dim3 grid((unsigned)((a.n + ROWS - 1) / ROWS));
  if constexpr (GRAD && G >= 512) {
    // A gradient that the 256 MB cache cannot keep beside the logits goes past it, and so do they (8192 x 32000 bf16: 217 us through
    // the caches, 196 past them; 2048 x 32000 fp32: 116 and 104); a smaller one stays there for the products that read it next.
    if ((double)a.n * a.V * sizeof(typename GsElt<T>::type) > 128e6)
      return gs_distill_regs_kernel<T, G, EP, LOSS, GRAD, true><<<grid, dim3(G), ds_lds(a.k), s>>>(a);
  }
  gs_distill_regs_kernel<T, G, EP, LOSS, GRAD, false><<<grid, dim3(G < 256 ? 256 : G), ROWS * ds_lds(a.k), s>>>(a);
}

// Rows that fit the registers are read once; a wave works on the shortest.  Where a choice is left, the fewest threads: several rows
// on a compute unit overlap one's loads with another's arithmetic and barriers (8192 x 32000 bf16: 512 threads of 64 logits
// 196 us, 1024 of 32 238; 2048 x 60000: 512 of 128 109 us, 1024 of 64 160).  Longer rows, and losses alone, which gain nothing
// from holding a long row, are walked (1024 x 131072 bf16, loss and gradient: 128 us held, 159 us walked twice).
template <int T, bool LOSS, bool GRAD>
void ds_stats(const DistillArgs& a, hipStream_t s) {
  const bool few = a.k <= 256;                            // (four rows' entries in a workgroup's LDS)
  if (few && a.V <= 64 * 8) return ds_regs<T, 64, 8, LOSS, GRAD>(a, s);
  if (few && a.V <= 64 * 32) return ds_regs<T, 64, 32, LOSS, GRAD>(a, s);
  if (a.V <= 256 * 32) return ds_regs<T, 256, 32, LOSS, GRAD>(a, s);
  if (a.V <= 512 * 32) return ds_regs<T, 512, 32, LOSS, GRAD>(a, s);
  if (a.V <= 512 * 64) return ds_regs<T, 512, 64, LOSS, GRAD>(a, s);
  if constexpr (T == GS_TYPE_F32) {
    if (GRAD && a.V <= 1024 * 64) return ds_regs<T, 1024, 64, LOSS, GRAD>(a, s);
  } else {
    if (GRAD && a.V <= 512 * 128) return ds_regs<T, 512, 128, LOSS, GRAD>(a, s);
    if (GRAD && a.V <= 1024 * 128) return ds_regs<T, 1024, 128, LOSS, GRAD>(a, s);
  }
  gs_distill_row_kernel<T, 1024, true, LOSS, GRAD><<<dim3((unsigned)a.n), dim3(1024), ds_lds(a.k), s>>>(a);
}

// A launch has fewer than 2^32 threads, and a row takes up to 1024 of them: more rows go in bands
constexpr long DS_BAND = 1L << 21;

template <int T>
int ds_launch(const DistillArgs& all, hipStream_t s) {
  typedef typename GsElt<T>::type E;
  for (long at = 0; at < all.n; at += DS_BAND) {
    DistillArgs a = all;
    a.n = std::min(all.n - at, DS_BAND);
    a.Z = (const E*)all.Z + at * all.ldz;
    a.tv = (const E*)all.tv + at * all.k;
    a.ti = all.ti + at * all.k;
    if (all.lse_in) a.lse_in = all.lse_in + at;
    if (all.w) a.w = all.w + at;
    if (all.loss) a.loss = all.loss + at;
    if (all.lse) a.lse = all.lse + at;
    if (all.dZ) a.dZ = (E*)all.dZ + at * all.ldd;
    if (!a.dZ) ds_stats<T, true, false>(a, s);
    else if (a.loss) ds_stats<T, true, true>(a, s);
    else gs_distill_row_kernel<T, 512, false, false, true><<<dim3((unsigned)a.n), dim3(512), ds_lds(a.k), s>>>(a);
    GS_LAUNCH_CHECK();
  }
  return GS_OK;
}

int ds_run(const char* who, DistillArgs a, int type, long n, hipStream_t s) {
  if (!gs_type_bytes(type)) GS_FAIL(GS_ERR_ARG, "%s: unknown element type %d", who, type);
  if (n < 0 || a.V < 1 || a.k < 1) GS_FAIL(GS_ERR_ARG, "%s: %ld rows of %d classes, %d teacher entries", who, n, a.V, a.k);
  if (a.k > DS_MAX_TOP) GS_FAIL(GS_ERR_UNSUPPORTED, "%s: at most %d teacher entries a row (got %d)", who, DS_MAX_TOP, a.k);
  if (n > 0x7fffffffL) GS_FAIL(GS_ERR_UNSUPPORTED, "%s: rows are counted in 32 bits", who);
  if (!(a.tau > 0.f) || !(a.tau < INFINITY)) GS_FAIL(GS_ERR_ARG, "%s: temperature %g", who, (double)a.tau);
  if (a.ldz < a.V || (a.dZ && a.ldd < a.V)) GS_FAIL(GS_ERR_ARG, "%s: a row stride is below the %d classes", who, a.V);
  if (!(1.f / a.tau * DS_LOG2E < INFINITY)) GS_FAIL(GS_ERR_ARG, "%s: temperature %g has no reciprocal in fp32", who, (double)a.tau);
  if (a.dZ && a.dZ == a.Z && a.ldd != a.ldz) GS_FAIL(GS_ERR_ARG, "%s: in place with row strides %ld and %ld", who, a.ldz, a.ldd);
  if (n == 0) return GS_OK;
  if (!a.Z || !a.tv || !a.ti) GS_FAIL(GS_ERR_ARG, "%s: null pointer", who);
  const int e = gs_type_bytes(type);
  const GsSpan z = gs_span(a.Z, n, a.ldz, a.V, e), dz = gs_span(a.dZ, n, a.ldd, a.V, e);
  const GsSpan in[] = {gs_span(a.tv, n * a.k, e), gs_span(a.ti, n * a.k, 4), gs_span(a.lse_in, n, 4), gs_span(a.w, n, 4)};
  const GsSpan out[] = {dz, gs_span(a.loss, n, 4), gs_span(a.lse, n, 4)};
  bool clash = a.dZ != a.Z && gs_overlap(dz, z);
  for (int o = 0; o < 3; ++o) {
    clash |= o > 0 && gs_overlap(out[o], z);
    for (const GsSpan& i : in) clash |= gs_overlap(out[o], i);
    for (int q = 0; q < o; ++q) clash |= gs_overlap(out[o], out[q]);
  }
  if (clash) GS_FAIL(GS_ERR_ARG, "%s: an output lies on another operand (only dZ may, on all of Z)", who);
  a.inv_hi = 1.f / a.tau;
  a.inv_lo = (float)(1.0 / (double)a.tau - (double)a.inv_hi);
  a.c_hi = (float)(1.4426950408889634 / (double)a.tau);
  a.c_lo = (float)(1.4426950408889634 / (double)a.tau - (double)a.c_hi);
  if (type == GS_TYPE_F32) return ds_launch<GS_TYPE_F32>(a, s);
  if (type == GS_TYPE_F16) return ds_launch<GS_TYPE_F16>(a, s);
  return ds_launch<GS_TYPE_BF16>(a, s);
}

}  // namespace

extern "C" int gs_distill_fwd(const void* Z, long ldz, int type, long n, int V, const void* top_val, const int* top_cls, int k, float tau,
                              float* loss, float* lse, gs_stream_t stream) {
  if (n > 0 && (!loss || !lse)) GS_FAIL(GS_ERR_ARG, "gs_distill_fwd: null pointer");
  DistillArgs a = {Z, ldz, n, V, k, top_val, top_cls, tau, 0.f, 0.f, 0.f, 0.f, nullptr, nullptr, loss, lse, nullptr, 0};
  return ds_run("gs_distill_fwd", a, type, n, (hipStream_t)stream);
}

extern "C" int gs_distill_bwd(const void* Z, long ldz, int type, long n, int V, const void* top_val, const int* top_cls, int k, float tau,
                              const float* lse, const float* d_loss, void* dZ, long ldd, gs_stream_t stream) {
  if (n > 0 && (!lse || !d_loss || !dZ)) GS_FAIL(GS_ERR_ARG, "gs_distill_bwd: null pointer");
  DistillArgs a = {Z, ldz, n, V, k, top_val, top_cls, tau, 0.f, 0.f, 0.f, 0.f, lse, d_loss, nullptr, nullptr, dZ, ldd};
  return ds_run("gs_distill_bwd", a, type, n, (hipStream_t)stream);
}

extern "C" int gs_distill_loss_grad(const void* Z, long ldz, int type, long n, int V, const void* top_val, const int* top_cls, int k,
                                    float tau, const float* d_loss, float* loss, void* dZ, long ldd, gs_stream_t stream) {
  if (n > 0 && (!d_loss || !loss || !dZ)) GS_FAIL(GS_ERR_ARG, "gs_distill_loss_grad: null pointer");
  DistillArgs a = {Z, ldz, n, V, k, top_val, top_cls, tau, 0.f, 0.f, 0.f, 0.f, nullptr, d_loss, loss, nullptr, dZ, ldd};
  return ds_run("gs_distill_loss_grad", a, type, n, (hipStream_t)stream);
}
