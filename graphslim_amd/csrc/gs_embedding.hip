// Embedding lookup with scaling, and the gradient of its table:
//   out[t] = s W[id_t]              (0 where id_t is no row of the table: padding)
//   dW[v]  = s sum_{t : id_t = v} dOut[t], in fp32, rounded once: sums of consecutive tokens, in ascending order, added in their order.
// Where a row's tokens are cut follows from the ids and the sizes, so two runs are bitwise equal.
#include <algorithm>

#include "gs_types.h"

namespace {

// Bound by HBM: the distinct rows are read, all output rows written, and the scale costs nothing beside that.  One thread takes two 16-byte
// pieces of output rows, half of all pieces apart, so that two dependent loads (id, row) are under way; the piece's row comes from a
// 32-bit division, since one in 64 bits costs more than the piece's traffic.
// 16383 ids, 50001 x 602 fp32: 11.3 us = 4.7 TB/s (a large copy reaches 4.9); 8 ids, 32000 x 1024 bf16: 8 us, a launch and its host call.
template <int T>
__global__ __launch_bounds__(256) void gs_embedding_fwd_kernel(const typename GsElt<T>::type* __restrict__ W, long ldw, long V, int F,
                                                               const int* __restrict__ ids, unsigned total, float scale,
                                                               typename GsElt<T>::type* __restrict__ out, long ldo, unsigned pieces) {
  typedef typename GsElt<T>::type E;
  constexpr int N = 16 / sizeof(E);
  const unsigned half = (total + 1) / 2, c0 = blockIdx.x * 256u + threadIdx.x;
  if (c0 >= half) return;
  float v[2][N];
  unsigned t[2];
  int f[2];
  long id[2];
  bool on[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned c = c0 + i * half;
    on[i] = c < total;
    t[i] = on[i] ? c / pieces : 0;
    f[i] = on[i] ? (int)(c - t[i] * pieces) * N : 0;
    id[i] = ids[t[i]];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[i][e] = 0.f;
    if (id[i] >= 0 && id[i] < V) gs_load<E, N>(W + id[i] * ldw + f[i], F - f[i], 0.f, v[i]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[i][e] *= scale;
    if (on[i]) gs_store<E, N>(out + t[i] * ldo + f[i], F - f[i], v[i]);
  }
}

// ---- the gradient ---------------------------------------------------------------------------------------------------------------
// The table is cut into buckets of R consecutive rows.  The tokens of a bucket, sorted by row (stable, so ascending within a row), are
// walked by the waves of one workgroup, each on columns of its own: a run of one row is summed in registers and written once, rows
// without tokens are written as zeros.
//   few tokens:  one launch, every workgroup picks its bucket's tokens out of all ids itself.
//   many:        gs_embedding_count / _place sort the tokens by bucket first; a bucket of more than EM_SPAN tokens (a frequent id) is
//                cut into spans with a workgroup each, whose sums gs_embedding_join adds in the spans' order.
constexpr int EM_TILE = 4096;      // ids per workgroup of the sort: four a thread, all loaded at once
// Tokens of a bucket per workgroup: fewer make more partial sums, more a longer walk of a frequent row (bf16, 30000 ids on 300 x 2000:
// 128, 256 and 512 tokens 62, 55 and 70 us; 32768 ids on 128000 x 2048: 169, 170 and 176 us).
constexpr int EM_SPAN = 256;
// Tiles up to which the sort's workgroups each add up all tiles' counts; beyond, a launch of its own makes prefix sums of them, since the
// adding grows with the square of the tokens (32000 rows of 16, fp32: 140 000 tokens 32 us either way, 1 000 000 100 against 92,
// 4 000 000 490 against 307).
constexpr int EM_SCAN = 64;
constexpr int EM_MAX_BUCKETS = 2048;
constexpr int EM_MAX_R = 1024;     // rows of a bucket at most
constexpr long EM_MAX_V = (long)EM_MAX_R * EM_MAX_BUCKETS;
constexpr long EM_FEW = 512;       // ids up to which many small workgroups do it: writing the empty rows is all the work (78 us = 5.3 TB/s
                                   // for 16 ids on 50000 x 2048 fp32)
constexpr long EM_DIRECT = 8192;   // tokens up to which one launch does it all (every workgroup reads all ids, 32 KB from its L2; three
                                   // launches more cost 10 us: 8192 ids on 32000 x 1024 bf16 take 31)

struct EmbPlan {
  int R, nb, nbp;      // rows per bucket (sorted: a power of two), buckets, rounded up to 8
  int tiles, extra;    // sort tiles; workgroups for the second and further spans
  bool direct;
  size_t cnt, start, xs, owner, list, ptrs, part, bytes;
};

EmbPlan emb_plan(long n, long V, int F) {
  EmbPlan p;
  p.direct = n <= EM_DIRECT;
  if (p.direct) {        // a bucket for each compute unit (few ids: four), of up to 64 rows
    p.R = (int)std::min(std::max(gs_cdiv(V, n <= EM_FEW ? 1024 : 256), 4), 64);
  } else {
    p.R = 4;
    while ((V + p.R - 1) / p.R > 1024 && p.R < 64) p.R *= 2;
    while ((V + p.R - 1) / p.R > EM_MAX_BUCKETS) p.R *= 2;
  }
  p.nb = gs_cdiv(V, p.R);
  p.tiles = gs_cdiv(n, EM_TILE);
  p.extra = (int)(n / EM_SPAN);
  size_t o = 0;
  auto take = [&](size_t bytes) { size_t at = o; o += (bytes + 255) / 256 * 256; return at; };
  p.nbp = (p.nb + 7) / 8 * 8;
  p.cnt = take((size_t)(p.tiles + 1) * p.nbp * 4);
  p.start = take((size_t)(p.nb + 1) * 4);
  p.xs = take((size_t)(p.nb + 1) * 4);
  p.owner = take((size_t)p.extra * 4);
  p.list = take((size_t)n * 8);
  p.ptrs = take((size_t)2 * p.extra * p.R * 4);
  p.part = take((size_t)2 * p.extra * (p.R < EM_SPAN ? p.R : EM_SPAN) * F * 4);
  p.bytes = p.direct ? 0 : o;
  return p;
}

// lanes of this wave whose `key` (below 2^bits) is mine, among those with `on`
__device__ __forceinline__ unsigned long long emb_match(int key, bool on, int bits) {
  unsigned long long m = __ballot(on);
  for (int b = 0; b < bits; ++b) {
    const bool set = (key >> b) & 1;
    const unsigned long long have = __ballot(set);
    m &= set ? have : ~have;
  }
  return m;
}

// an id's row in the V rows from id0 on, or -1
__device__ __forceinline__ int emb_row(int id, long id0, long V) {
  const long r = (long)id - id0;
  return id >= 0 && r >= 0 && r < V ? (int)r : -1;
}

// cnt[tile][bucket]: tokens of the tile in the bucket (rows of nbp = nb rounded up to 8 counts)
__global__ __launch_bounds__(1024) void gs_embedding_count_kernel(const int* __restrict__ ids, long n, long id0, long V, int rshift, int nbp,
                                                                  int* __restrict__ cnt) {
  __shared__ int h[EM_MAX_BUCKETS];
  constexpr int Q = EM_TILE / 1024;
  const long t0 = (long)blockIdx.x * EM_TILE;
  int id[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const long t = t0 + i * 1024 + threadIdx.x;
    id[i] = t < n ? emb_row(ids[t], id0, V) : -1;
  }
  for (int b = threadIdx.x; b < nbp; b += 1024) h[b] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q; ++i)
    if (id[i] >= 0) atomicAdd(&h[id[i] >> rshift], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < nbp; b += 1024) cnt[(long)blockIdx.x * nbp + b] = h[b];
}

// cnt[tile][bucket] becomes the count of the tiles before, cnt[tiles][bucket] that of all.  A workgroup takes 64 buckets, its waves
// consecutive parts of the tiles: every part is summed, then walked again from the sum of the parts before it.
__global__ __launch_bounds__(1024) void gs_embedding_scan_kernel(int* __restrict__ cnt, int tiles, int nbp) {
  __shared__ int sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.x * 64 + lane;
  const int per = (tiles + 15) / 16, t0 = min(wave * per, tiles), t1 = min(t0 + per, tiles);
  const bool on = b < nbp;
  int* c = cnt + b;
  int sum = 0;
  if (on) {
#pragma unroll 8
    for (int t = t0; t < t1; ++t) sum += c[(long)t * nbp];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (!on) return;
  int run = 0;
  for (int w = 0; w < wave; ++w) run += sums[w][lane];
  for (int t = t0; t < t1; t += 8) {
    int v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c[(long)min(t + j, t1 - 1) * nbp];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (t + j < t1) {
        c[(long)(t + j) * nbp] = run;
        run += v[j];
      }
  }
  if (wave == 15) c[(long)tiles * nbp] = run;
}

// Stable: a tile's place in a bucket follows from the counts of the tiles before it, a wave's from those of the waves before it, a
// lane's from the lanes before it.  start[b]: where bucket b begins in the list; xs[b]: further spans of the buckets before b; owner[e]:
// the bucket of further span e, or -1.
__global__ __launch_bounds__(1024) void gs_embedding_place_kernel(const int* __restrict__ ids, long n, long id0, long V, int rshift, int nb, int nbp,
                                                                  int bits, const int* __restrict__ cnt, int tiles,
                                                                  int* __restrict__ start, int* __restrict__ xs, int* __restrict__ owner,
                                                                  int extra, int2* __restrict__ list) {
  constexpr int W = 16, Q = EM_TILE / 1024, PER = EM_MAX_BUCKETS / 1024;
  static_assert(PER == 2 && EM_TILE < 65536, "two buckets a thread; places within a tile in 16 bits");
  __shared__ unsigned short pos[W][EM_MAX_BUCKETS];   // per wave: the next place of each bucket, from the tile's first one
  __shared__ int first[EM_MAX_BUCKETS];
  __shared__ int wsum[W], wext[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long t0 = (long)blockIdx.x * EM_TILE + wave * (EM_TILE / W) + lane;
  int id[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    id[i] = t0 + i * 64 < n ? emb_row(ids[t0 + i * 64], id0, V) : -1;
  }
  int before[PER] = {}, all[PER] = {};
  if (tid * PER < nbp && tiles > EM_SCAN) {
    const int2* c = (const int2*)cnt + tid;
    const int2 u = c[(long)blockIdx.x * (nbp / 2)], v = c[(long)tiles * (nbp / 2)];
    before[0] = u.x;
    before[1] = u.y;
    all[0] = v.x;
    all[1] = v.y;
  } else if (tid * PER < nbp) {
    const int2* c = (const int2*)cnt + tid;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
      const int2 u = c[(long)t * (nbp / 2)];
      const bool low = t < (int)blockIdx.x;
      all[0] += u.x;
      all[1] += u.y;
      before[0] += low ? u.x : 0;
      before[1] += low ? u.y : 0;
    }
  }
  for (int i = tid; i < W * EM_MAX_BUCKETS / 2; i += 1024) ((int*)pos)[i] = 0;
  const int spans[PER] = {all[0] > 0 ? (all[0] - 1) / EM_SPAN : 0, all[1] > 0 ? (all[1] - 1) / EM_SPAN : 0};
  const int mine = all[0] + all[1], ext = spans[0] + spans[1];
  int inc = mine, einc = ext;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(inc, o, 64), e = __shfl_up(einc, o, 64);
    if (lane >= o) { inc += a; einc += e; }
  }
  if (lane == 63) { wsum[wave] = inc; wext[wave] = einc; }
  __syncthreads();
  // counts of the wave's quarter thousand, stably numbered at once: a lane's number among its like, and the wave's total
  unsigned rank[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const bool on = id[i] >= 0;
    const int b = on ? id[i] >> rshift : 0;
    const unsigned long long same = emb_match(b, on, bits);
    rank[i] = 0;
    if (on) {
      volatile unsigned short* p = &pos[wave][b];
      const unsigned at = *p;
      rank[i] = at + __popcll(same & ((1ull << lane) - 1));
      if ((same >> lane) == 1) *p = (unsigned short)(at + __popcll(same));     // the last lane of its kind, after all have read
    }
    __builtin_amdgcn_wave_barrier();
  }
  int base = inc - mine, ebase = einc - ext;
  for (int w = 0; w < wave; ++w) { base += wsum[w]; ebase += wext[w]; }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int b = tid * PER + j;
    if (b >= nb) break;
    first[b] = base + before[j];
    unsigned at = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const unsigned c = pos[w][b];
      pos[w][b] = (unsigned short)at;
      at += c;
    }
    if (blockIdx.x == 0) {
      start[b] = base;
      xs[b] = ebase;
      for (int e = 0; e < spans[j]; ++e) owner[ebase + e] = b;
    }
    base += all[j];
    ebase += spans[j];
    if (blockIdx.x == 0 && b == nb - 1) {
      start[nb] = base;
      xs[nb] = ebase;
    }
  }
  if (blockIdx.x == 0) {                              // further spans that there are not
    int total = 0;
    for (int w = 0; w < W; ++w) total += wext[w];
    for (int e = total + tid; e < extra; e += 1024) owner[e] = -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q; ++i)
    if (id[i] >= 0) {
      const int b = id[i] >> rshift;
      list[first[b] + pos[wave][b] + rank[i]] = make_int2((int)(t0 + i * 64), id[i]);
    }
}

struct EmbSum {
  const int* ids;        // direct: all ids
  const int* start;      // sorted: as gs_embedding_place_kernel left them
  const int* xs;
  const int* owner;
  const int2* list;
  int* ptrs;             // [2 extra][R]: place of a row's sum in its span's slot or -1, where a bucket has several spans
  float* part;           // [2 extra][slot rows][F]: their sums
  const void* dout;
  long ldd;
  void* dW;
  long ldw;
  long n, id0, V;
  int F, R, rshift, nb, extra, slot_rows, cap, cw, cws, rbits;
  float scale;
  int accumulate;
};

// A lane's N columns begin at f0, a multiple of N; the last lane's would reach beyond the row, so it loads the row's last N columns
// (from f on) and stores those from f0 on.  So every load is a whole vector, and a batch of them stays in flight.
template <typename E, int N>
__device__ __forceinline__ void emb_store(E* __restrict__ row, int f, int f0, const float* __restrict__ v) {
  if (f == f0) {
    gs_store<E, N>(row + f, N, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (f + i >= f0) row[f + i] = (E)v[i];
  }
}

// A finished sum into its row of the table's gradient
template <typename EO, int N>
__device__ __forceinline__ void emb_write(EO* __restrict__ o, bool accumulate, float scale, int f, int f0, float* acc) {
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] *= scale;
  if (accumulate) {
    float old[N];
    gs_load<EO, N>(o + f, N, 0.f, old);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += old[i];
  }
  emb_store<EO, N>(o, f, f0, acc);
}

// One workgroup of W waves per span of a bucket's tokens (at most 64 W P) and 64 N cw columns: cw waves side by side on the columns, W / cw
// groups of them on consecutive parts of the sorted tokens, so that a frequent row is walked by several waves.  A run that crosses
// from one part into the next is summed by the wave that it begins in, from what the others leave in LDS, in order.
// U rows of dout are in flight per lane.  Blocks [0, extra) are the further spans, the longest work, and begin first.
// What bounds it: with many tokens HBM (dout read once, the table's gradient written once: 32768 ids on 128000 x 2048 bf16, 659 MB,
// 170 us = 3.9 TB/s with the sort and the join); with few, the walk of the most frequent row by one compute unit, whose loads' latency
// is what U hides (5001 ids on 10007 x 500 fp32: 21 us, of which 6 would be traffic; one row in flight took 48).
template <int T, int TO, int N, bool DIRECT, int W, int P, int U>
__global__ __launch_bounds__(W * 64) void gs_embedding_sum_kernel(EmbSum a) {
  typedef typename GsElt<T>::type E;
  typedef typename GsElt<TO>::type EO;
  typedef typename GsVec<E, N>::type V;
  constexpr int WS = W == 16 ? 4 : 3;
  static_assert(1 << WS == W, "a power of two");
  extern __shared__ int dyn[];
  int* ptr = dyn;                                      // [R + 1] where a row's tokens begin
  int* cnt = ptr + a.R + 1;                            // [W][R] per wave: tokens of a row, then the next one's place
  int* st = cnt + W * a.R;                             // [cap] tokens in order of their rows
  unsigned short* sr = (unsigned short*)(st + a.cap);  // [cap] their rows in the bucket
  unsigned short* place = sr + a.cap;                  // [R] rows with tokens before this one
  __shared__ float slot_sum[W][64][N];                 // a wave's part of a run that began before its part
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int b, span = 0, spans = 1, i0 = 0, i1 = (int)a.n, slot = 0;
  if (DIRECT) {
    b = blockIdx.x;
  } else {
    if ((int)blockIdx.x < a.extra) {
      slot = blockIdx.x;
      b = a.owner[slot];
      if (b < 0) return;
      span = slot - a.xs[b] + 1;
    } else {
      b = blockIdx.x - a.extra;
      slot = a.extra + a.xs[b];
    }
    spans = a.xs[b + 1] - a.xs[b] + 1;
    i0 = a.start[b] + span * EM_SPAN;
    i1 = min(i0 + EM_SPAN, a.start[b + 1]);
  }
  const long row0 = (long)b * a.R;
  const int rows = (int)min((long)a.R, a.V - row0);
  // stable counting sort of items [i0, i1) by row: each wave takes 64 P of them, in order
  int t[P], r[P];                                      // tokens, their rows in the bucket or -1
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int i = i0 + (wave * P + j) * 64 + lane;
    r[j] = -1;
    t[j] = i;
    if (i < i1) {
      long row;
      if (DIRECT) {
        row = emb_row(a.ids[i], a.id0, a.V);
      } else {
        const int2 v = a.list[i];
        t[j] = v.x;
        row = v.y;
      }
      if (row >= row0 && row < row0 + rows) r[j] = (int)(row - row0);
    }
  }
  for (int i = tid; i < W * a.R; i += W * 64) cnt[i] = 0;
  __syncthreads();
  unsigned short rank[P];                              // among the wave's items of the row
#pragma unroll
  for (int j = 0; j < P; ++j) {
    rank[j] = 0;
    if (!__ballot(r[j] >= 0)) continue;
    const unsigned long long same = emb_match(r[j], r[j] >= 0, a.rbits);
    if (r[j] >= 0) {
      volatile int* p = &cnt[wave * a.R + r[j]];
      const int at = *p;
      rank[j] = (unsigned short)(at + __popcll(same & ((1ull << lane) - 1)));
      if ((same >> lane) == 1) *p = at + __popcll(same);   // the last lane of its kind, after all have read (one wave, in order)
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if (wave == 0) {                                     // exclusive prefix, row by row and within a row wave by wave
    int run = 0, kept = 0;
    for (int base = 0; base < a.R; base += 64) {
      const int r = base + lane;
      int c[W], sum = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) { c[w] = r < a.R ? cnt[w * a.R + r] : 0; sum += c[w]; }
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) { const int v = __shfl_up(inc, o, 64); if (lane >= o) inc += v; }
      const unsigned long long have = __ballot(sum > 0);
      int at = run + inc - sum;
      if (r < a.R) {
        ptr[r] = at;
        place[r] = (unsigned short)(kept + __popcll(have & ((1ull << lane) - 1)));
#pragma unroll
        for (int w = 0; w < W; ++w) { cnt[w * a.R + r] = at; at += c[w]; }
      }
      run += __shfl(inc, 63, 64);
      kept += __popcll(have);
    }
    if (lane == 0) ptr[a.R] = run;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < P; ++j)
    if (r[j] >= 0) {
      const int to = cnt[wave * a.R + r[j]] + rank[j];
      st[to] = t[j];
      sr[to] = (unsigned short)r[j];
    }
  __syncthreads();
  const int total = ptr[a.R];
  const bool whole = spans == 1;
  if (!whole && blockIdx.y == 0)
    for (int r = tid; r < a.R; r += W * 64) a.ptrs[(long)slot * a.R + r] = ptr[r] < ptr[r + 1] ? place[r] : -1;

  const int tw = wave >> a.cws, gsh = WS - a.cws, groups = 1 << gsh;   // (powers of two: no division)
  const int f0 = (((int)blockIdx.y << a.cws) + (wave & (a.cw - 1))) * 64 * N + lane * N, f = min(f0, a.F - N);
  const bool on = f0 < a.F;
  auto part_at = [&](int g) { return (int)((unsigned)(total * g) >> gsh); };   // (total is at most EM_DIRECT)
  const int p0 = part_at(tw), p1 = part_at(tw + 1);
  const E* src = (const E*)a.dout + f;
  float* part = a.part + (long)slot * a.slot_rows * a.F;
  EO* table = (EO*)a.dW + row0 * a.ldw;
  const long ldd = a.ldd, ldw = a.ldw;
  const bool accumulate = a.accumulate != 0;
  const float scale = a.scale;
  if (whole && !accumulate && on) {                    // rows without tokens; their stores go out before the walk's loads return
    const float z[N] = {};
    for (int row = tw; row < rows; row += groups)
      if (ptr[row] == ptr[row + 1]) emb_store<EO, N>(table + row * ldw, f, f0, z);
  }
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  const int before = p0 > 0 ? __builtin_amdgcn_readfirstlane(sr[p0 - 1]) : -1;
  int cur = -1;                                        // row being summed
  bool foreign = false;                                // its run began before this part
  auto finish = [&]() {                                // the sum of row cur
    if (cur >= 0) {
      if (foreign) {
#pragma unroll
        for (int i = 0; i < N; ++i) slot_sum[wave][lane][i] = acc[i];
      } else if (on) {
        if (whole) emb_write<EO, N>(table + cur * ldw, accumulate, scale, f, f0, acc);
        else emb_store<float, N>(part + (long)place[cur] * a.F, f, f0, acc);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
    }
  };
  for (int base = p0; base < p1; base += U) {
    V v[U];
    int of[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int at = min(base + j, p1 - 1);
      const int token = __builtin_amdgcn_readfirstlane(st[at]);
      of[j] = __builtin_amdgcn_readfirstlane(sr[at]);
      v[j] = *(const V*)(src + token * ldd);
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (base + j < p1) {
        if (of[j] != cur) {
          finish();
          foreign = cur < 0 && of[j] == before;
          cur = of[j];
        }
        if constexpr (N == 1) {
          acc[0] += (float)v[j];
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] += (float)v[j][i];
        }
      }
    }
  }
  const bool open = p0 < p1 && p1 < total && __builtin_amdgcn_readfirstlane(sr[p1]) == cur;   // goes on in the next part
  if (!open || foreign) finish();
  __syncthreads();
  if (open && !foreign) {
    for (int g = tw + 1; g < groups; ++g) {
      const int q0 = part_at(g), q1 = part_at(g + 1);
      if (q0 == q1) continue;
      if (sr[q0] != cur) break;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += slot_sum[(g << a.cws) + (wave & (a.cw - 1))][lane][i];
      if (sr[q1 - 1] != cur) break;
    }
    finish();
  }
}

// Buckets of several spans: the sums of each row in the spans' order, a wave per row.  Blocks (e, ., .) work if e is a bucket's first
// further span.
template <int TO, int N>
__global__ __launch_bounds__(256) void gs_embedding_join_kernel(EmbSum a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e = blockIdx.x, b = a.owner[e];
  if (b < 0 || a.xs[b] != e) return;
  const int spans = a.xs[b + 1] - e + 1;
  const long row0 = (long)b * a.R;
  const int r = blockIdx.z * 4 + wave;
  if (r >= (int)min((long)a.R, a.V - row0)) return;
  const int f0 = blockIdx.y * 64 * N + lane * N, f = min(f0, a.F - N);
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  bool any = false;
  for (int base = 0; base < spans; base += 64) {
    const int s = base + lane;                         // a lane looks up one span's place for the row
    const int slot = s == 0 ? a.extra + e : e + s - 1;
    const int at = s < spans ? a.ptrs[(long)slot * a.R + r] : -1;
    unsigned long long have = __ballot(at >= 0);
    any |= have != 0;
    while (have) {
      constexpr int U = 4;
      float v[U][N];
      unsigned long long left = have;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int l = left ? __ffsll(left) - 1 : __ffsll(have) - 1;
        const long at_l = (long)__shfl(slot, l, 64) * a.slot_rows + __shfl(at, l, 64);
        gs_load<float, N>(a.part + at_l * a.F + f, N, 0.f, v[j]);
        left &= left - 1;
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (!have) break;
        have &= have - 1;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += v[j][i];
      }
    }
  }
  if (f0 < a.F && (any || !a.accumulate)) {
    typedef typename GsElt<TO>::type EO;
    emb_write<EO, N>((EO*)a.dW + (row0 + r) * a.ldw, a.accumulate != 0, a.scale, f, f0, acc);
  }
}

template <int T>
int emb_fwd(const void* W, long ldw, long V, int F, const int* ids, long n, float scale, void* out, long ldo, hipStream_t s) {
  typedef typename GsElt<T>::type E;
  const unsigned pieces = (unsigned)gs_cdiv(F, 16 / sizeof(E));
  const long band = std::max(1L, (1L << 31) / (long)pieces);          // rows of a launch: their pieces are counted in 32 bits
  for (long t0 = 0; t0 < n; t0 += band) {
    const unsigned total = (unsigned)(std::min(band, n - t0) * pieces);
    gs_embedding_fwd_kernel<T><<<dim3((total / 2 + 256) / 256), dim3(256), 0, s>>>((const E*)W, ldw, V, F, ids + t0, total, scale,
                                                                                  (E*)out + t0 * ldo, ldo, pieces);
    GS_LAUNCH_CHECK();
  }
  return GS_OK;
}

template <int T, int TO, int N, bool DIRECT, int W, int P, int U>
int emb_sum_launch(const EmbPlan& p, EmbSum a, hipStream_t s) {
  a.cw = 1;
  while (a.cw < W && a.cw * 64 * N < a.F) { a.cw *= 2; ++a.cws; }
  const unsigned gy = (unsigned)gs_cdiv(a.F, a.cw * 64 * N);
  a.cap = (int)std::min<long>(DIRECT ? std::max<long>(a.n, 1) : EM_SPAN, W * 64 * P);
  const size_t lds = (size_t)a.cap * 6 + (size_t)((W + 1) * p.R + 1) * 4 + (size_t)p.R * 2 + 2;
  gs_embedding_sum_kernel<T, TO, N, DIRECT, W, P, U><<<dim3((unsigned)((DIRECT ? 0 : p.extra) + p.nb), gy), dim3(W * 64), lds, s>>>(a);
  GS_LAUNCH_CHECK();
  return GS_OK;
}

template <int T, int TO, int N>
int emb_sum(const EmbPlan& p, EmbSum a, hipStream_t s) {
  static_assert(8 * 64 >= EM_FEW && 16 * 64 * 8 >= EM_DIRECT && 8 * 64 >= EM_SPAN, "a workgroup takes its items in one go");
  if (p.direct) return a.n <= EM_FEW ? emb_sum_launch<T, TO, N, true, 8, 1, 8>(p, a, s) : emb_sum_launch<T, TO, N, true, 16, 8, 16>(p, a, s);
  GS_TRY((emb_sum_launch<T, TO, N, false, 8, 1, 8>(p, a, s)));
  if (p.extra > 0) {
    gs_embedding_join_kernel<TO, N><<<dim3((unsigned)p.extra, (unsigned)gs_cdiv(a.F, 64 * N), (unsigned)gs_cdiv(p.R, 4)), dim3(256), 0, s>>>(a);
    GS_LAUNCH_CHECK();
  }
  return GS_OK;
}

template <int T, int TO>
int emb_bwd_rows(const void* dout, long ldd, const int* ids, long n, long id0, long V, int F, float scale, int accumulate, void* dW, long ldw,
            char* scratch, hipStream_t s) {
  const EmbPlan p = emb_plan(n, V, F);
  EmbSum a = {};
  a.ids = ids; a.dout = dout; a.ldd = ldd; a.dW = dW; a.ldw = ldw; a.n = n; a.id0 = id0; a.V = V; a.F = F; a.scale = scale; a.accumulate = accumulate;
  a.R = p.R; a.nb = p.nb; a.extra = p.extra; a.slot_rows = p.R < EM_SPAN ? p.R : EM_SPAN;
  while ((1 << a.rbits) < p.R) ++a.rbits;
  a.rshift = a.rbits;
  if (!p.direct) {
    int* start = (int*)(scratch + p.start);
    int* xs = (int*)(scratch + p.xs);
    int* owner = (int*)(scratch + p.owner);
    int2* list = (int2*)(scratch + p.list);
    int* cnt = (int*)(scratch + p.cnt);
    int bits = 0;
    while ((1 << bits) < p.nb) ++bits;
    gs_embedding_count_kernel<<<dim3((unsigned)p.tiles), dim3(1024), 0, s>>>(ids, n, id0, V, a.rshift, p.nbp, cnt);
    GS_LAUNCH_CHECK();
    if (p.tiles > EM_SCAN) {
      gs_embedding_scan_kernel<<<dim3((unsigned)gs_cdiv(p.nbp, 64)), dim3(1024), 0, s>>>(cnt, p.tiles, p.nbp);
      GS_LAUNCH_CHECK();
    }
    gs_embedding_place_kernel<<<dim3((unsigned)p.tiles), dim3(1024), 0, s>>>(ids, n, id0, V, a.rshift, p.nb, p.nbp, bits, cnt, p.tiles, start, xs, owner, p.extra, list);
    GS_LAUNCH_CHECK();
    a.start = start; a.xs = xs; a.owner = owner; a.list = list; a.ptrs = (int*)(scratch + p.ptrs); a.part = (float*)(scratch + p.part);
  }
  // columns per lane: 16 bytes of dout where the width has them, so that more waves share a frequent row
  constexpr int N = T == GS_TYPE_F32 ? 4 : 8;
  if (F >= 64 * N) return emb_sum<T, TO, N>(p, a, s);
  if (F >= 128) return emb_sum<T, TO, 2>(p, a, s);
  return emb_sum<T, TO, 1>(p, a, s);
}

// tables of more rows than the buckets hold: a band of rows after the other
template <int T, int TO>
int emb_bwd(const void* dout, long ldd, const int* ids, long n, long V, int F, float scale, int accumulate, void* dW, long ldw,
            char* scratch, hipStream_t s) {
  for (long v0 = 0; v0 < V; v0 += EM_MAX_V)
    GS_TRY((emb_bwd_rows<T, TO>(dout, ldd, ids, n, v0, std::min(V - v0, EM_MAX_V), F, scale, accumulate,
                                (typename GsElt<TO>::type*)dW + v0 * ldw, ldw, scratch, s)));
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
  const int e = gs_type_bytes(type);
  const GsSpan o = gs_span(out, n, ldo, F, e);
  if (gs_overlap(o, gs_span(W, V, ldw, F, e)) || gs_overlap(o, gs_span(ids, n, 4)))
    GS_FAIL(GS_ERR_ARG, "gs_embedding_fwd: the result lies on another operand");
  hipStream_t s = (hipStream_t)stream;
  if (type == GS_TYPE_F32) return emb_fwd<GS_TYPE_F32>(W, ldw, V, F, ids, n, scale, out, ldo, s);
  if (type == GS_TYPE_F16) return emb_fwd<GS_TYPE_F16>(W, ldw, V, F, ids, n, scale, out, ldo, s);
  return emb_fwd<GS_TYPE_BF16>(W, ldw, V, F, ids, n, scale, out, ldo, s);
}

extern "C" size_t gs_embedding_bwd_scratch_bytes(long n, long V, int F) {
  return n < 0 || V < 1 || F < 1 || n > 0x7fffffffL ? 0 : emb_plan(n, std::min(V, EM_MAX_V), F).bytes;
}

extern "C" int gs_embedding_bwd(const void* dout, long ldd, int type, const int* ids, long n, long V, int F, float scale, int accumulate,
                                void* dW, long ldw, int type_dw, void* scratch, gs_stream_t stream) {
  GS_TRY(emb_check("gs_embedding_bwd", n, V, F, type, ldd, ldw));
  if (type_dw != type && type_dw != GS_TYPE_F32)
    GS_FAIL(GS_ERR_ARG, "gs_embedding_bwd: the gradient is held in the type of d_out or in fp32 (got %d for %d)", type_dw, type);
  if (!dW || (n > 0 && (!dout || !ids))) GS_FAIL(GS_ERR_ARG, "gs_embedding_bwd: null pointer");
  const GsSpan w = gs_span(dW, V, ldw, F, gs_type_bytes(type_dw));
  if (n > 0 && (gs_overlap(w, gs_span(dout, n, ldd, F, gs_type_bytes(type))) || gs_overlap(w, gs_span(ids, n, 4))))
    GS_FAIL(GS_ERR_ARG, "gs_embedding_bwd: the gradient lies on another operand");
  const EmbPlan p = emb_plan(n, std::min(V, EM_MAX_V), F);
  if (((p.direct ? 0L : p.extra) + p.nb) * (p.direct ? 1024 : 512) > 0xffffffffL)
    GS_FAIL(GS_ERR_UNSUPPORTED, "gs_embedding_bwd: %ld ids are beyond one launch", n);
  if (gs_embedding_bwd_scratch_bytes(n, V, F) > 0 && (!scratch || ((size_t)scratch & 15)))
    GS_FAIL(GS_ERR_ARG, "gs_embedding_bwd: the scratch is missing or not 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  if (type == GS_TYPE_F32) return emb_bwd<GS_TYPE_F32, GS_TYPE_F32>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, (char*)scratch, s);
  if (type == GS_TYPE_F16)
    return type_dw == GS_TYPE_F16 ? emb_bwd<GS_TYPE_F16, GS_TYPE_F16>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, (char*)scratch, s)
                                  : emb_bwd<GS_TYPE_F16, GS_TYPE_F32>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, (char*)scratch, s);
  return type_dw == GS_TYPE_BF16 ? emb_bwd<GS_TYPE_BF16, GS_TYPE_BF16>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, (char*)scratch, s)
                                 : emb_bwd<GS_TYPE_BF16, GS_TYPE_F32>(dout, ldd, ids, n, V, F, scale, accumulate, dW, ldw, (char*)scratch, s);
}
