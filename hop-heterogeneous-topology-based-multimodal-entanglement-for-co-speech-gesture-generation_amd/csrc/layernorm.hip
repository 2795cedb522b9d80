// Layer normalisation with trainable weights, forward and backward (fp32, bf16 or fp16 storage; all arithmetic and statistics fp32).
//
//   mu = sum_d x / D      v = sum_d (x - mu)^2 / D      r = 1 / sqrt(v + eps)      xh = (x - mu) r      y = xh g + b
//   dx = r (g dy - mean_d(g dy) - xh mean_d(g dy xh))       dg = sum_rows dy xh       db = sum_rows dy
//
// Bound: HBM (8 / 22 operations per element against 4-8 / 6-12 bytes); measured, in a recorded graph: forward 8192 x 4096 fp32 41.8 us
// (6.5 TB/s of x and y together, some of it from the 256 MB cache), backward 85.6 (4.7 TB/s of x, dy, dx); 32768 x 1024 bf16 22.4 and
// 41.0; a large copy moves 5.2 TB/s.  Below some 10 MB the launches bound it: 4352 x 768 bf16 5.0 and 12.9 us (two launches), one window
// of 34 rows 3.0.  So each pass reads x (and dy) once: a row stays in the registers of one wave (up to 256 16-byte vectors) or of a
// workgroup of 256 (up to 512), 512 (1024) or 1024 threads (2048); wider rows are re-read (from the caches) by the looped form.
// The variance is taken around the mean, not as E x^2 - mu^2: the row is in registers, a second pass over it costs no memory.
// The weights' gradients are sums over the rows: a workgroup walks rows blockIdx, blockIdx + grid, ... and keeps its columns' sums in
// registers, leaves one partial row [2][D] in the workspace, and a second launch adds the partial rows in index order (no atomics:
// the same bits every time).
#include "t16_dev.h"

namespace hopmi {

// the sums of a row over the TPR threads that hold it; with more than one wave through LDS (two exchange areas used in turn: the
// second call's writes cannot meet the first call's reads, one barrier per call)
template <int TPR, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float* xch, int& phase) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
  if (TPR == 64) return;
  constexpr int W = TPR / 64;
  float* a = xch + (phase & 1) * 2 * W;
  phase ^= 1;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) a[k * W + (threadIdx.x >> 6)] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) s += a[k * W + w];
    v[k] = s;
  }
}

template <typename T, typename WT, int NV, int TPR>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void ln_fwd_kernel(const T* __restrict__ x, long long ldx, const WT* __restrict__ w,
                                                                       const WT* __restrict__ b, T* __restrict__ y,
                                                                       float* __restrict__ mean_out, float* __restrict__ rstd_out, int M,
                                                                       int D, float eps) {
  constexpr int V = Vec<T>::N, RPB = TPR == 64 ? 4 : 1;
  __shared__ float xch[4 * (TPR / 64)];
  int phase = 0;
  const int lane = threadIdx.x & (TPR - 1), vecs = D / V, tail = D - vecs * V, td = vecs * V + lane;
  const float invD = 1.f / (float)D;
  const long long step = (long long)gridDim.x * RPB;
  const long long row0 = (long long)blockIdx.x * RPB + (TPR == 64 ? threadIdx.x >> 6 : 0);
  u32x4_t nx[NV];
  float nt = 0.f;
  auto load = [&](long long row) {
    const T* p = x + row * ldx;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + TPR * i < vecs) nx[i] = ld16(p + (long long)(lane + TPR * i) * V);
    if (lane < tail) nt = to_f(p[td]);
  };
  if (row0 < M) load(row0);
  for (long long row = row0; row < M; row += step) {
    u32x4_t c[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) c[i] = nx[i];
    const float ct = nt;
    if (row + step < M) load(row + step);                    // the next row travels while this one is reduced
    float s[1] = {lane < tail ? ct : 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + TPR * i < vecs)
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += vget(c[i], e, x);
    row_sums<TPR, 1>(s, xch, phase);
    const float mu = s[0] * invD;
    float q[1] = {lane < tail ? (ct - mu) * (ct - mu) : 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + TPR * i < vecs)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = vget(c[i], e, x) - mu;
          q[0] = fmaf(d, d, q[0]);
        }
    row_sums<TPR, 1>(q, xch, phase);
    const float r = 1.f / sqrtf(q[0] * invD + eps);
    T* o = y + row * D;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + TPR * i < vecs) {
        const int d0 = (lane + TPR * i) * V;
        float f[V], g[V];
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (vget(c[i], e, x) - mu) * r;
        if (w != nullptr) {
          ldf<V>(w + d0, g);
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] *= g[e];
        }
        if (b != nullptr) {
          ldf<V>(b + d0, g);
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] += g[e];
        }
        st16(o + d0, vpack(f, x));
      }
    if (lane < tail) {
      float f = (ct - mu) * r;
      if (w != nullptr) f *= to_f(w[td]);
      if (b != nullptr) f += to_f(b[td]);
      o[td] = (T)f;
    }
    if (mean_out != nullptr && lane == 0) {
      mean_out[row] = mu;
      rstd_out[row] = r;
    }
  }
}

// rows wider than the register forms hold: one 1024-thread workgroup per row, the row re-read (from the caches) for each of the passes
template <typename T, typename WT>
__global__ __launch_bounds__(1024) void ln_fwd_loop_kernel(const T* __restrict__ x, long long ldx, const WT* __restrict__ w,
                                                           const WT* __restrict__ b, T* __restrict__ y,
                                                           float* __restrict__ mean_out, float* __restrict__ rstd_out, int M, int D,
                                                           float eps) {
  __shared__ float xch[4 * 16];
  int phase = 0;
  const float invD = 1.f / (float)D;
  for (long long row = blockIdx.x; row < M; row += gridDim.x) {
    const T* p = x + row * ldx;
    float s[1] = {0.f}, q[1] = {0.f};
    for (int d = threadIdx.x; d < D; d += 1024) s[0] += to_f(p[d]);
    row_sums<1024, 1>(s, xch, phase);
    const float mu = s[0] * invD;
    for (int d = threadIdx.x; d < D; d += 1024) {
      const float c = to_f(p[d]) - mu;
      q[0] = fmaf(c, c, q[0]);
    }
    row_sums<1024, 1>(q, xch, phase);
    const float r = 1.f / sqrtf(q[0] * invD + eps);
    for (int d = threadIdx.x; d < D; d += 1024) {
      float f = (to_f(p[d]) - mu) * r;
      if (w != nullptr) f *= to_f(w[d]);
      if (b != nullptr) f += to_f(b[d]);
      y[row * D + d] = (T)f;
    }
    if (mean_out != nullptr && threadIdx.x == 0) {
      mean_out[row] = mu;
      rstd_out[row] = r;
    }
  }
}

// part: [gridDim.x][2][D] sums of dy xh and of dy over the rows of each workgroup (null: not wanted); dx null: not wanted
template <typename T, typename WT, int NV, int TPR>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void ln_bwd_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy,
                                                                       const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                       const WT* __restrict__ w, T* __restrict__ dx,
                                                                       float* __restrict__ part, int M, int D) {
  constexpr int V = Vec<T>::N, RPB = TPR == 64 ? 4 : 1;
  __shared__ float xch[4 * (TPR / 64)];
  extern __shared__ float comb[];                            // TPR == 64: [4][2][D], the waves' column sums
  int phase = 0;
  const int lane = threadIdx.x & (TPR - 1), vecs = D / V, tail = D - vecs * V, td = vecs * V + lane;
  const float invD = 1.f / (float)D;
  const long long step = (long long)gridDim.x * RPB;
  const long long row0 = (long long)blockIdx.x * RPB + (TPR == 64 ? threadIdx.x >> 6 : 0);
  float dg[NV][V], db[NV][V], dgt = 0.f, dbt = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) dg[i][e] = db[i][e] = 0.f;
  u32x4_t nx[NV], ny[NV];
  float nxt = 0.f, nyt = 0.f, nmu = 0.f, nr = 0.f;
  auto load = [&](long long row) {
    const T *p = x + row * ldx, *g = dy + row * D;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + TPR * i < vecs) {
        nx[i] = ld16(p + (long long)(lane + TPR * i) * V);
        ny[i] = ld16(g + (long long)(lane + TPR * i) * V);
      }
    if (lane < tail) {
      nxt = to_f(p[td]);
      nyt = to_f(g[td]);
    }
    nmu = mean[row];
    nr = rstd[row];
  };
  auto weights = [&](int d0, float (&f)[V]) {
    if (w != nullptr) ldf<V>(w + d0, f);
    else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = 1.f;
    }
  };
  if (row0 < M) load(row0);
  for (long long row = row0; row < M; row += step) {
    u32x4_t cx[NV], cy[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      cx[i] = nx[i];
      cy[i] = ny[i];
    }
    const float cxt = nxt, cyt = nyt, mu = nmu, r = nr;
    if (row + step < M) load(row + step);
    float s[2] = {0.f, 0.f};                                 // sum g dy, sum g dy xh
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + TPR * i < vecs) {
        float wv[V];
        weights((lane + TPR * i) * V, wv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float g = vget(cy[i], e, x), xh = (vget(cx[i], e, x) - mu) * r;
          dg[i][e] = fmaf(g, xh, dg[i][e]);
          db[i][e] += g;
          const float gw = g * wv[e];
          s[0] += gw;
          s[1] = fmaf(gw, xh, s[1]);
        }
      }
    if (lane < tail) {
      const float xh = (cxt - mu) * r;
      dgt = fmaf(cyt, xh, dgt);
      dbt += cyt;
      const float gw = w != nullptr ? cyt * to_f(w[td]) : cyt;
      s[0] += gw;
      s[1] = fmaf(gw, xh, s[1]);
    }
    if (dx == nullptr) continue;                             // (uniform)
    row_sums<TPR, 2>(s, xch, phase);
    const float m0 = s[0] * invD, m1 = s[1] * invD;
    T* o = dx + row * D;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + TPR * i < vecs) {
        const int d0 = (lane + TPR * i) * V;
        float f[V], wv[V];
        weights(d0, wv);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = r * (vget(cy[i], e, x) * wv[e] - m0 - (vget(cx[i], e, x) - mu) * r * m1);
        st16(o + d0, vpack(f, x));
      }
    if (lane < tail) {
      const float xh = (cxt - mu) * r, gw = w != nullptr ? cyt * to_f(w[td]) : cyt;
      o[td] = (T)(r * (gw - m0 - xh * m1));
    }
  }
  if (part == nullptr) return;
  float* out = part + (long long)blockIdx.x * 2 * D;
  auto visit = [&](auto&& f) {                               // every column this thread holds, with its two sums
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (lane + TPR * i < vecs)
#pragma unroll
        for (int e = 0; e < V; ++e) f((lane + TPR * i) * V + e, dg[i][e], db[i][e]);
    if (lane < tail) f(td, dgt, dbt);
  };
  if (TPR == 64) {                                           // the four waves' sums meet in LDS, all threads add
    float* mine = comb + (threadIdx.x >> 6) * 2 * D;
    visit([&](int d, float a, float c) { mine[d] = a; mine[D + d] = c; });
    __syncthreads();
    for (int d = threadIdx.x; d < 2 * D; d += 256) out[d] = comb[d] + comb[2 * D + d] + comb[4 * D + d] + comb[6 * D + d];
  } else {
    visit([&](int d, float a, float c) { out[d] = a; out[D + d] = c; });
  }
}

template <typename T, typename WT>
__global__ __launch_bounds__(1024) void ln_bwd_loop_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           const WT* __restrict__ w, T* __restrict__ dx, int M, int D) {
  __shared__ float xch[4 * 16];
  int phase = 0;
  const float invD = 1.f / (float)D;
  for (long long row = blockIdx.x; row < M; row += gridDim.x) {
    const T *p = x + row * ldx, *g = dy + row * D;
    const float mu = mean[row], r = rstd[row];
    float s[2] = {0.f, 0.f};
    for (int d = threadIdx.x; d < D; d += 1024) {
      const float gw = to_f(g[d]) * (w != nullptr ? to_f(w[d]) : 1.f);
      s[0] += gw;
      s[1] = fmaf(gw, (to_f(p[d]) - mu) * r, s[1]);
    }
    row_sums<1024, 2>(s, xch, phase);
    for (int d = threadIdx.x; d < D; d += 1024) {
      const float gw = to_f(g[d]) * (w != nullptr ? to_f(w[d]) : 1.f);
      dx[row * D + d] = (T)(r * (gw - s[0] * invD - (to_f(p[d]) - mu) * r * (s[1] * invD)));
    }
  }
}

// column sums of the wide rows: workgroup (64 columns, row slice), four waves on every fourth row of the slice
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_cols_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ dy,
                                                          const float* __restrict__ mean, const float* __restrict__ rstd,
                                                          float* __restrict__ part, int M, int D) {
  __shared__ float red[2][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
  float a = 0.f, c = 0.f;
  if (d < D)
    for (long long row = (long long)blockIdx.y * 4 + wave; row < M; row += (long long)gridDim.y * 4) {
      const float g = to_f(dy[row * D + d]);
      a = fmaf(g, (to_f(x[row * ldx + d]) - mean[row]) * rstd[row], a);
      c += g;
    }
  red[0][wave][lane] = a;
  red[1][wave][lane] = c;
  __syncthreads();
  if (wave == 0 && d < D) {
    float* out = part + (long long)blockIdx.y * 2 * D;
    out[d] = red[0][0][lane] + red[0][1][lane] + red[0][2][lane] + red[0][3][lane];
    out[D + d] = red[1][0][lane] + red[1][1][lane] + red[1][2][lane] + red[1][3][lane];
  }
}

// out[c] = sum over the G partial rows, column c of [dg | db]: 16 waves take every 16th row of 64 columns, then meet in LDS
template <typename WT>
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float* __restrict__ part, int G, int D, WT* __restrict__ dg,
                                                         WT* __restrict__ db) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < 2 * D) {
    int g = wave;
    for (; g + 7 * 16 < G; g += 8 * 16) {                    // eight loads in flight
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(long long)(g + 16 * k) * 2 * D + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; g < G; g += 16) s += part[(long long)g * 2 * D + c];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && c < 2 * D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += red[k][lane];
    if (c < D) { if (dg != nullptr) dg[c] = (WT)t; }
    else if (db != nullptr) db[c - D] = (WT)t;
  }
}

constexpr int LN_WIDEST = 1 << 29;                           // (2 D and what is added to it count in 31 bits)

// which form a row width takes, by its number of 16-byte vectors: a wave up to 256, then two vectors per thread
static int ln_form(int D, int dtype) {
  const int vecs = D / (dtype == T_F32 ? 4 : 8);
  return vecs <= 256 ? 64 : vecs <= 512 ? 256 : vecs <= 1024 ? 512 : vecs <= 2048 ? 1024 : 0;
}
// Workgroups of a backward launch: rows in whole passes over an even grid.  More workgroups hide more latency and leave more partial rows:
// up to 1024 where a row is 128 vectors or fewer (32768 x 1024 bf16: 41.0 us against 44.0 on 512; 65536 x 256 fp32 36.6 / 45.0; 4352 x 768 bf16
// 12.9 / 13.8), up to 512 for wider ones (16384 x 2048 bf16: 45.2 us against 54.7 on 1024; 8192 x 4096 fp32 85.6 / 90.2).
static int ln_bwd_grid(int M, int D, int dtype) {
  const int form = ln_form(D, dtype), cap = D / (dtype == T_F32 ? 4 : 8) <= 128 ? 1024 : 512;
  const long long units = form == 64 ? ((long long)M + 3) / 4 : M;
  if (form == 0) return (int)(units < 64 ? units : 64);
  const long long passes = (units + cap - 1) / cap;
  return (int)((units + passes - 1) / passes);
}

template <typename T, typename WT, int NV, int TPR>
static void ln_fwd_go(const void* x, long long ldx, const void* w, const void* b, void* y, float* mean, float* rstd, int M, int D,
                      float eps, hipStream_t st) {
  const long long units = TPR == 64 ? ((long long)M + 3) / 4 : M;
  const int cap = TPR == 64 ? 2048 : TPR == 256 ? 1536 : TPR == 512 ? 1024 : 512;
  hipLaunchKernelGGL((ln_fwd_kernel<T, WT, NV, TPR>), dim3((unsigned)(units < cap ? units : cap)), dim3(TPR == 64 ? 256 : TPR), 0, st,
                     static_cast<const T*>(x), ldx, static_cast<const WT*>(w), static_cast<const WT*>(b), static_cast<T*>(y), mean, rstd, M, D, eps);
}

template <typename T, typename WT>
static void ln_fwd_typed(const void* x, long long ldx, const void* w, const void* b, void* y, float* mean, float* rstd, int M,
                         int D, float eps, int dtype, hipStream_t st) {
  const int vecs = D / Vec<T>::N, form = ln_form(D, dtype);
  if (form == 64 && vecs <= 64) ln_fwd_go<T, WT, 1, 64>(x, ldx, w, b, y, mean, rstd, M, D, eps, st);
  else if (form == 64 && vecs <= 128) ln_fwd_go<T, WT, 2, 64>(x, ldx, w, b, y, mean, rstd, M, D, eps, st);
  else if (form == 64) ln_fwd_go<T, WT, 4, 64>(x, ldx, w, b, y, mean, rstd, M, D, eps, st);
  else if (form == 256) ln_fwd_go<T, WT, 2, 256>(x, ldx, w, b, y, mean, rstd, M, D, eps, st);
  else if (form == 512) ln_fwd_go<T, WT, 2, 512>(x, ldx, w, b, y, mean, rstd, M, D, eps, st);
  else if (form == 1024) ln_fwd_go<T, WT, 2, 1024>(x, ldx, w, b, y, mean, rstd, M, D, eps, st);
  else
    hipLaunchKernelGGL((ln_fwd_loop_kernel<T, WT>), dim3(M < 512 ? M : 512), dim3(1024), 0, st, static_cast<const T*>(x), ldx, static_cast<const WT*>(w), static_cast<const WT*>(b),
                       static_cast<T*>(y), mean, rstd, M, D, eps);
}

template <typename T, typename WT, int NV, int TPR>
static void ln_bwd_go(const void* x, long long ldx, const void* dy, const float* mean, const float* rstd, const void* w, void* dx,
                      float* part, int M, int D, int grid, hipStream_t st) {
  const auto k = ln_bwd_kernel<T, WT, NV, TPR>;
  const size_t lds = TPR == 64 && part != nullptr ? 8 * D * sizeof(float) : 0;               // up to 66 KB
  static std::atomic<unsigned long long> told{0};
  allow_lds(reinterpret_cast<const void*>(k), 72 * 1024, told);
  hipLaunchKernelGGL(k, dim3(grid), dim3(TPR == 64 ? 256 : TPR), lds, st, static_cast<const T*>(x), ldx,
                     static_cast<const T*>(dy), mean, rstd, static_cast<const WT*>(w), static_cast<T*>(dx), part, M, D);
}

template <typename T, typename WT>
static void ln_bwd_typed(const void* x, long long ldx, const void* dy, const float* mean, const float* rstd, const void* w,
                         void* dx, float* part, int M, int D, int dtype, hipStream_t st) {
  const int vecs = D / Vec<T>::N, form = ln_form(D, dtype);
  if (form == 64 && vecs <= 64) ln_bwd_go<T, WT, 1, 64>(x, ldx, dy, mean, rstd, w, dx, part, M, D, ln_bwd_grid(M, D, dtype), st);
  else if (form == 64 && vecs <= 128) ln_bwd_go<T, WT, 2, 64>(x, ldx, dy, mean, rstd, w, dx, part, M, D, ln_bwd_grid(M, D, dtype), st);
  else if (form == 64) ln_bwd_go<T, WT, 4, 64>(x, ldx, dy, mean, rstd, w, dx, part, M, D, ln_bwd_grid(M, D, dtype), st);
  else if (form == 256) ln_bwd_go<T, WT, 2, 256>(x, ldx, dy, mean, rstd, w, dx, part, M, D, ln_bwd_grid(M, D, dtype), st);
  else if (form == 512) ln_bwd_go<T, WT, 2, 512>(x, ldx, dy, mean, rstd, w, dx, part, M, D, ln_bwd_grid(M, D, dtype), st);
  else if (form == 1024) ln_bwd_go<T, WT, 2, 1024>(x, ldx, dy, mean, rstd, w, dx, part, M, D, ln_bwd_grid(M, D, dtype), st);
  else {
    if (dx != nullptr)
      hipLaunchKernelGGL((ln_bwd_loop_kernel<T, WT>), dim3(M < 512 ? M : 512), dim3(1024), 0, st, static_cast<const T*>(x), ldx,
                         static_cast<const T*>(dy), mean, rstd, static_cast<const WT*>(w), static_cast<T*>(dx), M, D);
    if (part != nullptr)
      hipLaunchKernelGGL((ln_bwd_cols_kernel<T>), dim3((D + 63) / 64, ln_bwd_grid(M, D, dtype)), dim3(256), 0, st, static_cast<const T*>(x), ldx,
                         static_cast<const T*>(dy), mean, rstd, part, M, D);
  }
}

static int ln_check(const char* what, int dtype, int wdtype, int M, int D, long long ldx) {
  if (dtype < T_F32 || dtype > T_F16 || (wdtype != dtype && wdtype != T_F32)) {
    set_error("%s: dtype=%d, weights %d (0 fp32, 1 bf16, 2 fp16; weights of the same type or fp32)", what, dtype, wdtype);
    return HOPMI_EINVAL;
  }
  if (M < 1 || D < 1 || D > LN_WIDEST || ldx < D) { set_error("%s: bad sizes M=%d D=%d ldx=%lld", what, M, D, ldx); return HOPMI_EINVAL; }
  return HOPMI_OK;
}

// calls f(T{}, WT{}) with the storage types the codes stand for
template <typename F> static void ln_types(int dtype, int wdtype, F&& f) {
  if (dtype == T_F32) f(float{}, float{});
  else if (dtype == T_BF16 && wdtype == T_BF16) f(__bf16{}, __bf16{});
  else if (dtype == T_BF16) f(__bf16{}, float{});
  else if (wdtype == T_F16) f(_Float16{}, _Float16{});
  else f(_Float16{}, float{});
}

}  // namespace hopmi

using namespace hopmi;

extern "C" int hopmi_layernorm_fwd(const void* x, long long ldx, const void* weight, const void* bias, int wdtype, void* y, float* mean,
                                   float* rstd, int M, int D, float eps, int dtype, void* stream) {
  const int rc = ln_check("hopmi_layernorm_fwd", dtype, wdtype, M, D, ldx);
  if (rc != HOPMI_OK) return rc;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) { set_error("hopmi_layernorm_fwd: null pointer argument"); return HOPMI_EINVAL; }
  if (!(eps >= 0.f)) { set_error("hopmi_layernorm_fwd: eps=%g", (double)eps); return HOPMI_EINVAL; }
  ln_types(dtype, wdtype, [&](auto t, auto wt) {
    ln_fwd_typed<decltype(t), decltype(wt)>(x, ldx, weight, bias, y, mean, rstd, M, D, eps, dtype, static_cast<hipStream_t>(stream));
  });
  return check_launch("hopmi_layernorm_fwd");
}

extern "C" size_t hopmi_layernorm_bwd_ws_floats(int M, int D, int dtype) {
  if (M < 1 || D < 1 || D > LN_WIDEST || dtype < T_F32 || dtype > T_F16) return 0;
  return (size_t)ln_bwd_grid(M, D, dtype) * 2 * D;
}

extern "C" int hopmi_layernorm_bwd(const void* x, long long ldx, const void* dy, const float* mean, const float* rstd, const void* weight,
                                   int wdtype, void* dx, void* dweight, void* dbias, float* ws, int M, int D, int dtype, void* stream) {
  const int rc = ln_check("hopmi_layernorm_bwd", dtype, wdtype, M, D, ldx);
  if (rc != HOPMI_OK) return rc;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (!x || !dy || !mean || !rstd || (sums && !ws)) { set_error("hopmi_layernorm_bwd: null pointer argument"); return HOPMI_EINVAL; }
  if (!dx && !sums) return HOPMI_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* part = sums ? ws : nullptr;
  ln_types(dtype, wdtype, [&](auto t, auto wt) {
    using WT = decltype(wt);
    ln_bwd_typed<decltype(t), WT>(x, ldx, dy, mean, rstd, weight, dx, part, M, D, dtype, st);
    if (sums)
      hipLaunchKernelGGL((ln_reduce_kernel<WT>), dim3((2 * D + 63) / 64), dim3(1024), 0, st, part, ln_bwd_grid(M, D, dtype), D,
                         static_cast<WT*>(dweight), static_cast<WT*>(dbias));
  });
  return check_launch("hopmi_layernorm_bwd");
}
