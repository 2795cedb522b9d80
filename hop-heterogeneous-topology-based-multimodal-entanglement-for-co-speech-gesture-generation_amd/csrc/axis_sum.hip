// Sums over one axis of a dense tensor, in [outer][R][inner] -> out [outer][inner]: what the gradient of a broadcast operand is made of
// (linear_act's residual).  fp32 arithmetic in a fixed order, one rounding at the end: the same bits every time.
// Bound: one read of the input.  The axis is cut into groups of rows where outer x inner alone does not fill the chip; a group leaves one
// partial row, and a second launch of the same kernel adds them in order.  (A library's reduction over many blocks clears its
// counters by a memset, and a memset node in a recorded graph is not reliably ordered in front of the kernel behind it: replays
// have given the sums of other inputs.  Nothing has to be cleared here.)
// Two forms, by `inner`: from 64 on a wave reads 64 neighbouring columns of a row; below, a team of threads walks the group's
// contiguous stretch in steps of a multiple of `inner`, so a thread stays in one column, and a tree in LDS adds the threads of a column.
// Measured, bf16, us in a recorded graph: 4352 x 768 over the rows 7.6 (two launches), over the columns 4.1, over both 7.4; 16384 x 4096 over
// the rows 29 (4.6 TB/s), over the columns 22 (6.0 TB/s, part of it from the 256 MB cache); 300 x 72 over the rows 5.1.
#include "t16_dev.h"

#include <algorithm>
#include <type_traits>

namespace hopmi {

constexpr int AS_THREADS = 256, AS_BLOCKS = 1024;            // (workgroups that a launch of one group each aims for)

struct AxisSum {
  const void* in;
  void* out;                                                 // [outer][groups][inner]
  long long outer, R, inner, per;                            // group g: rows [g per, min(R, (g + 1) per))
  int groups;
};

template <typename T, typename O> __global__ __launch_bounds__(AS_THREADS) void axis_sum_cols_kernel(AxisSum A) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long strips = (A.inner + 63) / 64, items = A.outer * A.groups * strips;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const long long og = item / strips, i = (item - og * strips) * 64 + lane, o = og / A.groups, g = og - o * A.groups;
    const long long end = min(A.R, (g + 1) * A.per);
    float s = 0.f;
    if (i < A.inner) {
      const T* p = static_cast<const T*>(A.in) + o * A.R * A.inner + i;
      long long r = g * A.per + wave;
      for (; r + 3 * 4 < end; r += 4 * 4) {                  // four loads in flight
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = to_f(p[(r + 4 * k) * A.inner]);
#pragma unroll
        for (int k = 0; k < 4; ++k) s += v[k];
      }
      for (; r < end; r += 4) s += to_f(p[r * A.inner]);
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && i < A.inner) static_cast<O*>(A.out)[og * A.inner + i] = (O)(red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane]);
    __syncthreads();                                         // (red is written again in the next round)
  }
}

// TEAM threads per (outer index, group); inner < 64
template <typename T, typename O, int TEAM> __global__ __launch_bounds__(AS_THREADS) void axis_sum_rows_kernel(AxisSum A) {
  __shared__ float red[AS_THREADS];
  constexpr int TEAMS = AS_THREADS / TEAM;
  const int t = threadIdx.x % TEAM, inner = (int)A.inner, chunks = TEAM / inner, step = chunks * inner;
  float* mine = red + threadIdx.x - t;
  const long long items = A.outer * A.groups;
  for (long long base = (long long)blockIdx.x * TEAMS; base < items; base += (long long)gridDim.x * TEAMS) {
    const long long item = base + threadIdx.x / TEAM;
    float s = 0.f;
    if (item < items && t < step) {
      const long long o = item / A.groups, g = item - o * A.groups, r0 = g * A.per, n = (min(A.R, r0 + A.per) - r0) * inner;
      const T* p = static_cast<const T*>(A.in) + (o * A.R + r0) * inner;
      long long e = t;
      for (; e + 3LL * step < n; e += 4LL * step) {          // four loads in flight
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = to_f(p[e + k * step]);
#pragma unroll
        for (int k = 0; k < 4; ++k) s += v[k];
      }
      for (; e < n; e += step) s += to_f(p[e]);
    }
    mine[t] = s;
    __syncthreads();
    for (int c = chunks; c > 1; c = (c + 1) / 2) {           // (uniform: it depends on `inner` only)
      const int h = (c + 1) / 2;
      if (t < (c - h) * inner) mine[t] += mine[t + h * inner];
      __syncthreads();
    }
    if (item < items && t < inner) static_cast<O*>(A.out)[item * inner + t] = (O)mine[t];
    __syncthreads();
  }
}

// groups of at least 32 rows (columns form: eight per wave) or 2048 elements, as many as fill the chip
static int axis_groups(long long outer, long long R, long long inner) {
  const long long items = inner >= 64 ? outer * ((inner + 63) / 64) : outer, least = inner >= 64 ? 32 : (2048 + inner - 1) / inner;
  long long g = (AS_BLOCKS + items - 1) / items;
  g = std::min(g, (R + least - 1) / least);
  const long long per = (R + g - 1) / g;
  return (int)((R + per - 1) / per);
}

// The team of a narrow item: eight threads for up to 64 elements (70000 x 8 over the columns 4.0 us; a wave each 18.7), a wave up to 4096 (4352 x
// 2304 over the columns 5.6 us, 16384 x 4096 22; 256 threads each 7.8 and 29), 256 threads beyond.
template <typename T, typename O> static void axis_sum_go(const void* in, void* out, long long outer, long long R, long long inner, int groups, hipStream_t st) {
  const AxisSum A{in, out, outer, R, inner, (R + groups - 1) / groups, groups};
  auto grid = [](long long n) { return dim3((unsigned)std::min(n, 1LL << 16)); };
  if (inner >= 64) hipLaunchKernelGGL((axis_sum_cols_kernel<T, O>), grid(outer * groups * ((inner + 63) / 64)), dim3(AS_THREADS), 0, st, A);
  else if (A.per * inner > 4096) hipLaunchKernelGGL((axis_sum_rows_kernel<T, O, 256>), grid(outer * groups), dim3(AS_THREADS), 0, st, A);
  else if (inner <= 8 && A.per * inner <= 64) hipLaunchKernelGGL((axis_sum_rows_kernel<T, O, 8>), grid((outer * groups + 31) / 32), dim3(AS_THREADS), 0, st, A);
  else hipLaunchKernelGGL((axis_sum_rows_kernel<T, O, 64>), grid((outer * groups + 3) / 4), dim3(AS_THREADS), 0, st, A);
}

static bool axis_sides(long long outer, long long R, long long inner) {
  constexpr long long MOST = 1LL << 40;
  return outer >= 1 && R >= 1 && inner >= 1 && outer <= MOST && R <= MOST && inner <= MOST && outer <= MOST / R && outer * R <= MOST / inner;
}

}  // namespace hopmi

using namespace hopmi;

extern "C" size_t hopmi_axis_sum_ws_floats(long long outer, long long R, long long inner) {
  if (!axis_sides(outer, R, inner)) return 0;
  const int g = axis_groups(outer, R, inner);
  return g > 1 ? (size_t)outer * g * inner : 0;
}

extern "C" int hopmi_axis_sum(const void* in, int in_dtype, void* out, int out_dtype, long long outer, long long R, long long inner, float* ws,
                              void* stream) {
  if (!in || !out) { set_error("hopmi_axis_sum: null pointer argument"); return HOPMI_EINVAL; }
  if (!axis_sides(outer, R, inner)) {
    set_error("hopmi_axis_sum: [%lld][%lld][%lld] (sides of at least 1, up to 2^40 elements)", outer, R, inner);
    return HOPMI_EINVAL;
  }
  if (in_dtype < T_F32 || in_dtype > T_F16 || out_dtype < T_F32 || out_dtype > T_F16 || (in_dtype != T_F32 && out_dtype != T_F32 && in_dtype != out_dtype)) {
    set_error("hopmi_axis_sum: dtype=%d -> %d (0 fp32, 1 bf16, 2 fp16; one 16-bit type)", in_dtype, out_dtype);
    return HOPMI_EINVAL;
  }
  const int groups = axis_groups(outer, R, inner);
  if (groups > 1 && !ws) { set_error("hopmi_axis_sum: null workspace"); return HOPMI_EINVAL; }
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto typed = [&](auto f, int dtype) {
    if (dtype == T_F32) f(float{});
    else if (dtype == T_BF16) f(__bf16{});
    else f(_Float16{});
  };
  auto last = [&](const void* p, auto t, long long rows) {   // the launch that writes `out`
    using T = decltype(t);
    typed([&](auto o) {
      using O = decltype(o);
      if constexpr (std::is_same_v<T, float> || std::is_same_v<O, float> || std::is_same_v<T, O>) axis_sum_go<T, O>(p, out, outer, rows, inner, 1, st);
    }, out_dtype);
  };
  typed([&](auto t) {
    if (groups == 1) last(in, t, R);
    else {
      axis_sum_go<decltype(t), float>(in, ws, outer, R, inner, groups, st);
      last(ws, float{}, groups);
    }
  }, in_dtype);
  return check_launch("hopmi_axis_sum");
}
