// The global 2-norm of a list of gradient tensors and their clipping by it:
//
//   n = sqrt(sum over tensors and elements of g^2)        c = min(1, max_norm / (n + 1e-6))        g' = c g
//
// Bound: HBM.  The norm has to have read every value before the first can be scaled: one read of all gradients, then one read and one
// write where something is written -- in place only if c < 1 (scaling by 1 changes nothing), into other tensors always.
// Launch 1 (norm): the tensors are cut into chunks of 16 Ki elements, a workgroup takes chunks blockIdx, blockIdx + grid, ... and leaves
// ONE sum; launch 2 (scale): every workgroup adds these <= 1024 sums in index order itself (8 KB out of the caches: less than a third
// launch costs), forms c, and scales its chunks, the list's last ones first.  No atomics, nothing to clear, the same bits every time.
// Sums are held in 64 bits, so neither the length of the list nor the size of a gradient (|g| up to 3.4e38 squares to 1e77) limits it.
// The list travels in the kernels' arguments (several launches for longer lists): no device table, no copy, nothing that has to outlive the
// call, and a recording holds the addresses by itself.
// Measured (a large copy moves 5.2 TB/s): 65.8 M fp32 values in 172 tensors, nothing to scale: norm 38 us (6.9 TB/s, part of it from the
// 256 MB cache), the second launch 4; 160 M bf16 values into fp32: norm 87 us (320 MB, while the write-back of the last call's 640 MB of
// results is still under way; 3.7 TB/s), scale 178 us (960 MB: 5.4 TB/s); 1.1 M fp32 values in 40 tensors: 4.4 + 2.5 us, two launches.
// In place above the limit (both launches and the host's list): 65.8 M fp32 128 us, 790 MB, bf16 60-65, 1.1 M fp32 12.
#include "t16_dev.h"

namespace hopmi {

constexpr int GC_CHUNK = 16384;                    // elements per work item: 256 threads x 16 vectors of 4, x 8 of 8
constexpr int GC_GRID = 1024;                      // workgroups of the norm's launches at most = sums that the second launch adds

// a list of tensors as kernel arguments, up to 4 KB of them: 250 tensors that are read (and written in place), 165 with outputs
template <bool INTO> struct GcList {
  static constexpr int MAX = INTO ? 165 : 250;
  const void* in[MAX];
  unsigned start[MAX];                             // first chunk of the tensor; its type code in the top two bits
  unsigned tail[MAX];                              // elements in its last chunk
  int count;
  unsigned chunks;
  void* out[INTO ? MAX : 1];
};
static_assert(sizeof(GcList<false>) <= 4040 && sizeof(GcList<true>) <= 4040, "kernel arguments of 4 KB");

struct GcItem { int t; long long base; int cnt; int dt; };
template <bool INTO> __device__ __forceinline__ GcItem gc_find(const GcList<INTO>& L, unsigned chunk) {
  int lo = 0, hi = L.count - 1;                    // the last tensor that starts at or before the chunk
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((L.start[mid] & 0x3fffffffu) <= chunk) lo = mid; else hi = mid - 1;
  }
  const unsigned first = L.start[lo] & 0x3fffffffu, next = lo + 1 < L.count ? L.start[lo + 1] & 0x3fffffffu : L.chunks;
  return GcItem{lo, (long long)(chunk - first) * GC_CHUNK, chunk + 1 == next ? (int)L.tail[lo] : GC_CHUNK, (int)(L.start[lo] >> 30)};
}

// The squares of a vector.  fp32: each in 64 bits.  16-bit values: a square is exact in fp32 and eight are added there first, a relative
// error below 8 x 2^-24 of a sum of positive terms (a conversion and a 64-bit step per value would double the vector work) -- where that
// sum leaves fp32's comfortable range, or is 0, they are taken again in 64 bits.
template <typename T> __device__ __forceinline__ double gc_vec(const u32x4_t& v, const T* t) {
  constexpr int V = Vec<T>::N;
  if constexpr (V == 8) {
    float f = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) f = fmaf(vget(v, e, t), vget(v, e, t), f);
    if (f > 0x1p-60f && f < 0x1p100f) return (double)f;
  }
  double s = 0.0;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const double d = (double)vget(v, e, t);
    s = fma(d, d, s);
  }
  return s;
}
template <typename T> __device__ __forceinline__ double gc_squares(const T* p, int cnt) {
  constexpr int V = Vec<T>::N;
  double s = 0.0;
  const int vecs = cnt / V;
  int i = threadIdx.x;
  for (; i + 3 * 256 < vecs; i += 4 * 256) {       // four loads in flight
    u32x4_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = ld16(p + (i + 256 * k) * V);
#pragma unroll
    for (int k = 0; k < 4; ++k) s += gc_vec(v[k], p);
  }
  for (; i < vecs; i += 256) s += gc_vec(ld16(p + i * V), p);
  if ((int)threadIdx.x < cnt - vecs * V) {
    const double d = (double)to_f(p[vecs * V + threadIdx.x]);
    s = fma(d, d, s);
  }
  return s;
}

__device__ __forceinline__ double block_sum256(double s, double* xch) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) xch[threadIdx.x >> 6] = s;
  __syncthreads();
  return xch[0] + xch[1] + xch[2] + xch[3];
}

__global__ __launch_bounds__(256) void gc_norm_kernel(GcList<false> L, double* __restrict__ sums) {
  __shared__ double xch[4];
  double s = 0.0;
  for (unsigned c = blockIdx.x; c < L.chunks; c += gridDim.x) {
    const GcItem it = gc_find(L, c);
    if (it.dt == T_F32) s += gc_squares(static_cast<const float*>(L.in[it.t]) + it.base, it.cnt);
    else if (it.dt == T_BF16) s += gc_squares(static_cast<const __bf16*>(L.in[it.t]) + it.base, it.cnt);
    else s += gc_squares(static_cast<const _Float16*>(L.in[it.t]) + it.base, it.cnt);
  }
  s = block_sum256(s, xch);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// o = c p; T -> T in place (o == p), or T -> fp32
template <typename T, typename O> __device__ __forceinline__ void gc_scale(const T* p, O* o, int cnt, float c) {
  constexpr int V = Vec<T>::N, VO = Vec<O>::N;
  const int vecs = cnt / V;
  auto put = [&](int i, const u32x4_t& v) {
    float f[V];
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = c * vget(v, e, p);
#pragma unroll
    for (int k = 0; k < V / VO; ++k) st16(o + i * V + k * VO, vpack(f + k * VO, o));
  };
  int i = threadIdx.x;
  for (; i + 3 * 256 < vecs; i += 4 * 256) {       // four loads in flight
    u32x4_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = ld16(p + (i + 256 * k) * V);
#pragma unroll
    for (int k = 0; k < 4; ++k) put(i + 256 * k, v[k]);
  }
  for (; i < vecs; i += 256) put(i, ld16(p + i * V));
  if ((int)threadIdx.x < cnt - vecs * V) {
    const int t = vecs * V + threadIdx.x;
    o[t] = (O)(c * to_f(p[t]));
  }
}

template <bool INTO>
__global__ __launch_bounds__(256) void gc_scale_kernel(GcList<INTO> L, const double* __restrict__ sums, int nsums, float max_norm,
                                                       float* __restrict__ norm_out) {
  __shared__ double xch[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < nsums; i += 256) s += sums[i];
  const double n = sqrt(block_sum256(s, xch));
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)n;
  const double q = (double)max_norm / (n + 1e-6);
  // (a NaN norm gives a NaN factor, an infinite one 0, as the formula says; without a limit the norm is all that is wanted)
  const float c = q > 1.0 || __builtin_isinf(max_norm) ? 1.f : (float)q;
  if (!INTO && c == 1.f) return;
  for (unsigned k = blockIdx.x; k < L.chunks; k += gridDim.x) {
    const GcItem it = gc_find(L, L.chunks - 1 - k);              // from the end: what the norm read last is still in the caches
    auto scale = [&](auto type) {
      using T = decltype(type);
      const T* p = static_cast<const T*>(L.in[it.t]) + it.base;
      if constexpr (INTO) gc_scale(p, static_cast<float*>(L.out[it.t]) + it.base, it.cnt, c);
      else gc_scale(p, const_cast<T*>(p), it.cnt, c);
    };
    if (it.dt == T_F32) scale(float{});
    else if (it.dt == T_BF16) scale(__bf16{});
    else scale(_Float16{});
  }
}

// fills L with tensors [first, ...) of the list; returns the next one.  Empty tensors take no place.
struct GcArgs { const void* const* in; void* const* out; const long long* n; const int* dtypes; int count; };
template <bool INTO> static int gc_fill(GcList<INTO>& L, const GcArgs& A, int first) {
  L.count = 0;
  L.chunks = 0;
  int t = first;
  for (; t < A.count && L.count < GcList<INTO>::MAX; ++t) {
    if (A.n[t] == 0) continue;
    const long long c = (A.n[t] + GC_CHUNK - 1) / GC_CHUNK;
    if (L.chunks + c > 0x3fffffffLL) break;
    L.in[L.count] = A.in[t];
    if (INTO) L.out[L.count] = A.out[t];
    L.start[L.count] = L.chunks | ((unsigned)A.dtypes[t] << 30);
    L.tail[L.count] = (unsigned)(A.n[t] - (c - 1) * GC_CHUNK);
    ++L.count;
    L.chunks += (unsigned)c;
  }
  return t;
}
template <bool INTO> static void gc_scale_all(const GcArgs& A, const double* sums, int nsums, float max_norm, float* norm, hipStream_t st) {
  GcList<INTO> L;
  for (int k = 0, t = 0; k == 0 || t < A.count; ++k) {                         // (no values at all: the norm, 0, and nothing to scale)
    t = gc_fill(L, A, t);
    const unsigned g = L.chunks < 2048u ? (L.chunks > 0 ? L.chunks : 1u) : 2048u;
    hipLaunchKernelGGL((gc_scale_kernel<INTO>), dim3(g), dim3(256), 0, st, L, sums, nsums, max_norm, k == 0 ? norm : nullptr);
  }
}

}  // namespace hopmi

using namespace hopmi;

extern "C" size_t hopmi_grad_clip_ws_bytes(void) { return GC_GRID * sizeof(double); }

extern "C" int hopmi_grad_clip(const void* const* grads, void* const* outs, const long long* numels, const int* dtypes, int count,
                               float max_norm, float* norm, void* ws, void* stream) {
  if (count < 0 || (count > 0 && (!grads || !numels || !dtypes)) || !norm || !ws) {
    set_error("hopmi_grad_clip: null pointer argument / count=%d", count);
    return HOPMI_EINVAL;
  }
  if (!(max_norm >= 0.f)) { set_error("hopmi_grad_clip: max_norm=%g", (double)max_norm); return HOPMI_EINVAL; }
  for (int t = 0; t < count; ++t)
    if (numels[t] < 0 || numels[t] > GC_CHUNK * 0x3ffffff0LL || dtypes[t] < T_F32 || dtypes[t] > T_F16 ||
        (numels[t] > 0 && (!grads[t] || (outs != nullptr && !outs[t])))) {
      set_error("hopmi_grad_clip: tensor %d: n=%lld dtype=%d, or a null pointer", t, numels[t], dtypes[t]);
      return HOPMI_EINVAL;
    }
  const GcArgs A{grads, outs, numels, dtypes, count};
  GcList<false> L;
  int lists = 0;
  for (int t = 0; t < count; ++lists) {
    t = gc_fill(L, A, t);
    if (L.count == 0) break;
  }
  // every launch of the norm gets its share of the sums' places
  if (lists > GC_GRID / 8) { set_error("hopmi_grad_clip: %d tensors are more than one call takes", count); return HOPMI_EINVAL; }
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* sums = static_cast<double*>(ws);
  int nsums = 0;
  for (int k = 0, t = 0; k < lists; ++k) {
    t = gc_fill(L, A, t);
    const int cap = GC_GRID / lists, g = L.chunks < (unsigned)cap ? (int)L.chunks : cap;
    hipLaunchKernelGGL(gc_norm_kernel, dim3(g), dim3(256), 0, st, L, sums + nsums);
    nsums += g;
  }
  if (outs != nullptr) gc_scale_all<true>(A, sums, nsums, max_norm, norm, st);
  else gc_scale_all<false>(A, sums, nsums, max_norm, norm, st);
  return check_launch("hopmi_grad_clip");
}
