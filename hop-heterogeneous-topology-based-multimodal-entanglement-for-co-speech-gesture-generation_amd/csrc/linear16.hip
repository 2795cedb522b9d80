// Matrix products of 16-bit operands (bf16 or fp16, fp32 accumulation) with bias, activation and residual in the epilogue, and the
// products of their backward pass:
//
//   forward    z = X W^T + b,  Y = act(z) + R              X [M][K], W [N][K]: both contiguous along the contraction
//   backward   dz = dY act'(z),  db = sum_rows dz          (one element-wise pass; dz rounded once, to the operands' type)
//              dX = dz W                                   W [N][K] contiguous along the RESULT's columns
//              dW = dz^T X                                 both contiguous along the result's sides, contraction over the rows
//
// One kernel covers the three: each operand's tile is staged into LDS by LDS-DMA (global_load_lds, 16 bytes per lane, no registers in
// between) in the order in which it lies in memory, and read as MFMA fragments either straight (contraction-contiguous: ds_read_b128)
// or through the transposing LDS read (ds_read_b64_tr_b16), so no operand is ever transposed in memory.
// v_mfma_f32_16x16x32: lane 16 q + n holds A[n][8 q ..], B[8 q ..][n] and D[4 q + r][n].  The result's COLUMNS are put on D's rows, so a
// lane ends with four consecutive columns of one row (a 16-byte LDS write); through LDS every thread then gets eight columns of a row,
// and every access of the epilogue is 16 bytes.
// LDS images are swizzled through the SOURCE address of each lane's 16 bytes (the DMA's LDS side is fixed: lane l at base + 16 l):
//   contraction-contiguous tile [rows][64]: 128-byte rows, 16-byte chunk c at c ^ ((row >> 1) & 7): the sixteen lanes that a 16-byte read serves
//   together (0-3, 12-15, 20-23, 24-27, ...) lie on sixteen different slots
//   result-contiguous tile [64][cols]: mn_swizzle() below: the eight rows that one half wave reads lie on eight different 32-byte groups
// Edges: rows past the end are clamped to the last one (their results are not stored); contraction indices past the end read 16 bytes
// of zeros instead, on both operands.  Operands whose rows do not start on 16 bytes, or end inside one, are copied once into rows
// padded with zeros, both in one launch (2171 x 1021 and 427 x 1021 fp16: 6.2 us).
// Bound: the matrix cores for large products, launch, first loads and the epilogue's bytes for small ones.  Measured, bf16, us (2 M N K
// over the time; the same product of the BLAS library on the same card; a product of 8192^3 runs there at 1590 TFLOP/s):
//   16384 x 4096 x 4096   x w^T 405 (1357 TFLOP/s; library 365)   dX 408 (1347; 420)   dW 405 (1357; 470)
//   4352 x 768 -> 2304    x w^T 24.1 (640; 26.8)                   dX 22.9 (672; 25.4)  dW 29.9 (515; 36.3)
//   one row, 768 -> 2304  3.6 (few-row form: 3.5 MB of W)          34 rows, 768 -> 768 with bias and residual 5.2 (recorded: 3.1, 4.7)
// With bias, gelu, residual and the kept pre-activation (three more streams of the result's size) 16384 x 4096 x 4096 takes 470-490,
// 4352 x 768 -> 2304 32.
#include "t16_dev.h"

#include <algorithm>
#include <type_traits>

namespace hopmi {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_SILU = 3 };

__device__ __attribute__((aligned(16))) const unsigned g_zero16[4] = {0, 0, 0, 0};

typedef __bf16 bfrag __attribute__((ext_vector_type(8)));
typedef _Float16 hfrag __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x4 mfma16x32(u32x4_t a, u32x4_t b, f32x4 c, const __bf16*) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bfrag, a), __builtin_bit_cast(bfrag, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16x32(u32x4_t a, u32x4_t b, f32x4 c, const _Float16*) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hfrag, a), __builtin_bit_cast(hfrag, b), c, 0, 0, 0);
}

// The normal distribution's tail, Phi(-u) for u >= 0, = exp(-u^2 / 2) Q(t) with t = 1 / (1 + p u): Q is e^{x^2} erfc(x) / 2 at x = u / sqrt 2,
// a smooth function that a polynomial in t without constant term (Q -> 0 with t) meets to 5e-6 of its value on 0 <= u <= 14 (least
// largest relative error, fitted against 64-bit values); beyond, exp(-u^2 / 2) is 0 in fp32.  RELATIVE accuracy far below the result's
// rounding (2^-9 / 2^-12) also in the tail.  The epilogue of a product with a short contraction is bound by these instructions (15 per
// gelu, two of them at a quarter of the rate).
__device__ __forceinline__ float gauss_tail(float u, float e) {      // e = exp(-u^2 / 2)
  const float t = __builtin_amdgcn_rcpf(fmaf(0.31f, u, 1.f));
  float q = fmaf(-0.07392919063568115f, t, 0.18044988811016083f);
  q = fmaf(q, t, 0.01574617065489292f);
  q = fmaf(q, t, 0.13342832028865814f);
  q = fmaf(q, t, 0.12044187635183334f);
  q = fmaf(q, t, 0.12386061996221542f);
  return q * (t * e);
}
// With u = |z|: gelu(z) = max(z, 0) - u Phi(-u), silu(z) = max(z, 0) - u e^-u / (1 + e^-u), one expression for both signs, which keeps the
// negative tails (e^-u as a square, whose root stays in fp32's normal range as far as u e^-u does).  u is bounded where the tail is 0, so
// the limits z and 0 come out at the infinities too; minimum and maximum are the forms that pass a NaN on.
__device__ __forceinline__ float bounded(float z, float most) { return __builtin_elementwise_minimum(fabsf(z), most); }
__device__ __forceinline__ float act_fwd(float z, int act) {
  if (act == ACT_NONE) return z;
  const float top = __builtin_elementwise_maximum(z, 0.f);
  if (act == ACT_GELU) {
    const float u = bounded(z, 14.f);
    return fmaf(-u, gauss_tail(u, __builtin_amdgcn_exp2f(u * u * -0.72134752044448170f)), top);
  }
  if (act == ACT_SILU) {
    const float u = bounded(z, 170.f), h = __builtin_amdgcn_exp2f(u * -0.72134752044448170f);
    return fmaf(-(u * h) * h, __builtin_amdgcn_rcpf(fmaf(h, h, 1.f)), top);
  }
  return top;
}
// g act'(z).  relu selects: what arrives at an inactive unit is dropped, an infinity or a NaN too (0 times it would be NaN).
__device__ __forceinline__ float act_bwd(float g, float z, int act) {
  if (act == ACT_NONE) return g;
  if (act == ACT_RELU) return z > 0.f ? g : 0.f;
  float d;                                         // act'(-u); act'(u) = 1 - act'(-u)
  if (act == ACT_GELU) {
    const float u = bounded(z, 14.f), e = __builtin_amdgcn_exp2f(u * u * -0.72134752044448170f);
    d = fmaf(u * -0.3989422804014327f, e, gauss_tail(u, e));         // Phi(-u) - u phi(u)
  } else {
    const float u = bounded(z, 170.f), h = __builtin_amdgcn_exp2f(u * -0.72134752044448170f), e = h * h;
    const float r = __builtin_amdgcn_rcpf(1.f + e), s = e * r;       // the sigmoids of u and of -u
    d = s * fmaf(-u, r, 1.f);
  }
  return g * (z > 0.f ? 1.f - d : d);
}

// V (4 or 8) consecutive elements at any element address
template <typename T, int V> __device__ __forceinline__ void ldv(const T* p, float (&f)[V]) {
  u32x4_t w = {0, 0, 0, 0};
  if constexpr (V == 8) w = ld16(p);
  else {
    const u32x2_any v = *reinterpret_cast<const u32x2_any*>(p);
    w[0] = v[0];
    w[1] = v[1];
  }
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = vget(w, e, p);
}
template <typename T, int V> __device__ __forceinline__ void stv(T* p, const float (&f)[V]) {
  if constexpr (V == 8) st16(p, vpack(f, p));
  else {
    u32x2_any v;
    v[0] = pk2(f[0], f[1], p);
    v[1] = pk2(f[2], f[3], p);
    *reinterpret_cast<u32x2_any*>(p) = v;
  }
}

template <typename T> struct Epi16 {
  T* C; long long ldc;
  const T* bias;                 // [N] or null
  const T* res; long long ldr;   // [M][N] or null
  T* z; long long ldz;           // pre-activation values for the backward pass, or null (rounded to the operands' type: what dY act'(z)
                                 // loses by it is a third of what the rounding of dz itself loses)
  int act;
};
// columns col .. col + V - 1 of a row, of which `left` (>= 1) exist
template <int V, typename T> __device__ __forceinline__ void epilogue16(const Epi16<T>& E, long long row, int col, int left, float (&f)[V]) {
  const bool whole = left >= V;
  float b[V], r[V];
#pragma unroll
  for (int e = 0; e < V; ++e) b[e] = r[e] = 0.f;
  if (E.bias != nullptr) {
    if (whole) ldv(E.bias + col, b);
    else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left) b[e] = to_f(E.bias[col + e]);
    }
  }
  if (E.res != nullptr) {
    const T* p = E.res + row * E.ldr + col;
    if (whole) ldv(p, r);
    else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left) r[e] = to_f(p[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] += b[e];
  if (E.z != nullptr) {
    T* p = E.z + row * E.ldz + col;
    if (whole) stv(p, f);
    else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < left) p[e] = (T)f[e];
    }
  }
  if (E.act != ACT_NONE) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = act_fwd(f[e], E.act);
  }
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] += r[e];
  T* p = E.C + row * E.ldc + col;
  if (whole) stv(p, f);
  else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) p[e] = (T)f[e];
  }
}

template <typename T> struct Gemm16 {
  const T* A; long long lda;     // the result's rows:    [M][K] (KA) or [K][M]
  const T* B; long long ldb;     // the result's columns: [N][K] (KB) or [K][N]
  int M, N, K;
  Epi16<T> E;
  float* part;                   // contraction split over several workgroups: fp32 partial results [splits][M][N], else null
  int tiles_m, tiles_n, splits;
};

constexpr int G16_BK = 64;       // contraction per step, two MFMAs': rows of 128 bytes, whole lines, from every operand layout (with half of
                                 // it the L2s' request rate was the bound: 64-byte requests, 80 % of the slots taken)

// the 32-byte group of a result-contiguous tile's row k that holds its group 0 (group p: at p ^ this); rows of 128 bytes lie two to a line
template <int R> __device__ __forceinline__ int mn_swizzle(int k) {
  return R == 64 ? ((k >> 1) & 1) | ((k >> 3) & 1) << 1 : (k & 3) | ((k >> 3) & 1) << 2;
}

// Staging of one operand's tile of R rows (KC: [R][64], else [64][R]) by NW waves, and its fragments.
template <typename T, int R, int NW, bool KC> struct Tile16 {
  static constexpr int BK = G16_BK, BYTES = R * BK * 2;
  static constexpr int NI = BYTES / 1024 / NW;     // 1 KiB DMA instructions per wave and step
  static constexpr int CPR = BK / 8;               // 16-byte chunks per row (KC)
  static constexpr int LPR = KC ? CPR : R / 8;     // lanes per tile row in memory order
  static_assert(64 % LPR == 0 && NI * NW * 1024 == BYTES, "whole rows per instruction, whole instructions per wave");
  const char* base;                                // uniform; advances by one step
  long long adv;
  unsigned off[NI];                                // this lane's bytes from base

  __device__ __forceinline__ void init(const T* p, long long ld, int r0, int r_total, int k0, int lane, int wave) {
    base = reinterpret_cast<const char*>(KC ? p + (long long)r0 * ld + k0 : p + (long long)k0 * ld + r0);
    adv = KC ? BK * 2 : BK * 2 * ld;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = (i * NW + wave) * (64 / LPR) + lane / LPR, s = lane % LPR;
      if (KC) {
        const int rc = min(row, r_total - 1 - r0);             // (r_total > r0)
        off[i] = (unsigned)(rc * ld * 2 + (s ^ ((row >> 1) & 7)) * 16);
      } else {
        const int c = ((((s >> 1) ^ mn_swizzle<R>(row)) << 1) | (s & 1)) * 8;
        const int cc = min(c, ((r_total - r0 + 7) & ~7) - 8);  // (whole chunks: the operand's rows are padded to 8)
        off[i] = (unsigned)(row * ld * 2 + cc * 2);
      }
    }
  }
  // instruction i of a whole step's DMA into `lds`; advance() after the last
  __device__ __forceinline__ void issue(char* lds, int wave, int i) const {
#ifdef __HIP_DEVICE_COMPILE__                      // (the host pass has no such type)
    const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, -1, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)(lds + (i * NW + wave) * 1024), 16, off[i], 0, 0, 0);
#endif
  }
  __device__ __forceinline__ void advance() { base += adv; }
  // ... of a step of which only `left` contraction indices exist (KC: rounded up to 8); zeros behind them
  __device__ __forceinline__ void load_edge(char* lds, int left, int lane, int wave) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = (i * NW + wave) * (64 / LPR) + lane / LPR;
      const int k = KC ? ((lane % LPR) ^ ((row >> 1) & 7)) * 8 : row;
      const char* src = k < left ? base + off[i] : reinterpret_cast<const char*>(g_zero16);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                       (__attribute__((address_space(3))) void*)(lds + (i * NW + wave) * 1024), 16, 0, 0);
    }
    base += adv;
  }
};

// The transposing LDS read: of the 16 lanes that share q, lane n addresses four elements of row n >> 2 and receives column n's four rows.
// (restrict on the pointer is what tells the compiler's wait counting that the read does not touch what a DMA in flight writes: without
// it every such read waited for ALL outstanding DMA, and the steps were not pipelined at all.)
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ s16x4 read_transposed(lds_s16x4* __restrict__ p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }

// the fragment of 16-row block b of a staged tile, contraction half h
template <typename T, int R, bool KC>
__device__ __forceinline__ u32x4_t frag16(const char* lds, int b, int h, int n, int q) {
  if (KC) return *reinterpret_cast<const u32x4_t*>(lds + (b * 16 + n) * 128 + (((h * 4 + q) ^ (n >> 1)) << 4));
  const int sw = mn_swizzle<R>(8 * q + (n >> 2));  // (the same for all the contraction indices this lane addresses)
  const char* a = lds + (h * 32 + 8 * q + (n >> 2)) * (R * 2) + (n & 3) * 8 + ((b ^ sw) << 5);
  const s16x4 lo = read_transposed((lds_s16x4*)a), hi = read_transposed((lds_s16x4*)(a + 4 * R * 2));
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 l = __builtin_bit_cast(u2, lo), h2 = __builtin_bit_cast(u2, hi);
  return u32x4_t{l[0], l[1], h2[0], h2[1]};
}

// s_waitcnt vmcnt(N) lgkmcnt(0), as the builtin (the compiler's own counting then knows of it), and the barrier, with nothing moved across
template <int N> __device__ __forceinline__ void wait_and_meet() {
  static_assert(N < 64, "six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | 7 << 4 | (N >> 4) << 14);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ST LDS buffers of one step each, and two sets of fragment registers: the products of a step's half run on fragments that were read
// during the half before, so neither the DMA (ST - 1 steps ahead) nor the LDS reads are waited for in a wave's own time.  One barrier per
// step, between its halves: there, every wave has read all of this step (its buffer takes step s + ST) and step s + 1 has landed (the
// younger DMA stays in flight: counted).
template <typename T, int BM, int BN, int WR, int WC, int ST, bool KA, bool KB>
__device__ __forceinline__ void gemm16_tile(const Gemm16<T>& G, int id, char* lds) {
  constexpr int NW = WR * WC, RB = BM / WR / 16, CB = BN / WC / 16, BK = G16_BK;
  using TA = Tile16<T, BM, NW, KA>;
  using TB = Tile16<T, BN, NW, KB>;
  constexpr int SB = TA::BYTES + TB::BYTES, NI = TA::NI + TB::NI;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, q = lane >> 4;
  const int wr = wave / WC, wc = wave % WC;
  // workgroups go to the eight XCDs in turn: give each XCD one contiguous stretch of the tile order, and walk that order in groups of
  // eight tile rows, so that what an L2 holds is used by its own workgroups
  const int tiles = G.tiles_m * G.tiles_n, total = tiles * G.splits;
  {
    const int per = total / 8, rem = total % 8, x = id % 8, i = id / 8;
    id = x * per + min(x, rem) + i;
  }
  const int split = id / tiles;
  id -= split * tiles;
  const int per_group = 8 * G.tiles_n, g = id / per_group, first = g * 8, size = min(8, G.tiles_m - first);
  const int tm = first + (id - g * per_group) % size, tn = (id - g * per_group) / size;
  const int r0 = tm * BM, c0 = tn * BN;
  const int all = (G.K + BK - 1) / BK;
  const int s0 = (int)((long long)all * split / G.splits), steps = (int)((long long)all * (split + 1) / G.splits) - s0;
  TA ta;
  TB tb;
  ta.init(G.A, G.lda, r0, G.M, s0 * BK, lane, wave);
  tb.init(G.B, G.ldb, c0, G.N, s0 * BK, lane, wave);
  f32x4 acc[RB][CB];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < CB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto load_any = [&](char* to, int s) {           // step s of this workgroup, which may be the contraction's last
    const int left = G.K - (s0 + s) * BK;
    if (left >= BK) {
#pragma unroll
      for (int i = 0; i < TA::NI; ++i) ta.issue(to, wave, i);
#pragma unroll
      for (int i = 0; i < TB::NI; ++i) tb.issue(to + TA::BYTES, wave, i);
      ta.advance();
      tb.advance();
    } else {
      ta.load_edge(to, KA ? (left + 7) & ~7 : left, lane, wave);
      tb.load_edge(to + TA::BYTES, KB ? (left + 7) & ~7 : left, lane, wave);
    }
  };
  u32x4_t fa0[RB], fb0[CB], fa1[RB], fb1[CB];
  // reads half h of the tiles at `from`; with `to`, a whole step's DMA goes between the reads
  auto fetch = [&](const char* from, int h, u32x4_t (&a)[RB], u32x4_t (&b)[CB], auto dma, char* to) {
#pragma unroll
    for (int i = 0; i < RB + CB; ++i) {
      if (i < RB) a[i] = frag16<T, BM, KA>(from, wr * RB + i, h, n, q);
      else b[i - RB] = frag16<T, BN, KB>(from + TA::BYTES, wc * CB + i - RB, h, n, q);
      if constexpr (decltype(dma)::value) {
#pragma unroll
        for (int k = i * NI / (RB + CB); k < (i + 1) * NI / (RB + CB); ++k) {
          if (k < TA::NI) ta.issue(to, wave, k);
          else tb.issue(to + TA::BYTES, wave, k - TA::NI);
        }
      }
    }
    if constexpr (decltype(dma)::value) {
      ta.advance();
      tb.advance();
    }
  };
  auto multiply = [&](const u32x4_t (&a)[RB], const u32x4_t (&b)[CB], auto dma) {
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) acc[i][j] = mfma16x32(b[j], a[i], acc[i][j], G.A);
    constexpr int NR = RB + CB, PER = RB * CB / NR > 0 ? RB * CB / NR : 1;
#pragma unroll
    for (int k = 0; k < NR; ++k) {                 // the reads and the DMA spread between the products
      __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
      if (k < RB ? KA : KB) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      else __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      if constexpr (decltype(dma)::value) {
        if ((k + 1) * NI / NR > k * NI / NR) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      }
    }
  };
  constexpr std::true_type with_dma{};
  constexpr std::false_type no_dma{};
  char *cur = lds, *nxt = lds + SB;
  auto advance = [&] {
    cur = nxt;
    nxt = nxt + SB == lds + ST * SB ? lds : nxt + SB;
  };
#pragma unroll
  for (int k = 0; k < ST; ++k)
    if (k < steps) load_any(lds + k * SB, k);
  if (steps >= ST) wait_and_meet<NI * (ST - 1)>();
  else wait_and_meet<0>();
  fetch(cur, 0, fa0, fb0, no_dma, nullptr);
  int s = 0;
  for (; s + ST + 1 < steps; ++s) {                // (steps that load whole ones)
    fetch(cur, 1, fa1, fb1, no_dma, nullptr);
    multiply(fa0, fb0, no_dma);
    wait_and_meet<NI * (ST - 2)>();
    fetch(nxt, 0, fa0, fb0, with_dma, cur);
    multiply(fa1, fb1, with_dma);
    advance();
  }
#pragma unroll 1
  for (; s < steps; ++s) {                         // the last ST + 1: the contraction's end may be in what they load
    fetch(cur, 1, fa1, fb1, no_dma, nullptr);
    multiply(fa0, fb0, no_dma);
    if (s + ST - 1 < steps) wait_and_meet<NI * (ST - 2)>();
    else wait_and_meet<0>();
    if (s + ST < steps) load_any(cur, s + ST);
    fetch(nxt, 0, fa0, fb0, no_dma, nullptr);      // (past the last step: values that nothing uses)
    multiply(fa1, fb1, no_dma);
    advance();
  }
  // The results leave through LDS, 16 rows of every wave at a time: a thread then has eight consecutive columns, the same ones in every
  // row it meets (their bias is loaded once), a wave whole lines, and the epilogue's code is there twice, not once per register.  The
  // residual of the next 16 rows travels meanwhile.  (The last reads of the buffers are awaited first; no DMA is in flight any more.)
  constexpr int LDC = BN + 4, VR = BN / 8, ROWS = WR * 16, RPT = ROWS * VR / (64 * NW);
  static_assert(ROWS * LDC * 4 <= ST * SB && (64 * NW) % VR == 0 && RPT * 64 * NW == ROWS * VR, "the staged rows fit the buffers and the threads");
  float* stage = reinterpret_cast<float*>(lds);
  const Epi16<T>& E = G.E;
  const int vc = threadIdx.x % VR * 8, col = c0 + vc, left = G.N - col;
  auto row_of = [&](int i, int k) {
    const int sr = threadIdx.x / VR + k * (64 * NW / VR);
    return (long long)r0 + (sr / 16 * RB + i) * 16 + sr % 16;
  };
  const bool lean = left >= 8 && G.part == nullptr;
  float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (lean && E.bias != nullptr) ldv(E.bias + col, b);
  u32x4_t rn[RPT];
  auto residual = [&](int i) {
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const long long row = row_of(i, k);
      rn[k] = lean && E.res != nullptr && row < G.M ? ld16(E.res + row * E.ldr + col) : u32x4_t{0, 0, 0, 0};
    }
  };
  residual(0);
#pragma unroll 1
  for (int i = 0; i < RB; ++i) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RB; ++k)
      if (k == i) {
#pragma unroll
        for (int j = 0; j < CB; ++j) *reinterpret_cast<f32x4*>(&stage[(wr * 16 + n) * LDC + (wc * CB + j) * 16 + 4 * q]) = acc[k][j];
      }
    u32x4_t rc[RPT];
#pragma unroll
    for (int k = 0; k < RPT; ++k) rc[k] = rn[k];
    if (i + 1 < RB) residual(i + 1);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RPT; ++k) {
      const long long row = row_of(i, k);
      if (row >= G.M || left <= 0) continue;
      const float* p = &stage[(threadIdx.x / VR + k * (64 * NW / VR)) * LDC + vc];
      const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
      float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      if (lean) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += b[e];
        if (E.z != nullptr) stv(E.z + row * E.ldz + col, f);
        if (E.act != ACT_NONE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = act_fwd(f[e], E.act);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += vget(rc[k], e, G.A);
        stv(E.C + row * E.ldc + col, f);
      } else if (G.part != nullptr) {
        float* o = G.part + ((long long)split * G.M + row) * G.N + col;
        if (left >= 8) {
          st16(o, vpack(f, o));
          st16(o + 4, vpack(f + 4, o));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < left) o[e] = f[e];
        }
      } else {
        for (int h = 0; h < 2; ++h) {              // (the result's last columns)
          float g[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) g[e] = h ? f[4 + e] : f[e];
          if (left > 4 * h) epilogue16<4>(E, row, col + 4 * h, left - 4 * h, g);
        }
      }
    }
  }
}

template <typename T, int BM, int BN, int WR, int WC, int ST, bool KA, bool KB>
__global__ __launch_bounds__(64 * WR * WC, 2) void gemm16_kernel(Gemm16<T> G) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  gemm16_tile<T, BM, BN, WR, WC, ST, KA, KB>(G, blockIdx.x, lds);
}

// out[c] = the sum of G partial rows in column c; NW waves take every NW-th row of 64 columns from c0 on, sixteen loads in flight, and
// meet in `red` [NW][64]
template <int NW, typename T> __device__ __forceinline__ void colsum16(const float* part, int G, int N, T* out, int c0, float* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = c0 + lane;
  float s = 0.f;
  if (c < N) {
    int g = wave;
    for (; g + 15 * NW < G; g += 16 * NW) {
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = part[(long long)(g + k * NW) * N + c];
#pragma unroll
      for (int k = 0; k < 16; ++k) s += v[k];
    }
    for (; g < G; g += NW) s += part[(long long)g * N + c];
  }
  red[wave * 64 + lane] = s;
  __syncthreads();
  if (wave == 0 && c < N) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) t += red[k * 64 + lane];
    out[c] = (T)t;
  }
}

// The two products of a backward pass and the bias gradient's last sums in one launch: dz is all they wait for, and none of them fills
// the chip evenly at ordinary sizes.  The product with the longer contraction first, then the other, the sums last.  Measured against the
// three launches, bf16, us: 4352 x 768 x 2304 (rows x inputs x outputs) 47 / 60, 4352 x 768 x 768 24 / 35, 600 x 4096 x 1024 19 / 30, 34 x 768 x 768
// 5.8 / 10.5, 64 x 64 x 64 3.4 / 7.6.
template <typename T> struct Pair16 {
  Gemm16<T> dx, dw;                                // layouts 1 and 2
  int dx_first, n0, n01;                           // workgroups of the first product, of both
  const float* part; int groups, n;                // partial column sums [groups][n]
  T* dbias;
};
template <typename T, int BM, int BN, int WR, int WC, int ST>
__global__ __launch_bounds__(64 * WR * WC, 2) void gemm16_pair_kernel(Pair16<T> P) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int id = blockIdx.x;
  if (id >= P.n01) colsum16<WR * WC>(P.part, P.groups, P.n, P.dbias, (id - P.n01) * 64, reinterpret_cast<float*>(lds));
  else {
    const bool first = id < P.n0;
    const int mine = first ? id : id - P.n0;
    if (first == (P.dx_first != 0)) gemm16_tile<T, BM, BN, WR, WC, ST, true, false>(P.dx, mine, lds);
    else gemm16_tile<T, BM, BN, WR, WC, ST, false, false>(P.dw, mine, lds);
  }
}

// the partial results of a split contraction, added in split order, through the same epilogue; four columns per thread
template <typename T>
__global__ __launch_bounds__(256) void gemm16_join_kernel(const float* __restrict__ part, int splits, int M, int N, Epi16<T> E) {
  const int q4 = (N + 3) / 4;
  const long long total = (long long)M * q4, plane = (long long)M * N;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long row = i / q4;
    const int col = (int)(i - row * q4) * 4, left = N - col;
    const float* p = part + row * N + col;
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    if (left >= 4) {
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const u32x4_t v = ld16(p + s * plane);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] += __uint_as_float(v[e]);
      }
    } else {
      for (int s = 0; s < splits; ++s) {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < left) f[e] += p[s * plane + e];
      }
    }
    epilogue16<4>(E, row, col, left, f);
  }
}

// Few rows (M <= 64): bound by reading W once.  A workgroup takes 16 columns of the result for all rows; its eight waves share the
// contraction in stretches of 128 (256 contiguous bytes of each of 16 rows of W per wave and stretch), straight from memory into MFMA
// operands at any alignment, and add their partial tiles through LDS.
constexpr int FEW_ROWS = 64, FEW_WAVES = 8;
template <typename T, int MB>
__global__ __launch_bounds__(64 * FEW_WAVES) void gemm16_few_kernel(Gemm16<T> G) {
  __shared__ float red[FEW_WAVES][MB][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, q = lane >> 4;
  const int c0 = blockIdx.x * 16;
  const T* wp = G.B + (long long)min(c0 + n, G.N - 1) * G.ldb + 8 * q;
  const T* xp[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) xp[m] = G.A + (long long)min(m * 16 + n, G.M - 1) * G.lda + 8 * q;
  f32x4 acc[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  // eight elements from contraction index k on, zeros past the end
  auto tail8 = [&](const T* p, int k) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = k + e < G.K ? to_f(p[e]) : 0.f;
    return vpack(f, p);
  };
  u32x4_t w[2][4], x[2][MB][4];                    // a stretch's operands and, on their way, the next one's
  auto load = [&](int k0, u32x4_t (&w)[4], u32x4_t (&x)[MB][4]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) w[s] = ld16(wp + k0 + 32 * s);
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int s = 0; s < 4; ++s) x[m][s] = ld16(xp[m] + k0 + 32 * s);
  };
  auto multiply = [&](const u32x4_t (&w)[4], const u32x4_t (&x)[MB][4]) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int m = 0; m < MB; ++m) acc[m] = mfma16x32(w[s], x[m][s], acc[m], G.A);
  };
  constexpr int STRIDE = FEW_WAVES * 128;
  int k0 = wave * 128;
  if (k0 + 128 <= G.K) load(k0, w[0], x[0]);
  for (; k0 + 128 <= G.K; k0 += 2 * STRIDE) {
    if (k0 + STRIDE + 128 <= G.K) load(k0 + STRIDE, w[1], x[1]);
    multiply(w[0], x[0]);
    if (k0 + STRIDE + 128 > G.K) { k0 += STRIDE; break; }
    if (k0 + 2 * STRIDE + 128 <= G.K) load(k0 + 2 * STRIDE, w[0], x[0]);
    multiply(w[1], x[1]);
  }
  for (int k = k0; k < G.K && k < k0 + 128; k += 32) {         // the contraction's end, if it lies in this wave's last stretch
    const int kl = k + 8 * q;
    const u32x4_t we = kl + 8 <= G.K ? ld16(wp + k) : tail8(wp + k, kl);
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const u32x4_t xe = kl + 8 <= G.K ? ld16(xp[m] + k) : tail8(xp[m] + k, kl);
      acc[m] = mfma16x32(we, xe, acc[m], G.A);
    }
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][m][n][4 * q + r] = acc[m][r];
  __syncthreads();
  for (int i = threadIdx.x; i < MB * 64; i += 64 * FEW_WAVES) {
    const int row = i >> 2, c = (i & 3) * 4, left = G.N - c0 - c;
    if (row >= G.M || left <= 0) continue;
    float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < FEW_WAVES; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] += red[w][row >> 4][row & 15][c + e];
    epilogue16<4>(G.E, row, c0 + c, left, f);
  }
}

// dz = dY act'(z) (rows padded with zeros to ldd, a multiple of 8; null: not wanted) and the partial column sums of the UNROUNDED dz of
// each row group, part [gridDim.y][N] (null: not wanted).  dz is rounded to the operands' type because the products' matrix instructions
// take 16-bit operands; in two parts it would double both.  The gradients' error against 64 bits grows by it from 0.0017 to 0.0024 of
// their norm in bf16, from 0.00021 to 0.00030 in fp16.  A wave takes 512 columns of every fourth row of its group.  Bound: HBM (two
// reads, one write): 16384 x 4096 bf16 gelu 77 us (5.2 TB/s), 4352 x 2304 14.7 (4.1).  Six workgroups per CU with one row at a time hide the
// latency best: with two rows in flight per wave (more registers) 80 and 17.4, with four 87 and 18.7; on eight or four workgroups per CU
// 81 and 14.7, 78 and 16.2.
template <typename T>
__global__ __launch_bounds__(256) void act_bwd16_kernel(const T* __restrict__ dy, long long ldy, const T* __restrict__ z, long long ldz,
                                                        T* __restrict__ dz, long long ldd, float* __restrict__ part, int M, int N, int act) {
  __shared__ float red[3][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 512 + lane * 8, left = N - col;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const long long first = (long long)blockIdx.y * 4 + wave, step = (long long)gridDim.y * 4;
  auto finish = [&](long long row, float (&g)[8], const u32x4_t& zv) {
    if (act != ACT_NONE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = act_bwd(g[e], vget(zv, e, dy), act);
    }
    if (dz != nullptr) st16(dz + row * ldd + col, vpack(g, dy));
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] += g[e];
  };
  if (left >= 8) {
    for (long long row = first; row < M; row += step) {
      const u32x4_t gv = ld16(dy + row * ldy + col);
      u32x4_t zv;                                                // (finish() looks at it where there is an activation)
      if (act != ACT_NONE) zv = ld16(z + row * ldz + col);
      float g[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = vget(gv, e, dy);
      finish(row, g, zv);
    }
  } else if (left > 0) {                                         // the rows' ends (those of z and dz are padded to 8)
    for (long long row = first; row < M; row += step) {
      float g[8];
      const T* p = dy + row * ldy + col;
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = e < left ? to_f(p[e]) : 0.f;
      u32x4_t zv = act != ACT_NONE ? ld16(z + row * ldz + col) : u32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) zv[w] &= (2 * w < left ? 0xffffu : 0u) | (2 * w + 1 < left ? 0xffff0000u : 0u);   // (z's padding holds anything)
      finish(row, g, zv);
    }
  }
  if (part == nullptr) return;
  if (wave > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) red[wave - 1][lane * 8 + e] = s[e];
  }
  __syncthreads();
  if (wave == 0 && left > 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) part[(long long)blockIdx.y * N + col + e] = s[e] + red[0][lane * 8 + e] + red[1][lane * 8 + e] + red[2][lane * 8 + e];
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void colsum16_join_kernel(const float* __restrict__ part, int G, int N, T* __restrict__ out) {
  __shared__ float red[16 * 64];
  colsum16<16>(part, G, N, out, blockIdx.x * 64, red);
}

// rows of N 16-bit elements at any stride and alignment -> rows of ldp (a multiple of 8) elements, zeros behind the N-th (bits are moved,
// whatever they stand for); one or two of them in a launch (workgroups from `first` on take the second)
struct Pad16 { const unsigned short* src; long long lds; unsigned short* dst; long long ldp; int M, N; };
__global__ __launch_bounds__(256) void pad16_kernel(Pad16 A, Pad16 B, unsigned first) {
  const bool second = blockIdx.x >= first;
  const Pad16& P = second ? B : A;
  const unsigned block = second ? blockIdx.x - first : blockIdx.x, blocks = second ? gridDim.x - first : first;
  const int vecs = (int)(P.ldp / 8), N = P.N;
  const long long total = (long long)P.M * vecs;
  for (long long i = (long long)block * 256 + threadIdx.x; i < total; i += (long long)blocks * 256) {
    const long long row = i / vecs;
    const int col = (int)(i - row * vecs) * 8;
    const unsigned short* p = P.src + row * P.lds + col;
    u32x4_t v = {0, 0, 0, 0};
    if (col + 8 <= N) v = ld16(p);
    else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < N) v[e >> 1] |= (unsigned)p[e] << (16 * (e & 1));
    }
    st16(P.dst + row * P.ldp + col, v);
  }
}

// ---- geometry
// Five tile forms.  What a product costs is the rounds it takes to put its workgroups on the chip, the steps of each, and, where the
// contraction is split, the join; no one form is best: 16384 x 4096 x 4096 takes 407 us in tiles of 256 x 256, 445 / 456 / 549 in 192 x 128 /
// 128 x 128 (two buffers) / 128 x 128 (four); 4352 x 2304 x 768 27.0 / 23.8 / 27.2 / 31.9 and 30.7 in 64 x 64; 4352 x 768 x 2304 - / 32.4 / 27.2 /
// 23.0 / 31.1; 512 x 768 x 768 - / 14.0 / 10.7 / 10.9 / 7.3.  So the choice is by a model of that cost, us, whose constants were fitted to
// such times (24 products, all layouts, 1 to 16384 workgroups: within 15 % of nearly all of them):
//   start     launch, first DMA, and the first tile's end
//   alone     a step where a CU holds one workgroup;  together: where it holds as many as fit, for all of them
//   end       a round's epilogue
struct Form16 { int bm, bn, slots; float start, alone, together, end; };
static constexpr Form16 FORMS16[] = {{256, 256, 256, 8.f, 1.55f, 1.55f, 1.f},     // 8 waves, 128 KB of LDS: one workgroup per CU
                                     {192, 128, 512, 6.f, 0.69f, 1.35f, 1.5f},    // not for result-contiguous A (rows of 192)
                                     {128, 128, 512, 4.5f, 0.62f, 0.89f, 2.5f},
                                     {128, 128, 256, 5.f, 0.47f, 0.47f, 1.5f},    // four buffers: one workgroup per CU, DMA three steps ahead
                                     {64, 64, 512, 3.f, 0.18f, 0.35f, 0.8f}};
struct Plan16 { int form, tiles_m, tiles_n, splits; float us; };
static Plan16 plan16(int M, int N, int K, int layout) {
  const int steps = (K + G16_BK - 1) / G16_BK;
  Plan16 best{0, 0, 0, 0, 0.f};
  for (int f = 0; f < 5; ++f) {
    if (f == 1 && layout == 2) continue;
    const Form16& F = FORMS16[f];
    const int threads = f == 0 ? 512 : 256;
    const long long tm = ((long long)M + F.bm - 1) / F.bm, tn = ((long long)N + F.bn - 1) / F.bn, tiles = tm * tn;
    // (more splits than fill the chip once, or steps of fewer than four, never pay: the join reads every partial result again)
    for (int sp = 1; sp <= 32 && (sp == 1 || (tiles * sp <= F.slots && steps / sp >= 4)); sp += sp < 4 ? 1 : sp / 2) {
      if (tiles * sp * threads >= 1LL << 32) break;          // (more than a launch counts)
      const long long wgs = tiles * sp, rounds = wgs / F.slots, rest = wgs - rounds * F.slots;
      const float n = (float)((steps + sp - 1) / sp);
      float t = F.start + (float)rounds * (n * F.together + F.end);
      if (rest > 0) t += n * (rest > 256 ? F.together : F.alone) + F.end;
      if (sp > 1) t += 4.f + 8.f * (float)sp * (float)M * (float)N / 12e6f;
      if (best.splits == 0 || t < best.us) best = Plan16{f, (int)tm, (int)tn, sp, t};
    }
  }
  return best;
}

// The two products of a backward pass in one launch: a form, the splits of each, and the model's time.  The workgroups of the longer
// steps come first, so a slot takes one after the other: `a` of `na` steps, then `b` of `nb`.
struct PlanPair16 { int form, dx_first; Plan16 dx, dw; float us; };
static float pair_steps(long long a, long long na, long long b, long long nb, long long slots) {
  if (a + b <= slots) return (float)std::max(na, nb);
  const long long t0 = a / slots * na, busy = a % slots, t1 = busy > 0 ? t0 + na : t0;      // slots - busy are free at t0, busy at t1
  auto first = [&](long long from) {                                                        // the first end, in steps of nb from `from`, by which b are done
    long long lo = 0, hi = (t1 - t0) / nb + (b + slots - 1) / slots + 1;
    while (lo < hi) {
      const long long mid = (lo + hi) / 2, t = from + mid * nb;
      const long long done = (t - t0) / nb * (slots - busy) + (t > t1 ? (t - t1) / nb * busy : 0);
      if (done >= b) hi = mid; else lo = mid + 1;
    }
    return from + lo * nb;
  };
  return (float)std::max(std::min(first(t0), first(t1)), t1);
}
static PlanPair16 plan_pair16(int M, int N, int K) {
  const int s1 = (N + G16_BK - 1) / G16_BK, s2 = (M + G16_BK - 1) / G16_BK;                 // dX [M][K] over N, dW [N][K] over M
  PlanPair16 best{-1, 0, {}, {}, 0.f};
  for (int f = 2; f < 5; ++f) {                    // (products that fill the chip in larger tiles gain nothing from each other)
    const Form16& F = FORMS16[f];
    const long long m1 = ((long long)M + F.bm - 1) / F.bm, m2 = ((long long)N + F.bm - 1) / F.bm, n1 = ((long long)K + F.bn - 1) / F.bn;
    for (int p1 = 1; p1 <= 4 && (p1 == 1 || (m1 * n1 * p1 <= F.slots && s1 / p1 >= 4)); p1 *= 2)
      for (int p2 = 1; p2 <= 32 && (p2 == 1 || (m2 * n1 * p2 <= F.slots && s2 / p2 >= 4)); p2 += p2 < 4 ? 1 : p2 / 2) {
        const long long w1 = m1 * n1 * p1, w2 = m2 * n1 * p2, l1 = (s1 + p1 - 1) / p1, l2 = (s2 + p2 - 1) / p2;
        if ((w1 + w2 + N) * 512 >= 1LL << 32) continue;                                     // (more than a launch counts)
        const bool first = l1 >= l2;
        const float n = first ? pair_steps(w1, l1, w2, l2, F.slots) : pair_steps(w2, l2, w1, l1, F.slots);
        const float more = (float)((w1 + w2 - 1) / F.slots);                                // rounds behind the first: each fills its buffers again
        float t = F.start + n * (w1 + w2 > 256 ? F.together : F.alone) + F.end * (more + 1.f) + more * (F.slots > 256 ? 2.f : 3.f);
        if (p1 > 1) t += 4.f + 8.f * (float)p1 * (float)M * (float)K / 12e6f;
        if (p2 > 1) t += 4.f + 8.f * (float)p2 * (float)N * (float)K / 12e6f;
        if (best.form < 0 || t < best.us)
          best = PlanPair16{f, first, {f, (int)m1, (int)n1, p1, t}, {f, (int)m2, (int)n1, p2, t}, t};
      }
  }
  return best;
}

// Up to 64 rows of x w^T: the few-row form where the models find it faster (its own: a start, and per stretch of the contraction W's
// fragment and each row's), and wherever the operands do not lie as tiles need them.  Measured, few rows / tiles, us: one row of 768 x 768
// 3.2 / 5.2, of 4096 x 4096 8.7 / 10.8; 34 rows of 768 x 768 4.8 / 5.6, of 2304 -> 768 9.1 / 7.6, of 4096 x 4096 15.7 / 11.8; 64 rows of 128 x 128 3.2 /
// 3.9, of 768 x 768 5.9 / 5.6; one row of 1024 -> 16384, four workgroups per CU, 9.1 / 8.4.
static bool few16(int M, int N, int K, const Plan16& p) {
  const float per_k = 1.05e-3f + 5.2e-5f * (float)M, rounds = (float)((N + 16 * 256 - 1) / (16 * 256));
  return p.splits == 0 || 2.5f + rounds * (float)K * per_k <= p.us - 0.2f;
}

template <typename T, int BM, int BN, int WR, int WC, int ST, bool KA, bool KB> static void gemm16_go(const Gemm16<T>& G, hipStream_t st) {
  constexpr int bytes = ST * (BM + BN) * G16_BK * 2;
  const auto k = gemm16_kernel<T, BM, BN, WR, WC, ST, KA, KB>;
  static std::atomic<unsigned long long> told{0};
  allow_lds(reinterpret_cast<const void*>(k), bytes, told);
  hipLaunchKernelGGL(k, dim3((unsigned)(G.tiles_m * G.tiles_n * G.splits)), dim3(64 * WR * WC), bytes, st, G);
}
template <typename T> static void gemm16_join(const Gemm16<T>& G, const Plan16& p, const float* ws, hipStream_t st) {
  if (p.splits < 2) return;
  const long long work = (long long)G.M * ((G.N + 3) / 4), blocks = (work + 255) / 256;
  hipLaunchKernelGGL((gemm16_join_kernel<T>), dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, ws, p.splits, G.M, G.N, G.E);
}
template <typename T> static void gemm16_run(Gemm16<T> G, int layout, bool few, const Plan16& p, float* ws, hipStream_t st) {
  if (few) {
    const dim3 grid((G.N + 15) / 16), block(64 * FEW_WAVES);
    if (G.M <= 16) hipLaunchKernelGGL((gemm16_few_kernel<T, 1>), grid, block, 0, st, G);
    else if (G.M <= 32) hipLaunchKernelGGL((gemm16_few_kernel<T, 2>), grid, block, 0, st, G);
    else if (G.M <= 48) hipLaunchKernelGGL((gemm16_few_kernel<T, 3>), grid, block, 0, st, G);
    else hipLaunchKernelGGL((gemm16_few_kernel<T, 4>), grid, block, 0, st, G);
    return;
  }
  G.tiles_m = p.tiles_m;
  G.tiles_n = p.tiles_n;
  G.splits = p.splits;
  G.part = p.splits > 1 ? ws : nullptr;
  auto go = [&](auto ka, auto kb) {
    constexpr bool KA = decltype(ka)::value, KB = decltype(kb)::value;
    if (p.form == 0) gemm16_go<T, 256, 256, 2, 4, 2, KA, KB>(G, st);
    else if (p.form == 1) {
      if constexpr (KA) gemm16_go<T, 192, 128, 2, 2, 2, KA, KB>(G, st);
    } else if (p.form == 2) gemm16_go<T, 128, 128, 2, 2, 2, KA, KB>(G, st);
    else if (p.form == 3) gemm16_go<T, 128, 128, 2, 2, 4, KA, KB>(G, st);
    else gemm16_go<T, 64, 64, 2, 2, 4, KA, KB>(G, st);
  };
  if (layout == 0) go(std::true_type{}, std::true_type{});
  else if (layout == 1) go(std::true_type{}, std::false_type{});
  else go(std::false_type{}, std::false_type{});
  gemm16_join(G, p, ws, st);
}

template <typename T, int BM, int BN, int WR, int WC, int ST> static void pair16_go(const Pair16<T>& P, hipStream_t st) {
  constexpr int bytes = ST * (BM + BN) * G16_BK * 2;
  const auto k = gemm16_pair_kernel<T, BM, BN, WR, WC, ST>;
  static std::atomic<unsigned long long> told{0};
  allow_lds(reinterpret_cast<const void*>(k), bytes, told);
  hipLaunchKernelGGL(k, dim3((unsigned)(P.n01 + (P.dbias != nullptr ? (P.n + 63) / 64 : 0))), dim3(64 * WR * WC), bytes, st, P);
}
template <typename T> static void pair16_run(Pair16<T> P, const PlanPair16& p, float* ws, hipStream_t st) {
  float* ws2 = p.dx.splits > 1 ? ws + (size_t)p.dx.splits * P.dx.M * P.dx.N : ws;
  auto set = [&](Gemm16<T>& G, const Plan16& q, float* part) {
    G.tiles_m = q.tiles_m;
    G.tiles_n = q.tiles_n;
    G.splits = q.splits;
    G.part = q.splits > 1 ? part : nullptr;
    return q.tiles_m * q.tiles_n * q.splits;
  };
  const int w1 = set(P.dx, p.dx, ws), w2 = set(P.dw, p.dw, ws2);
  P.dx_first = p.dx_first;
  P.n0 = p.dx_first ? w1 : w2;
  P.n01 = w1 + w2;
  if (p.form == 2) pair16_go<T, 128, 128, 2, 2, 2>(P, st);
  else if (p.form == 3) pair16_go<T, 128, 128, 2, 2, 4>(P, st);
  else pair16_go<T, 64, 64, 2, 2, 4>(P, st);
  gemm16_join(P.dx, p.dx, ws, st);
  gemm16_join(P.dw, p.dw, ws2, st);
}

// rows of `cols` elements as tiles are staged from them: 16-byte addresses and ends, and a stride whose 256 rows an offset of 32 bits spans
static bool g16_direct(const void* p, long long ld, int cols) {
  return !((reinterpret_cast<uintptr_t>(p) & 15) | (ld & 7) | (cols & 7)) && ld <= 1 << 22;
}
// sides whose sums with a tile's count in 31 bits
static bool g16_sides(int M, int N, int K) {
  constexpr int MOST = 1 << 30;
  return M >= 1 && N >= 1 && K >= 1 && M <= MOST && N <= MOST && K <= MOST;
}
static int act_bwd_groups(int M, int N) {
  const int strips = (N + 511) / 512;
  const long long quads = ((long long)M + 3) / 4;
  long long g = 1536 / strips;
  g = g < 1 ? 1 : g;
  return (int)(quads < g ? quads : g);
}

}  // namespace hopmi

using namespace hopmi;

extern "C" size_t hopmi_gemm16_ws_floats(int M, int N, int K, int layout) {
  if (!g16_sides(M, N, K) || layout < 0 || layout > 2) return 0;
  const Plan16 p = plan16(M, N, K, layout);
  if (layout == 0 && M <= FEW_ROWS && few16(M, N, K, p)) return 0;
  return p.splits > 1 ? (size_t)p.splits * M * N : 0;
}

extern "C" int hopmi_gemm16_form(int M, int N, int K, int layout, int* form, int* splits) {
  if (!g16_sides(M, N, K) || layout < 0 || layout > 2 || !form || !splits) {
    set_error("hopmi_gemm16_form: M=%d N=%d K=%d (sides of 1 to 2^30) layout=%d, or a null pointer", M, N, K, layout);
    return HOPMI_EINVAL;
  }
  const Plan16 p = plan16(M, N, K, layout);
  const bool few = layout == 0 && M <= FEW_ROWS && few16(M, N, K, p);
  *form = few || p.splits == 0 ? -1 : p.form;
  *splits = few ? 1 : p.splits;
  return HOPMI_OK;
}

extern "C" int hopmi_gemm16_direct(const void* p, long long ld, int cols) { return g16_direct(p, ld, cols) ? 1 : 0; }

extern "C" int hopmi_gemm16(const void* A, long long lda, const void* B, long long ldb, int layout, void* C, long long ldc, const void* bias,
                            const void* res, long long ldr, void* z, long long ldz, int act, int M, int N, int K, int dtype, float* ws,
                            void* stream) {
  if (!A || !B || !C) { set_error("hopmi_gemm16: null pointer argument"); return HOPMI_EINVAL; }
  if (M < 1 || N < 1 || K < 1 || layout < 0 || layout > 2 || act < ACT_NONE || act > ACT_SILU) {
    set_error("hopmi_gemm16: M=%d N=%d K=%d layout=%d activation=%d", M, N, K, layout, act);
    return HOPMI_EINVAL;
  }
  if (!g16_sides(M, N, K)) { set_error("hopmi_gemm16: M=%d N=%d K=%d (sides of up to 2^30) are more tiles than a launch counts", M, N, K); return HOPMI_EINVAL; }
  if (dtype != T_BF16 && dtype != T_F16) { set_error("hopmi_gemm16: dtype=%d (1 bf16, 2 fp16)", dtype); return HOPMI_EINVAL; }
  const int ca = layout == 2 ? M : K, cb = layout == 0 ? K : N;
  if (lda < ca || ldb < cb || ldc < N || (res && ldr < N) || (z && ldz < N)) { set_error("hopmi_gemm16: a row stride below the row's length"); return HOPMI_EINVAL; }
  const Plan16 p = plan16(M, N, K, layout);
  const bool tiled = g16_direct(A, lda, 0) && g16_direct(B, ldb, 0) && lda >= ((ca + 7) & ~7) && ldb >= ((cb + 7) & ~7);
  // (rows whose last vector is not whole may be followed by anything where rows run along the contraction: the few-row form then)
  const bool few = layout == 0 && M <= FEW_ROWS && (!tiled || (K & 7) || few16(M, N, K, p));
  if (!few && !tiled) {
    set_error("hopmi_gemm16: operands need rows on 16 bytes that end on 16 bytes, with strides up to 2^22 elements (hopmi_pad16)");
    return HOPMI_EINVAL;
  }
  if (!few && p.splits == 0) { set_error("hopmi_gemm16: M=%d N=%d are more tiles than a launch counts", M, N); return HOPMI_EINVAL; }
  if (!few && p.splits > 1 && !ws) { set_error("hopmi_gemm16: null workspace"); return HOPMI_EINVAL; }
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    Gemm16<T> G;
    G.A = static_cast<const T*>(A); G.lda = lda;
    G.B = static_cast<const T*>(B); G.ldb = ldb;
    G.M = M; G.N = N; G.K = K;
    G.E = Epi16<T>{static_cast<T*>(C), ldc, static_cast<const T*>(bias), static_cast<const T*>(res), ldr, static_cast<T*>(z), ldz, act};
    G.part = nullptr; G.tiles_m = G.tiles_n = G.splits = 1;
    gemm16_run(G, layout, few, p, ws, st);
  };
  if (dtype == T_BF16) go(__bf16{}); else go(_Float16{});
  return check_launch("hopmi_gemm16");
}

// What the backward pass launches: the pair, or (form < 0) two products of their own and the bias gradient's sums (3 us of their own
// beside the products), by the models of both: products in 256 x 256 tiles fill the chip by themselves, and short contractions of many
// tiles are better off in forms of their own (128 rows of 4096 x 4096: 34 us in three launches, 40 as a pair).
struct Backward16 { PlanPair16 pair; Plan16 dx, dw; size_t floats; };
static Backward16 plan_backward16(int M, int N, int K) {
  Backward16 b;
  b.dx = plan16(M, K, N, 1);
  b.dw = plan16(N, K, M, 2);
  b.pair = plan_pair16(M, N, K);
  if (b.pair.form >= 0 && b.pair.us > b.dx.us + b.dw.us + 3.f) b.pair.form = -1;
  const Plan16 &x = b.pair.form >= 0 ? b.pair.dx : b.dx, &w = b.pair.form >= 0 ? b.pair.dw : b.dw;
  b.floats = (x.splits > 1 ? (size_t)x.splits * M * K : 0) + (w.splits > 1 ? (size_t)w.splits * N * K : 0);
  return b;
}

extern "C" size_t hopmi_linear16_bwd_ws_floats(int M, int N, int K) { return g16_sides(M, N, K) ? plan_backward16(M, N, K).floats : 0; }

extern "C" int hopmi_linear16_bwd_form(int M, int N, int K, int* pair, int* dx_form, int* dx_splits, int* dw_form, int* dw_splits) {
  if (!g16_sides(M, N, K) || !pair || !dx_form || !dx_splits || !dw_form || !dw_splits) {
    set_error("hopmi_linear16_bwd_form: M=%d N=%d K=%d (sides of 1 to 2^30), or a null pointer", M, N, K);
    return HOPMI_EINVAL;
  }
  const Backward16 b = plan_backward16(M, N, K);
  *pair = b.pair.form >= 0;
  const Plan16 &x = *pair ? b.pair.dx : b.dx, &w = *pair ? b.pair.dw : b.dw;
  *dx_form = x.splits == 0 ? -1 : x.form;
  *dx_splits = x.splits;
  *dw_form = w.splits == 0 ? -1 : w.form;
  *dw_splits = w.splits;
  return HOPMI_OK;
}

extern "C" int hopmi_linear16_bwd(const void* dz, long long lddz, const void* w, long long ldw, const void* x, long long ldx, void* dx,
                                  void* dw, const float* part, void* dbias, int M, int N, int K, int dtype, float* ws, void* stream) {
  if (!dz || !w || !x || !dx || !dw || (dbias && !part)) { set_error("hopmi_linear16_bwd: null pointer argument"); return HOPMI_EINVAL; }
  if (!g16_sides(M, N, K) || (dtype != T_BF16 && dtype != T_F16)) {
    set_error("hopmi_linear16_bwd: M=%d N=%d K=%d (sides of 1 to 2^30) dtype=%d (1 bf16, 2 fp16)", M, N, K, dtype);
    return HOPMI_EINVAL;
  }
  const int n8 = (N + 7) & ~7, k8 = (K + 7) & ~7;
  if (!g16_direct(dz, lddz, 0) || !g16_direct(w, ldw, 0) || !g16_direct(x, ldx, 0) || lddz < n8 || ldw < k8 || ldx < k8) {
    set_error("hopmi_linear16_bwd: operands need rows on 16 bytes that end on 16 bytes, with strides up to 2^22 elements (hopmi_pad16)");
    return HOPMI_EINVAL;
  }
  const Backward16 b = plan_backward16(M, N, K);
  if (b.floats > 0 && !ws) { set_error("hopmi_linear16_bwd: null workspace"); return HOPMI_EINVAL; }
  if (b.pair.form < 0 && (b.dx.splits == 0 || b.dw.splits == 0)) {
    set_error("hopmi_linear16_bwd: M=%d N=%d K=%d are more tiles than a launch counts", M, N, K);
    return HOPMI_EINVAL;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    auto product = [&](const void* A, long long lda, const void* B, long long ldb, void* C, int m, int k) {
      Gemm16<T> G;
      G.A = static_cast<const T*>(A); G.lda = lda;
      G.B = static_cast<const T*>(B); G.ldb = ldb;
      G.M = m; G.N = K; G.K = k;
      G.E = Epi16<T>{static_cast<T*>(C), K, nullptr, nullptr, 0, nullptr, 0, ACT_NONE};
      G.part = nullptr; G.tiles_m = G.tiles_n = G.splits = 1;
      return G;
    };
    const Gemm16<T> X = product(dz, lddz, w, ldw, dx, M, N), W = product(dz, lddz, x, ldx, dw, N, M);
    const int groups = act_bwd_groups(M, N);
    T* db = static_cast<T*>(dbias);
    if (b.pair.form >= 0) {
      pair16_run(Pair16<T>{X, W, 0, 0, 0, part, groups, N, db}, b.pair, ws, st);
      return;
    }
    if (db != nullptr) hipLaunchKernelGGL((colsum16_join_kernel<T>), dim3((N + 63) / 64), dim3(1024), 0, st, part, groups, N, db);
    gemm16_run(X, 1, false, b.dx, ws, st);
    gemm16_run(W, 2, false, b.dw, b.dx.splits > 1 ? ws + (size_t)b.dx.splits * M * K : ws, st);
  };
  if (dtype == T_BF16) go(__bf16{}); else go(_Float16{});
  return check_launch("hopmi_linear16_bwd");
}

static bool pad16_fits(const void* src, long long lds, const void* dst, long long ldp, int M, int N) {
  if (src && dst && g16_sides(M, N, 1) && lds >= N && ldp >= N && ldp <= 1LL << 31 && !(ldp & 7) && !(reinterpret_cast<uintptr_t>(dst) & 15)) return true;
  set_error("hopmi_pad16: M=%d N=%d strides %lld -> %lld, or a null or unaligned pointer", M, N, lds, ldp);
  return false;
}
static unsigned pad16_blocks(long long ldp, int M) {
  const long long blocks = ((long long)M * (ldp / 8) + 255) / 256;
  return (unsigned)(blocks < 4096 ? blocks : 4096);
}
extern "C" int hopmi_pad16(const void* src, long long lds_, void* dst, long long ldp, int M, int N, void* stream) {
  if (!pad16_fits(src, lds_, dst, ldp, M, N)) return HOPMI_EINVAL;
  const Pad16 P{static_cast<const unsigned short*>(src), lds_, static_cast<unsigned short*>(dst), ldp, M, N};
  const unsigned blocks = pad16_blocks(ldp, M);
  hipLaunchKernelGGL(pad16_kernel, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream), P, P, blocks);
  return check_launch("hopmi_pad16");
}
extern "C" int hopmi_pad16_two(const void* src, long long lds_, void* dst, long long ldp, int M, int N, const void* src2, long long lds2,
                               void* dst2, long long ldp2, int M2, int N2, void* stream) {
  if (!pad16_fits(src, lds_, dst, ldp, M, N) || !pad16_fits(src2, lds2, dst2, ldp2, M2, N2)) return HOPMI_EINVAL;
  const Pad16 P{static_cast<const unsigned short*>(src), lds_, static_cast<unsigned short*>(dst), ldp, M, N};
  const Pad16 Q{static_cast<const unsigned short*>(src2), lds2, static_cast<unsigned short*>(dst2), ldp2, M2, N2};
  const unsigned first = pad16_blocks(ldp, M), blocks = first + pad16_blocks(ldp2, M2);
  hipLaunchKernelGGL(pad16_kernel, dim3(blocks), dim3(256), 0, static_cast<hipStream_t>(stream), P, Q, first);
  return check_launch("hopmi_pad16_two");
}

extern "C" size_t hopmi_act_bwd16_ws_floats(int M, int N) { return !g16_sides(M, N, 1) ? 0 : (size_t)act_bwd_groups(M, N) * N; }

extern "C" int hopmi_act_bwd16(const void* dy, long long ldy, const void* z, long long ldz, void* dz, long long ldd, void* dbias, float* ws,
                               int act, int M, int N, int dtype, void* stream) {
  if (!dy || !g16_sides(M, N, 1) || ldy < N || act < ACT_NONE || act > ACT_SILU || (dtype != T_BF16 && dtype != T_F16) || (act != ACT_NONE && !z) ||
      (z && ldz < ((N + 7) & ~7)) || (dz && (ldd < N || (ldd & 7))) || (dbias && !ws)) {
    set_error("hopmi_act_bwd16: M=%d N=%d activation=%d dtype=%d, a bad stride, or a null pointer", M, N, act, dtype);
    return HOPMI_EINVAL;
  }
  if (!dz && !ws) return HOPMI_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int groups = act_bwd_groups(M, N);
  auto go = [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((act_bwd16_kernel<T>), dim3((N + 511) / 512, groups), dim3(256), 0, st, static_cast<const T*>(dy), ldy,
                       static_cast<const T*>(z), ldz, static_cast<T*>(dz), ldd, ws, M, N, act);
    if (dbias)
      hipLaunchKernelGGL((colsum16_join_kernel<T>), dim3((N + 63) / 64), dim3(1024), 0, st, ws, groups, N, static_cast<T*>(dbias));
  };
  if (dtype == T_BF16) go(__bf16{}); else go(_Float16{});
  return check_launch("hopmi_act_bwd16");
}
