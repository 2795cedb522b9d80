// One fused WaveNet layer of the HOP graph-wavenet block (reference: model/gwnet.py:181-237), forward:
//
//   r^      = BN_{i-1}(y_{i-1})                      applied ON LOAD as r^ = y*scale + shift (identity for layer 0)
//   u       = tanh(Wf0 r^[t] + Wf1 r^[t+d] + bf) * sigmoid(Wg0 r^[t] + Wg1 r^[t+d] + bg)     gwnet.py:186-200
//   utail   = u[last 4 frames]                       the only part of the skip path that reaches the output
//   y_i     = Wm.[u; uA1; uA2] + bm + r^[t+d]        graph conv + residual, gwnet.py:224-233 (pre-BN)
//   stats   = per-channel sum / sum of squares of y_i (BatchNorm2d batch statistics, gwnet.py:237)
//
// replacing ~15 aten launches and 10 activation round trips per layer by one kernel: the activation tile
// is read once (two time taps), everything between lives in LDS/registers, y_i is written once.
//
// Work decomposition: the output rows (clip b, frame t', node v) are flat, row = slab*V + v with
// slab = b*T_out + t'; a workgroup of 8 waves takes tiles of S consecutive output slabs (<= 80 rows): wave (w, h)
// owns output channels 16 w + [0, 16) of the 16-row MFMA tiles of row half h.  The two channel contractions (gated TCN,
// K = 2 taps x 64; graph conv, K = 192) run as three-term products of scaled fp16 hi/lo operands on v_mfma_f32_16x16x32_f16
// (f16_dev.h: 22 significand bits per operand -- fp32-equivalent -- at 5.3x the fp32 matrix rate; rounds 2-4 carried bf16 hi/lo
// pairs, 2^-16 per product); their weight operands are split MFMA fragments with one power-of-two scale per output channel,
// prepared once per forward pass for all layers (hopmi_wn_prepare_weights) and held in registers (112 VGPRs); the activations
// are scaled (one power of two per tile row, found over both taps by the 16 lanes that hold the row; a fixed one for the gate
// activations, which are bounded by 1, and their node mixes, bounded through the mix matrices' column sums) and split once when
// the tile is committed to LDS.  The node mix (K = V) stays on the exact-fp32 MFMA.
// Per tile: two tap panels HBM -> registers -> normalise -> split -> LDS; TCN; gate (hardware exp); skip tail;
// node mix; contraction; epilogue adds bias + residual, stores y and accumulates the BatchNorm partial sums.  A tiny
// second kernel turns the per-(workgroup, half) partials into mean / rstd / running stats / the next layer's
// scale+shift in a fixed order (reproducible).  Nothing is saved for the backward: it recomputes the gates from xin.
#include <hip/hip_ext.h>

#define HOPMI_FILE_ID 7          // (diagnostic build: common.h, split_check)
#include "attn_dev.h"
#include "f16_dev.h"
#include "io_dev.h"
#include "wn_dev.h"

namespace hopmi {

constexpr int WN_FIN_G = 16;     // workgroups of the BatchNorm finalisation (wn_bn_finalize_kernel)

// gate non-linearities on the hardware exp and reciprocal (v_exp_f32, v_rcp_f32 through __builtin_amdgcn_rcpf: 1 ulp;
// __frcp_rn expands to the ten-instruction IEEE division sequence): absolute error ~1e-7, far inside the 1e-3 bar
__device__ __forceinline__ float sigmoid_(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }
__device__ __forceinline__ float tanh_(float x) { return 2.f * __builtin_amdgcn_rcpf(1.f + __expf(-2.f * x)) - 1.f; }
// u = tanh(a) sigmoid(g) = (1 - e^-2a) / ((1 + e^-2a)(1 + e^-g)) with ONE reciprocal; the exponents are clamped so that
// the denominator stays finite (tanh(-22) = -1 and sigmoid(-44) = 8e-20 to fp32 precision)
__device__ __forceinline__ float gate_(float a, float g) {
  const float ea = __expf(fminf(-2.f * a, 44.f)), eg = __expf(fminf(-g, 44.f));
  return (1.f - ea) * __builtin_amdgcn_rcpf((1.f + ea) * (1.f + eg));
}

// ---- weight images -----------------------------------------------------------------------------------------------
constexpr int WN_MAX_LAYERS = 8;
struct WeightPtrs { const float* wf[WN_MAX_LAYERS]; const float* wg[WN_MAX_LAYERS]; const float* wm[WN_MAX_LAYERS]; };

// one thread = one (hi, lo) pair of 16-byte fragment units: 8 consecutive-k weights of one output channel, scaled by the power
// of two that puts the largest magnitude of the channel's whole row (both taps of a TCN matrix: 128 weights; Wm: 192) in
// [2^14, 2^15); the thread that holds a row's first unit also writes the row's inverse scale behind the fragments
__global__ __launch_bounds__(256) void wn_prepare_weights_kernel(WeightPtrs P, u32x4* __restrict__ img) {
  constexpr int PAIRS = WIMG_UNITS / 2;                     // 3584 per layer
  const int layer = blockIdx.y;
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= PAIRS) return;
  const int lane = t & 63, n = lane & 15, q = lane >> 4;
  u32x4* out = img + (size_t)layer * WIMGH_UNITS;
  float* inv_out = reinterpret_cast<float*>(out + WIMG_UNITS);
  float v[8];
  int unit, inv_at;
  const float* rowp;
  int row_n4;
  bool first;
  if (t < WIMG_TCN_UNITS / 2) {
    const int ks = (t >> 6) & 3, gate = (t >> 8) & 1, w = t >> 9;
    rowp = (gate ? P.wg[layer] : P.wf[layer]) + (size_t)(16 * w + n) * C * 2;      // Conv2d layout [out][in][1][tap]: 128 floats
    row_n4 = 2 * C / 4;
    const float* src = rowp + (32 * (ks & 1) + 8 * q) * 2 + (ks >> 1);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = src[2 * e];
    unit = (((w * 2 + gate) * 4 + ks) * 2) * 64 + lane;
    inv_at = gate * C + 16 * w + n;
    first = ks == 0 && q == 0;
  } else {
    const int u = t - WIMG_TCN_UNITS / 2;
    const int wks = u >> 6, ks = wks % 6, w = wks / 6;
    rowp = P.wm[layer] + (size_t)(16 * w + n) * K3;
    row_n4 = K3 / 4;
    const float* src = rowp + 32 * ks + 8 * q;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = src[e];
    unit = WIMG_TCN_UNITS + ((w * 6 + ks) * 2) * 64 + lane;
    inv_at = 2 * C + 16 * w + n;
    first = ks == 0 && q == 0;
  }
  float m = 0.f;
  for (int i = 0; i < row_n4; ++i) m = absmax4(m, reinterpret_cast<const float4*>(rowp)[i]);
  const float sc = scale_for_absmax(m);
  const Split8 s = split8h(make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]), sc);
  out[unit] = s.hi;
  out[unit + 64] = s.lo;
  if (first) inv_out[inv_at] = inv_pow2(sc);
}

// per-thread description of the NIT rows this thread streams in a tile (the idx -> row map is the same
// for the load phase and the skip-tail store phase)
template <int NIT>
struct RowMap {
  int in0[NIT];     // float4 index of the tap-0 source row start (+ c4), clamped into the tensor
  int tail[NIT];    // float4 index into utail (+ c4) or -1
  bool ok[NIT];     // row < R
};

constexpr int WN_THREADS = 512;
constexpr int wn_rows_nit(int mt) { return ((16 * mt + 4) * 16 + WN_THREADS - 1) / WN_THREADS; }

// Node mix of the slabs s = h, h + 2, ... of a tile, wave (w, h) doing channels [16w, 16w+16): reads u (fp32) from
// U[row][LDD], writes the split results next to u in the contraction operand images:
//   Hb[s*V + node][64*(1+blk) + c] = sum_v A{blk+1}[v][node] * U[s*V + v][c]
// The product is taken transposed, D[i = channel][j = stacked node m], so a lane ends up with 4 consecutive channels of
// one node: one 8-byte store per part.  Stacked nodes m >= 2V of the padded N go to the dump row.
template <int KS, int MTN, bool HOLD>
__device__ __forceinline__ void node_mix2(const float* U, __bf16* Hh, __bf16* Hl, const float* AT, const GcnGeom& g, int nsl,
                                          int dump_row, int w, int h, int q, int j, float sh) {
  // HOLD: the mix matrix fragments stay in registers for all slabs of the tile (small V: many slabs per tile);
  // !HOLD: they are read from LDS next to each MFMA (V = 42: one slab per tile, 66 registers would buy nothing)
  const int V = g.V;
  float am[HOLD ? MTN : 1][HOLD ? KS : 1];
  int woff[MTN];
#pragma unroll
  for (int mt = 0; mt < MTN; ++mt) {
    if (HOLD) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) am[mt][ks] = AT[(4 * ks + q) * g.ldA + 16 * mt + j];   // B[k = v][n = m]
    }
    const int m = 16 * mt + j;
    const int blk = (m >= V) ? 1 : 0;
    woff[mt] = (m < 2 * V) ? ((m - blk * V) * HS + C * (1 + blk) + 16 * w + 4 * q) : -1;     // relative to the slab's first row
  }
  const int dump = dump_row * HS + C + 16 * w + 4 * q;
  // SGN slabs per iteration: SGN * MTN independent accumulator chains keep the matrix pipe fed while the LDS reads of
  // the group and the previous group's split + stores are in flight
  constexpr int SGN = HOLD ? 2 : 1;
  int s = h;
  for (; s + 2 * (SGN - 1) < nsl; s += 2 * SGN) {
    float xb[SGN][KS];
#pragma unroll
    for (int sg = 0; sg < SGN; ++sg)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) xb[sg][ks] = U[((s + 2 * sg) * V + 4 * ks + q) * LDD + 16 * w + j];   // A[i = c][k = v]
#pragma unroll
    for (int mt = 0; mt < MTN; ++mt) {
      f32x4 acc[SGN];
#pragma unroll
      for (int sg = 0; sg < SGN; ++sg) acc[sg] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const float b = HOLD ? am[mt][ks] : AT[(4 * ks + q) * g.ldA + 16 * mt + j];
#pragma unroll
        for (int sg = 0; sg < SGN; ++sg) acc[sg] = mfma16(xb[sg][ks], b, acc[sg]);
      }
#pragma unroll
      for (int sg = 0; sg < SGN; ++sg) {
        const int off = woff[mt] >= 0 ? (s + 2 * sg) * V * HS + woff[mt] : dump;
        const Split4 sp = split4h(acc[sg][0] * sh, acc[sg][1] * sh, acc[sg][2] * sh, acc[sg][3] * sh);
        *reinterpret_cast<u32x2*>(Hh + off) = sp.hi;
        *reinterpret_cast<u32x2*>(Hl + off) = sp.lo;
      }
    }
  }
  for (; s < nsl; s += 2) {                            // leftover slab of this half
    float xb[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) xb[ks] = U[(s * V + 4 * ks + q) * LDD + 16 * w + j];
#pragma unroll
    for (int mt = 0; mt < MTN; ++mt) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) acc = mfma16(xb[ks], HOLD ? am[mt][ks] : AT[(4 * ks + q) * g.ldA + 16 * mt + j], acc);
      const int off = woff[mt] >= 0 ? s * V * HS + woff[mt] : dump;
      const Split4 sp = split4h(acc[0] * sh, acc[1] * sh, acc[2] * sh, acc[3] * sh);
      *reinterpret_cast<u32x2*>(Hh + off) = sp.hi;
      *reinterpret_cast<u32x2*>(Hl + off) = sp.lo;
    }
  }
}

// any V (runtime loops)
__device__ __forceinline__ void node_mix2_generic(const float* U, __bf16* Hh, __bf16* Hl, const float* AT, const GcnGeom& g,
                                                  int nsl, int w, int h, int q, int j, float sh) {
  const int V = g.V;
  const int ksteps = g.KP >> 2, mt_n = g.MP >> 4;
  for (int s = h; s < nsl; s += 2) {
    const float* us = U + (s * V + q) * LDD + 16 * w + j;
    for (int mt = 0; mt < mt_n; ++mt) {
      const float* at = AT + q * g.ldA + 16 * mt + j;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      for (int ks = 0; ks < ksteps; ++ks) acc = mfma16(us[4 * ks * LDD], at[4 * ks * g.ldA], acc);
      const int m = 16 * mt + j;
      if (m < 2 * V) {
        const int blk = (m >= V) ? 1 : 0;
        const int off = (s * V + m - blk * V) * HS + C * (1 + blk) + 16 * w + 4 * q;
        const Split4 sp = split4h(acc[0] * sh, acc[1] * sh, acc[2] * sh, acc[3] * sh);
        *reinterpret_cast<u32x2*>(Hh + off) = sp.hi;
        *reinterpret_cast<u32x2*>(Hl + off) = sp.lo;
      }
    }
  }
}

// Weight fragments are loaded from the L2-resident image per tile -- the TCN set behind the tile's activation loads, the
// graph-conv set behind the TCN phase -- so that neither is loop-carried (112-163 VGPRs, no spills).  MULTI = the
// workgroup walks several tiles (plain loop, loads at the top of every iteration); !MULTI = the grid covers the launch,
// one tile per workgroup: straight-line code whose first loads are issued before anything else.
// GCN = false: the gate-only form (TCN + gate, no graph conv: what the backward uses to regenerate the gate values).
// TS = storage type of the activation tensors xin, y and utail (float or __bf16, io_dev.h): read / written 4 channels at a time,
// all arithmetic in fp32 (the bf16 form of BASELINE.json configs 2 / 4: y is rounded once, when it is stored).
template <int MT, bool MULTI, bool GCN, typename TS>
__global__ __launch_bounds__(WN_THREADS) void wn_layer_fwd_kernel(const TS* __restrict__ xin, const float* __restrict__ scsh,
                                                                  const u32x4* __restrict__ wimg,
                                                                  const float* __restrict__ bfp, const float* __restrict__ bgp,
                                                                  const float* __restrict__ prep,
                                                                  const float* __restrict__ bm, TS* __restrict__ y,
                                                                  float* __restrict__ fs, TS* __restrict__ utail,
                                                                  float* __restrict__ stats_part, LayerGeom L, int utail_ld4) {
  constexpr int do_gcn = GCN ? 1 : 0;
  extern __shared__ __attribute__((aligned(16))) float smem[];
  HOPMI_STAMP(0);
  const GcnGeom& g = L.g;
  constexpr int NIT = wn_rows_nit(MT);
  constexpr int MTH = (MT + 1) / 2;                // 16-row tiles per row half
  constexpr int rows_lds = 16 * MT + 4;            // == g.rows_lds; a constant here so that the image offsets are immediates
  // LDS: four split activation images (tap 0/1 x hi/lo), u in fp32 (node-mix operand, skip tail), the split
  // contraction operand images u | uA1 | uA2 (hi, lo), the mix matrix
  __bf16* R0h = reinterpret_cast<__bf16*>(smem);   // [rows_lds][RS]
  __bf16* R0l = R0h + rows_lds * RS;
  __bf16* R1h = R0l + rows_lds * RS;
  __bf16* R1l = R1h + rows_lds * RS;
  float* U = reinterpret_cast<float*>(R1l + rows_lds * RS);       // [rows_lds][LDD]
  __bf16* Hh = reinterpret_cast<__bf16*>(U + rows_lds * LDD);     // [rows_lds][HS]
  __bf16* Hl = Hh + rows_lds * HS;
  float* AT = reinterpret_cast<float*>(Hl + rows_lds * HS);       // [KP][ldA]
  float* RSI = AT + g.KP * g.ldA;                                 // [rows_lds] inverse of the tap panels' row scales
  // (the wave index is wave-uniform: as a scalar it keeps every per-wave base address out of the vector registers)
  int tid = threadIdx.x;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), w = wv & 3, h = wv >> 2;
  int lane = tid & 63, q = lane >> 4, j = lane & 15, c4 = tid & 15;     // (re-derived per tile in the MULTI loop, see there)
  const int V = g.V;
  const int shift4 = L.d * V * 16;                 // tap-1 row offset in float4 units

  // Issue order of the prologue: the FIRST tile's activation loads (HBM latency), then the weight fragments, biases and
  // the mix image (L2): vmcnt retires in order, so the tile can be committed while the weights are still in flight.
  RowMap<NIT> rm;
  float4 x0r[NIT], x1r[NIT];
  auto issue_tile = [&](int tile) {
    const int slab0 = tile * g.S;
    const int R = min(g.S, L.n_slabs - slab0) * V;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int row = (tid >> 4) + (WN_THREADS / 16) * it;
      const int rc = min(row, R - 1);
      const int s = (int)((rc + 0.5f) * L.invV);
      const int v = rc - s * V;
      const int slab = slab0 + s;
      const int b = (int)((slab + 0.5f) * L.invT);
      const int tp = slab - b * L.T_out;
      rm.ok[it] = row < R;
      rm.in0[it] = ((b * L.T_in + tp) * V + v) * 16 + c4;
      rm.tail[it] = (utail != nullptr && rm.ok[it] && tp >= L.T_out - 4) ? ((b * 4 + tp - (L.T_out - 4)) * V + v) * utail_ld4 + c4 : -1;
      x0r[it] = ld4(xin + 4 * (size_t)rm.in0[it]);
      x1r[it] = ld4(xin + 4 * (size_t)(rm.in0[it] + shift4));
    }
  };
  if (!MULTI) issue_tile(blockIdx.x);

  // ---- weights: the wave's split A-operand fragments, straight from the prepared image (L2-resident) ---------------
  u32x4 wt[2][4][2];                               // [gate f/g][k step: tap = ks>>1][hi/lo]
  u32x4 wm[6][2];                                  // [k step][hi/lo]
  auto load_wt = [&]() {
    const u32x4* tp = wimg + (size_t)(w * 2) * 4 * 2 * 64 + lane;
#pragma unroll
    for (int gate = 0; gate < 2; ++gate)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int part = 0; part < 2; ++part) wt[gate][ks][part] = tp[((gate * 4 + ks) * 2 + part) * 64];
  };
  if (!MULTI) load_wt();
  auto load_wm = [&]() {
    const u32x4* mp = wimg + WIMG_TCN_UNITS + (size_t)(w * 6) * 2 * 64 + lane;
#pragma unroll
    for (int ks = 0; ks < 6; ++ks)
#pragma unroll
      for (int part = 0; part < 2; ++part) wm[ks][part] = mp[(ks * 2 + part) * 64];
  };
  // MFMA products are taken transposed (D[i = channel][j = row]): a lane holds 4 consecutive channels
  // 16w + 4q + r of one row, so gate outputs, u, the split images and y move as 8/16-byte LDS / global accesses
  const float4 bf4 = *reinterpret_cast<const float4*>(bfp + 16 * w + 4 * q);
  const float4 bg4 = *reinterpret_cast<const float4*>(bgp + 16 * w + 4 * q);
  float4 bias4 = make_float4(0.f, 0.f, 0.f, 0.f);
  if (do_gcn) bias4 = *reinterpret_cast<const float4*>(bm + 16 * w + 4 * q);
  // inverse weight scales of this lane's 4 output channels (behind the fragments in the image); the operand scale of the
  // contraction images u | uA1 | uA2 (behind the mix images in `prep`: hopmi_gcn_prepare bounds the mixes by the column sums)
  const float* winv = reinterpret_cast<const float*>(wimg + WIMG_UNITS);
  const float4 isf4 = *reinterpret_cast<const float4*>(winv + 16 * w + 4 * q);
  const float4 isg4 = *reinterpret_cast<const float4*>(winv + C + 16 * w + 4 * q);
  float4 ism4 = make_float4(0.f, 0.f, 0.f, 0.f);
  float sh = H_UNIT_SCALE;
  if (do_gcn) {
    const float* ptr = prep + g.KP * g.ldA + g.K2P * g.ldB;
    sh = ptr[0];
    const float ish = ptr[1];
    const float4 t = *reinterpret_cast<const float4*>(winv + 2 * C + 16 * w + 4 * q);
    ism4 = make_float4(t.x * ish, t.y * ish, t.z * ish, t.w * ish);
  }
  const float4 sc4 = reinterpret_cast<const float4*>(scsh)[c4];
  const float4 sh4 = reinterpret_cast<const float4*>(scsh + C)[c4];
  f32x4 st1 = {0.f, 0.f, 0.f, 0.f}, st2 = {0.f, 0.f, 0.f, 0.f};   // BatchNorm partial sums of channels 16w + 4q + r
  // the 4 padding rows behind the tile are read by the node mix's K padding (times zero): keep them finite
  for (int idx = tid; idx < 4 * C; idx += WN_THREADS) U[(16 * MT + idx / C) * LDD + idx % C] = 0.f;
  if (GCN) {
    // the mix image -> LDS (plain copy loop: a register array staged across the loads ended up in scratch).  Its loads are
    // the youngest in flight, so the wait also covers the tile's activation loads -- which the commit below needs anyway.
    // Eight loads in flight per thread and round trip: one load per iteration made the V = 42 image (20 KB+) 23 us of a
    // 39 us launch (tools/probes/wn_stamps.py).
    const int at_n4 = (g.KP * g.ldA) >> 2;
    for (int idx0 = tid; idx0 < at_n4; idx0 += 8 * WN_THREADS) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int idx = idx0 + u * WN_THREADS;
        v[u] = reinterpret_cast<const float4*>(prep)[min(idx, at_n4 - 1)];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int idx = idx0 + u * WN_THREADS;
        if (idx < at_n4) reinterpret_cast<float4*>(AT)[idx] = v[u];
      }
    }
  }

  for (int tile = blockIdx.x; tile < g.ntiles; tile += gridDim.x) {
    HOPMI_STAMP(1);
    const int slab0 = tile * g.S;
    const int nsl = min(g.S, L.n_slabs - slab0);
    const int R = nsl * V;
    const size_t orow0 = (size_t)slab0 * V;        // first flat output row of the tile

    // ---- phase 0: stream both tap panels, normalise, split, commit to LDS -------------------------
    if (MULTI) {
      // every address below derives from the lane index: hiding it from the optimiser per iteration keeps the (dozens of)
      // loop-invariant address registers from being hoisted out of the loop and held across all phases
      asm volatile("" : "+v"(tid));
      lane = tid & 63; q = lane >> 4; j = lane & 15; c4 = tid & 15;
      issue_tile(tile);
      load_wt();
    }
    __syncthreads();                               // previous tile's LDS fully consumed
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int row = (tid >> 4) + (WN_THREADS / 16) * it;
      if (row < rows_lds) {
        float4 a = x0r[it], b2 = x1r[it];
        a = make_float4(a.x * sc4.x + sh4.x, a.y * sc4.y + sh4.y, a.z * sc4.z + sh4.z, a.w * sc4.w + sh4.w);
        b2 = make_float4(b2.x * sc4.x + sh4.x, b2.y * sc4.y + sh4.y, b2.z * sc4.z + sh4.z, b2.w * sc4.w + sh4.w);
        if (!rm.ok[it]) { a = make_float4(0.f, 0.f, 0.f, 0.f); b2 = a; }
        // one power-of-two scale per output row over BOTH taps (they meet in one accumulator): the row's 128 values sit in
        // the 16 lanes of a DPP row
        const float rs = scale_for_absmax(row16_max(absmax4(absmax4(0.f, a), b2)));
        const Split4 sa = split4h(a.x * rs, a.y * rs, a.z * rs, a.w * rs), sb = split4h(b2.x * rs, b2.y * rs, b2.z * rs, b2.w * rs);
        const int off = row * RS + 4 * c4;
        *reinterpret_cast<u32x2*>(R0h + off) = sa.hi;
        *reinterpret_cast<u32x2*>(R0l + off) = sa.lo;
        *reinterpret_cast<u32x2*>(R1h + off) = sb.hi;
        *reinterpret_cast<u32x2*>(R1l + off) = sb.lo;
        if (c4 == 0) RSI[row] = inv_pow2(rs);
      }
    }
    __syncthreads();
    HOPMI_STAMP(2);

    // ---- phase 1: gated TCN (two taps, two gates) as split products, gate, u -> LDS ---------------------
    {
      f32x4 af[MTH], ag[MTH];
#pragma unroll
      for (int i = 0; i < MTH; ++i) { af[i] = {0.f, 0.f, 0.f, 0.f}; ag[i] = {0.f, 0.f, 0.f, 0.f}; }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const __bf16* rh = ((ks >> 1) ? R1h : R0h) + j * RS + 32 * (ks & 1) + 8 * q;      // B[k = 32(ks&1) + 8q + e][j = row]
        const __bf16* rl = ((ks >> 1) ? R1l : R0l) + j * RS + 32 * (ks & 1) + 8 * q;
        u32x4 bh[MTH], bl[MTH];
#pragma unroll
        for (int i = 0; i < MTH; ++i) {
          const int mt = min(h * MTH + i, MT - 1);
          bh[i] = *reinterpret_cast<const u32x4*>(rh + 16 * mt * RS);
          bl[i] = *reinterpret_cast<const u32x4*>(rl + 16 * mt * RS);
        }
#pragma unroll
        for (int i = 0; i < MTH; ++i) {
          af[i] = mfma_h3(wt[0][ks][0], wt[0][ks][1], bh[i], bl[i], af[i]);
          ag[i] = mfma_h3(wt[1][ks][0], wt[1][ks][1], bh[i], bl[i], ag[i]);
        }
      }
      HOPMI_STAMP(3);
      if (do_gcn) {                                      // lands behind the gate / node-mix phases
        __builtin_amdgcn_sched_barrier(0);               // (not above the TCN: its fragments are still live there)
        load_wm();
      }
      // af[i][r] = filter pre-activation of row 16 mt + j, channel 16w + 4q + r
#pragma unroll
      for (int i = 0; i < MTH; ++i) {
        const int mt = h * MTH + i;
        if (mt < MT) {
          const int row = 16 * mt + j;
          const float ir = RSI[row];
          // pre-activations in real units: accumulator x (1 / row scale) x (1 / output channel's weight scale) + bias
          const float4 pf = make_float4(af[i][0] * (isf4.x * ir) + bf4.x, af[i][1] * (isf4.y * ir) + bf4.y, af[i][2] * (isf4.z * ir) + bf4.z,
                                        af[i][3] * (isf4.w * ir) + bf4.w);
          const float4 pg = make_float4(ag[i][0] * (isg4.x * ir) + bg4.x, ag[i][1] * (isg4.y * ir) + bg4.y, ag[i][2] * (isg4.z * ir) + bg4.z,
                                        ag[i][3] * (isg4.w * ir) + bg4.w);
          const float4 u = make_float4(gate_(pf.x, pg.x), gate_(pf.y, pg.y), gate_(pf.z, pg.z), gate_(pf.w, pg.w));
          *reinterpret_cast<float4*>(U + row * LDD + 16 * w + 4 * q) = u;
          const Split4 su = split4h(u.x * sh, u.y * sh, u.z * sh, u.w * sh);
          *reinterpret_cast<u32x2*>(Hh + row * HS + 16 * w + 4 * q) = su.hi;
          *reinterpret_cast<u32x2*>(Hl + row * HS + 16 * w + 4 * q) = su.lo;
          if (fs != nullptr && row < R) {                        // diagnostic output only
            const float4 f = make_float4(tanh_(pf.x), tanh_(pf.y), tanh_(pf.z), tanh_(pf.w));
            const float4 sg = make_float4(sigmoid_(pg.x), sigmoid_(pg.y), sigmoid_(pg.z), sigmoid_(pg.w));
            float* fp = fs + (orow0 + row) * (2 * C) + 16 * w + 4 * q;
            *reinterpret_cast<float4*>(fp) = f;
            *reinterpret_cast<float4*>(fp + C) = sg;
          }
        }
      }
    }
    __syncthreads();
    HOPMI_STAMP(4);

    // ---- skip tail: last 4 frames of u, LDS -> HBM as whole 256-B rows ------------------------------
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int row = (tid >> 4) + (WN_THREADS / 16) * it;
      if (rm.tail[it] >= 0) st4(utail + 4 * (size_t)rm.tail[it], *reinterpret_cast<const float4*>(U + row * LDD + 4 * c4));
    }

    if (do_gcn) {
      // ---- phase 2: node mix (exact fp32 MFMA, K = V) -> split images -------------------------------------------------
      const int dump_row = rows_lds - 1;
      if (V == 9) node_mix2<3, 2, true>(U, Hh, Hl, AT, g, nsl, dump_row, w, h, q, j, sh);              // TED
      else if (V == 42) node_mix2<11, 6, false>(U, Hh, Hl, AT, g, nsl, dump_row, w, h, q, j, sh);       // TED-Expressive
      else node_mix2_generic(U, Hh, Hl, AT, g, nsl, w, h, q, j, sh);
      __syncthreads();
      HOPMI_STAMP(5);
      // ---- phase 3: channel contraction (K = 192, split products) + bias + residual, y store, BatchNorm sums ------
      f32x4 acc[MTH];
#pragma unroll
      for (int i = 0; i < MTH; ++i) acc[i] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 6; ++ks) {
        u32x4 bh[MTH], bl[MTH];
#pragma unroll
        for (int i = 0; i < MTH; ++i) {
          const int mt = min(h * MTH + i, MT - 1);
          bh[i] = *reinterpret_cast<const u32x4*>(Hh + (16 * mt + j) * HS + 32 * ks + 8 * q);
          bl[i] = *reinterpret_cast<const u32x4*>(Hl + (16 * mt + j) * HS + 32 * ks + 8 * q);
        }
#pragma unroll
        for (int i = 0; i < MTH; ++i) acc[i] = mfma_h3(wm[ks][0], wm[ks][1], bh[i], bl[i], acc[i]);
      }
      HOPMI_STAMP(6);
#pragma unroll
      for (int i = 0; i < MTH; ++i) {
        const int mt = h * MTH + i;
        const int row = 16 * mt + j;
        if (mt < MT && row < R) {
          const float4 res = join4h(*reinterpret_cast<const u32x2*>(R1h + row * RS + 16 * w + 4 * q),
                                    *reinterpret_cast<const u32x2*>(R1l + row * RS + 16 * w + 4 * q), RSI[row]);   // gwnet.py:233
          const f32x4 yv = {acc[i][0] * ism4.x + bias4.x + res.x, acc[i][1] * ism4.y + bias4.y + res.y, acc[i][2] * ism4.z + bias4.z + res.z,
                            acc[i][3] * ism4.w + bias4.w + res.w};
          if (y != nullptr) st4(y + (orow0 + row) * C + 16 * w + 4 * q, make_float4(yv[0], yv[1], yv[2], yv[3]));
          st1 += yv;
          st2 += yv * yv;
        }
      }
    }
    if (!MULTI) break;                             // (nothing is loop-carried: registers)
  }

  HOPMI_STAMP(7);
  if (stats_part != nullptr) {
    // sum over the 16 rows j of the DPP row (xor 1, 2, 4, 8), fixed order; one partial per (workgroup, row half)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        st1[r] += __shfl_xor(st1[r], o);
        st2[r] += __shfl_xor(st2[r], o);
      }
    }
    if (j == 0) {
      float* p = stats_part + (size_t)(blockIdx.x * 2 + h) * 2 * C;
      *reinterpret_cast<f32x4*>(p + 16 * w + 4 * q) = st1;
      *reinterpret_cast<f32x4*>(p + C + 16 * w + 4 * q) = st2;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0)                         // arrival counter of wn_bn_finalize_kernel (behind its tail)
      *reinterpret_cast<int*>(stats_part + (size_t)gridDim.x * 2 * 2 * C + (size_t)WN_FIN_G * 2 * C * 2) = 0;
  }
}

// BatchNorm2d training-mode finalisation (gwnet.py:237; torch semantics: biased variance normalises, unbiased variance feeds
// running_var, momentum 0.1) from the per-workgroup partial rows of the layer kernel.  A single workgroup adding 512 rows
// is bound by the memory requests one CU can keep in flight (~20 us measured, more than the layer kernel itself): the rows
// are summed by WN_FIN_G workgroups (fixed order inside each), and the last one to arrive adds the WN_FIN_G sums in index
// order and finalises -- bitwise reproducible, no waiting anywhere.  `tail` (behind the partial rows in ws): WN_FIN_G x 256
// doubles + the arrival counter (zeroed by the layer kernel, left at zero again here).
__global__ __launch_bounds__(256) void wn_bn_finalize_kernel(const float* __restrict__ part, int nblk, double n,
                                                             const float* __restrict__ gamma, const float* __restrict__ beta,
                                                             float* __restrict__ running_mean, float* __restrict__ running_var,
                                                             float momentum, float eps, float* __restrict__ scsh_out,
                                                             float* __restrict__ mean_rstd_out, double* tail) {
  __shared__ double red[2][2 * C];
  __shared__ int last;
  const int col = threadIdx.x & 127, half = threadIdx.x >> 7, g = blockIdx.x;
  int* counter = reinterpret_cast<int*>(tail + (size_t)WN_FIN_G * 2 * C);
  {
    // rows g + WN_FIN_G (2 k + half), k = 0, 1, ...: up to 16 per thread, all loads in flight at once
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int b = g + WN_FIN_G * (2 * u + half);
      v[u] = (b < nblk) ? part[(size_t)b * 2 * C + col] : 0.f;
    }
    double acc = 0.0;
#pragma unroll
    for (int u = 0; u < 16; ++u) acc += (double)v[u];
    for (int b = g + WN_FIN_G * (32 + half); b < nblk; b += 2 * WN_FIN_G) acc += (double)part[(size_t)b * 2 * C + col];   // (grids beyond 256)
    red[half][col] = acc;
  }
  __syncthreads();
  if (threadIdx.x < 2 * C) {
    const double sum = red[0][threadIdx.x] + red[1][threadIdx.x];
    __hip_atomic_store(tail + (size_t)g * 2 * C + threadIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const int seen = __hip_atomic_fetch_add(counter, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    last = seen == WN_FIN_G - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (threadIdx.x < 2 * C) {
    double t = 0.0;
#pragma unroll
    for (int k = 0; k < WN_FIN_G; ++k) t += __hip_atomic_load(tail + (size_t)k * 2 * C + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    red[0][threadIdx.x] = t;
  }
  if (threadIdx.x == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (threadIdx.x < C) {
    const int c = threadIdx.x;
    const double s1 = red[0][c], s2 = red[0][C + c];
    const double mean = s1 / n;
    double var = s2 / n - mean * mean;
    if (var < 0.0) var = 0.0;
    const float rstd = (float)(1.0 / sqrt(var + (double)eps));
    const float sc = gamma[c] * rstd;
    const double unbiased = n > 1.0 ? var * n / (n - 1.0) : var;
    scsh_out[c] = sc;
    scsh_out[C + c] = beta[c] - (float)mean * sc;
    mean_rstd_out[c] = (float)mean;
    mean_rstd_out[C + c] = rstd;
    mean_rstd_out[2 * C + c] = (float)unbiased;
    if (running_mean != nullptr) {
      running_mean[c] = running_update(running_mean[c], (float)mean, momentum);
      running_var[c] = running_update(running_var[c], (float)unbiased, momentum);
    }
  }
}

// the same running-statistics update once more, from the (mean, rstd, unbiased variance) a finalisation left behind
__global__ __launch_bounds__(64) void wn_bn_replay_kernel(const float* __restrict__ stats, float* __restrict__ running_mean,
                                                          float* __restrict__ running_var, float momentum) {
  const int c = threadIdx.x;
  running_mean[c] = running_update(running_mean[c], stats[c], momentum);
  running_var[c] = running_update(running_var[c], stats[2 * C + c], momentum);
}

// forward tiling: one 8-wave workgroup per CU, tiles of up to 80 rows, sized so that the grid covers the launch in one
// round whenever it can (the weight fragments are loaded once per workgroup)
constexpr int WN_GRID_DEFAULT = 256, WN_FWD_MAX_MT = WN_MAX_MT;
static LayerGeom make_fwd_geom(int B, int T_in, int V, int d) {
  return make_layer_geom(B, T_in, V, d, wn_env_int("HOPMI_WN_GRID", WN_GRID_DEFAULT), wn_env_int("HOPMI_WN_MAXMT", WN_FWD_MAX_MT));
}

static int wn_grid(const LayerGeom& L) {
  const int cap = wn_env_int("HOPMI_WN_GRID", WN_GRID_DEFAULT);
  return L.g.ntiles < cap ? L.g.ntiles : cap;
}

static size_t wn_fwd_lds_bytes(const GcnGeom& g) {
  return (size_t)g.rows_lds * (4 * RS + 2 * HS) * sizeof(__bf16) + ((size_t)g.rows_lds * (LDD + 1) + (size_t)g.KP * g.ldA) * sizeof(float);
}

static thread_local hipEvent_t t_ev_start = nullptr, t_ev_stop = nullptr;    // hopmi_time_next_launch

// the pending measurement events of this host thread (null unless hopmi_time_next_launch armed them), handed to ONE launch
hipEvent_t wn_take_timing_events(hipEvent_t* stop) {
  const hipEvent_t e0 = t_ev_start;
  *stop = t_ev_stop;
  t_ev_start = t_ev_stop = nullptr;
  return e0;
}

template <int MT, typename TS>
static int launch_wn_fwd(const TS* xin, const float* scsh, const u32x4* wimg, const float* bf, const float* bg,
                         const float* prep, const float* bm, TS* y, float* fs, TS* utail, int utail_ld, float* part,
                         const LayerGeom& L, int do_gcn, int grid, hipStream_t st) {
  const size_t lds = wn_fwd_lds_bytes(L.g);
  static bool attr_done = false;                         // > 64 KiB of dynamic LDS needs the attribute once per kernel
  if (!attr_done) {
    const void* fns[] = {reinterpret_cast<const void*>(&wn_layer_fwd_kernel<MT, true, true, TS>),
                         reinterpret_cast<const void*>(&wn_layer_fwd_kernel<MT, false, true, TS>),
                         reinterpret_cast<const void*>(&wn_layer_fwd_kernel<MT, true, false, TS>),
                         reinterpret_cast<const void*>(&wn_layer_fwd_kernel<MT, false, false, TS>)};
    for (const void* fn : fns)
      if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) (void)hipGetLastError();
    attr_done = true;
  }
  hipEvent_t e1 = nullptr;
  const hipEvent_t e0 = wn_take_timing_events(&e1);      // null unless a measurement asked for this launch
  const bool multi = L.g.ntiles > grid;
#define HOPMI_WN_LAUNCH(MULTI_, GCN_)                                                                                          \
  hipExtLaunchKernelGGL((wn_layer_fwd_kernel<MT, MULTI_, GCN_, TS>), dim3(grid), dim3(WN_THREADS), lds, st, e0, e1, 0, xin, scsh, wimg, bf, \
                        bg, prep, bm, y, fs, utail, part, L, utail_ld / 4)
  if (do_gcn) { if (multi) HOPMI_WN_LAUNCH(true, true); else HOPMI_WN_LAUNCH(false, true); }
  else { if (multi) HOPMI_WN_LAUNCH(true, false); else HOPMI_WN_LAUNCH(false, false); }
#undef HOPMI_WN_LAUNCH
  return HOPMI_OK;
}

}  // namespace hopmi

using namespace hopmi;

#ifdef HOPMI_STAMPS
extern "C" int hopmi_debug_set_stamps_wn(long long* p) {
  return hipMemcpyToSymbol(HIP_SYMBOL(g_stamps), &p, sizeof(p)) == hipSuccess ? 0 : -1;
}
#endif

extern "C" int hopmi_time_next_launch(void* start_event, void* stop_event) {
  if ((start_event == nullptr) != (stop_event == nullptr)) { set_error("hopmi_time_next_launch: need both events or none"); return HOPMI_EINVAL; }
  t_ev_start = static_cast<hipEvent_t>(start_event);
  t_ev_stop = static_cast<hipEvent_t>(stop_event);
  return HOPMI_OK;
}

// Measurement hook: an empty kernel launched exactly like a WaveNet-layer kernel (same grid / block, the same
// hopmi_time_next_launch start/stop events).  What its events report is the floor of that timing method: on MI355X /
// ROCm 7.2 ~3.9 us for a kernel that does nothing (rocprofv3's kernel trace shows the same 3.6 us average for it).
__global__ void wn_noop_kernel() {}

extern "C" int hopmi_noop_launch(void* stream) {
  const hipEvent_t e0 = t_ev_start, e1 = t_ev_stop;
  t_ev_start = t_ev_stop = nullptr;
  hipExtLaunchKernelGGL(wn_noop_kernel, dim3(WN_GRID_DEFAULT), dim3(WN_THREADS), 0, static_cast<hipStream_t>(stream), e0, e1, 0);
  return check_launch("hopmi_noop_launch");
}

extern "C" size_t hopmi_wn_weight_image_bytes(int n_layers) {
  return (n_layers > 0 && n_layers <= WN_MAX_LAYERS) ? (size_t)n_layers * WIMGH_UNITS * sizeof(u32x4) : 0;
}

extern "C" int hopmi_wn_prepare_weights(const float* const* wf, const float* const* wg, const float* const* Wm, int n_layers,
                                        void* image, void* stream) {
  if (n_layers <= 0 || n_layers > WN_MAX_LAYERS || !wf || !wg || !Wm || !image) {
    set_error("hopmi_wn_prepare_weights: need 1..%d layers and non-null pointer tables / image", WN_MAX_LAYERS);
    return HOPMI_EINVAL;
  }
  WeightPtrs P{};
  for (int l = 0; l < n_layers; ++l) {
    if (!wf[l] || !wg[l] || !Wm[l]) { set_error("hopmi_wn_prepare_weights: null weight pointer for layer %d", l); return HOPMI_EINVAL; }
    P.wf[l] = wf[l]; P.wg[l] = wg[l]; P.wm[l] = Wm[l];
  }
  hipLaunchKernelGGL(wn_prepare_weights_kernel, dim3((WIMG_UNITS / 2 + 255) / 256, n_layers), dim3(256), 0,
                     static_cast<hipStream_t>(stream), P, static_cast<u32x4*>(image));
  return check_launch("hopmi_wn_prepare_weights");
}

extern "C" size_t hopmi_wn_layer_ws_floats(int B, int T_in, int V, int dilation) {
  if (wn_validate(B, T_in, V, dilation)) return 0;
  const LayerGeom L = make_fwd_geom(B, T_in, V, dilation);
  // one (sum, sum of squares) row per (workgroup, row half) + the finalisation's tail (WN_FIN_G x 256 doubles, counter)
  return (size_t)wn_grid(L) * 2 * 2 * C + (size_t)WN_FIN_G * 2 * C * 2 + 4;
}

template <typename TS>
static int wn_layer_fwd_impl(const TS* xin, const float* scsh_in, const void* wimg, const float* bf, const float* bg,
                             const float* prep, const float* bm, TS* y, float* fs, TS* utail, int utail_ld, float* ws, int B, int T_in,
                             int V, int dilation, int do_gcn, void* stream) {
  if (int e = wn_validate(B, T_in, V, dilation)) return e;
  if (!xin || !scsh_in || !wimg || !bf || !bg) { set_error("hopmi_wn_layer_fwd: null pointer argument"); return HOPMI_EINVAL; }
  if (utail != nullptr && (utail_ld < C || (utail_ld & 3))) { set_error("hopmi_wn_layer_fwd: utail_ld=%d must be a multiple of 4 and >= 64", utail_ld); return HOPMI_EINVAL; }
  if (do_gcn && (!prep || !bm)) { set_error("hopmi_wn_layer_fwd: do_gcn needs prep, bm"); return HOPMI_EINVAL; }
  const bool stats = ws != nullptr;
  if (stats && !do_gcn) { set_error("hopmi_wn_layer_fwd: batch statistics (ws) need do_gcn"); return HOPMI_EINVAL; }
  const LayerGeom L = make_fwd_geom(B, T_in, V, dilation);
  if (wn_fwd_lds_bytes(L.g) > 160 * 1024) { set_error("hopmi_wn_layer_fwd: internal: tile needs %zu bytes of LDS", wn_fwd_lds_bytes(L.g)); return HOPMI_EINVAL; }
  const int grid = wn_grid(L);
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* part = stats ? ws : nullptr;
  const u32x4* img = static_cast<const u32x4*>(wimg);
  switch (L.g.mtiles) {
    case 1: launch_wn_fwd<1, TS>(xin, scsh_in, img, bf, bg, prep, bm, y, fs, utail, utail_ld, part, L, do_gcn, grid, st); break;
    case 2: launch_wn_fwd<2, TS>(xin, scsh_in, img, bf, bg, prep, bm, y, fs, utail, utail_ld, part, L, do_gcn, grid, st); break;
    case 3: launch_wn_fwd<3, TS>(xin, scsh_in, img, bf, bg, prep, bm, y, fs, utail, utail_ld, part, L, do_gcn, grid, st); break;
    case 4: launch_wn_fwd<4, TS>(xin, scsh_in, img, bf, bg, prep, bm, y, fs, utail, utail_ld, part, L, do_gcn, grid, st); break;
    case 5: launch_wn_fwd<5, TS>(xin, scsh_in, img, bf, bg, prep, bm, y, fs, utail, utail_ld, part, L, do_gcn, grid, st); break;
    default: set_error("hopmi_wn_layer_fwd: internal: %d m-tiles", L.g.mtiles); return HOPMI_EINVAL;
  }
  return check_launch("hopmi_wn_layer_fwd");
}

extern "C" int hopmi_wn_layer_fwd(const float* xin, const float* scsh_in, const void* wimg, const float* bf, const float* bg,
                                  const float* prep, const float* bm, float* y, float* fs, float* utail,
                                  int utail_ld, float* ws, int B, int T_in, int V, int dilation, int do_gcn, void* stream) {
  return wn_layer_fwd_impl<float>(xin, scsh_in, wimg, bf, bg, prep, bm, y, fs, utail, utail_ld, ws, B, T_in, V, dilation, do_gcn, stream);
}

extern "C" int hopmi_wn_layer_fwd_dt(const void* xin, const float* scsh_in, const void* wimg, const float* bf, const float* bg,
                                     const float* prep, const float* bm, void* y, float* fs, void* utail, int utail_ld, float* ws,
                                     int B, int T_in, int V, int dilation, int do_gcn, int dtype, void* stream) {
  if (dtype == HOPMI_F32)
    return wn_layer_fwd_impl<float>(static_cast<const float*>(xin), scsh_in, wimg, bf, bg, prep, bm, static_cast<float*>(y), fs,
                                    static_cast<float*>(utail), utail_ld, ws, B, T_in, V, dilation, do_gcn, stream);
  if (dtype == HOPMI_BF16)
    return wn_layer_fwd_impl<__bf16>(static_cast<const __bf16*>(xin), scsh_in, wimg, bf, bg, prep, bm, static_cast<__bf16*>(y), fs,
                                     static_cast<__bf16*>(utail), utail_ld, ws, B, T_in, V, dilation, do_gcn, stream);
  set_error("hopmi_wn_layer_fwd_dt: dtype %d (0 = fp32, 1 = bf16)", dtype);
  return HOPMI_EINVAL;
}

extern "C" int hopmi_wn_bn_finalize(const float* ws, const float* gamma, const float* beta, float* running_mean,
                                    float* running_var, float momentum, float eps, float* scsh_out, float* mean_rstd_out,
                                    int B, int T_in, int V, int dilation, void* stream) {
  if (int e = wn_validate(B, T_in, V, dilation)) return e;
  if (!ws || !gamma || !beta || !scsh_out || !mean_rstd_out) { set_error("hopmi_wn_bn_finalize: null pointer argument"); return HOPMI_EINVAL; }
  const LayerGeom L = make_fwd_geom(B, T_in, V, dilation);
  double* tail = reinterpret_cast<double*>(const_cast<float*>(ws) + (size_t)wn_grid(L) * 2 * 2 * C);
  hipLaunchKernelGGL(wn_bn_finalize_kernel, dim3(WN_FIN_G), dim3(256), 0, static_cast<hipStream_t>(stream), ws, 2 * wn_grid(L),
                     (double)L.n_slabs * V, gamma, beta, running_mean, running_var, momentum, eps, scsh_out, mean_rstd_out, tail);
  return check_launch("hopmi_wn_bn_finalize");
}

extern "C" int hopmi_wn_bn_replay(const float* mean_rstd, float* running_mean, float* running_var, float momentum, void* stream) {
  if (!mean_rstd || !running_mean || !running_var) { set_error("hopmi_wn_bn_replay: null pointer argument"); return HOPMI_EINVAL; }
  hipLaunchKernelGGL(wn_bn_replay_kernel, dim3(1), dim3(64), 0, static_cast<hipStream_t>(stream), mean_rstd, running_mean,
                     running_var, momentum);
  return check_launch("hopmi_wn_bn_replay");
}

HOPMI_SPLIT_STATUS_SETTER(wavenet)
