// Linear in 16 bits: y = r + alpha act(x W^T + bias), or r + alpha act(g) u of gated weights (linear.h); x [M, K] as it
// lies, fp32 sums on v_mfma_f32_16x16x32, one rounding.
//
// Weights are kept in the order of the matrix core's fragments, 64 packed rows x 64 k = 8 KB pieces [pieces][K / 64][2][4 j]
// [64 lanes][16 bytes]: lane l of fragment j of half i holds packed row 16 ((l % 16) / 4) + 4 j + l % 4 of the 64, k = 32 i +
// 8 (l / 16) .. + 7, zeros past N and K. Dealt that way four fragments leave a lane 16 consecutive packed rows for one row of
// x: in a gated linear the gates and the up values of 8 outputs.
//
// Up to 16 rows of x the weights' bytes bound it and 8 waves divide K (few); small products run without barriers, both
// operands straight to registers (some); the rest goes through tiles in LDS, of 64 x 128 to 256 x 256 outputs.
#include <type_traits>

#include "linear.h"

namespace esm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

DEV f32x4 mfma_l16(half8 a, half8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
DEV f32x4 mfma_l16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <class V8>
DEV V8 bload8(rsrc_t r, int voff, int soff) {
  return __builtin_bit_cast(V8, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}

// ---- few rows -------------------------------------------------------------------------------------
// A workgroup takes 16 NJ packed weight rows (NJ fragments of a piece) for all, at most 16, rows of x; its 8 waves deal the
// blocks of 128 k among them, the next block's loads in flight, and sum through LDS. Bound by the weights' bytes: one row, 2,560
// -> 10,240 gated, 52 MB in 11.3 us from HBM, 4.65 TB/s (a large copy runs 5.1), 10.1 where part of them lies in the cache behind L2.
constexpr int kL16Waves = 8;
template <class V8, int NJ>
__global__ __launch_bounds__(64 * kL16Waves) void linear16_few_kernel(L16Args p) {
  constexpr int kPad = 16 * NJ + 4, kSteps = 4;  // (16 rows of sums cover the LDS banks); steps of 32 k in a block
  __shared__ __align__(16) float red[kL16Waves][16][kPad];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Kb = (p.K + 63) / 64, blocks = (Kb + 1) / 2;
  const int ng = blockIdx.x / (4 / NJ), j0 = blockIdx.x % (4 / NJ) * NJ;
  const int m = lane & 15;
  const rsrc_t rw = make_rsrc((const char*)p.w + (size_t)ng * Kb * 8192);
  const rsrc_t rx = make_rsrc_n(p.x, (uint32_t)(2 * ((p.M - 1) * p.x_st + p.K)));
  const uint32_t xo = m < p.M ? (uint32_t)(2 * (m * p.x_st + 8 * (lane >> 4))) : kOOB;
  struct Block {
    V8 w[kSteps][NJ], x[kSteps];
  };
  const auto load = [&](Block& b, int kb) {
    kb = min(kb, blocks - 1);  // (past the last: that one again, not used)
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      // (an odd count of 64s ends inside the block: zeros behind it, by the offset that the range is checked against)
      const int wo = 2 * kb + i / 2 < Kb ? 16 * lane : (int)kOOB;
#pragma unroll
      for (int j = 0; j < NJ; j++) b.w[i][j] = bload8<V8>(rw, wo, kb * 16384 + 4096 * i + 1024 * (j0 + j));
      const int k = 128 * kb + 32 * i;
      b.x[i] = bload8<V8>(rx, (int)(k + 8 * (lane >> 4) < p.K ? xo + 2u * (uint32_t)k : kOOB), 0);
    }
  };
  f32x4 acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const auto take = [&](const Block& b) {
#pragma unroll
    for (int i = 0; i < kSteps; i++)
#pragma unroll
      for (int j = 0; j < NJ; j++) acc[j] = mfma_l16(b.w[i][j], b.x[i], acc[j]);
  };
  Block b0, b1;
  if (wave < blocks) load(b0, wave);
  for (int kb = wave; kb < blocks; kb += 2 * kL16Waves) {
    load(b1, kb + kL16Waves);
    __builtin_amdgcn_sched_barrier(0);
    take(b0);
    __builtin_amdgcn_sched_barrier(0);
    if (kb + kL16Waves >= blocks) break;
    load(b0, kb + 2 * kL16Waves);
    __builtin_amdgcn_sched_barrier(0);
    take(b1);
    __builtin_amdgcn_sched_barrier(0);
  }
  // lane's sums: row m, packed rows 16 (lane / 16) + 4 (j0 + j) + e -> column 4 NJ (lane / 16) + 4 j + e
#pragma unroll
  for (int j = 0; j < NJ; j++) *reinterpret_cast<f32x4*>(&red[wave][m][4 * NJ * (lane >> 4) + 4 * j]) = acc[j];
  __syncthreads();
  end_few<V8, NJ, kL16Waves, kPad>(p.end, &red[0][0][0], p.M, ng, j0, threadIdx.x, 64 * kL16Waves);
}

// ---- some rows --------------------------------------------------------------------------------------
// A workgroup takes 16 MB rows of x by a piece of 64 packed weight rows; its 8 waves deal the blocks of 64 k among them, the
// next block's fragments in flight, and sum through LDS. Bound by the latency of a wave's few blocks and the sum: 64 rows,
// 5,120 -> 2,560 13.6 us, of which the 26 MB of weights need 5; 24 rows, 2,560 -> 7,680 9.8.
constexpr int kL16Pad = 68;
template <class V8, int MB>
__global__ __launch_bounds__(64 * kL16Waves) void linear16_some_kernel(L16Args p) {
  __shared__ __align__(16) float red[kL16Waves][16 * MB * kL16Pad];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Kb = (p.K + 63) / 64;
  // row tiles run fastest: those that share weights are on one XCD at one time
  const int t = xcd_remap(blockIdx.x, gridDim.x), ng = t / p.mtiles, row0 = (t - ng * p.mtiles) * 16 * MB;
  const rsrc_t rw = make_rsrc((const char*)p.w + (size_t)ng * Kb * 8192);
  const rsrc_t rx = make_rsrc((const uint16_t*)p.x + row0 * p.x_st);
  uint32_t xo[MB];
#pragma unroll
  for (int b = 0; b < MB; b++) {
    const int r = min(16 * b + (lane & 15), p.M - 1 - row0);  // (rows past the last: that one again, not stored)
    xo[b] = (uint32_t)(2 * (r * p.x_st + 8 * (lane >> 4)));
  }
  struct Block {
    V8 w[2][4], x[2][MB];
  };
  const auto load = [&](Block& k, int kb) {
    kb = min(kb, Kb - 1);
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
      for (int j = 0; j < 4; j++) k.w[i][j] = bload8<V8>(rw, 16 * lane, kb * 8192 + 4096 * i + 1024 * j);
      const bool in = 64 * kb + 32 * i + 8 * (lane >> 4) < p.K;
#pragma unroll
      for (int b = 0; b < MB; b++) k.x[i][b] = bload8<V8>(rx, (int)(in ? xo[b] : kOOB), 2 * (64 * kb + 32 * i));
    }
  };
  f32x4 acc[MB][4];
#pragma unroll
  for (int b = 0; b < MB; b++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const auto take = [&](const Block& k) {
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int b = 0; b < MB; b++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[b][j] = mfma_l16(k.w[i][j], k.x[i][b], acc[b][j]);
  };
  Block k0, k1;
  if (wave < Kb) load(k0, wave);
  for (int kb = wave; kb < Kb; kb += 2 * kL16Waves) {
    // (the compiler would sink the next block's loads behind this block's products, and each wave wait for its own)
    load(k1, kb + kL16Waves);
    __builtin_amdgcn_sched_barrier(0);
    take(k0);
    __builtin_amdgcn_sched_barrier(0);
    if (kb + kL16Waves >= Kb) break;
    load(k0, kb + 2 * kL16Waves);
    __builtin_amdgcn_sched_barrier(0);
    take(k1);
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int b = 0; b < MB; b++)
#pragma unroll
    for (int j = 0; j < 4; j++)
      *reinterpret_cast<f32x4*>(&red[wave][(16 * b + (lane & 15)) * kL16Pad + 16 * (lane >> 4) + 4 * j]) = acc[b][j];
  __syncthreads();
  end_lds<V8, kL16Pad>(p.end, red[0], kL16Waves, 16 * MB * kL16Pad, 16 * MB, row0, p.M, ng, threadIdx.x, 64 * kL16Waves);
}

// ---- tiles of up to 192 rows ----------------------------------------------------------------------
// Workgroup tile of 16 MB WM rows of x by WN pieces of weights, WM x WN waves of 16 MB x 64 each. A step is 64 k: both
// operands come by direct loads into a ring of S slots, S - 1 steps ahead. Rows of x land 128 bytes a row, 16-byte chunk c of row
// r at c ^ (r % 8), so that a load takes whole lines of memory and a fragment's rows lie in different banks. Bound by what fills
// LDS and by tiles too few for the CUs: 238 rows, 5,120 -> 2,560 in 64 x 256, K in six, 18.1 us and 4.8 for its splits' sum (a library's
// product 21.6), 1,000 rows, 2,560 -> 2,560 in 64 x 256 24.2 (23.7).
template <class V8, int MB, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN) void linear16_tiles_kernel(L16Args p) {
  constexpr int NW = WM * WN, kX = 2048 * MB * WM, kW = 8192 * WN, kSlot = kX + kW;  // bytes a slot
  constexpr int kLoadsX = kX / 1024 / NW, kLoadsW = kW / 1024 / NW, kLoads = kLoadsX + kLoadsW;
  static_assert(kLoadsX * NW * 1024 == kX && kLoadsW * NW * 1024 == kW, "whole loads per wave");
  static_assert((S - 2) * kLoads < 64, "loads in flight the counter can tell");
  __shared__ __align__(1024) char lds[S * kSlot];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN, Kb = (p.K + 63) / 64;
  // workgroups in groups of 8 row tiles, so that those running together share both operands' pieces in L2
  int t = xcd_remap(blockIdx.x, gridDim.x);
  const int tiles = p.mtiles * p.ntiles, split = t / tiles;
  t -= split * tiles;
  const int group = t / (8 * p.ntiles), in = t - group * 8 * p.ntiles, gm = min(8, p.mtiles - 8 * group);
  const int mt = 8 * group + in % gm, nt = in / gm;
  const int kb0 = Kb * split / p.splits, kb1 = Kb * (split + 1) / p.splits;
  const int m0 = mt * 16 * MB * WM, ng0 = nt * WN, row0 = m0 + 16 * MB * wm;
  const dma_src_t rx = dma_src((const uint16_t*)p.x + m0 * p.x_st, kBufRange);
  const dma_src_t rw = dma_src((const char*)p.w + (size_t)ng0 * Kb * 8192, kBufRange);
  const uint32_t base = lds_address(lds);
  // where this lane reads x from: row lane / 8 of a load's 8, the chunk that lands at place lane % 8 of it
  const int chunk = (lane & 7) ^ (lane >> 3);
  uint32_t xo[kLoadsX];
#pragma unroll
  for (int i = 0; i < kLoadsX; i++) {
    const int r = min(8 * (wave * kLoadsX + i) + (lane >> 3), p.M - 1 - m0);  // (rows past the last: that one again)
    xo[i] = (uint32_t)(2 * (r * p.x_st + 8 * chunk));
  }
  const auto load = [&](int kb, int slot, int i) {
    const uint32_t at = base + slot * kSlot;
    if (i < kLoadsX) {
      const int u = wave * kLoadsX + i;
      dma16(rx, at + 1024 * u, 64 * kb + 8 * chunk < p.K ? xo[i < kLoadsX ? i : 0] : kOOB, 128u * (uint32_t)kb);
    } else {
      const int u = wave * kLoadsW + i - kLoadsX, r = min(u >> 3, p.pieces - 1 - ng0);
      dma16(rw, at + kX + 1024 * u, 16 * lane, (uint32_t)(r * Kb + kb) * 8192u + 1024u * (u & 7));
    }
  };
  f32x4 acc[MB][4];
#pragma unroll
  for (int i = 0; i < MB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int n = kb1 - kb0;
#pragma unroll
  for (int i = 0; i < S - 1; i++)
#pragma unroll
    for (int u = 0; u < kLoads; u++) load(min(kb0 + i, kb1 - 1), i, u);  // (past the last block: loaded again, not used)
  // this lane's chunk of a row in LDS, of either half of the 64 k
  const int sw0 = 16 * ((lane >> 4) ^ (lane & 7)), sw1 = 16 * ((4 + (lane >> 4)) ^ (lane & 7));
  for (int i = 0, slot = 0; i < n; i++, slot = slot + 1 == S ? 0 : slot + 1) {
    constexpr int kLeft = (S - 2) * kLoads;
    __builtin_amdgcn_s_waitcnt(0x0F70 | (kLeft & 15) | ((kLeft >> 4) << 14));  // vmcnt(kLeft): this block's loads are in
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
    const int kn = min(kb0 + i + S - 1, kb1 - 1), next = slot == 0 ? S - 1 : slot - 1;
    const char* xs = lds + slot * kSlot + 2048 * MB * wm + 128 * (lane & 15);
    const char* ws = lds + slot * kSlot + kX + 8192 * wn + 16 * lane;
    // Loads of a later block are spread over the step; the next 16 rows' fragment is read before the matrix
    // instructions of these, the second half's weights during the first's.
    constexpr int kSpread = (kLoads + 2 * MB - 1) / (2 * MB);
    const auto xf = [&](int u) {  // rows 16 (u % MB) .., half u / MB
      return *reinterpret_cast<const V8*>(xs + 2048 * (u % MB) + (u < MB ? sw0 : sw1));
    };
    V8 w[4], wn2[4], x = xf(0), xn;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = *reinterpret_cast<const V8*>(ws + 1024 * j);
#pragma unroll
    for (int u = 0; u < 2 * MB; u++) {
      if (u + 1 < 2 * MB) xn = xf(u + 1);
      if (u >= MB - 2 && u < MB) {  // (MB >= 2)
        const int j = 2 * (u - (MB - 2));
        wn2[j] = *reinterpret_cast<const V8*>(ws + 4096 + 1024 * j);
        wn2[j + 1] = *reinterpret_cast<const V8*>(ws + 4096 + 1024 * (j + 1));
      }
#pragma unroll
      for (int l = kSpread * u; l < kSpread * (u + 1); l++)
        if (l < kLoads) load(kn, next, l);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; j++) acc[u % MB][j] = mfma_l16(w[j], x, acc[u % MB][j]);
      __builtin_amdgcn_sched_barrier(0);
      x = xn;
      if (u == MB - 1)
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = wn2[j];
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this slot's reads are back before the next barrier frees it
    __asm__ volatile("" ::: "memory");
  }
  wait_vm(0);  // no load of this workgroup outlives it, or lands on what end_tile keeps in LDS
  __syncthreads();
  const int ng = ng0 + wn;
  if (ng >= p.pieces) return;
  if (p.part) {
#pragma unroll
    for (int b = 0; b < MB; b++) {
      const int m = row0 + 16 * b + (lane & 15);
      if (m < p.M) part16(p.part, (long long)split * p.M + m, p.pieces, ng, lane >> 4, acc[b]);
    }
  } else {
    end_tile<V8>(p.end, p.M, row0, ng, lane, acc, lds + 8192 * wave);
  }
}

// ---- tiles of 256 x 256 ---------------------------------------------------------------------------
// The same in steps of 32 k, of which LDS holds four where it holds two of 64. Rows of x land 64 bytes a row, 16-byte chunk c of
// row r at c ^ (-(r / 4) % 4), so that the 16 lanes that LDS serves at a time, rows of two chunks, cover the banks (with c ^ (r /
// 4 % 4) two of them met, a fifth of the cycles, which the clock made up for: the time was the same). A step's first fragments
// are read at the end of the step before it, behind the products, as the barrier between them stands for the slot after the next:
// with the slot itself the waves would leave each barrier only to wait for LDS. Bound by the matrix cores' power, 69% busy below
// 1.6 GHz: 8,192 x 8,192 x 8,192 in 800 to 890 us by the box, up to 1.37 PFLOP/s (a library's product 785 on the fastest); 3,481 x
// 2,560 x 7,680 128 to 135 us (121).
template <class V8, int MB, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN) void linear16_large_kernel(L16Args p) {
  constexpr int NW = WM * WN, kX = 1024 * MB * WM, kW = 4096 * WN, kSlot = kX + kW;  // bytes a slot
  constexpr int kLoadsX = kX / 1024 / NW, kLoadsW = kW / 1024 / NW, kLoads = kLoadsX + kLoadsW;
  constexpr int R = MB % 4 == 0 ? 4 : MB % 3 == 0 ? 3 : 2;  // fragments of x in registers, R - 1 of them ahead
  static_assert(kLoadsX * NW * 1024 == kX && kLoadsW * NW * 1024 == kW, "whole loads per wave");
  static_assert(S >= 4 && (S - 2) * kLoads < 64, "a slot behind the next; loads in flight the counter can tell");
  static_assert(S * kSlot >= 8192 * NW, "end_tile's part of LDS");
  __shared__ __align__(1024) char lds[S * kSlot];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN, Ks = 2 * ((p.K + 63) / 64);  // (weights are whole 64s, zeros past K)
  int t = xcd_remap(blockIdx.x, gridDim.x);
  const int tiles = p.mtiles * p.ntiles, split = t / tiles;
  t -= split * tiles;
  const int group = t / (8 * p.ntiles), in = t - group * 8 * p.ntiles, gm = min(8, p.mtiles - 8 * group);
  const int mt = 8 * group + in % gm, nt = in / gm;
  const int k0 = Ks * split / p.splits, k1 = Ks * (split + 1) / p.splits;
  const int m0 = mt * 16 * MB * WM, ng0 = nt * WN, row0 = m0 + 16 * MB * wm;
  const dma_src_t rx = dma_src((const uint16_t*)p.x + m0 * p.x_st, kBufRange);
  const dma_src_t rw = dma_src((const char*)p.w + (size_t)ng0 * Ks * 4096, kBufRange);
  const uint32_t base = lds_address(lds);
  // where this lane reads x from: row lane / 4 of a load's 16, the chunk that lands at place lane % 4 of it
  const int chunk = (lane & 3) ^ (-(lane >> 4) & 3);
  uint32_t xo[kLoadsX];
#pragma unroll
  for (int i = 0; i < kLoadsX; i++) {
    const int r = min(16 * (wave * kLoadsX + i) + (lane >> 2), p.M - 1 - m0);  // (rows past the last: that one again)
    xo[i] = (uint32_t)(2 * (r * p.x_st + 8 * chunk));
  }
  const auto load = [&](int k, int slot, int i) {
    const uint32_t at = base + slot * kSlot;
    if (i < kLoadsX) {
      dma16(rx, at + 1024 * (wave * kLoadsX + i), 32 * k + 8 * chunk < p.K ? xo[i < kLoadsX ? i : 0] : kOOB, 64u * (uint32_t)k);
    } else {
      const int u = wave * kLoadsW + i - kLoadsX, r = min(u >> 2, p.pieces - 1 - ng0);
      dma16(rw, at + kX + 1024 * u, 16 * lane, (uint32_t)(r * Ks + k) * 4096u + 1024u * (u & 3));
    }
  };
  f32x4 acc[MB][4];
#pragma unroll
  for (int i = 0; i < MB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int n = k1 - k0;
#pragma unroll
  for (int i = 0; i < S - 1; i++)
#pragma unroll
    for (int u = 0; u < kLoads; u++) load(min(k0 + i, k1 - 1), i, u);  // (past the last step: loaded again, not used)
  const int mine = kX + 4096 * wn + 16 * lane, rows = 1024 * MB * wm + 64 * (lane & 15) + 16 * ((lane >> 4) ^ (-(lane >> 2) & 3));
  const auto weight = [&](int slot, int j) { return *reinterpret_cast<const V8*>(lds + slot * kSlot + mine + 1024 * j); };
  const auto row = [&](int slot, int b) { return *reinterpret_cast<const V8*>(lds + slot * kSlot + rows + 1024 * b); };
  V8 wa[4], wb[4], x[R];
  constexpr int kLeft = (S - 3) * kLoads;
  const auto settle = [&]() {  // the loads of all slots but the last S - 3 asked for are in, every wave's
    __builtin_amdgcn_s_waitcnt(0x0F70 | (kLeft & 15) | ((kLeft >> 4) << 14));
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
  };
  // One step from slot: its weights are in w, the first R - 1 fragments of x in x; the next step's go to nw and x.
  const auto step = [&](int i, int slot, V8 (&w)[4], V8 (&nw)[4]) {
    settle();
    const int kn = min(k0 + i + S - 1, k1 - 1), last = slot == 0 ? S - 1 : slot - 1, next = slot + 1 == S ? 0 : slot + 1;
    constexpr int kSpread = (kLoads + MB - 1) / MB;
#pragma unroll
    for (int b = 0; b < MB; b++) {
#pragma unroll
      for (int j = 0; j < 4; j++) acc[b][j] = mfma_l16(w[j], x[b % R], acc[b][j]);
      __builtin_amdgcn_sched_barrier(0);
      const int f = b + R - 1;  // the fragment to read now
      x[f % R] = f < MB ? row(slot, f) : row(next, f - MB);
      if (MB >= 4 ? b >= MB - 4 : true) {
        constexpr int kPer = MB >= 4 ? 1 : 4 / MB;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
          const int jj = (MB >= 4 ? b - (MB - 4) : b * kPer) + j;
          nw[jj] = weight(next, jj);
        }
      }
#pragma unroll
      for (int l = kSpread * b; l < kSpread * (b + 1); l++)
        if (l < kLoads) load(kn, last, l);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // before the first step: slot 0 is in
  __builtin_amdgcn_s_waitcnt(0x0F70 | (((S - 2) * kLoads) & 15) | ((((S - 2) * kLoads) >> 4) << 14));
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __asm__ volatile("" ::: "memory");
#pragma unroll
  for (int j = 0; j < 4; j++) wa[j] = weight(0, j);
#pragma unroll
  for (int b = 0; b < R - 1; b++) x[b] = row(0, b);
  int slot = 0;
  const auto after = [&]() { slot = slot + 1 == S ? 0 : slot + 1; };
  int i = 0;
  for (; i + 1 < n; i += 2) {  // (the weights' registers change places)
    step(i, slot, wa, wb);
    after();
    step(i + 1, slot, wb, wa);
    after();
  }
  if (i < n) step(i, slot, wa, wb);
  wait_vm(0);  // no load of this workgroup outlives it, or lands on what end_tile keeps in LDS
  __syncthreads();
  const int ng = ng0 + wn;
  if (ng >= p.pieces) return;
  if (p.part) {
#pragma unroll
    for (int b = 0; b < MB; b++) {
      const int m = row0 + 16 * b + (lane & 15);
      if (m < p.M) part16(p.part, (long long)split * p.M + m, p.pieces, ng, lane >> 4, acc[b]);
    }
  } else {
    end_tile<V8>(p.end, p.M, row0, ng, lane, acc, lds + 8192 * wave);
  }
}

// ---- weights ------------------------------------------------------------------------------------
// [N, K] into the fragment order, a thread 16 bytes; gated: fragments 0 and 2 of a piece from the first half of the rows, 1
// and 3 from the second.
__global__ __launch_bounds__(256) void linear16_pack_kernel(const uint16_t* __restrict__ w, uint16_t* __restrict__ out, int N, int K,
                                                            int pieces, int gated) {
  const int Kb = (K + 63) / 64, F = N / 2;
  const size_t total = (size_t)pieces * Kb * 512;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const int u = (int)(i % 512), l = u & 63, j = (u >> 6) & 3, half = u >> 8;
    const size_t piece = i / 512;
    const int kb = (int)(piece % Kb), ng = (int)(piece / Kb), k = 64 * kb + 32 * half + 8 * (l >> 4);
    const int g = (l & 15) >> 2, e = l & 3;
    const int o = gated ? 32 * ng + 8 * g + 4 * (j >> 1) + e : 64 * ng + 16 * g + 4 * j + e;
    const bool ok = k < K && o < (gated ? F : N);
    u32x4 v = {0, 0, 0, 0};
    if (ok) v = *reinterpret_cast<const u32x4*>(w + (size_t)(gated && (j & 1) ? F + o : o) * K + k);
    *reinterpret_cast<u32x4*>(out + 8 * i) = v;
  }
}

template <class V8, int MB, int WM, int WN, int S>
static hipError_t launch_tiles16(L16Args a, hipStream_t s) {
  a.mtiles = (a.M + 16 * MB * WM - 1) / (16 * MB * WM);
  a.ntiles = (a.pieces + WN - 1) / WN;
  const dim3 grid((unsigned)((size_t)a.mtiles * a.ntiles * a.splits)), block(64 * WM * WN);
  if constexpr (MB == 8) {
    ESM_LAUNCH((linear16_large_kernel<V8, MB, WM, WN, S>), grid, block, 0, s, a);
  } else {
    ESM_LAUNCH((linear16_tiles_kernel<V8, MB, WM, WN, S>), grid, block, 0, s, a);
  }
  return hipGetLastError();
}

template <class V8, int MB>
static hipError_t launch_some16(L16Args a, hipStream_t s) {
  a.mtiles = (a.M + 16 * MB - 1) / (16 * MB);
  ESM_LAUNCH((linear16_some_kernel<V8, MB>), dim3((unsigned)((size_t)a.mtiles * a.pieces)), dim3(64 * kL16Waves), 0, s, a);
  return hipGetLastError();
}

// The tiles: rows, pieces of 64 packed weight rows, workgroups on a CU; us per workgroup and per 64 k of it.
static const struct L16Tile { int rows, pieces, per_cu; double start, step; } kL16Tile[] = {
    {64, 2, 2, 2.5, 0.41}, {64, 4, 1, 2.5, 0.58}, {128, 2, 1, 2.5, 0.60}, {128, 4, 1, 3.5, 0.76}, {192, 4, 1, 4.0, 1.15}, {256, 4, 1, 4.5, 1.47}};

L16Size linear16_size(int tile) { return L16Size{kL16Tile[tile].rows, 64 * kL16Tile[tile].pieces}; }

template <class V8>
static hipError_t launch_linear16_t(const L16Args& a, int form, int mb, hipStream_t s) {
  if (form == kL16Few) {
    const dim3 grid(a.pieces * (4 / mb)), block(64 * kL16Waves);
    switch (mb) {
      case 4: ESM_LAUNCH((linear16_few_kernel<V8, 4>), grid, block, 0, s, a); break;
      case 2: ESM_LAUNCH((linear16_few_kernel<V8, 2>), grid, block, 0, s, a); break;
      default: ESM_LAUNCH((linear16_few_kernel<V8, 1>), grid, block, 0, s, a); break;
    }
    return hipGetLastError();
  }
  if (form == kL16Some) return mb == 1 ? launch_some16<V8, 1>(a, s) : launch_some16<V8, 3>(a, s);
  hipError_t e;
  switch (mb) {  // (kL16Tile's order)
    case 0: e = launch_tiles16<V8, 2, 2, 2, 3>(a, s); break;
    case 1: e = launch_tiles16<V8, 2, 2, 4, 4>(a, s); break;
    case 2: e = launch_tiles16<V8, 4, 2, 2, 5>(a, s); break;
    case 3: e = launch_tiles16<V8, 4, 2, 4, 3>(a, s); break;
    case 4: e = launch_tiles16<V8, 6, 2, 4, 2>(a, s); break;
    default: e = launch_tiles16<V8, 8, 2, 4, 4>(a, s); break;
  }
  if (e != hipSuccess || !a.part) return e;
  return launch_linear_join<V8>(a.part, a.end, a.M, a.pieces, a.splits, s);
}

hipError_t launch_linear16(const L16Args& a, bool bf16, const L16Plan& plan, hipStream_t s) {
  return bf16 ? launch_linear16_t<bf16x8>(a, plan.form, plan.mb, s) : launch_linear16_t<half8>(a, plan.form, plan.mb, s);
}

// Which form: the lowest of estimated times, from measurements of the kernels alone (us; rows, K -> N):
//   some, 16 rows a workgroup  24, 2560 -> 7680 9.8; 64, 5120 -> 2560 13.6     48 rows  238, 2560 -> 2560 14.2; 238, 5120 -> 2560 23.7
//   64 x 128   238, 2560 -> 7680 19.3; 300 30.2; 512, 5120 -> 2560 in three splits 22.8 and 4.6 for the join
//   64 x 256   1000, 2560 -> 2560 24.7; 512, 2560 -> 7680 32.6       128 x 128  512, 2560 -> 7680 29.0; 700, 4096 -> 4096 37.4
//   128 x 256  2000, 5120 -> 2560 60.3; 1000, 10240 -> 2560 in three splits 56.1 and 6.9
//   192 x 256  3481, 2560 -> 2560 48.7; 1500, 2560 -> 7680 62.2      256 x 256  3481, 2560 -> 7680 129; 8192, 8192 -> 8192 794
L16Plan linear16_plan(int M, int K, int N, bool gated, int cus) {
  const long long pieces = linear_pieces(N, gated);
  // Few rows: the most weight rows a workgroup (16, 32, 64) that still give more than half the CUs one (one row, 2560 -> 2560 4.1 /
  // 4.6 / 6.4, 16 rows, 2560 -> 10240 15.8 / 15.5 / 12.7, 4096 -> 4096 9.2 / 11.0 / 14.8).
  L16Plan p{kL16Few, 4, 1};
  const int least = gated ? 2 : 1;  // (a gate and its up value in one workgroup)
  while (p.mb > least && 16LL * pieces * (4 / p.mb) < 9LL * cus) p.mb /= 2;
  if (M <= 16) return p;
  const int Kb = (K + 63) / 64;
  double best = 1e30;
  for (int mb : {1, 3}) {
    if ((M + 16LL * mb - 1) / (16 * mb) * pieces > cus) continue;  // (a second round takes as long as the first)
    const double c = 2.6 + (Kb + 7) / 8 * (0.5 + 0.6 * mb);
    if (c < best) best = c, p = L16Plan{kL16Some, mb, 1};
  }
  for (int i = 0; i < (int)(sizeof kL16Tile / sizeof kL16Tile[0]); i++) {
    const L16Tile& t = kL16Tile[i];
    for (int sp = 1; sp <= kL16MaxSplits && (sp == 1 || 4 * sp <= Kb); sp++) {
      const long long wgs = (M + t.rows - 1) / t.rows * ((pieces + t.pieces - 1) / t.pieces) * sp, each = (long long)cus * t.per_cu;
      if (sp > 1 && wgs > each) break;  // splits only fill one round
      // two on a CU take 1.6 times as long as one
      const double rounds = wgs <= cus ? 1 : (double)((wgs + each - 1) / each) * (t.per_cu == 2 ? 1.6 : 1);
      double c = rounds * (t.start + t.step * ((Kb + sp - 1) / sp));
      if (sp > 1) c += 3.5 + 1.5e-6 * sp * M * 64.0 * pieces;  // writing and summing the partials
      if (c < best) best = c, p = L16Plan{kL16Tiles, i, sp};
    }
  }
  return p;
}

hipError_t launch_linear16_pack(const void* w, void* out, int N, int K, bool gated, hipStream_t s) {
  const int pieces = linear_pieces(N, gated);
  const size_t blocks = ((size_t)pieces * ((K + 63) / 64) * 512 + 255) / 256;
  ESM_LAUNCH(linear16_pack_kernel, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, (const uint16_t*)w, (uint16_t*)out,
             N, K, pieces, (int)gated);
  return hipGetLastError();
}

}  // namespace esm
