// Linear with weights in e4m3 (one fp32 scale per 128 x 128 block) on the fp8 matrix cores:
//   r = 448 / max(amax, 2^-96), xq = e4m3(x r), sx = max(amax, 2^-96) / 448   per row of x and 128 columns
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in b} xq[m, k] wq[n, k]
// The inner sums run in v_mfma_f32_16x16x128_f8f6f4, whose depth is one scale block: each result is taken with
// its two scales into an fp32 accumulator. Rounded are x (to e4m3, the operator's definition), y, and what the
// matrix core cuts: it aligns 8 consecutive products to the largest's exponent and drops what lies 13 binary places
// below (measured; v_mfma_f32_16x16x32_fp8_fp8 does the same at a third of the rate, 1.39 against 4.46 PFLOP/s), about
// 2^-12 of y, below half a step of fp16; from there on sums are fp32.
//
// Both operands are kept in the order of the matrix core's fragments, so every load is 1 KB of consecutive bytes
// and LDS reads have no bank conflicts:
//   codes: 64 weight rows x 128 k = 8 KB pieces [N / 64][K / 128][4 j][2][64 lanes][16 bytes]; lane l of fragment j
//     holds weight row 16 ((l % 16) / 4) + 4 j + l % 4 of the 64, k = 32 (l / 16) + 16 half .. + 15. With the rows
//     dealt that way the four fragments leave a lane 16 consecutive outputs of one row of x.
//   x: 16 rows x 128 k = 2 KB pieces [M / 16][K / 128][2][64 lanes][16 bytes], the same k order.
// Up to 16 rows of x one launch does it all (f8_few_kernel: bound by the codes' bytes); beyond, x goes through
// f8_quantize_kernel, then f8_some_kernel (some hundred rows: no barriers, operands straight to registers) or
// f8_gemm_kernel (tiles through LDS by loads that write it directly).
// The same kernels take x already in e4m3 (add_norm's rows; CODED), and end as linear.h has it, with a bias, an activation or
// gate and a residual (END): y = r + alpha act(z + bias).
#include <type_traits>

#include "linear.h"

namespace esm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// e4m3 x e4m3 -> fp32, 16 x 16 x 128 (a: 16 weight rows, b: 16 rows of x; 32 bytes a lane each). Result: column
// (row of x) lane % 16, rows 4 (lane / 16) + register.
DEV f32x4 mfma_f8(i32x8 a, i32x8 b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// Largest magnitude of 8 values as their 16-bit pattern without the sign: NaN above infinity above the rest.
DEV uint32_t top_bits(u16x8 v) {
  u16x8 a = v & (uint16_t)0x7fff;
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) m = max(m, (uint32_t)a[e]);
  return m;
}
template <class V8>
DEV float bits_value(uint32_t b) {
  V8 v{};
  u16x8 u = __builtin_bit_cast(u16x8, v);
  u[0] = (uint16_t)b;
  return (float)__builtin_bit_cast(V8, u)[0];
}
// 8 values times r as 8 codes (round to nearest even; r keeps them within 448).
template <class V8>
DEV void f8_codes(V8 v, float r, int& lo, int& hi) {
  lo = __builtin_amdgcn_cvt_pk_fp8_f32((float)v[0] * r, (float)v[1] * r, 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32((float)v[2] * r, (float)v[3] * r, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32((float)v[4] * r, (float)v[5] * r, 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32((float)v[6] * r, (float)v[7] * r, hi, true);
}

// ---- x to e4m3 --------------------------------------------------------------------------------
// A thread takes 16 values of a row; the 8 threads of a row's block share its maximum. Bound by bytes, small ones by a
// launch and one latency: 8192 x 8192 47 us, 4.4 TB/s; 3481 x 2560 6.9, 238 x 5120 2.0 to 3.5 (with four blocks a
// thread 8.1 and 2.7 to 4.3).
template <class V8>
__global__ __launch_bounds__(256) void f8_quantize_kernel(const uint16_t* __restrict__ x, long long st, uint8_t* __restrict__ xq,
                                                          float* __restrict__ sx, int M, int K, int Mp) {
  const int Kb = (K + 127) / 128, t = threadIdx.x;
  const int c = t & 7, m = 32 * blockIdx.x + (t >> 3), kb = blockIdx.y, k = 128 * kb + 16 * c;
  if (m >= Mp) return;
  u16x8 a = {}, b = {};
  if (m < M && k < K) {
    const u16x8* src = reinterpret_cast<const u16x8*>(x + m * st + k);
    a = src[0];
    b = src[1];
  }
  uint32_t top = max(top_bits(a), top_bits(b));
  const auto other = [&](auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, decltype(ctrl)::value, 0xf, 0xf, false);
  };
  top = max(top, other(std::integral_constant<int, 0xB1>{}));   // quad_perm(1, 0, 3, 2)
  top = max(top, other(std::integral_constant<int, 0x4E>{}));   // quad_perm(2, 3, 0, 1)
  top = max(top, other(std::integral_constant<int, 0x141>{}));  // row_half_mirror
  float r, s;
  f8_scale(bits_value<V8>(top), r, s);
  int q[4];
  f8_codes(__builtin_bit_cast(V8, a), r, q[0], q[1]);
  f8_codes(__builtin_bit_cast(V8, b), r, q[2], q[3]);
  uint8_t* dst = xq + ((size_t)(m >> 4) * Kb + kb) * 2048 + (c & 1) * 1024 + (16 * (c >> 1) + (m & 15)) * 16;
  *reinterpret_cast<i32x4*>(dst) = i32x4{q[0], q[1], q[2], q[3]};
  if (c == 0) sx[(size_t)kb * Mp + m] = s;
}

// Fragment at soff + 16 lane of a buffer whose every read is in range.
DEV i32x4 bload_i4(rsrc_t r, int voff, int soff) {
  return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 0));
}
DEV i32x8 bload_frag(rsrc_t r, int voff, int soff) {
  const i32x4 lo = bload_i4(r, voff, soff), hi = bload_i4(r, voff, soff + 1024);
  return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// The weight scales of a piece: of its even and its odd fragments (gated: the gates' and the up values').
struct PieceScales {
  const float *even, *odd;
};
DEV PieceScales piece_scales(const F8Args& p, int ng, int Kb) {
  if (!p.end.gated) return PieceScales{p.sw + (size_t)(ng >> 1) * Kb, p.sw + (size_t)(ng >> 1) * Kb};
  return PieceScales{p.sw + (size_t)(ng >> 2) * Kb, p.sw + (size_t)((p.end.No + 32 * ng) >> 7) * Kb};
}

// ---- few rows: everything in one launch ------------------------------------------------------------
// A workgroup takes 16 NJ weight rows for all (at most 16) rows of x; its 8 waves deal the blocks of 128 k among
// them (the next block's loads in flight), bring x to e4m3 in registers (32 values of one row a lane) and sum
// through LDS. Bound by the codes' bytes and a launch's ramp: one row of 2560 -> 10240 5.1 to 6.0 us, 5.1 to 4.4 TB/s.
constexpr int kFewWaves = 8;
template <class V8, int NJ, bool END, bool CODED>
__global__ __launch_bounds__(64 * kFewWaves) void f8_few_kernel(F8Args p) {
  constexpr int kPad = 16 * NJ + 4;  // (16 rows of sums cover the LDS banks)
  __shared__ __align__(16) float red[kFewWaves][16][kPad];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Kb = (p.K + 127) / 128;
  const int ng = blockIdx.x / (4 / NJ), j0 = blockIdx.x % (4 / NJ) * NJ;  // 64-row piece, first fragment in it
  const int m = lane & 15, kl = 32 * (lane >> 4);
  const rsrc_t rw = make_rsrc(p.wq + (size_t)ng * Kb * 8192 + j0 * 2048);
  const uint16_t* xr = (const uint16_t*)p.x + (m < p.M ? m : 0) * p.x_st;
  const PieceScales sw = piece_scales(p, ng, Kb);
  const rsrc_t rx = make_rsrc(p.xq);
  f32x4 acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Block {
    i32x8 w[NJ], xq;
    u16x8 x[4];
    float sw, sw1, sx;
  };
  const auto load = [&](Block& b, int kb) {
    kb = min(kb, Kb - 1);
#pragma unroll
    for (int j = 0; j < NJ; j++) b.w[j] = bload_frag(rw, 16 * lane, kb * 8192 + 2048 * j);
    if constexpr (CODED) {  // (rows past the last: whatever is there, not stored)
      b.xq = bload_frag(rx, 16 * lane, kb * 2048);
      b.sx = p.sx[(size_t)kb * p.Mp + m];
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int k = 128 * kb + kl + 8 * i;
        b.x[i] = u16x8{};
        if (m < p.M && k < p.K) b.x[i] = *reinterpret_cast<const u16x8*>(xr + k);
      }
    }
    b.sw = sw.even[kb];
    if (END) b.sw1 = sw.odd[kb];
  };
  const auto take = [&](const Block& b) {
    i32x8 xf;
    float s;
    if constexpr (CODED) {
      xf = b.xq;
      s = b.sx;
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) top = max(top, top_bits(b.x[i]));
      top = max(top, (uint32_t)__shfl_xor((int)top, 16));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32));
      float r;
      f8_scale(bits_value<V8>(top), r, s);
      int q[8];
#pragma unroll
      for (int i = 0; i < 4; i++) f8_codes(__builtin_bit_cast(V8, b.x[i]), r, q[2 * i], q[2 * i + 1]);
      xf = i32x8{q[0], q[1], q[2], q[3], q[4], q[5], q[6], q[7]};
    }
    const float s1 = END ? s * b.sw1 : 0.f;
    s *= b.sw;
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const f32x4 d = mfma_f8(b.w[j], xf);
#pragma unroll
      for (int e = 0; e < 4; e++) acc[j][e] = fmaf(END && (j & 1) ? s1 : s, d[e], acc[j][e]);
    }
  };
  Block b0, b1;
  if (wave < Kb) load(b0, wave);
  for (int kb = wave; kb < Kb; kb += 2 * kFewWaves) {
    load(b1, kb + kFewWaves);
    take(b0);
    if (kb + kFewWaves >= Kb) break;
    load(b0, kb + 2 * kFewWaves);
    take(b1);
  }
  // lane's outputs: row m, weight rows 16 (lane / 16) + 4 (j0 + j) + e of the piece -> column 4 NJ (lane / 16) + 4 j + e
#pragma unroll
  for (int j = 0; j < NJ; j++)
    *reinterpret_cast<f32x4*>(&red[wave][m][4 * NJ * (lane >> 4) + 4 * j]) = acc[j];
  __syncthreads();
  if constexpr (END) {
    end_few<V8, NJ, kFewWaves, kPad>(p.end, &red[0][0][0], p.M, ng, j0, threadIdx.x, 64 * kFewWaves);
    return;
  }
  for (int i = threadIdx.x; i < 16 * 16 * NJ; i += 64 * kFewWaves) {
    const int mm = i / (16 * NJ), c = i % (16 * NJ);
    float sum = red[0][mm][c];
#pragma unroll
    for (int w = 1; w < kFewWaves; w++) sum += red[w][mm][c];
    const int n = 64 * ng + 16 * (c / (4 * NJ)) + 4 * j0 + c % (4 * NJ);
    if (mm < p.M && n < p.N) {
      if (p.part)
        p.part[(size_t)mm * p.N + n] = sum;
      else {
        V8 v{};
        v[0] = (decltype(+v[0]))sum;
        ((uint16_t*)p.y)[(size_t)mm * p.N + n] = __builtin_bit_cast(u16x8, v)[0];
      }
    }
  }
}

// ---- some rows: no barriers, K divided between the waves ---------------------------------------------
// A workgroup takes 16 MB RW rows of x by 64 weight rows; its 8 waves deal the blocks of 128 k among them (RW = 2:
// four waves to each half of the rows), read both operands' fragments straight from memory (the next block's in
// flight) and sum through LDS. Through LDS tiles a step of this size is a chain of latencies (0.47 us at
// 64 x 128 x 128, whatever its neighbours do). One workgroup of 64 rows lies on a CU (240 registers), so 128 rows serve
// where 64 would need a second round: 238 rows 2560 -> 7680 11.0 -> 9.7 us, 512 rows 5120 -> 2560 18.4 -> 15.7. Bound by L2:
// 238 rows 5120 -> 2560 in tiles of 48 8.0 us, 14 TB/s of fragments.
constexpr int kSomeWaves = 8, kSomePad = 68;  // (rows of sums 68 floats apart: 16 of them cover the LDS banks)
template <class V8, int MB, int RW, bool END>
__global__ __launch_bounds__(64 * kSomeWaves) void f8_some_kernel(F8Args p) {
  constexpr int KW = kSomeWaves / RW;  // waves that share K; RW tiles of 16 MB rows
  __shared__ __align__(16) float red[kSomeWaves][16 * MB * kSomePad];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rg = wave / KW, kw = wave % KW;
  const int Kb = (p.K + 127) / 128, Mb = p.Mp / 16;
  // row tiles run fastest: those that share weights are on one XCD at one time
  const int t = xcd_remap(blockIdx.x, gridDim.x), ng = t / p.mtiles, mbt = (t - ng * p.mtiles) * MB * RW, mb0 = min(mbt + rg * MB, Mb - 1);
  const rsrc_t rw = make_rsrc(p.wq + (size_t)ng * Kb * 8192), rx = make_rsrc(p.xq + (size_t)mb0 * Kb * 2048);
  const rsrc_t rs = make_rsrc(p.sx);
  const PieceScales sw = piece_scales(p, ng, Kb);
  struct Block {
    i32x8 w[4], x[MB];
    float s[MB], sw, sw1;
  };
  const auto load = [&](Block& k, int kb) {
    kb = min(kb, Kb - 1);
#pragma unroll
    for (int j = 0; j < 4; j++) k.w[j] = bload_frag(rw, 16 * lane, kb * 8192 + 2048 * j);
#pragma unroll
    for (int b = 0; b < MB; b++) {  // (row blocks past the last: that one again, not stored)
      const int r = min(b, Mb - 1 - mb0);
      k.x[b] = bload_frag(rx, 16 * lane, (r * Kb + kb) * 2048);
      k.s[b] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, 4 * (lane & 15), 4 * (kb * p.Mp + 16 * (mb0 + r)), 0));
    }
    k.sw = sw.even[kb];
    if (END) k.sw1 = sw.odd[kb];
  };
  f32x4 acc[MB][4];
#pragma unroll
  for (int b = 0; b < MB; b++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const auto take = [&](const Block& k) {
#pragma unroll
    for (int b = 0; b < MB; b++) {
      const float s = k.s[b] * k.sw, s1 = END ? k.s[b] * k.sw1 : 0.f;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const f32x4 d = mfma_f8(k.w[j], k.x[b]);
#pragma unroll
        for (int e = 0; e < 4; e++) acc[b][j][e] = fmaf(END && (j & 1) ? s1 : s, d[e], acc[b][j][e]);
      }
    }
  };
  Block k0, k1;
  if (kw < Kb) load(k0, kw);
  for (int kb = kw; kb < Kb; kb += 2 * KW) {
    load(k1, kb + KW);
    take(k0);
    if (kb + KW >= Kb) break;
    load(k0, kb + 2 * KW);
    take(k1);
  }
#pragma unroll
  for (int b = 0; b < MB; b++)
#pragma unroll
    for (int j = 0; j < 4; j++)
      *reinterpret_cast<f32x4*>(&red[wave][(16 * b + (lane & 15)) * kSomePad + 16 * (lane >> 4) + 4 * j]) = acc[b][j];
  __syncthreads();
  if constexpr (END) {
#pragma unroll
    for (int g = 0; g < RW; g++)
      end_lds<V8, kSomePad>(p.end, red[g * KW], KW, 16 * MB * kSomePad, 16 * MB, 16 * (mbt + MB * g), p.M, ng, threadIdx.x,
                            64 * kSomeWaves);
    return;
  }
  for (int i = threadIdx.x; i < RW * 16 * MB * 8; i += 64 * kSomeWaves) {  // 8 columns of a row each
    const int ri = i >> 3, c = 8 * (i & 7), m = 16 * mbt + ri, n = 64 * ng + c;
    if (m >= p.M || n >= p.N) continue;
    const int g = ri / (16 * MB) * KW, r = ri % (16 * MB);
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll
    for (int w = 0; w < KW; w++) {
      a += *reinterpret_cast<const f32x4*>(&red[g + w][r * kSomePad + c]);
      b += *reinterpret_cast<const f32x4*>(&red[g + w][r * kSomePad + c + 4]);
    }
    if (p.part) {
      *reinterpret_cast<f32x4*>(p.part + (size_t)m * p.N + n) = a;
      *reinterpret_cast<f32x4*>(p.part + (size_t)m * p.N + n + 4) = b;
    } else {
      V8 v;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        v[e] = (decltype(+v[e]))a[e];
        v[4 + e] = (decltype(+v[e]))b[e];
      }
      *reinterpret_cast<V8*>((uint16_t*)p.y + (size_t)m * p.N + n) = v;
    }
  }
}

// ---- many rows ----------------------------------------------------------------------------------
// Workgroup tile of 16 MB WM rows of x by 64 WN weight rows, WM x WN waves of 16 MB x 64 each. A step is one
// block of 128 k: x and weight pieces and each wave's row scales come by direct loads into a ring of S slots. Bound by
// the matrix cores' power and the LDS reads that feed them (a wave's 16 MB x 64 reads MB + 4 fragments for 4 MB
// products): 8192 x 8192 x 8192 435 to 500 us by the clock, 2.5 to 2.2 PFLOP/s; 3481 x 2560 x 7680 72 us, 1.9.
template <class V8, int MB, int WM, int WN, int S, bool END>
__global__ __launch_bounds__(64 * WM * WN) void f8_gemm_kernel(F8Args p) {
  constexpr int NW = WM * WN, kX = 2048 * MB * WM, kW = 8192 * WN, kScales = 1024;  // bytes a slot
  constexpr int kSlot = kX + kW + NW * kScales;
  constexpr int kLoadsX = kX / 1024 / NW, kLoadsW = kW / 1024 / NW, kLoads = kLoadsX + kLoadsW + 1;
  static_assert(kLoadsX * NW * 1024 == kX && kLoadsW * NW * 1024 == kW, "whole loads per wave");
  static_assert((S - 2) * kLoads < 64, "loads in flight the counter can tell");
  __shared__ __align__(1024) char lds[S * kSlot];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN, Kb = (p.K + 127) / 128;
  // workgroups in groups of 8 row tiles, so that those running together share both operands' pieces in L2
  int t = xcd_remap(blockIdx.x, gridDim.x);
  const int tiles = p.mtiles * p.ntiles, split = t / tiles;
  t -= split * tiles;
  const int group = t / (8 * p.ntiles), in = t - group * 8 * p.ntiles, gm = min(8, p.mtiles - 8 * group);
  const int mt = 8 * group + in % gm, nt = in / gm;
  const int kb0 = Kb * split / p.splits, kb1 = Kb * (split + 1) / p.splits;  // (below 2^13 x 16)
  const int mb0 = mt * MB * WM, ng0 = nt * WN, Mb = p.Mp / 16, Ng = p.pieces;
  const int row0 = 16 * (mb0 + MB * wm);  // this wave's first row
  const dma_src_t rx = dma_src(p.xq + (size_t)mb0 * Kb * 2048, kBufRange), rw = dma_src(p.wq + (size_t)ng0 * Kb * 8192, kBufRange);
  const dma_src_t rs = dma_src(p.sx + min(row0, p.Mp - 16), kBufRange);
  const uint32_t base = lds_address(lds);
  // load number i of this wave's kLoads for a block: pieces of x, pieces of the weights, its rows' scales
  const auto load = [&](int kb, int slot, int i) {
    const uint32_t at = base + slot * kSlot;
    if (i < kLoadsX) {  // (row blocks past the last: that one again, not stored)
      const int u = wave * kLoadsX + i, r = min(u >> 1, Mb - 1 - mb0);  // KB u of the slot: row block u / 2, half u % 2
      dma16(rx, at + 1024 * u, 16 * lane, (uint32_t)(r * Kb + kb) * 2048u + 1024u * (u & 1));
    } else if (i < kLoadsX + kLoadsW) {
      const int u = wave * kLoadsW + i - kLoadsX, r = min(u >> 3, Ng - 1 - ng0);
      dma16(rw, at + kX + 1024 * u, 16 * lane, (uint32_t)(r * Kb + kb) * 8192u + 1024u * (u & 7));
    } else {  // (past the last row: the next block's scales, or the 1 KB behind the last's)
      dma16(rs, at + kX + kW + kScales * wave, 16 * lane, 4u * (uint32_t)p.Mp * (uint32_t)kb);
    }
  };
  f32x4 acc[MB][4];
#pragma unroll
  for (int i = 0; i < MB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const PieceScales sw = piece_scales(p, min(ng0 + wn, Ng - 1), Kb);
  const int n = kb1 - kb0;
  // This wave's weight scales of 64 blocks, one a lane: a load per block would wait for every tile in flight. (The
  // empty assembly has the wait here, not at each use.)
  float sws, sws1 = 0.f;
  const auto load_scales = [&](int i) {
    sws = i + lane < n ? sw.even[kb0 + i + lane] : 0.f;
    __asm__ volatile("" : "+v"(sws));
    if (END) {
      sws1 = i + lane < n ? sw.odd[kb0 + i + lane] : 0.f;
      __asm__ volatile("" : "+v"(sws1));
    }
  };
  const auto frag = [&](const char* src) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(src), hi = *reinterpret_cast<const i32x4*>(src + 1024);
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  load_scales(0);
#pragma unroll
  for (int i = 0; i < S - 1; i++)
#pragma unroll
    for (int u = 0; u < kLoads; u++) load(min(kb0 + i, kb1 - 1), i, u);  // (past the last block: loaded again, not used)
  for (int i = 0, slot = 0; i < n; i++, slot = slot + 1 == S ? 0 : slot + 1) {
    constexpr int kLeft = (S - 2) * kLoads;
    if (i > 0 && (i & 63) == 0) load_scales(i);
    __builtin_amdgcn_s_waitcnt(0x0F70 | (kLeft & 15) | ((kLeft >> 4) << 14));  // vmcnt(kLeft): this block's loads are in
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
    const int kn = min(kb0 + i + S - 1, kb1 - 1), next = slot == 0 ? S - 1 : slot - 1;
    const char* at = lds + slot * kSlot;
    const char* xs = at + 2048 * MB * wm + 16 * lane;
    const float* ss = reinterpret_cast<const float*>(at + kX + kW + kScales * wave) + (lane & 15);
    const float swk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sws), i & 63));
    const float swk1 = END ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sws1), i & 63)) : 0.f;
    // Loads of a later block are spread over the step: issued at once by all waves they keep every one of them from its
    // first LDS read until the last is out (72 of 1 KB at 64 bytes a cycle).
    constexpr int kSpread = (kLoads + (MB < 5 ? MB : 5) - 1) / (MB < 5 ? MB : 5);
    // The fragment and scale of the next 16 rows are read, and the last 16 rows' results taken into the sums, between
    // the matrix instructions of these.
    i32x8 w[4], x = frag(xs), xn;
    float s = ss[0], sn = 0.f, sp = 0.f, sp1 = 0.f;
    f32x4 d[4], dp[4];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = frag(at + kX + 8192 * wn + 2048 * j + 16 * lane);
#pragma unroll
    for (int b = 0; b <= MB; b++) {
      if (b + 1 < MB) {
        xn = frag(xs + 2048 * (b + 1));
        sn = ss[16 * (b + 1)];
      }
#pragma unroll
      for (int u = kSpread * b; u < kSpread * (b + 1); u++)
        if (u < kLoads) load(kn, next, u);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (b < MB) d[j] = mfma_f8(w[j], x);
        if (b > 0) {
#pragma unroll
          for (int e = 0; e < 4; e++) acc[b - 1][j][e] = fmaf(END && (j & 1) ? sp1 : sp, dp[j][e], acc[b - 1][j][e]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) dp[j] = d[j];
      x = xn;
      sp = swk * s;
      if (END) sp1 = swk1 * s;
      s = sn;
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this slot's reads are back before the next barrier frees it
    __asm__ volatile("" ::: "memory");
  }
  wait_vm(0);  // no load of this workgroup outlives it
  if constexpr (END) {
    __syncthreads();  // (or lands on what end_tile keeps in LDS)
    const int ng = ng0 + wn;
    if (ng >= Ng) return;
    if (!p.part) {
      end_tile<V8>(p.end, p.M, row0, ng, lane, acc, lds + 8192 * wave);
      return;
    }
#pragma unroll
    for (int b = 0; b < MB; b++) {
      const int m = row0 + 16 * b + (lane & 15);
      if (m < p.M) part16(p.part, (long long)split * p.M + m, Ng, ng, lane >> 4, acc[b]);
    }
    return;
  }
  // lane: row lane % 16 of each block, columns 16 (lane / 16) .. + 15 of the 64
  const int col = 64 * (ng0 + wn) + 16 * (lane >> 4);
#pragma unroll
  for (int b = 0; b < MB; b++) {
    const int m = row0 + 16 * b + (lane & 15);
    if (m >= p.M) continue;
    if (p.part) {
      float* dst = p.part + ((size_t)split * p.M + m) * p.N + col;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (col + 4 * j < p.N) *reinterpret_cast<f32x4*>(dst + 4 * j) = acc[b][j];
    } else {
      uint16_t* dst = (uint16_t*)p.y + (size_t)m * p.N + col;
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        V8 v;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          v[e] = (decltype(+v[e]))acc[b][j][e];
          v[4 + e] = (decltype(+v[e]))acc[b][j + 1][e];
        }
        if (col + 4 * j < p.N) *reinterpret_cast<V8*>(dst + 4 * j) = v;
      }
    }
  }
}

// Sum of the splits in their order, one rounding.
template <class V8>
__global__ __launch_bounds__(256) void f8_reduce_kernel(const float* __restrict__ part, uint16_t* __restrict__ y, size_t n8, int splits) {
  for (size_t c = (size_t)blockIdx.x * 256 + threadIdx.x; c < n8; c += (size_t)gridDim.x * 256) {
    f32x4 a = *reinterpret_cast<const f32x4*>(part + 8 * c), b = *reinterpret_cast<const f32x4*>(part + 8 * c + 4);
    for (int s = 1; s < splits; s++) {
      const float* src = part + 8 * (c + s * n8);
      a += *reinterpret_cast<const f32x4*>(src);
      b += *reinterpret_cast<const f32x4*>(src + 4);
    }
    V8 v;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      v[e] = (decltype(+v[e]))a[e];
      v[4 + e] = (decltype(+v[e]))b[e];
    }
    *reinterpret_cast<V8*>(y + 8 * c) = v;
  }
}

// ---- weights ------------------------------------------------------------------------------------
// Codes [N, K] into the fragment order, zeros past N and K: a thread writes 16 bytes.
__global__ __launch_bounds__(256) void f8_pack_kernel(const uint8_t* __restrict__ q, uint8_t* __restrict__ out, int N, int K) {
  const int Kb = (K + 127) / 128;
  const size_t total = (size_t)((N + 63) / 64) * Kb * 512;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const int u = (int)(i % 512), l = u & 63, half = (u >> 6) & 1, j = u >> 7;
    const size_t piece = i / 512;
    const int kb = (int)(piece % Kb);
    const size_t n = 64 * (piece / Kb) + 16 * ((l & 15) >> 2) + 4 * j + (l & 3);
    const int k = 128 * kb + 32 * (l >> 4) + 16 * half;
    i32x4 v = {0, 0, 0, 0};
    if (n < (size_t)N && k < K) v = *reinterpret_cast<const i32x4*>(q + n * K + k);
    *reinterpret_cast<i32x4*>(out + 16 * i) = v;
  }
}

// fp32 weights to codes and scales, a workgroup per 128 x 128 block (the same rule as x's blocks of a row, the
// scale rounded to fp32 before it divides, as other tools make such weights).
__global__ __launch_bounds__(256) void f8_quantize_weight_kernel(const float* __restrict__ w, uint8_t* __restrict__ q,
                                                                 float* __restrict__ sw, int N, int K) {
  __shared__ uint32_t red[4];
  const int Kb = (K + 127) / 128, kb = blockIdx.x % Kb, nb = blockIdx.x / Kb, t = threadIdx.x;
  const int k = 128 * kb + 4 * (t & 31), n0 = 128 * nb + (t >> 5);
  uint32_t top = 0;
  for (int i = 0; i < 16; i++) {
    const int n = n0 + 8 * i;
    if (n >= N || k >= K) continue;
    const u32x4 v = *reinterpret_cast<const u32x4*>(w + (size_t)n * K + k);
#pragma unroll
    for (int e = 0; e < 4; e++) top = max(top, v[e] & 0x7fffffffu);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  if ((t & 63) == 0) red[t >> 6] = top;
  __syncthreads();
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  float r, s;
  f8_scale(__builtin_bit_cast(float, top), r, s);
  if (t == 0) sw[blockIdx.x] = s;
  for (int i = 0; i < 16; i++) {
    const int n = n0 + 8 * i;
    if (n >= N || k >= K) continue;
    const f32x4 v = *reinterpret_cast<const f32x4*>(w + (size_t)n * K + k);
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] / s, v[1] / s, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] / s, v[3] / s, c, true);
    *reinterpret_cast<int*>(q + (size_t)n * K + k) = c;
  }
}

template <class V8, bool END, int MB, int WM, int WN, int S>
static hipError_t launch_gemm(F8Args a, hipStream_t s) {
  a.mtiles = (a.M + 16 * MB * WM - 1) / (16 * MB * WM);
  a.ntiles = (a.pieces + WN - 1) / WN;
  ESM_LAUNCH((f8_gemm_kernel<V8, MB, WM, WN, S, END>), dim3((unsigned)((size_t)a.mtiles * a.ntiles * a.splits)), dim3(64 * WM * WN), 0,
             s, a);
  return hipGetLastError();
}

template <class V8, bool END, int MB, int RW>
static hipError_t launch_some(F8Args a, hipStream_t s) {
  a.mtiles = (a.Mp / 16 + MB * RW - 1) / (MB * RW);
  ESM_LAUNCH((f8_some_kernel<V8, MB, RW, END>), dim3((unsigned)((size_t)a.mtiles * a.pieces)), dim3(64 * kSomeWaves), 0, s, a);
  return hipGetLastError();
}

template <class V8, bool END, bool CODED>
static hipError_t launch_few(const F8Args& a, int mb, hipStream_t s) {
  const dim3 grid(a.pieces * (4 / mb)), block(64 * kFewWaves);
  switch (mb) {
    case 4: ESM_LAUNCH((f8_few_kernel<V8, 4, END, CODED>), grid, block, 0, s, a); break;
    case 2: ESM_LAUNCH((f8_few_kernel<V8, 2, END, CODED>), grid, block, 0, s, a); break;
    default: ESM_LAUNCH((f8_few_kernel<V8, 1, END, CODED>), grid, block, 0, s, a); break;
  }
  return hipGetLastError();
}

template <class V8, bool END>
static hipError_t launch_f8_t(const F8Args& a, int form, int mb, hipStream_t s) {
  hipError_t e;
  if (form == kF8Few) {
    if constexpr (END)
      if (a.coded) return launch_few<V8, true, true>(a, mb, s);
    return launch_few<V8, END, false>(a, mb, s);
  }
  if (!a.coded) {
    ESM_LAUNCH((f8_quantize_kernel<V8>), dim3((a.Mp + 31) / 32, (a.K + 127) / 128), dim3(256), 0, s,
               (const uint16_t*)a.x, a.x_st, a.xq, a.sx, a.M, a.K, a.Mp);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (form == kF8Some) switch (mb) {
      case 1: return launch_some<V8, END, 1, 1>(a, s);
      case 2: return launch_some<V8, END, 2, 1>(a, s);
      case 3: return launch_some<V8, END, 3, 1>(a, s);
      case 4: return launch_some<V8, END, 4, 1>(a, s);
      default: return launch_some<V8, END, 4, 2>(a, s);
    }
  switch (mb) {
    case 2: e = launch_gemm<V8, END, 2, 2, 4, 2>(a, s); break;
    case 4: e = launch_gemm<V8, END, 4, 2, 4, 2>(a, s); break;
    case 6: e = launch_gemm<V8, END, 6, 2, 4, 2>(a, s); break;
    default: e = launch_gemm<V8, END, 8, 2, 4, 2>(a, s); break;
  }
  if (e != hipSuccess || !a.part) return e;
  if constexpr (END) return launch_linear_join<V8>(a.part, a.end, a.M, a.pieces, a.splits, s);
  if (!a.y) return e;
  const size_t n8 = (size_t)a.M * a.N / 8, blocks = (n8 + 255) / 256;
  ESM_LAUNCH((f8_reduce_kernel<V8>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, a.part, (uint16_t*)a.y, n8,
             a.splits);
  return hipGetLastError();
}

hipError_t launch_f8_linear(const F8Args& a, bool bf16, const F8Plan& plan, hipStream_t s) {
  if (a.end.on) return bf16 ? launch_f8_t<bf16x8, true>(a, plan.form, plan.mb, s) : launch_f8_t<half8, true>(a, plan.form, plan.mb, s);
  return bf16 ? launch_f8_t<bf16x8, false>(a, plan.form, plan.mb, s) : launch_f8_t<half8, false>(a, plan.form, plan.mb, s);
}

// Which form, its row blocks and splits: the lowest of estimated times, from these measurements (us, kernel alone,
// K = 2560 -> N = 7680 unless said; some: 64 x 64 tiles without barriers; 64, 128, 192, 256: LDS tiles of that many rows):
//   M = 238   some 9.7, 64 rows 18       M = 512   some 23, 64: 18.6, 128: 22, 256: 32
//   M = 1000  some 44, 64: 36, 128: 24, 192: 27, 256: 33     M = 1500  128: 44, 192: 31, 256: 33
//   M = 2000  128: 46, 192: 55, 256: 38    M = 3481  128: 90, 192: 86, 256: 70
//   5120 -> 2560 at M = 238  some 8.0, LDS tiles with K split 15 and 4 for the sum; at M = 512  some 15.7, 64 rows in two
//   splits 21 and 5; at M = 1000  some 31, 64 rows 33, 128 rows in three splits 25 and 6
F8Plan f8_plan(int M, int K, int N, int cus, bool gated) {
  // Few rows: the most weight rows a workgroup (16, 32 or 64) that still give more than half the CUs one, as each
  // workgroup reads x whole and few workgroups in flight leave the codes' loads waiting (us, 64 / 32 / 16 rows, M = 1 to 16:
  // 2560 -> 10240 5.1 to 6.3 / 6.3 to 9.4 / 8.2 to 12.2, 2560 -> 7680 4.9 to 6.3 / 4.5 to 5.7 / 6.2 to 8.8,
  // 2560 -> 2560 - / 4.8 to 5.6 / 4.2 to 5.3, 5120 -> 2560 - / 7.2 to 8.3 / 6.8 to 7.9, 8192 -> 8192 12.3 to 16 / 11.5 to 13.2 / 18).
  // Up to 16 rows, as x brought to e4m3 apart costs 3 us (16 rows of 2560 -> 10240 6.3 against 3 + 4.4, 5120 -> 2560 7.9
  // against 2.5 + 6.2), and a second block of 16 here 16 us.
  F8Plan p{kF8Few, 4, 1};
  const int least = gated ? 2 : 1;  // (a gate and its up value in one workgroup)
  while (p.mb > least && 16LL * ((N + 63) / 64) * (4 / p.mb) < 9LL * cus) p.mb /= 2;
  if (M <= 16) return p;
  const int Kb = (K + 127) / 128;
  // Some rows: the fewest rows a workgroup (16 to 64) whose tiles fit one to a CU; else 32 where two rounds take them
  // all, else 128 if those fit, else rounds of 64 (us, 16 / 32 / 48 / 64 rows a workgroup: 64 rows
  // 5120 -> 2560 5.7 / 6.5 / 7.8 / 9.1, 238 rows - / 11.3 / 8.0 / 9.5, 96 rows 2560 -> 7680 - / 7.5 / 5.5 / 6.2, 24 rows
  // 2560 -> 10240 5.4 / 4.6 / 4.9 / 5.6, 96 rows 9.3 / 8.0 / 9.3 / 10.8 and 9.1 in 128; two of 32 rows on a CU at once would take
  // 128 registers, which spill: 10.3).
  const long long pieces = (N + 63) / 64;
  const auto tiles = [&](int mb) { return ((M + 15) / 16 + mb - 1) / mb * pieces; };
  p.form = kF8Some;
  for (p.mb = 1; p.mb < 5 && tiles(p.mb) > cus;) p.mb++;
  double best = 2.5 + Kb * (0.03 + 0.045 * p.mb);
  if (p.mb == 5) {
    p.mb = tiles(2) <= 2 * cus ? 2 : tiles(8) <= cus ? 8 : 4;
    best = 2.5 + Kb * (p.mb == 2 ? 0.28 : p.mb == 8 ? 0.38 : 1.2e-3 * (double)tiles(4) * cus / 256);
  }
  const struct { int mb; double step; } forms[] = {{2, 0.78}, {4, 1.0}, {6, 1.25}, {8, 1.55}};  // us a block of k
  for (const auto& f : forms)
    for (int sp = 1; sp <= kF8MaxSplits && (sp == 1 || 4 * sp <= Kb); sp++) {
      const long long wgs = (long long)((M + 32 * f.mb - 1) / (32 * f.mb)) * ((N + 255) / 256) * sp, rounds = (wgs + cus - 1) / cus;
      if (sp > 1 && rounds > 1) break;  // splits only fill one round
      double c = rounds * (2.5 + f.step * ((Kb + sp - 1) / sp));
      if (sp > 1) c += 3.0 + 8.0 * sp * M * N / 4.0e6;  // writing and summing the partials
      if (c < best) {
        best = c;
        p = F8Plan{kF8Tiles, f.mb, sp};
      }
    }
  return p;
}

hipError_t launch_f8_pack(const uint8_t* q, uint8_t* out, int N, int K, hipStream_t s) {
  const size_t blocks = ((size_t)((N + 63) / 64) * ((K + 127) / 128) * 512 + 255) / 256;
  ESM_LAUNCH(f8_pack_kernel, dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, s, q, out, N, K);
  return hipGetLastError();
}

hipError_t launch_f8_quantize_weight(const float* w, uint8_t* q, float* sw, int N, int K, hipStream_t s) {
  ESM_LAUNCH(f8_quantize_weight_kernel, dim3((unsigned)((size_t)((N + 127) / 128) * ((K + 127) / 128))), dim3(256), 0, s, w, q, sw, N, K);
  return hipGetLastError();
}

}  // namespace esm
