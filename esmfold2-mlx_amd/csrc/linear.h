// The end of a linear: y = r + alpha act(z), or r + alpha act(g) u of gated weights, with z (g, u) the products' fp32
// sums and a bias. fp32 throughout, one rounding to the 16-bit output.
//
// Both linears (16-bit and e4m3) leave a lane 16 consecutive packed weight rows 16 g + 4 j + e of a piece of 64 (g = lane /
// 16, j the fragment, e the register) for one row of x. Gated weights are packed so that fragments 0 and 2 hold gate rows and
// 1 and 3 the up rows of the same outputs: output 32 piece + 8 g + 4 (j / 2) + e. A gate and its up value meet in a lane.
#pragma once

#include "common.h"
#include "kernels.h"

namespace esm {

// gelu(z) = z P(z), P the normal distribution function: 1 - P(|z|) = (t (a1 + t (a2 + ...))) e^(-z^2 / 2) / 2 with
// t = 1 / (1 + p |z| / sqrt 2), off by 0.75e-7 at most in exact arithmetic (Abramowitz and Stegun, 7.1.26; half of its bound on
// erf). In fp32, with reciprocal and power off by a step, P is off by 5.5e-7 at most, near z = 0, and by 1.8e-7 below z = -1.
DEV float gelu_erf(float z) {
  const float a = fabsf(z), t = __builtin_amdgcn_rcpf(fmaf(a, 0.3275911f * 0.70710678f, 1.f));
  float q = fmaf(t, 1.061405429f, -1.453152027f);
  q = fmaf(t, q, 1.421413741f);
  q = fmaf(t, q, -0.284496736f);
  q = fmaf(t, q, 0.254829592f);
  const float tail = 0.5f * t * q * __builtin_amdgcn_exp2f(-0.72134752f * z * z);
  return z * (z > 0.f ? 1.f - tail : tail);
}
DEV float silu(float z) { return z * sigmoidf_fast(z); }
// 0.5 z (1 + tanh u) = z sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3)
DEV float gelu_tanh(float z) {
  return z * sigmoidf_fast(1.5957691216f * z * fmaf(0.044715f * z, z, 1.f));
}

// All values of a lane by one activation, chosen once for all.
template <int N>
DEV void activate(f32x4 (&v)[N], int act) {
  const auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) v[i][e] = f(v[i][e]);
  };
  switch (act) {
    case kActRelu: each([](float z) { return z < 0.f ? 0.f : z; }); break;  // (NaN stays)
    case kActGelu: each(gelu_erf); break;
    case kActGeluTanh: each(gelu_tanh); break;
    case kActSilu: each(silu); break;
    default: break;
  }
}

// 8 outputs n .. n + 7 (n < the row's outputs, a multiple of 8) of row m: scaled, the residual's added, rounded, stored.
template <class V8>
DEV void put8(const LinearEnd& p, long long m, int n, f32x4 a, f32x4 b) {
  if (p.res) {
    const V8 r = *reinterpret_cast<const V8*>((const uint16_t*)p.res + m * p.r_st + n);
#pragma unroll
    for (int e = 0; e < 4; e++) {
      a[e] = fmaf(p.alpha, a[e], (float)r[e]);
      b[e] = fmaf(p.alpha, b[e], (float)r[4 + e]);
    }
  } else if (p.alpha != 1.f) {
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] *= p.alpha, b[e] *= p.alpha;
  }
  V8 v;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    v[e] = (decltype(+v[e]))a[e];
    v[4 + e] = (decltype(+v[e]))b[e];
  }
  *reinterpret_cast<V8*>((uint16_t*)p.y + m * p.No + n) = v;
}
// The same for 4 outputs (8 bytes).
template <class V8>
DEV void put4(const LinearEnd& p, long long m, int n, f32x4 a) {
  typedef decltype(__builtin_shufflevector(V8{}, V8{}, 0, 1, 2, 3)) V4;
  if (p.res) {
    const V4 r = *reinterpret_cast<const V4*>((const uint16_t*)p.res + m * p.r_st + n);
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] = fmaf(p.alpha, a[e], (float)r[e]);
  } else if (p.alpha != 1.f) {
#pragma unroll
    for (int e = 0; e < 4; e++) a[e] *= p.alpha;
  }
  V4 v;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = (decltype(+v[e]))a[e];
  *reinterpret_cast<V4*>((uint16_t*)p.y + m * p.No + n) = v;
}
DEV f32x4 bias4(const LinearEnd& p, int n) {  // (n a multiple of 4, anything past the last reads none)
  return p.bias && n < p.Nb ? *reinterpret_cast<const f32x4*>(p.bias + n) : f32x4{0.f, 0.f, 0.f, 0.f};
}

// 16 packed columns of row m from column 16 g of piece `ng` on, in fragment order.
template <class V8>
DEV void end16(const LinearEnd& p, long long m, int ng, int g, f32x4 (&v)[4]) {
  if (p.gated) {
    const int n = 32 * ng + 8 * g;
    if (n >= p.No) return;
    f32x4 a[2] = {v[0] + bias4(p, n), v[2] + bias4(p, n + 4)};
    const f32x4 u[2] = {v[1] + bias4(p, p.No + n), v[3] + bias4(p, p.No + n + 4)};
    activate(a, p.act);
    put8<V8>(p, m, n, a[0] * u[0], a[1] * u[1]);
  } else {
    const int n = 64 * ng + 16 * g;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] += bias4(p, n + 4 * j);
    activate(v, p.act);
    if (n < p.No) put8<V8>(p, m, n, v[0], v[1]);
    if (n + 8 < p.No) put8<V8>(p, m, n + 8, v[2], v[3]);
  }
}

// The accumulators of a wave: rows row0 + 16 b + lane % 16 by a piece of 64 packed columns. They pass through LDS (8 KB of
// the wave's own, two row blocks at a time) into one rolled loop: unrolled over the registers, the activations' code and
// values would spill (148 registers of 256).
template <class V8, int MB>
DEV void end_tile(const LinearEnd& p, int M, int row0, int ng, int lane, const f32x4 (&acc)[MB][4], char* lds) {
  f32x4* own = reinterpret_cast<f32x4*>(lds) + lane;
  static_assert(MB % 2 == 0, "pairs of row blocks");
#pragma unroll
  for (int i = 0; i < MB; i += 2) {
#pragma unroll
    for (int u = 0; u < 8; u++) own[64 * u] = acc[i + (u >> 2)][u & 3];
#pragma unroll 1
    for (int b = 0; b < 2; b++) {
      const int m = row0 + 16 * (i + b) + (lane & 15);
      f32x4 v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = own[64 * (4 * b + j)];
      if (m < M) end16<V8>(p, m, ng, lane >> 4, v);
    }
  }
}

// fp32 partials of packed columns (rows of 64 pieces) into their row: columns 16 g .. of a piece, as end16 takes them.
DEV void part16(float* part, long long row, int pieces, int ng, int g, const f32x4 (&v)[4]) {
  float* dst = part + (row * pieces + ng) * 64 + 16 * g;
#pragma unroll
  for (int j = 0; j < 4; j++) *reinterpret_cast<f32x4*>(dst + 4 * j) = v[j];
}

// The sum of the splits in their order and the end of the linear: a thread takes 16 packed columns of a row. Bound by a launch
// and two latencies: 238 rows of 2,560 4.8 us.
template <class V8>
__global__ __launch_bounds__(256) void linear_join_kernel(const float* __restrict__ part, LinearEnd p, int M, int pieces, int splits) {
  const size_t each = (size_t)M * pieces * 4, step = each * 16;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < each; i += (size_t)gridDim.x * 256) {
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = *reinterpret_cast<const f32x4*>(part + 16 * i + 4 * j);
    for (int s = 1; s < splits; s++)
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += *reinterpret_cast<const f32x4*>(part + s * step + 16 * i + 4 * j);
    const size_t piece = i >> 2, m = piece / pieces;
    end16<V8>(p, (long long)m, (int)(piece - m * pieces), (int)(i & 3), v);
  }
}

// Partials of `rows` rows x one piece that lie in LDS, `waves` copies of 64 columns kPad floats apart: summed in their order, ended.
template <class V8, int kPad>
DEV void end_lds(const LinearEnd& p, const float* red, int copies, int stride, int rows, long long m0, int M, int ng, int first,
                 int threads) {
  for (int i = first; i < rows * 4; i += threads) {
    const int r = i >> 2, g = i & 3;
    if (m0 + r >= M) continue;
    f32x4 v[4] = {};
    for (int w = 0; w < copies; w++)
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] += *reinterpret_cast<const f32x4*>(red + w * stride + r * kPad + 16 * g + 4 * j);
    end16<V8>(p, m0 + r, ng, g, v);
  }
}

// The sums of fragments j0 .. j0 + NJ - 1 of a piece for at most 16 rows, `WAVES` copies in LDS: column 4 NJ g + 4 j + e of a
// row is packed row 16 g + 4 (j0 + j) + e. A thread takes 4 outputs, so that few rows still give many threads work.
template <class V8, int NJ, int WAVES, int kPad>
DEV void end_few(const LinearEnd& p, const float* red, int M, int ng, int j0, int first, int threads) {
  const int each = p.gated ? 2 * NJ : 4 * NJ;  // groups of 4 outputs of a row
  for (int i = first; i < 16 * each; i += threads) {
    const int m = i / each, u = i - m * each;
    if (m >= M) continue;
    const auto sum = [&](int c) {
      f32x4 v = *reinterpret_cast<const f32x4*>(red + m * kPad + c);
#pragma unroll
      for (int w = 1; w < WAVES; w++) v += *reinterpret_cast<const f32x4*>(red + (16 * w + m) * kPad + c);
      return v;
    };
    int n;
    f32x4 z[1];
    if (p.gated) {
      if constexpr (NJ >= 2) {
        const int g = u / (NJ / 2), j = u - g * (NJ / 2), c = 4 * NJ * g + 8 * j;
        n = 32 * ng + 8 * g + 4 * (j0 / 2 + j);
        if (n >= p.No) continue;
        z[0] = sum(c) + bias4(p, n);
        activate(z, p.act);
        z[0] *= sum(c + 4) + bias4(p, p.No + n);
      } else {
        return;  // (a gate and its up value stand in different workgroups: not planned)
      }
    } else {
      const int g = u / NJ, j = u - g * NJ;
      n = 64 * ng + 16 * g + 4 * (j0 + j);
      if (n >= p.No) continue;
      z[0] = sum(4 * NJ * g + 4 * j) + bias4(p, n);
      activate(z, p.act);
    }
    put4<V8>(p, m, n, z[0]);
  }
}

template <class V8>
static hipError_t launch_linear_join(const float* part, const LinearEnd& end, int M, int pieces, int splits, hipStream_t s) {
  const size_t blocks = ((size_t)M * pieces * 4 + 255) / 256;
  ESM_LAUNCH((linear_join_kernel<V8>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, part, end, M, pieces, splits);
  return hipGetLastError();
}

}  // namespace esm
