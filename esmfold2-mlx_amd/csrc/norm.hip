// Residual addition and norm of the sum, one pass over rows of D values:
//   s = x + alpha y                          (fp32; written back in x's type, fp32 or 16-bit)
//   h = s / sqrt(mean(s^2) + eps) w          rms; layer: (s - mean) / sqrt(mean((s - mean)^2) + eps) w; + b
// with h rounded once to the 16-bit type, or once to e4m3 by the rule of the e4m3 linear (per row and 128 columns:
// r = 448 / max(amax, 2^-96), code = e4m3(h r), scale = max(amax, 2^-96) / 448) in the order that linear's matrix cores
// take, so that it starts without a pass of its own over the rows. The norm takes s before its rounding to x's type.
//
// W waves take a row, a lane NIT pieces of 8 values, kept in registers between the sums and the output: every value
// is read once. Bound by bytes: 16,384 rows of 8,192 in 215 us, 5.0 TB/s where a large copy runs 5.1; 3,481 rows of 2,560, fp32 to
// e4m3, 23.7 us, 4.1 TB/s; small calls by a launch and two latencies, 8 rows of 4,096 4.0 us. Each wave's mean and squares about it are
// joined as  mean = sum n_w mean_w / n,  M2 = sum M2_w + n_w (mean_w - mean)^2  with one barrier.
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace esm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kNormWaves = 16;  // most waves of a workgroup

template <class V8, bool X32, bool F8, int NIT>
__global__ __launch_bounds__(64 * kNormWaves) void add_norm_kernel(AddNormArgs p) {
  __shared__ float red[kNormWaves][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int W = p.waves, r = wave / W, w = wave - r * W;  // row of the workgroup, wave of the row
  const long long row = (long long)blockIdx.x * p.rows + r;
  const bool live = row < p.T;
  const int width = F8 ? p.Kb * 128 : p.D;  // (e4m3: whole blocks, zeros behind the row)
  int col[NIT];
  float s[NIT][8];
#pragma unroll
  for (int it = 0; it < NIT; it++) {
    col[it] = 8 * ((it * W + w) * 64 + lane);
    const bool ok = live && col[it] < p.D;
    V8 yv{};
    if (X32) {
      f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
      if (ok) {
        const float* src = (const float*)p.x + row * p.x_st + col[it];
        a = *reinterpret_cast<const f32x4*>(src);
        b = *reinterpret_cast<const f32x4*>(src + 4);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) s[it][e] = a[e], s[it][4 + e] = b[e];
    } else {
      V8 a{};
      if (ok) a = *reinterpret_cast<const V8*>((const uint16_t*)p.x + row * p.x_st + col[it]);
#pragma unroll
      for (int e = 0; e < 8; e++) s[it][e] = (float)a[e];
    }
    if (p.y) {
      if (ok) yv = *reinterpret_cast<const V8*>((const uint16_t*)p.y + row * p.y_st + col[it]);
#pragma unroll
      for (int e = 0; e < 8; e++) s[it][e] = fmaf(p.alpha, (float)yv[e], s[it][e]);
    }
  }
  if (p.s) {
#pragma unroll
    for (int it = 0; it < NIT; it++) {
      if (!live || col[it] >= p.D) continue;
      if (X32) {
        float* dst = (float*)p.s + row * p.s_st + col[it];
        *reinterpret_cast<f32x4*>(dst) = f32x4{s[it][0], s[it][1], s[it][2], s[it][3]};
        *reinterpret_cast<f32x4*>(dst + 4) = f32x4{s[it][4], s[it][5], s[it][6], s[it][7]};
      } else {
        V8 v;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (decltype(+v[e]))s[it][e];
        *reinterpret_cast<V8*>((uint16_t*)p.s + row * p.s_st + col[it]) = v;
      }
    }
  }
  // (values past the row are zeros; about a mean they would count, and are left out)
  float mean = 0.f, m2 = 0.f;
  const auto values_of = [&](int w) {
    int n = 0;
    for (int it = 0; it < NIT; it++) n += min(max(p.D - 512 * (it * W + w), 0), 512);
    return (float)n;
  };
  if (p.layer) {
    float t = 0.f;
#pragma unroll
    for (int it = 0; it < NIT; it++)
#pragma unroll
      for (int e = 0; e < 8; e++) t += s[it][e];
    mean = wave_total(t) / fmaxf(values_of(w), 1.f);
  }
  {
    float t = 0.f;
#pragma unroll
    for (int it = 0; it < NIT; it++) {
      if (col[it] >= p.D) continue;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float d = s[it][e] - mean;
        t = fmaf(d, d, t);
      }
    }
    m2 = wave_total(t);
  }
  const float inv = 1.f / (float)p.D;
  if (W > 1) {
    if (lane == 0) red[wave][0] = mean, red[wave][1] = m2;
    __syncthreads();
    const int i = lane & 15;
    const float a = i < W ? red[r * W + i][0] : 0.f, b = i < W ? red[r * W + i][1] : 0.f;
    float d = 0.f;
    if (p.layer) {
      const float n = i < W ? values_of(i) : 0.f;
      mean = row16_sum(n * a) * inv;
      d = n * (a - mean) * (a - mean);
    }
    m2 = row16_sum(b + d);
  }
  const float rs = rsqrtf(m2 * inv + p.eps);
  if (!live) return;
#pragma unroll
  for (int it = 0; it < NIT; it++) {
    if (col[it] >= width) continue;
    float h[8];
    const bool ok = !F8 || col[it] < p.D;
    f32x4 w0 = {1.f, 1.f, 1.f, 1.f}, w1 = w0, b0 = {0.f, 0.f, 0.f, 0.f}, b1 = b0;
    if (ok && p.w) w0 = *reinterpret_cast<const f32x4*>(p.w + col[it]), w1 = *reinterpret_cast<const f32x4*>(p.w + col[it] + 4);
    if (ok && p.b) b0 = *reinterpret_cast<const f32x4*>(p.b + col[it]), b1 = *reinterpret_cast<const f32x4*>(p.b + col[it] + 4);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float v = fmaf((s[it][e] - mean) * rs, e < 4 ? w0[e & 3] : w1[e & 3], e < 4 ? b0[e & 3] : b1[e & 3]);
      h[e] = ok ? v : 0.f;
    }
    if constexpr (F8) {
      // the 16 lanes of a data-parallel row hold 128 columns; NaN and infinity are the largest, and make all 128 NaN
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) top = max(top, __builtin_bit_cast(uint32_t, h[e]) & 0x7fffffffu);
      const auto other = [&](auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, decltype(ctrl)::value, 0xf, 0xf, false);
      };
      top = max(top, other(std::integral_constant<int, 0x128>{}));  // row_ror:8, 4, 2, 1
      top = max(top, other(std::integral_constant<int, 0x124>{}));
      top = max(top, other(std::integral_constant<int, 0x122>{}));
      top = max(top, other(std::integral_constant<int, 0x121>{}));
      float f, scale;
      f8_scale(__builtin_bit_cast(float, top), f, scale);
      int lo = __builtin_amdgcn_cvt_pk_fp8_f32(h[0] * f, h[1] * f, 0, false);
      lo = __builtin_amdgcn_cvt_pk_fp8_f32(h[2] * f, h[3] * f, lo, true);
      int hi = __builtin_amdgcn_cvt_pk_fp8_f32(h[4] * f, h[5] * f, 0, false);
      hi = __builtin_amdgcn_cvt_pk_fp8_f32(h[6] * f, h[7] * f, hi, true);
      const int kb = col[it] >> 7, c = (col[it] >> 4) & 7, m = (int)(row & 15);
      uint8_t* dst = p.hq + ((size_t)(row >> 4) * p.Kb + kb) * 2048 + (c & 1) * 1024 + (16 * (c >> 1) + m) * 16 + (col[it] & 8);
      *reinterpret_cast<u32x2*>(dst) = u32x2{(uint32_t)lo, (uint32_t)hi};
      if ((lane & 15) == 0) p.sx[(size_t)kb * p.Mp + row] = scale;
    } else {
      V8 v;
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = (decltype(+v[e]))h[e];
      *reinterpret_cast<V8*>((uint16_t*)p.h + row * p.h_st + col[it]) = v;
    }
  }
}

template <class V8, bool X32, bool F8>
static hipError_t launch_norm_t(AddNormArgs a, hipStream_t st) {
  // Rows enough to fill the GPU: up to 8 pieces a lane, few waves a row; few rows: as many waves as the row has pieces
  const int width = F8 ? a.Kb * 128 : a.D, units = (width + 511) / 512;  // 64 lanes' pieces
  const bool few = a.T < 1024;
  int nit = few ? (units + kNormWaves - 1) / kNormWaves : 8;
  if (!few) {  // the fewest idle lanes, then the most pieces a lane
    int best = 1 << 30;
    for (int n : {8, 5, 4, 3, 2, 1}) {
      const int w = (units + n - 1) / n;
      if (w <= kNormWaves && w * n - units < best) best = w * n - units, nit = n;
    }
  }
  if (nit > 5) nit = 8;
  a.waves = (units + nit - 1) / nit;
  a.rows = few ? 1 : max(1, (F8 ? 8 : 4) / a.waves);
  const dim3 grid((unsigned)((a.T + a.rows - 1) / a.rows)), block(64 * a.waves * a.rows);
  switch (nit) {
    case 1: ESM_LAUNCH((add_norm_kernel<V8, X32, F8, 1>), grid, block, 0, st, a); break;
    case 2: ESM_LAUNCH((add_norm_kernel<V8, X32, F8, 2>), grid, block, 0, st, a); break;
    case 3: ESM_LAUNCH((add_norm_kernel<V8, X32, F8, 3>), grid, block, 0, st, a); break;
    case 4: ESM_LAUNCH((add_norm_kernel<V8, X32, F8, 4>), grid, block, 0, st, a); break;
    case 5: ESM_LAUNCH((add_norm_kernel<V8, X32, F8, 5>), grid, block, 0, st, a); break;
    case 8: ESM_LAUNCH((add_norm_kernel<V8, X32, F8, 8>), grid, block, 0, st, a); break;
    default: return hipErrorInvalidValue;  // (D is bounded by the caller)
  }
  return hipGetLastError();
}

hipError_t launch_add_norm(const AddNormArgs& a, bool bf16, bool x32, hipStream_t s) {
  const auto launch = [&](auto v, auto x) {
    typedef decltype(v) V8;
    constexpr bool X32 = decltype(x)::value;
    return a.hq ? launch_norm_t<V8, X32, true>(a, s) : launch_norm_t<V8, X32, false>(a, s);
  };
  if (bf16) return x32 ? launch(bf16x8{}, std::true_type{}) : launch(bf16x8{}, std::false_type{});
  return x32 ? launch(half8{}, std::true_type{}) : launch(half8{}, std::false_type{});
}

}  // namespace esm
