// Norm of queries and keys with the rotation of each row's position, one pass:
//   y = norm(x) * w        rms: x / sqrt(mean(x^2) + eps); layer: the same of x - mean(x); or none;
//                          over each head, or over the row of all its heads (q and k apart)
//   (a, b) -> (a cos - b sin, b cos + a sin)   of the first `rot` values of each head, pairs (i, i + rot/2)
//                                              or (2i, 2i + 1); the others pass through
// with the angle position * freq[i], freq in radians and fp64: at a position of 10^6 an fp32 angle is off by
// 0.06 rad, so the product and its reduction to one revolution are fp64 and the hardware's sine and cosine take
// the fraction. Statistics, norm and rotation are fp32, rounded once to the 16-bit output.
//
// A lane owns 16 values of a head, its 8 pairs, as two 16-byte pieces, so that a rotation stays within the
// lane; 2^lph lanes make a head and a wave takes 64 / 2^lph heads at a time. Memory bound: what matters is
// that a wave has its loads in flight before the angles, which depend on the row alone and are used for
// each of the wave's NIT groups of heads. 16,384 rows of 32 + 8 heads of 128 73 us, 4.6 TB/s; 3,481 rows of 40 + 40
// heads of 64 over the row 20 us, 3.6 TB/s (two barriers for the row's sums); 8 rows 3.4 us.
#include "common.h"
#include "kernels.h"

namespace esm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kRopeWaves = 16;  // most waves of a workgroup

// Sum over the 2^lph lanes of a head (lph uniform): within four lanes by quad permutes, then by the mirrors of
// 8 and 16 lanes, which reach the other half once each quad (each eight) holds one value.
DEV float head_sum(float v, int lph) {
  if (lph > 0) v += dpp_f32<0xB1>(v);   // quad_perm(1, 0, 3, 2)
  if (lph > 1) v += dpp_f32<0x4E>(v);   // quad_perm(2, 3, 0, 1)
  if (lph > 2) v += dpp_f32<0x141>(v);  // row_half_mirror
  if (lph > 3) v += dpp_f32<0x140>(v);  // row_mirror
  return v;
}

// Sums of q's and k's parts over the workgroup.
DEV void row_sum(float& sq, float& sk, float (*red)[kRopeWaves], int nw) {
  sq = row16_sum(sq);
  sk = row16_sum(sk);
  sq += __shfl_xor(sq, 16);
  sk += __shfl_xor(sk, 16);
  sq += __shfl_xor(sq, 32);
  sk += __shfl_xor(sk, 32);
  const int w = threadIdx.x >> 6;
  __syncthreads();  // red is reused by consecutive calls
  if ((threadIdx.x & 63) == 0) {
    red[0][w] = sq;
    red[1][w] = sk;
  }
  __syncthreads();
  sq = red[0][0];
  sk = red[1][0];
  for (int i = 1; i < nw; i++) {
    sq += red[0][i];
    sk += red[1][i];
  }
}

template <class V8, bool ROW, int NIT>
__global__ __launch_bounds__(64 * kRopeWaves) void qk_norm_rope_kernel(QkRopeArgs p) {
  __shared__ float red[2][kRopeWaves];
  const size_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int lph = p.lph, hpw = 64 >> lph;             // heads per wave and pass
  const int c = lane & ((1 << lph) - 1), hl = lane >> lph;
  const bool turn = 16 * c < p.rot;
  // the two pieces of this lane: its pairs' first and second values (half layout), or 16 values in a row
  const int o1 = turn && !p.interleaved ? 8 * c : 16 * c;
  const int o2 = turn && !p.interleaved ? o1 + p.rot / 2 : o1 + 8;
  const bool ok1 = o1 < p.d, ok2 = o2 < p.d;
  const int g0 = (blockIdx.y * nw + wave) * NIT;      // first group of heads of this wave

  V8 x1[NIT], x2[NIT];
  int head[NIT];
#pragma unroll
  for (int it = 0; it < NIT; it++) {
    const int hh = (g0 + it) * hpw + hl;
    head[it] = hh < p.H + p.Hk ? hh : -1;
    const bool isk = hh >= p.H;
    const char* src = (const char*)(isk ? p.k : p.q) +
                      2 * (row * (size_t)(isk ? p.k_st : p.q_st) + (size_t)(isk ? hh - p.H : hh) * (isk ? p.k_sh : p.q_sh));
    x1[it] = x2[it] = V8{};
    if (head[it] >= 0 && ok1) x1[it] = *reinterpret_cast<const V8*>(src + 2 * o1);
    if (head[it] >= 0 && ok2) x2[it] = *reinterpret_cast<const V8*>(src + 2 * o2);
  }

  // sine and cosine of the lane's pairs 8c .. 8c + 7
  float sn[8], cs[8];
  if (turn) {
    const double pos = p.pos64 ? (double)p.pos64[row] : p.pos32 ? (double)p.pos32[row] : (double)row;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      double rev = pos * p.freq[8 * c + e] * 0.15915494309189533577;
      rev -= floor(rev);
      sn[e] = __builtin_amdgcn_sinf((float)rev) * p.gain;
      cs[e] = __builtin_amdgcn_cosf((float)rev) * p.gain;
    }
  }

  float a[NIT][8], b[NIT][8];
#pragma unroll
  for (int it = 0; it < NIT; it++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      a[it][e] = (float)x1[it][e];
      b[it][e] = (float)x2[it][e];
    }
  if (p.norm) {
    float mean[NIT], rstd[NIT];
    // mean of f over each head, or over q's and k's rows
    const auto reduce = [&](auto part, float (&out)[NIT]) {
      if constexpr (ROW) {
        float sq = 0.f, sk = 0.f;
#pragma unroll
        for (int it = 0; it < NIT; it++) {
          const float s = part(it);
          sq += head[it] >= 0 && head[it] < p.H ? s : 0.f;
          sk += head[it] >= p.H ? s : 0.f;
        }
        row_sum(sq, sk, red, nw);
        sq /= (float)(p.H * p.d);
        sk /= (float)(p.Hk * p.d);
#pragma unroll
        for (int it = 0; it < NIT; it++) out[it] = head[it] >= p.H ? sk : sq;
      } else {
#pragma unroll
        for (int it = 0; it < NIT; it++) out[it] = head_sum(part(it), lph) / (float)p.d;
      }
    };
    if (p.norm == kNormLayer) {
      reduce(
          [&](int it) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) s += a[it][e] + b[it][e];  // (pieces past the head hold zeros)
            return s;
          },
          mean);
#pragma unroll
      for (int it = 0; it < NIT; it++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
          a[it][e] -= mean[it];
          b[it][e] -= mean[it];
        }
    }
    reduce(
        [&](int it) {
          float s = 0.f, t = 0.f;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            s += a[it][e] * a[it][e];
            t += b[it][e] * b[it][e];
          }
          return (ok1 ? s : 0.f) + (ok2 ? t : 0.f);
        },
        rstd);
#pragma unroll
    for (int it = 0; it < NIT; it++) {
      if (head[it] < 0) continue;
      const float r = rsqrtf(rstd[it] + p.eps);
      const bool isk = head[it] >= p.H;
      const float* w = isk ? p.k_w : p.q_w;
      f32x4 wa0 = {1.f, 1.f, 1.f, 1.f}, wa1 = wa0, wb0 = wa0, wb1 = wa0;  // (no weight: 1)
      if (w) {
        w += (size_t)(isk ? head[it] - p.H : head[it]) * (isk ? p.kw_sh : p.qw_sh);
        if (ok1) wa0 = *reinterpret_cast<const f32x4*>(w + o1), wa1 = *reinterpret_cast<const f32x4*>(w + o1 + 4);
        if (ok2) wb0 = *reinterpret_cast<const f32x4*>(w + o2), wb1 = *reinterpret_cast<const f32x4*>(w + o2 + 4);
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        a[it][e] = a[it][e] * r * (e < 4 ? wa0[e & 3] : wa1[e & 3]);
        b[it][e] = b[it][e] * r * (e < 4 ? wb0[e & 3] : wb1[e & 3]);
      }
    }
  }
#pragma unroll
  for (int it = 0; it < NIT; it++) {
    if (head[it] < 0) continue;
    V8 y1, y2;
    if (turn && p.interleaved) {  // pair e: values 2e, 2e + 1 of the 16
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float u = 2 * e < 8 ? a[it][(2 * e) & 7] : b[it][(2 * e) & 7];
        const float v = 2 * e < 8 ? a[it][(2 * e + 1) & 7] : b[it][(2 * e + 1) & 7];
        const float ru = u * cs[e] - v * sn[e], rv = v * cs[e] + u * sn[e];
        if (2 * e < 8) {
          y1[(2 * e) & 7] = ru;
          y1[(2 * e + 1) & 7] = rv;
        } else {
          y2[(2 * e) & 7] = ru;
          y2[(2 * e + 1) & 7] = rv;
        }
      }
    } else if (turn) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        y1[e] = a[it][e] * cs[e] - b[it][e] * sn[e];
        y2[e] = b[it][e] * cs[e] + a[it][e] * sn[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        y1[e] = a[it][e];
        y2[e] = b[it][e];
      }
    }
    const bool isk = head[it] >= p.H;
    char* dst = (char*)(isk ? p.ko : p.qo) +
                2 * (row * (size_t)(isk ? p.ko_st : p.qo_st) +
                     (size_t)(isk ? head[it] - p.H : head[it]) * (isk ? p.ko_sh : p.qo_sh));
    if (ok1) *reinterpret_cast<V8*>(dst + 2 * o1) = y1;
    if (ok2) *reinterpret_cast<V8*>(dst + 2 * o2) = y2;
  }
}

template <class V8, bool ROW>
static hipError_t launch_rope_t(const QkRopeArgs& a, int groups, hipStream_t s) {
  // Over the row one workgroup takes all heads; over each head a workgroup takes up to four waves' groups. With
  // rows enough to fill the GPU a wave takes several groups for its angles (16,384 rows of 32 + 8 heads of 128: one
  // group a wave 81, two 74, three 85 us; 3,481 rows of 40 + 40 heads of 64 over the row: 22.8, 20.8, 20.1).
  const int need = ROW ? (groups + kRopeWaves - 1) / kRopeWaves : 1, want = a.T < 512 ? 1 : ROW ? 3 : 2;
  const int nit = need > want ? need : want < groups ? want : groups;
  const int per = (groups + nit - 1) / nit, gy = ROW ? 1 : (per + 3) / 4, waves = (per + gy - 1) / gy;
  const dim3 grid(a.T, gy), block(64 * waves);
  switch (nit) {
    case 1: ESM_LAUNCH((qk_norm_rope_kernel<V8, ROW, 1>), grid, block, 0, s, a); break;
    case 2: ESM_LAUNCH((qk_norm_rope_kernel<V8, ROW, 2>), grid, block, 0, s, a); break;
    case 3: ESM_LAUNCH((qk_norm_rope_kernel<V8, ROW, 3>), grid, block, 0, s, a); break;
    case 4: ESM_LAUNCH((qk_norm_rope_kernel<V8, ROW, 4>), grid, block, 0, s, a); break;
    default: return hipErrorInvalidValue;  // (heads are bounded by the caller)
  }
  return hipGetLastError();
}

static int lanes_log2(int d) {
  int lph = 0;
  while ((16 << lph) < d) lph++;
  return lph;
}

bool qk_norm_rope_row_fits(int heads, int d) { return heads <= (64 >> lanes_log2(d)) * kRopeWaves * 4; }

hipError_t launch_qk_norm_rope(QkRopeArgs a, bool bf16, bool row, hipStream_t s) {
  a.lph = lanes_log2(a.d);
  const int hpw = 64 >> a.lph, groups = (a.H + a.Hk + hpw - 1) / hpw;
  if (bf16) return row ? launch_rope_t<bf16x8, true>(a, groups, s) : launch_rope_t<bf16x8, false>(a, groups, s);
  return row ? launch_rope_t<half8, true>(a, groups, s) : launch_rope_t<half8, false>(a, groups, s);
}

}  // namespace esm
