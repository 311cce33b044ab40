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
// each of the wave's NIT groups of heads. 16,384 rows of 32 + 8 heads of 128 68 us, 4.9 TB/s; 3,481 rows of 40 + 40
// heads of 64 over the row 17.1 us, 4.2 TB/s (vector work bounds it beside the bytes); 8 rows 3.4 us.
#include <type_traits>

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

// kFull: the head's lanes are all filled (d = 16 2^lph), and q and k both have weights or neither has: no lane's values
// or weights are guarded. kPlain: and all turn in the half layout (rot = d). The guards took a third of the instructions,
// which bound the norm over the row (3,481 rows of 40 + 40 heads of 64 19.1 -> 17.1 us).
enum : int { kGuarded = 0, kFull = 1, kPlain = 2 };
template <class V8, bool ROW, int NIT, int FORM>
__global__ __launch_bounds__(64 * kRopeWaves) void qk_norm_rope_kernel(QkRopeArgs p) {
  constexpr bool FULL = FORM != kGuarded, PLAIN = FORM == kPlain;
  __shared__ __align__(16) float red[kRopeWaves][4];
  const size_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int lph = p.lph, hpw = 64 >> lph;             // heads per wave and pass
  const int c = lane & ((1 << lph) - 1), hl = lane >> lph;
  const bool turn = PLAIN || 16 * c < p.rot;
  // the two pieces of this lane: its pairs' first and second values (half layout), or 16 values in a row
  const int o1 = PLAIN || (turn && !p.interleaved) ? 8 * c : 16 * c;
  const int o2 = PLAIN || (turn && !p.interleaved) ? o1 + p.rot / 2 : o1 + 8;
  const bool ok1 = FULL || o1 < p.d, ok2 = FULL || o2 < p.d;
  const int g0 = (blockIdx.y * nw + wave) * NIT;      // first group of heads of this wave

  V8 x1[NIT], x2[NIT];
  int head[NIT], hk[NIT];                             // the lane's head (-1: none), its number among q's or k's
  bool isk[NIT];
#pragma unroll
  for (int it = 0; it < NIT; it++) {
    const int hh = (g0 + it) * hpw + hl, last = p.H + p.Hk - 1;
    head[it] = hh <= last ? hh : -1;
    isk[it] = hh >= p.H;
    hk[it] = min(hh, last) - (isk[it] ? p.H : 0);     // (past the last head: that one again, not counted or stored)
    const char* src = (const char*)(isk[it] ? p.k : p.q) +
                      2 * (row * (size_t)(isk[it] ? p.k_st : p.q_st) + (size_t)hk[it] * (isk[it] ? p.k_sh : p.q_sh));
    if constexpr (FULL) {
      x1[it] = *reinterpret_cast<const V8*>(src + 2 * o1);
      x2[it] = *reinterpret_cast<const V8*>(src + 2 * o2);
    } else {
      x1[it] = x2[it] = V8{};
      if (ok1) x1[it] = *reinterpret_cast<const V8*>(src + 2 * o1);
      if (ok2) x2[it] = *reinterpret_cast<const V8*>(src + 2 * o2);
    }
  }

  // The norm's weights are asked for with the values (16,384 rows of 32 + 8 heads of 128, all turned, 64 -> 62 us); over
  // the row, where a wave takes three groups, they would take the registers of a second workgroup (20 -> 26 us).
  f32x4 wt[ROW ? 1 : NIT][4];
  const bool weighted = p.norm && p.q_w;              // (FULL: k's too)
  const auto weights = [&](int it) {
    f32x4* t = wt[ROW ? 0 : it];
    const float* w = (isk[it] ? p.k_w : p.q_w);
    if constexpr (!FULL) {
      t[0] = t[1] = t[2] = t[3] = f32x4{1.f, 1.f, 1.f, 1.f};  // (no weight: 1)
      if (!p.norm || !w) return;
    } else if (!weighted) {
      return;
    }
    w += (size_t)hk[it] * (isk[it] ? p.kw_sh : p.qw_sh);
    if (ok1) t[0] = *reinterpret_cast<const f32x4*>(w + o1), t[1] = *reinterpret_cast<const f32x4*>(w + o1 + 4);
    if (ok2) t[2] = *reinterpret_cast<const f32x4*>(w + o2), t[3] = *reinterpret_cast<const f32x4*>(w + o2 + 4);
  };
  if constexpr (!ROW)
#pragma unroll
    for (int it = 0; it < NIT; it++) weights(it);

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

  // The values stay in 16 bits until they are turned: in fp32 through the sums they would take twice the registers.
  float off[NIT], rs[NIT];  // y = x rs + off
#pragma unroll
  for (int it = 0; it < NIT; it++) off[it] = 0.f, rs[it] = 1.f;
  if (p.norm) {
    const bool layer = p.norm == kNormLayer;
    const auto sum = [&](int it) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) s += (float)x1[it][e] + (float)x2[it][e];  // (pieces past the head hold zeros)
      return s;
    };
    const auto squares = [&](int it, float m) {
      float s = 0.f, t = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float u = (float)x1[it][e] - m, v = (float)x2[it][e] - m;
        s = fmaf(u, u, s);
        t = fmaf(v, v, t);
      }
      return (ok1 ? s : 0.f) + (ok2 ? t : 0.f);
    };
    if constexpr (ROW) {
      // Over q's and k's rows with one barrier: each wave's mean and its squares about that, joined, a wave a lane, as
      //   mean = sum_w n_w mean_w / n,  M2 = sum_w M2_w + n_w (mean_w - mean)^2
      const auto values_of = [&](int w, int from, int to) {  // how many wave w has of the heads from .. to - 1
        const int a = w * NIT * hpw;
        return (float)(max(0, min(a + NIT * hpw, to) - max(a, from)) * p.d);
      };
      const float nq = values_of(wave, 0, p.H), nk = values_of(wave, p.H, p.H + p.Hk);
      float mq = 0.f, mk = 0.f;
      if (layer) {
        float sq = 0.f, sk = 0.f;
#pragma unroll
        for (int it = 0; it < NIT; it++) {
          const float s = head[it] >= 0 ? sum(it) : 0.f;
          sq += isk[it] ? 0.f : s;
          sk += isk[it] ? s : 0.f;
        }
        mq = wave_total(sq) / fmaxf(nq, 1.f), mk = wave_total(sk) / fmaxf(nk, 1.f);
      }
      float vq = 0.f, vk = 0.f;
#pragma unroll
      for (int it = 0; it < NIT; it++) {
        const float s = head[it] >= 0 ? squares(it, isk[it] ? mk : mq) : 0.f;
        vq += isk[it] ? 0.f : s;
        vk += isk[it] ? s : 0.f;
      }
      vq = wave_total(vq), vk = wave_total(vk);
      if (lane == 0) *reinterpret_cast<f32x4*>(red[wave]) = f32x4{mq, mk, vq, vk};
      __syncthreads();
      const int w = lane & 15;
      f32x4 part = {0.f, 0.f, 0.f, 0.f};
      if (w < nw) part = *reinterpret_cast<const f32x4*>(red[w]);
      const float iq = 1.f / (float)(p.H * p.d), ik = 1.f / (float)(p.Hk * p.d);
      float aq = 0.f, ak = 0.f;
      if (layer) {
        const float cq = values_of(w, 0, p.H), ck = values_of(w, p.H, p.H + p.Hk);
        aq = row16_sum(cq * part[0]) * iq, ak = row16_sum(ck * part[1]) * ik;
        part[2] = fmaf(cq * (part[0] - aq), part[0] - aq, part[2]);
        part[3] = fmaf(ck * (part[1] - ak), part[1] - ak, part[3]);
      }
      const float rq = rsqrtf(row16_sum(part[2]) * iq + p.eps), rk = rsqrtf(row16_sum(part[3]) * ik + p.eps);
#pragma unroll
      for (int it = 0; it < NIT; it++) rs[it] = isk[it] ? rk : rq, off[it] = -(isk[it] ? ak * rk : aq * rq);
    } else {
      const float inv = 1.f / (float)p.d;
#pragma unroll
      for (int it = 0; it < NIT; it++) {
        const float mean = layer ? head_sum(sum(it), lph) * inv : 0.f;
        rs[it] = rsqrtf(head_sum(squares(it, mean), lph) * inv + p.eps);
        off[it] = -mean * rs[it];
      }
    }
  }
#pragma unroll
  for (int it = 0; it < NIT; it++) {
    if (head[it] < 0) continue;
    if constexpr (ROW) weights(it);
    const f32x4* w = wt[ROW ? 0 : it];
    float a[8], b[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      a[e] = fmaf((float)x1[it][e], rs[it], off[it]);
      b[e] = fmaf((float)x2[it][e], rs[it], off[it]);
    }
    if (!FULL || weighted) {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        a[e] *= w[e >> 2][e & 3];
        b[e] *= w[2 + (e >> 2)][e & 3];
      }
    }
    V8 y1, y2;
    if (!PLAIN && turn && p.interleaved) {  // pair e: values 2e, 2e + 1 of the 16
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float u = 2 * e < 8 ? a[(2 * e) & 7] : b[(2 * e) & 7];
        const float v = 2 * e < 8 ? a[(2 * e + 1) & 7] : b[(2 * e + 1) & 7];
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
        y1[e] = a[e] * cs[e] - b[e] * sn[e];
        y2[e] = b[e] * cs[e] + a[e] * sn[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        y1[e] = a[e];
        y2[e] = b[e];
      }
    }
    char* dst = (char*)(isk[it] ? p.ko : p.qo) +
                2 * (row * (size_t)(isk[it] ? p.ko_st : p.qo_st) + (size_t)hk[it] * (isk[it] ? p.ko_sh : p.qo_sh));
    if (ok1) *reinterpret_cast<V8*>(dst + 2 * o1) = y1;
    if (ok2) *reinterpret_cast<V8*>(dst + 2 * o2) = y2;
  }
}

template <class V8, bool ROW, int FORM>
static hipError_t launch_rope_t(const QkRopeArgs& a, int groups, hipStream_t s) {
  // Over the row one workgroup takes all heads; over each head a workgroup takes up to four waves' groups. With
  // rows enough to fill the GPU a wave takes several groups for its angles, three over the row or where that leaves fewer
  // idle than two (us for 1, 2, 3: 16,384 rows of 32 + 8 heads of 128, half turned 76, 70, 69, all turned 69, 62, 60; of 20 + 4
  // heads of 80 29.4, 30.1, 27.5; 3,481 rows of 40 + 40 heads of 64 over the row 20.7, 18.5, 17.1).
  const int need = ROW ? (groups + kRopeWaves - 1) / kRopeWaves : 1;
  const int want = a.T < 512 ? 1 : ROW || (groups + 2) / 3 * 3 < (groups + 1) / 2 * 2 ? 3 : 2;
  const int nit = need > want ? need : want < groups ? want : groups;
  const int per = (groups + nit - 1) / nit, gy = ROW ? 1 : (per + 3) / 4, waves = (per + gy - 1) / gy;
  const dim3 grid(a.T, gy), block(64 * waves);
  switch (nit) {
    case 1: ESM_LAUNCH((qk_norm_rope_kernel<V8, ROW, 1, FORM>), grid, block, 0, s, a); break;
    case 2: ESM_LAUNCH((qk_norm_rope_kernel<V8, ROW, 2, FORM>), grid, block, 0, s, a); break;
    case 3: ESM_LAUNCH((qk_norm_rope_kernel<V8, ROW, 3, FORM>), grid, block, 0, s, a); break;
    case 4: ESM_LAUNCH((qk_norm_rope_kernel<V8, ROW, 4, FORM>), grid, block, 0, s, a); break;
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
  const bool full = a.d == 16 << a.lph && (!a.norm || !a.q_w == !a.k_w), plain = full && a.rot == a.d && !a.interleaved;
  const auto launch = [&](auto v, auto r) {
    typedef decltype(v) V8;
    constexpr bool ROW = decltype(r)::value;
    if (plain) return launch_rope_t<V8, ROW, kPlain>(a, groups, s);
    return full ? launch_rope_t<V8, ROW, kFull>(a, groups, s) : launch_rope_t<V8, ROW, kGuarded>(a, groups, s);
  };
  if (bf16) return row ? launch(bf16x8{}, std::true_type{}) : launch(bf16x8{}, std::false_type{});
  return row ? launch(half8{}, std::true_type{}) : launch(half8{}, std::false_type{});
}

}  // namespace esm
