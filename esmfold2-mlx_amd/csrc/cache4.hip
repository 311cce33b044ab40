// Keys and values in 4 bits, in pages of 64 keys, and the attention that reads them.
//
// x ~ s (c - z) per key (or value) and group of 64 values of a head: s the least bf16 value, 2^-96 or more, of which 15 reach
// over the group's range and 120 to its farthest value from zero; z = rint(-min / s), c = clamp(rint(x / s) + z, 0, 15). A
// group that holds a NaN or an infinity, or whose range passes fp32, reads as NaN (s is).
//
// The matrix cores take codes as they are: in bf16 0x4180 | c << 3 is 16 + c, in fp16 0x4c00 | c << 6, one instruction for
// two codes and a shift. Products with 16 + c and with -(16 + z) cancel in fp32, and s multiplies what comes out (keys) or the
// probability that goes in (values):
//   S^T[key][row] = sum_g s_kg (sum_d (16 + c_kd) q_d - (16 + z_kg) Q_g),  Q_g = sum_d q_d
//   O^T[d][row]  += sum_k (16 + c_kd) P_kg - (16 + z_kg) P_kg,             P_kg = p_k s_kg, rounded
// both by v_mfma_f32_16x16x32: a wave holds 16 rows of queries (or RT times 16), a row a lane (lane % 16) of every
// accumulator, and takes 32 keys at a time. P is bf16 whatever the type, as its range is p's times the values', and kept as the
// sum of two bf16 values, 16 bits of it: with the first alone bf16's output was off by 0.0023 of itself on long contexts,
// where its own rounding is 0.0017 (the second costs 4 to 8% of a token's time, 24 to 31% of a prompt's). No operand passes
// through LDS: the cache lies in the order the matrix cores take (HD = 64 or 128, the head size filled up). A page's head is
// 8 chunks of 8 keys, one after the other, so that whoever writes 8 keys writes whole lines of memory; key 4 b + e of chunk g is row 4 g + e of block b of the 32 keys' first
// product, and slot 4 b + e of lane group g in the second:
//   key codes    [2 b][4 lane groups][4 e][HD / 8 bytes]: lane group l's dword t: dims 32 t + 8 l + {0 .. 7}, the dword's nibble i
//                dim 2 i, nibble 4 + i dim 2 i + 1
//   value codes  [HD / 64][16 dims][16 bytes]: a byte is one key's dims 32 p + row (low) and 16 more (high), 8 bytes a pair p of
//                the two; key 4 b + e is byte {0, 2, 1, 3}[e] of dword b
//   key steps    [2 b][groups of 64 values][4 e] words s << 16 | 16 + z (in the type's own 16 bits)
//   value steps  [groups][8 keys] s (bf16), then the same of -(16 + z) (bf16)
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace esm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// Bytes of 8 keys of a page and head, and of their parts.
template <int HD>
struct Page {
  static constexpr int kGroups = HD / 64, kCodes = 8 * HD / 2, kSteps = 8 * kGroups * 4;
  static constexpr int kValCodesAt = kCodes, kKeyStepsAt = 2 * kCodes, kValStepsAt = kKeyStepsAt + kSteps;
  static constexpr int kChunk = kValStepsAt + kSteps, kBytes = 8 * kChunk;
};
static_assert(Page<64>::kBytes == cache4_page_bytes(64) && Page<128>::kBytes == cache4_page_bytes(128), "a page's size");

DEV uint32_t bf16_bits(float v) { return __builtin_bit_cast(uint32_t, v) >> 16; }  // (of values that bf16 holds)

// ---- writing ------------------------------------------------------------------------------------
// rint(x / s) without a division, of which eight a lane would bound the writing. x has at most 11 binary places and s 8, so x /
// s lies on k + 1/2 or 2^-12 from it at least; x inv, off by 2^-22 of itself, |x / s| <= 120, is first rounded to 2^-13, which
// leaves a tie a tie and nothing else one, then to the even whole number. Both roundings are those of an addition that leaves the
// whole number in the low bits of its result.
constexpr float kWhole = 12582912.f;  // 1.5 2^23
DEV float whole_steps(float x, float inv13) {  // inv13: 2^13 / s; the number is the result's distance from kWhole
  const float n = fmaf(x, inv13, kWhole) - kWhole;
  return fmaf(n, 0x1p-13f, kWhole);
}
// Step and zero of a group from its least and largest value (apart by infinity where it holds a NaN or an infinity: s is NaN).
DEV void four_bit_step(float lo, float hi, float& s, float& inv13, float& z) {
  const float far = fmaxf(fabsf(lo), fabsf(hi)), range = hi - lo;
  const auto reaches = [&](float t) { return (15.f * t >= range) & (120.f * t >= far) & (t >= 0x1p-96f); };
  uint32_t b = __builtin_bit_cast(uint32_t, fmaxf(fmaxf(range * (1.f / 15.f), far * (1.f / 120.f)), 0x1p-96f)) & 0xffff0000u;
  // (the products may be off by a step of fp32 either way)
  const bool less = reaches(__builtin_bit_cast(float, b - 0x10000u)), enough = reaches(__builtin_bit_cast(float, b));
  b = less ? b - 0x10000u : enough ? b : b + 0x10000u;
  s = __builtin_bit_cast(float, b);
  inv13 = __builtin_amdgcn_rcpf(s) * 0x1p13f;
  z = whole_steps(-lo, inv13) - kWhole;
  if (!(range < INFINITY)) s = __builtin_bit_cast(float, 0x7fc00000u), inv13 = 0.f, z = 0.f;
}
// 8 values' codes, a byte each.
DEV void eight_codes(const float (&v)[8], float inv13, float z, uint32_t (&bytes)[2]) {
  const int zero = __builtin_bit_cast(int, kWhole), zi = (int)z;
  int u[8];
#pragma unroll
  for (int e = 0; e < 8; e++) u[e] = min(max(__builtin_bit_cast(int, whole_steps(v[e], inv13)) + zi, zero), zero + 15);
#pragma unroll
  for (int i = 0; i < 2; i++) {  // (the low bytes of four)
    const uint32_t a = __builtin_amdgcn_perm(u[4 * i + 1], u[4 * i], 0x0c0c0400u), b = __builtin_amdgcn_perm(u[4 * i + 3], u[4 * i + 2], 0x04000c0cu);
    bytes[i] = a | b;
  }
}

// Eight keys of a sequence that make a chunk of a page (those at the ends of the call's rows may be of other calls): key k's
// row is row + k for from <= k < to. page: -1 where it is none of the cache's, or the rows stand before the sequence's first
// place or behind its table, or in no sequence.
struct Eight {
  int row, from, to, page, chunk;
};
// Groups there may be of T rows in n sequences: a sequence's first and last may be incomplete, so may those of no sequence.
static long long eight_groups(long long T, int n) { return T / 8 + 2LL * n + 4; }
DEV bool find_eight(const Cache4Args& p, int what, int lane, Eight& f) {
  int before = 0, end = 0, start = 0;
  for (int i0 = 0; i0 < p.n; i0 += 64) {
    const int i = min(i0 + lane, p.n - 1);
    const int a = min(max(p.cu[i], 0), p.T), nq = min(max(p.cu[i + 1], a), p.T) - a;
    const long long first = (long long)p.lens[i] - nq, lead = first & 7;  // (may be negative)
    const int groups = i0 + lane < p.n && nq > 0 ? (int)((lead + nq + 7) >> 3) : 0, sum = wave_scan(groups);
    const uint64_t hit = __ballot(what < before + sum);
    if (hit) {
      const int w = __builtin_ctzll(hit), seq = i0 + w;
      const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, w); };
      const int g = what - before - of(sum - groups), nqw = of(nq), leadw = of((int)lead);
      const long long pos = (((long long)of((int)(first >> 32)) << 32) | (uint32_t)of((int)first)) - leadw + 8LL * g;
      f.row = of(a) - leadw + 8 * g;
      f.from = max(0, leadw - 8 * g);
      f.to = min(8, leadw + nqw - 8 * g);
      f.page = -1;
      f.chunk = (int)(pos & 63) >> 3;
      if (pos >= 0 && pos < (long long)p.width * kCache4Page) f.page = p.table[(size_t)seq * p.width + (pos >> 6)];
      if (f.page < 0 || f.page >= p.pages) f.page = -1;
      return g >= 0 && f.row + f.from >= 0 && f.row + f.to <= p.T;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    if (i0 == 0) start = __builtin_amdgcn_readlane(a, 0);
    end = __builtin_amdgcn_readlane(a + nq, 63);
  }
  // rows of no sequence: behind the last, then before the first
  int g = what - before;
  f.page = -1, f.chunk = 0, f.from = 0;
  f.row = end + 8 * g;
  f.to = min(8, p.T - f.row);
  if (f.to > 0) return g >= 0;
  f.row = 8 * (g - (p.T - end + 7) / 8);
  f.to = min(8, start - f.row);
  return f.row >= 0 && f.to > 0;
}

// A wave takes the eight keys (or their values) of 64 / (HD / 2) heads, four at a time: HD / 8 lanes a key, a lane 8 of its
// values.
template <int HD>
struct EightLanes {
  static constexpr int kLanes = HD / 8, kHeads = 64 / (4 * kLanes);
  int c, k, item;  // 8 values of keys k and 4 + k of an item (the keys' heads, then the values')
  DEV EightLanes(int lane) : c(lane % kLanes), k(lane / kLanes & 3), item((blockIdx.y * 4 + (threadIdx.x >> 6)) * kHeads + lane / (4 * kLanes)) {}
  DEV bool in(const Eight& f, int b) const { return 4 * b + k >= f.from && 4 * b + k < f.to; }
  // The wave's next item, of those that a group's workgroups deal among them.
  DEV bool next(int items) {
    item += 4 * gridDim.y * kHeads;
    return __builtin_amdgcn_readfirstlane(item) < items;
  }
  // Bytes of 8 dims (a, b: 4 each) of one key a lane, to two dims (x, y) of the four keys a lane, 2 k and 2 k + 1 of the 8, in
  // the order of a value dword (keys 0, 2, 1, 3); and back. Exchanges with the lanes of keys k ^ 2 and k ^ 1.
  DEV void gather(uint32_t a, uint32_t b, uint32_t& x, uint32_t& y) const {
    const bool up = k & 2, odd = k & 1;
    const uint32_t v = __shfl_xor(up ? a : b, 2 * kLanes);
    const uint32_t m = up ? v : a, n = up ? b : v;  // four dims of keys k % 2 and k % 2 + 2
    const uint32_t lo = (m & 0xffff) | (n << 16), hi = (m >> 16) | (n & 0xffff0000u);
    const uint32_t w = __shfl_xor(odd ? lo : hi, kLanes);
    const uint32_t r = odd ? w : lo, q = odd ? hi : w;  // two dims of keys 0 and 2, of 1 and 3
    x = __builtin_amdgcn_perm(q, r, 0x06040200u);
    y = __builtin_amdgcn_perm(q, r, 0x07050301u);
  }
  DEV void scatter(uint32_t x, uint32_t y, uint32_t& a, uint32_t& b) const {
    const bool up = k & 2, odd = k & 1;
    const uint32_t r = __builtin_amdgcn_perm(y, x, 0x05010400u), q = __builtin_amdgcn_perm(y, x, 0x07030602u);
    const uint32_t w = __shfl_xor(odd ? r : q, kLanes);
    const uint32_t lo = odd ? w : r, hi = odd ? q : w;
    const uint32_t m = (lo & 0xffff) | (hi << 16), n = (lo >> 16) | (hi & 0xffff0000u);
    const uint32_t v = __shfl_xor(up ? m : n, 2 * kLanes);
    a = up ? v : m;
    b = up ? n : v;
  }
};
template <int N>
DEV uint32_t lanes_on(uint32_t v) {  // of the lane N further in the 16
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x100 + N, 0xf, 0xf, true);  // row_shl:N (past the 16: 0)
}

// One item of a wave: x, the lane's 8 values of either key, to their places. Where all eight keys are new, lanes join what
// lies together and write 8 and 16 bytes.
template <class V8, int HD>
DEV void hold_eight(const Cache4Args& p, const Eight& f, const EightLanes<HD>& at, const V8 (&x)[2]) {
  typedef Page<HD> P;
  const int c = at.c, g = c >> 3;  // group
  const bool val = at.item >= p.Hk, live = at.item < 2 * p.Hk, all = f.from == 0 && f.to == 8;
  const int h = live ? at.item - (val ? p.Hk : 0) : 0;
  char* chunk = (char*)p.data + ((size_t)f.page * p.Hk + h) * P::kBytes + f.chunk * P::kChunk;
  uint32_t own[2][2], joined[2][2], x4[2], y4[2];
  float s[2], z[2];
#pragma unroll
  for (int b = 0; b < 2; b++) {
    const bool in = live && at.in(f, b) && 8 * c < p.d;
    float v[8], lo = INFINITY, hi = -INFINITY, inv;
#pragma unroll
    for (int e = 0; e < 8; e++) {  // (NaN stays)
      v[e] = (float)x[b][e];
      lo = __builtin_elementwise_minimum(lo, v[e]);
      hi = __builtin_elementwise_maximum(hi, v[e]);
    }
    if (!in) lo = INFINITY, hi = -INFINITY;
    const auto over = [&](auto ctrl) {
      const auto other = [&](float t) {
        return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, t), decltype(ctrl)::value, 0xf, 0xf, true));
      };
      lo = __builtin_elementwise_minimum(lo, other(lo)), hi = __builtin_elementwise_maximum(hi, other(hi));
    };
    over(std::integral_constant<int, 0xB1>{});   // quad_perm(1, 0, 3, 2)
    over(std::integral_constant<int, 0x4E>{});   // quad_perm(2, 3, 0, 1)
    over(std::integral_constant<int, 0x141>{});  // row_half_mirror: 8 lanes, a group
    if (lo > hi) lo = hi = 0.f;  // (a group past the head's values)
    four_bit_step(lo, hi, s[b], inv, z[b]);
    eight_codes(v, inv, z[b], own[b]);
  }
  if (__any(val)) {  // a lane of low nibbles (c / 2 even) joins the high ones of the lane two further: 8 dims of a pair
#pragma unroll
    for (int b = 0; b < 2; b++) {
#pragma unroll
      for (int i = 0; i < 2; i++) joined[b][i] = own[b][i] | lanes_on<2>(own[b][i]) << 4;
      if (all) at.gather(joined[b][0], joined[b][1], x4[b], y4[b]);
    }
  }
  uint32_t xn[2], yn[2];  // the second pair's
  if (all && __any(val)) {
#pragma unroll
    for (int b = 0; b < 2; b++) xn[b] = lanes_on<4>(x4[b]), yn[b] = lanes_on<4>(y4[b]);
  }
  uint32_t w[2][HD / 32];
#pragma unroll
  for (int b = 0; b < 2; b++) {  // dims 0, 2, 4, 6 in the low half's nibbles, 1, 3, 5, 7 in the high half's
    const uint32_t p0 = own[b][0] | own[b][0] >> 12, p1 = own[b][1] | own[b][1] >> 12;  // (bytes: 0 and 2, 1 and 3, ...)
    w[b][0] = __builtin_amdgcn_perm(p1, p0, 0x05010400u);
    w[b][1] = lanes_on<4>(w[b][0]);
    if constexpr (HD == 128) w[b][2] = lanes_on<8>(w[b][0]), w[b][3] = lanes_on<12>(w[b][0]);
  }
  if (!live) return;
  if (!val) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
      // dims 8 c = 32 (c / 4) + 8 (c % 4)
      char* dst = chunk + ((b * 4 + (c & 3)) * 4 + at.k) * (HD / 8);
      if (all) {
        if (c < 4) {
          if constexpr (HD == 128) {
            *reinterpret_cast<u32x4*>(dst) = u32x4{w[b][0], w[b][1], w[b][2], w[b][3]};
          } else {
            *reinterpret_cast<u32x2*>(dst) = u32x2{w[b][0], w[b][1]};
          }
        }
      } else if (at.in(f, b)) {
        *reinterpret_cast<uint32_t*>(dst + 4 * (c >> 2)) = w[b][0];
      }
      if ((c & 7) == 0 && at.in(f, b)) {
        const uint32_t zb = std::is_same<V8, bf16x8>::value ? bf16_bits(16.f + z[b])
                                                            : (uint32_t)__builtin_bit_cast(uint16_t, (half_t)(16.f + z[b]));
        *reinterpret_cast<uint32_t*>(chunk + P::kKeyStepsAt + ((b * P::kGroups + g) * 4 + at.k) * 4) =
            (__builtin_bit_cast(uint32_t, s[b]) & 0xffff0000u) | zb;
      }
    }
    return;
  }
  if (!(c & 2)) {
    const int pair = c >> 2, dim = 8 * (c & 1);  // of the pair's low 16
    char* dst = chunk + P::kValCodesAt + ((pair >> 1) * 16 + dim) * 16 + 8 * (pair & 1);
    if (all) {
      if (!(pair & 1)) {
        *reinterpret_cast<u32x4*>(dst + 16 * (2 * at.k)) = u32x4{x4[0], x4[1], xn[0], xn[1]};
        *reinterpret_cast<u32x4*>(dst + 16 * (2 * at.k + 1)) = u32x4{y4[0], y4[1], yn[0], yn[1]};
      }
    } else {
      const int byte = (0x3120 >> (4 * at.k)) & 3;
#pragma unroll
      for (int b = 0; b < 2; b++)
        if (at.in(f, b))
#pragma unroll
          for (int e = 0; e < 8; e++) dst[16 * e + 4 * b + byte] = (char)(joined[b][e >> 2] >> (8 * (e & 3)));
    }
  }
  if ((c & 7) == 0) {
    uint16_t* st = reinterpret_cast<uint16_t*>(chunk + P::kValStepsAt) + 8 * g + at.k;
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (at.in(f, b)) {
        st[4 * b] = (uint16_t)(__builtin_bit_cast(uint32_t, s[b]) >> 16);
        st[8 * P::kGroups + 4 * b] = (uint16_t)bf16_bits(-(16.f + z[b]));
      }
  }
}
// With rows enough to fill the GPU one workgroup takes all heads of its eight keys, the next one's values asked for before this
// one's work: 8,287 rows of 8 heads of 128 in 16.5 us, 43 MB, bound by its 22 vector instructions a value of a lane (with 30 18.0,
// with divisions, and a branch for their ties, 23 us however the codes were stored). 64 single tokens 4.1 us: a launch and the
// latencies of starts, table and rows.
template <class V8, int HD>
__global__ __launch_bounds__(256) void cache4_write_kernel(Cache4Args p) {
  const int lane = threadIdx.x & 63;
  Eight f;
  if (!find_eight(p, blockIdx.x, lane, f) || f.page < 0) return;
  EightLanes<HD> at(lane);
  if (__builtin_amdgcn_readfirstlane(at.item) >= 2 * p.Hk) return;
  V8 x[2];
  const char *kr[2], *vr[2];  // this lane's part of the rows' first heads
  bool in[2];
#pragma unroll
  for (int b = 0; b < 2; b++) {
    in[b] = at.in(f, b) && 8 * at.c < p.d;
    const long long row = in[b] ? f.row + 4 * b + at.k : 0;
    kr[b] = (const char*)p.k + 2 * (row * p.k_st + 8 * at.c);
    vr[b] = (const char*)p.v + 2 * (row * p.v_st + 8 * at.c);
  }
  const auto load = [&]() {
    const bool val = at.item >= p.Hk;
    const long long head = 2 * (long long)(at.item - (val ? p.Hk : 0)) * (val ? p.v_sh : p.k_sh);
#pragma unroll
    for (int b = 0; b < 2; b++) {
      x[b] = V8{};
      if (in[b] && at.item < 2 * p.Hk) x[b] = *reinterpret_cast<const V8*>((val ? vr[b] : kr[b]) + head);
    }
  };
  load();
  for (bool more = true; more;) {
    const EightLanes<HD> now = at;
    const V8 y[2] = {x[0], x[1]};
    more = at.next(2 * p.Hk);
    if (more) load();
    hold_eight<V8, HD>(p, f, now, y);
  }
}

// What the rows' places hold, as 16-bit values (rounded once): the inverse of the above. Rows without a place are 0. The
// same 8,287 rows 10.9 us, 4 TB/s, bound by memory.
template <class V8, int HD>
DEV void give_four(const Cache4Args& p, const Eight& f, const EightLanes<HD>& at, int b) {
  typedef Page<HD> P;
  const int c = at.c, g = c >> 3;
  const bool val = at.item >= p.Hk, live = at.item < 2 * p.Hk, mine = live && at.in(f, b) && 8 * c < p.d;
  const int h = live ? at.item - (val ? p.Hk : 0) : 0;
  V8* dst = reinterpret_cast<V8*>((uint16_t*)(val ? p.vo : p.ko) + ((size_t)(mine ? f.row + 4 * b + at.k : 0) * p.Hk + h) * p.d + (mine ? 8 * c : 0));
  if (f.page < 0) {
    if (mine) *dst = V8{};
    return;
  }
  const char* chunk = (const char*)p.data + ((size_t)f.page * p.Hk + h) * P::kBytes + f.chunk * P::kChunk;
  float s, z;
  uint32_t code[8];
  if (val) {  // (a head's lanes exchange their bytes)
    const int pair = c >> 2, dim = 8 * (c & 1);
    const char* src = chunk + P::kValCodesAt + ((pair >> 1) * 16 + dim) * 16 + 8 * (pair & 1) + 4 * b;
    uint32_t bytes[2];
    at.scatter(*reinterpret_cast<const uint32_t*>(src + 16 * (2 * at.k)), *reinterpret_cast<const uint32_t*>(src + 16 * (2 * at.k + 1)),
               bytes[0], bytes[1]);  // (the lanes of high nibbles read the same bytes)
#pragma unroll
    for (int e = 0; e < 8; e++) code[e] = (bytes[e >> 2] >> (8 * (e & 3) + 2 * (c & 2))) & 15;
    const uint16_t* st = reinterpret_cast<const uint16_t*>(chunk + P::kValStepsAt) + 8 * g + 4 * b + at.k;
    s = __builtin_bit_cast(float, (uint32_t)st[0] << 16);
    z = -__builtin_bit_cast(float, (uint32_t)st[8 * P::kGroups] << 16) - 16.f;
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(chunk + ((b * 4 + (c & 3)) * 4 + at.k) * (HD / 8) + 4 * (c >> 2));
#pragma unroll
    for (int e = 0; e < 8; e++) code[e] = (w >> (4 * (e >> 1) + 16 * (e & 1))) & 15;
    const uint32_t st = *reinterpret_cast<const uint32_t*>(chunk + P::kKeyStepsAt + ((b * P::kGroups + g) * 4 + at.k) * 4);
    s = __builtin_bit_cast(float, st & 0xffff0000u);
    z = std::is_same<V8, bf16x8>::value ? __builtin_bit_cast(float, st << 16) - 16.f
                                        : (float)__builtin_bit_cast(half_t, (uint16_t)st) - 16.f;
  }
  if (!mine) return;
  V8 y;
#pragma unroll
  for (int e = 0; e < 8; e++) y[e] = (decltype(+y[e]))(s * ((float)code[e] - z));
  *dst = y;
}
template <class V8, int HD>
__global__ __launch_bounds__(256) void cache4_read_kernel(Cache4Args p) {
  const int lane = threadIdx.x & 63;
  Eight f;
  if (!find_eight(p, blockIdx.x, lane, f)) return;
  EightLanes<HD> at(lane);
  if (__builtin_amdgcn_readfirstlane(at.item) >= 2 * p.Hk) return;
  do {
#pragma unroll
    for (int b = 0; b < 2; b++)
      if (4 * b < f.to && 4 * b + 4 > f.from) give_four<V8, HD>(p, f, at, b);
  } while (at.next(2 * p.Hk));
}

// ---- attention --------------------------------------------------------------------------------------
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
struct F16Keys {
  typedef half8 v8;
  typedef half4 v4;
  typedef half_t elem;
  static constexpr uint32_t kMask = 0x03c003c0u, kMagic = 0x4c004c00u;
  static constexpr int kUp = 6;      // a code's place in the 16 bits
  static DEV f32x4 mfma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static DEV float zero_of(uint32_t w) { return (float)__builtin_bit_cast(half_t, (uint16_t)w); }
};
struct B16Keys {
  typedef bf16x8 v8;
  typedef bf16x4 v4;
  typedef __bf16 elem;
  static constexpr uint32_t kMask = 0x00780078u, kMagic = 0x41804180u;
  static constexpr int kUp = 3;
  static DEV f32x4 mfma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static DEV float zero_of(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
};
DEV f32x4 mfma_b16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// Mask and exponent that make 16 + c of a code, in registers of their own (hidden from the compiler, which would otherwise
// write them into a v_and and a v_or instead of one v_and_or).
template <uint32_t MASK, uint32_t MAGIC>
struct Unpack {
  uint32_t mask, magic;
  DEV Unpack() : mask(MASK), magic(MAGIC) {
    __asm__ volatile("" : "+s"(mask));
    __asm__ volatile("" : "+v"(magic));
  }
  // The two codes at bits AT of each half of w; UP: a code's place in the 16 bits.
  template <int AT, int UP>
  DEV uint32_t two(uint32_t w) const {
    return ((AT > UP ? w >> (AT > UP ? AT - UP : 0) : w << (UP > AT ? UP - AT : 0)) & mask) | magic;
  }
};
typedef Unpack<B16Keys::kMask, B16Keys::kMagic> UnpackB;
template <class T, class U>
DEV typename T::v8 key_codes(const U& u, uint32_t w) {
  return __builtin_bit_cast(typename T::v8, u32x4{u.template two<0, T::kUp>(w), u.template two<4, T::kUp>(w), u.template two<8, T::kUp>(w),
                                                  u.template two<12, T::kUp>(w)});
}
template <bool HIGH>
DEV bf16x8 value_codes(const UnpackB& u, uint32_t a, uint32_t b) {  // slots 0 .. 3 and 4 .. 7 of the pair's low or high dims
  constexpr int A = HIGH ? 4 : 0;
  return __builtin_bit_cast(bf16x8, u32x4{u.two<A, 3>(a), u.two<A + 8, 3>(a), u.two<A, 3>(b), u.two<A + 8, 3>(b)});
}

// Largest and sum over the four lanes that hold a row (those of one lane % 16).
DEV float row_max4(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
DEV float row_sum4(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// A work item is a (sequence, tile of 16 RT rows, chunk of keys) of one key head; chunks are as many whole passes of 256 keys
// as spread all sequences' keys over p.target workgroups of a head. Each workgroup, and the join, finds the same from the
// lengths on the device, so that lengths may change between two replays of one graph.
constexpr int kPass = 4 * kCache4Page;  // keys of a workgroup's pass, a page a wave
struct Item {
  int seq, q0, nq, nk, tile, chunk, chunks, keys, slot;  // keys: of a chunk; slot: where its partials go
};
template <bool BY_ROW>  // what: the item's number, or a row of q (then tile, chunk and slot are the caller's to find)
DEV bool find_item4(const Cache4Args& p, int rows, int what, int lane, Item& it) {
  const int most = p.width * kCache4Page;
  const auto spans = [&](int i0, int& a, int& nq, int& nk, int& tiles) {
    const int i = min(i0 + lane, p.n - 1);
    a = min(max(p.cu[i], 0), p.T);
    nq = min(max(p.cu[i + 1], a), p.T) - a;
    nk = min(max(p.lens[i], 0), most);
    tiles = i0 + lane < p.n ? (nq * p.G + rows - 1) / rows : 0;
  };
  int a, nq, nk, tiles;
  it.keys = 1 << 30;
  spans(0, a, nq, nk, tiles);
  if (p.divide) {
    float passes = 0.f;  // (whole numbers below 2^24, or so many that a few do not count)
    for (int i0 = 0;;) {
      passes += wave_total((float)tiles * (float)((nk + kPass - 1) / kPass));
      if ((i0 += 64) >= p.n) break;
      spans(i0, a, nq, nk, tiles);
    }
    // (two passes at least, and a 256th of the longest there may be: kCache4MaxChunks)
    it.keys = kPass * max(max(2, (int)ceilf(passes / (float)p.target)), (most + kPass * kCache4MaxChunks - 1) / (kPass * kCache4MaxChunks));
    if (p.n > 64) spans(0, a, nq, nk, tiles);
  }
  int before = 0;
  for (int i0 = 0;;) {
    const int chunks = max(1, (nk + it.keys - 1) / it.keys), items = tiles * chunks, sum = wave_scan(items);
    const uint64_t hit = __ballot(BY_ROW ? i0 + lane < p.n && what >= a && what < a + nq : what < before + sum);
    if (hit) {
      const int w = __builtin_ctzll(hit);
      const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, w); };
      it.seq = i0 + w, it.q0 = of(a), it.nq = of(nq), it.nk = of(nk), it.chunks = of(chunks);
      it.slot = before + of(sum - items);
      if (!BY_ROW) {
        const int at = what - it.slot;
        it.tile = at / it.chunks, it.chunk = at - it.tile * it.chunks;
        it.slot = what;
        return at >= 0 && it.tile < of(tiles);  // (starts that do not ascend: nothing outside)
      }
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    if ((i0 += 64) >= p.n) return false;
    spans(i0, a, nq, nk, tiles);
  }
}

constexpr float kFar4 = 1024.f;   // least exponent of a row's maximum that its scores are made relative to
constexpr float kGrow4 = 8.f;     // log2: what p may reach before its row is rescaled

template <class T, int HD, int RT>
struct Rows4 {
  typedef typename T::v8 v8;
  static constexpr int G = HD / 64;
  v8 q[RT][HD / 32];
  float qs[RT][G];       // sums of a group's query values
  f32x4 o[RT][HD / 16];  // lane: row lane % 16, dims 16 i + 4 (lane / 16) + e
  float m[RT], l[RT];    // running maximum of the unscaled scores, this lane's part of the sum
  Unpack<T::kMask, T::kMagic> ku;
  UnpackB vu;
  int lim[RT];           // last key the row sees

  // 32 keys' operands of this lane.
  struct Keys {
    uint32_t kc[2][HD / 32], vc[HD / 16];
    u32x4 ks[2][G], vs[G], vz[G];
  };
  static DEV void load_keys(Keys& k, const char* page, int half, int lane) {
    typedef Page<HD> P;
    const int g = lane >> 4, r = lane & 15;
    const char* codes = page + (4 * half + (r >> 2)) * P::kChunk + (4 * g + (r & 3)) * (HD / 8);
    const char* steps = page + (4 * half + g) * P::kChunk + P::kKeyStepsAt;
#pragma unroll
    for (int b = 0; b < 2; b++) {
      if constexpr (HD == 128) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(codes + 2 * HD * b);
#pragma unroll
        for (int t = 0; t < 4; t++) k.kc[b][t] = v[t];
      } else {
        const u32x2 v = *reinterpret_cast<const u32x2*>(codes + 2 * HD * b);
        k.kc[b][0] = v[0], k.kc[b][1] = v[1];
      }
#pragma unroll
      for (int i = 0; i < G; i++) k.ks[b][i] = *reinterpret_cast<const u32x4*>(steps + (b * G + i) * 16);
    }
  }
  static DEV void load_values(Keys& k, const char* page, int half, int lane) {
    typedef Page<HD> P;
    const char* chunk = page + (4 * half + (lane >> 4)) * P::kChunk;
#pragma unroll
    for (int i = 0; i < G; i++) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(chunk + P::kValCodesAt + (16 * i + (lane & 15)) * 16);
#pragma unroll
      for (int t = 0; t < 4; t++) k.vc[4 * i + t] = v[t];
      k.vs[i] = *reinterpret_cast<const u32x4*>(chunk + P::kValStepsAt + 16 * i);
      k.vz[i] = *reinterpret_cast<const u32x4*>(chunk + P::kValStepsAt + 16 * (G + i));
    }
  }

  DEV void grow(int r, float mx, float c) {
    const float mn = fmaxf(m[r], mx), ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f((m[r] - ref) * c);
    m[r] = mn;
    l[r] *= alpha;
#pragma unroll
    for (int i = 0; i < HD / 16; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) o[r][i][e] *= alpha;
  }

  // The 32 keys from key0 of the sequence on; MASKED: some row may not see some of them. Unseen keys may hold anything. The
  // registers of keys, then of values, take the next 32 keys' (`next`, `half`) as soon as they have been read.
  template <bool MASKED>
  DEV void step(Keys& k, int key0, float c, int lane, const char* next, int half) {
    const int g = lane >> 4;
    f32x4 s[RT][2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
      if (b) __builtin_amdgcn_sched_barrier(0);
      f32x4 acc[RT][G];
#pragma unroll
      for (int t = 0; t < HD / 32; t++) {
        const v8 kc = key_codes<T>(ku, k.kc[b][t]);
#pragma unroll
        for (int r = 0; r < RT; r++) acc[r][t >> 1] = T::mfma(kc, q[r][t], t & 1 ? acc[r][t >> 1] : f32x4{0.f, 0.f, 0.f, 0.f});
      }
#pragma unroll
      for (int r = 0; r < RT; r++) s[r][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < G; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t w = k.ks[b][i][e];
          const float st = __builtin_bit_cast(float, w & 0xffff0000u), z = T::zero_of(w);
#pragma unroll
          for (int r = 0; r < RT; r++) s[r][b][e] = fmaf(st, fmaf(-z, qs[r][i], acc[r][i][e]), s[r][b][e]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_keys(k, next, half, lane);
    __builtin_amdgcn_sched_barrier(0);
    if (MASKED) {
#pragma unroll
      for (int r = 0; r < RT; r++)
#pragma unroll
        for (int j = 0; j < 8; j++)
          s[r][j >> 2][j & 3] = key0 + 8 * g + j <= lim[r] ? s[r][j >> 2][j & 3] : -INFINITY;
    }
    float p[RT][8];
#pragma unroll
    for (int r = 0; r < RT; r++) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; j++) mx = fmaxf(mx, s[r][j >> 2][j & 3]);
      if (__any((mx - m[r]) * c > kGrow4)) grow(r, row_max4(mx), c);
      const float mc = m[r] * c;
      const bool far = !(fabsf(mc) < kFar4);
      float base = mc;
      if (__any(far)) {  // (see packed.hip: large exponents, and rows that have seen nothing)
        const float ref = far && m[r] != -INFINITY ? m[r] : 0.f;
        base = far ? 0.f : mc;
#pragma unroll
        for (int j = 0; j < 8; j++) s[r][j >> 2][j & 3] -= ref;
      }
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        p[r][j] = __builtin_amdgcn_exp2f(fmaf(s[r][j >> 2][j & 3], c, -base));
        sum += p[r][j];
      }
      l[r] += sum;
    }
#pragma unroll
    for (int i = 0; i < G; i++) {
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 hi[RT], lo[RT];
#pragma unroll
      for (int r = 0; r < RT; r++) {
        u32x4 h4, l4;  // (two values a conversion)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const uint32_t w = k.vs[i][j >> 1];
          f32x2 v = {p[r][j] * __builtin_bit_cast(float, w << 16), p[r][j + 1] * __builtin_bit_cast(float, w & 0xffff0000u)};
          if (MASKED) {
            v[0] = key0 + 8 * g + j <= lim[r] ? v[0] : 0.f;
            v[1] = key0 + 8 * g + j + 1 <= lim[r] ? v[1] : 0.f;
          }
          const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
          v[0] -= __builtin_bit_cast(float, h << 16);
          v[1] -= __builtin_bit_cast(float, h & 0xffff0000u);
          h4[j >> 1] = h;
          l4[j >> 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
        }
        hi[r] = __builtin_bit_cast(bf16x8, h4);
        lo[r] = __builtin_bit_cast(bf16x8, l4);
      }
      const bf16x8 z = __builtin_bit_cast(bf16x8, k.vz[i]);
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const uint32_t a = k.vc[4 * i + 2 * (u >> 1)], b = k.vc[4 * i + 2 * (u >> 1) + 1];
        const bf16x8 v = u & 1 ? value_codes<true>(vu, a, b) : value_codes<false>(vu, a, b);
#pragma unroll
        for (int r = 0; r < RT; r++) {
          f32x4& acc = o[r][4 * i + u];
          acc = mfma_b16(v, hi[r], acc);
          acc = mfma_b16(z, hi[r], acc);
          acc = mfma_b16(v, lo[r], acc);
          acc = mfma_b16(z, lo[r], acc);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_values(k, next, half, lane);
  }
};

// A workgroup takes 16 RT rows (query, head of the group; row = query G + head) of a sequence and key head and one chunk of
// its keys, a page a wave in turn, the next 32 keys' operands in flight; the waves' results are joined through LDS. Bound by the
// cache's bytes, of which a wave has 32 keys' in flight, where contexts are long (32 of 8,000 to 24,400 keys, 8 key heads of 128,
// 597 MB in 126 us, 4.7 TB/s of a copy's 5.1), else by a launch, latencies one after the other (lengths, table, first page) and 355
// vector and 40 matrix instructions a wave for 32 keys and 16 rows: 8 tokens, 38 MB 16.6 us; 16 x 5 tokens, 21 MB in three tiles a
// sequence 20.7; 2,048 causal rows on 16,384 keys 1.28 ms, 0.45 PFLOP/s. (64 keys in flight a wave took all registers: 32 contexts
// 40% slower, 8 tokens 60%; more chunks than target's 256 a head cost more than they fill.)
template <class T, int HD, int RT>
__global__ __launch_bounds__(256, RT == 2 ? 2 : 3) void cache4_attention_kernel(Cache4Args p) {
  typedef Page<HD> P;
  typedef Rows4<T, HD, RT> R;
  constexpr int kRows = 16 * RT;
  __shared__ __align__(16) f32x4 lds[4][RT][HD / 16][64];
  __shared__ float ml[4][2][kRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = blockIdx.x % p.Hk;
  Item it;
  if (!find_item4<false>(p, kRows, blockIdx.x / p.Hk, lane, it)) return;
  const int rows = it.nq * p.G, row0 = kRows * it.tile;
  R w;
#pragma unroll
  for (int r = 0; r < RT; r++) {
    const int row = row0 + 16 * r + (lane & 15), i = row / p.G, h = row - i * p.G;
    const bool ok = row < rows;
    const char* src = (const char*)p.q + 2 * ((long long)(it.q0 + (ok ? i : 0)) * p.q_st + (long long)(hk * p.G + h) * p.q_sh);
#pragma unroll
    for (int t = 0; t < HD / 32; t++) {
      const int c = 32 * t + 8 * (lane >> 4);
      w.q[r][t] = typename T::v8{};
      if (ok && c < p.d) w.q[r][t] = *reinterpret_cast<const typename T::v8*>(src + 2 * c);
    }
    w.m[r] = -INFINITY;
    w.l[r] = 0.f;
    w.lim[r] = p.causal && ok ? min(it.nk - 1, i + it.nk - it.nq) : it.nk - 1;
#pragma unroll
    for (int u = 0; u < HD / 16; u++) w.o[r][u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // keys seen by the tile's first row and by its last
  const auto seen = [&](int row) { return p.causal ? max(min(it.nk, min(row, rows - 1) / p.G + it.nk - it.nq + 1), 0) : it.nk; };
  const int whole = seen(row0), first = it.chunk * it.keys, last = min(seen(row0 + kRows - 1), min(first + min(it.keys, it.nk), it.nk));
  const int page0 = first / kCache4Page + wave, pages = (last + kCache4Page - 1) / kCache4Page;  // of this chunk, this wave's first
  const int* table = p.table + (size_t)it.seq * p.width;
  const char* base = (const char*)p.data + (size_t)hk * P::kBytes;
  // this wave's pages of 64 turns, one a lane
  int ids = -1;
  const auto page_of = [&](int turn) {
    if ((turn & 63) == 0) {
      const int i = page0 + 4 * (turn + lane);
      ids = i < pages ? table[i] : -1;
    }
    return __builtin_amdgcn_readlane(ids, turn & 63);
  };
  const auto at = [&](int id) { return base + (size_t)(id >= 0 && id < p.pages ? id : 0) * p.Hk * P::kBytes; };
  if (page0 < pages) {
    typename R::Keys k;
    int id = page_of(0);
    const char* page = at(id);
    R::load_keys(k, page, 0, lane);
    R::load_values(k, page, 0, lane);
    __builtin_amdgcn_sched_barrier(0);  // (q's sums while the first keys are on their way)
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int i = 0; i < R::G; i++) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (int e = 0; e < 8; e++) t += (float)w.q[r][2 * i + j][e];
        w.qs[r][i] = row_sum4(t);
      }
    bool good = id >= 0 && id < p.pages;  // (a page of no cache: not seen)
    int u = 0, pg = page0;                // halves of pages
    // to the next half: what its step takes, and where the one behind it lies (behind the last page: that one again, not used)
    const auto next = [&](bool& seen, int& key0) {
      seen = good;
      key0 = kCache4Page * pg + 32 * (u & 1);
      if (u & 1) {
        pg += 4;
        id = pg < pages ? page_of((u + 1) >> 1) : id;
        page = at(id);
        good = id >= 0 && id < p.pages;
      }
      u++;
    };
    bool seen;
    int key0;
    while (pg < pages && good && kCache4Page * pg + 32 * (u & 1) + 32 <= whole) {  // every row sees all 32
      next(seen, key0);
      w.template step<false>(k, key0, p.scale_log2, lane, page, u & 1);
    }
    while (pg < pages) {
      next(seen, key0);
      if (seen) {
        w.template step<true>(k, key0, p.scale_log2, lane, page, u & 1);
      } else {
        R::load_keys(k, page, u & 1, lane);
        R::load_values(k, page, u & 1, lane);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RT; r++) {
    const float l = row_sum4(w.l[r]);
    if (lane < 16) ml[wave][0][16 * r + lane] = w.m[r], ml[wave][1][16 * r + lane] = l;
#pragma unroll
    for (int u = 0; u < HD / 16; u++) lds[wave][r][u][lane] = w.o[r][u];
  }
  __syncthreads();
  const bool part = it.chunks > 1;
  const size_t slot = (size_t)it.slot * p.Hk + hk;
#pragma unroll 1
  for (int u = wave; u < RT * (HD / 16); u += 4) {  // 16 rows x 16 dims
    const int r = u / (HD / 16), db = u - r * (HD / 16), rr = 16 * r + (lane & 15), row = row0 + rr;
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 4; v++) M = fmaxf(M, ml[v][0][rr]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const float sc = __builtin_amdgcn_exp2f((ml[v][0][rr] - ref) * p.scale_log2);
      L = fmaf(sc, ml[v][1][rr], L);
      const f32x4 x = lds[v][r][db][lane];
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] = fmaf(sc, x[e], acc[e]);
    }
    if (row >= rows) continue;
    const int col = 16 * db + 4 * (lane >> 4), i = row / p.G, h = row - i * p.G;
    if (part) {
      if (db == 0 && lane < 16) {
        p.part_ml[2 * (slot * kRows + rr)] = M;
        p.part_ml[2 * (slot * kRows + rr) + 1] = L;
      }
      *reinterpret_cast<f32x4*>(p.part_o + (slot * kRows + rr) * HD + col) = acc;
    } else if (col < p.d) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      typename T::v4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = (typename T::elem)(acc[e] * inv);
      *reinterpret_cast<typename T::v4*>((char*)p.o + 2 * ((long long)(it.q0 + i) * p.o_st + (long long)(hk * p.G + h) * p.o_sh + col)) = y;
    }
  }
}

// The chunks of one (query, head) row: a thread takes one chunk's m and l, then groups of HD / 4 lanes sum O over every
// 1024 / HD-th chunk, joined through LDS. 4.2 to 5.3 us: a launch and three latencies.
template <class T, int HD>
__global__ __launch_bounds__(256) void cache4_join_kernel(Cache4Args p, int rows) {
  __shared__ float weight[256], red[2][4];
  __shared__ __align__(16) float sums[4][HD];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, H = p.G * p.Hk;
  const int q = blockIdx.x / H, head = blockIdx.x - q * H, hk = head / p.G;
  Item it;
  if (!find_item4<true>(p, rows, q, lane, it) || it.chunks == 1) return;
  const int row = (q - it.q0) * p.G + head - hk * p.G, tile = row / rows, rr = row - tile * rows;
  const size_t slot0 = (size_t)it.slot + (size_t)tile * it.chunks;
  if (it.slot < 0 || slot0 + it.chunks > (size_t)p.items) return;  // (starts that do not ascend)
  const auto at = [&](int j) { return ((slot0 + j) * p.Hk + hk) * rows + rr; };
  const bool live = t < it.chunks;  // (kCache4MaxChunks of them at most)
  const float m = live ? p.part_ml[2 * at(t)] : -INFINITY, l = live ? p.part_ml[2 * at(t) + 1] : 0.f;
  float M = m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
  if (lane == 0) red[0][wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float sc = __builtin_amdgcn_exp2f((m - (M == -INFINITY ? 0.f : M)) * p.scale_log2);
  weight[t] = live ? sc : 0.f;
  const float L4 = wave_total(live ? sc * l : 0.f);
  if (lane == 0) red[1][wave] = L4;
  __syncthreads();
  const float L = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  constexpr int kCols = HD / 4, kSide = 256 / kCols;
  const int col = 4 * (t % kCols), side = t / kCols;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int j = side; j < it.chunks; j += kSide) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(p.part_o + at(j) * HD + col);
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] = fmaf(weight[j], x[e], acc[e]);
  }
#pragma unroll
  for (int o = kCols; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], o);
  if (lane < kCols) *reinterpret_cast<f32x4*>(&sums[wave][col]) = acc;
  __syncthreads();
  if (t < kCols && col < p.d) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
    typename T::v4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = (typename T::elem)((sums[0][col + e] + sums[1][col + e] + sums[2][col + e] + sums[3][col + e]) * inv);
    *reinterpret_cast<typename T::v4*>((char*)p.o + 2 * ((long long)q * p.o_st + (long long)head * p.o_sh + col)) = y;
  }
}

// Rows of a tile by the mean rows of a sequence; keys divided unless the table holds few or the tiles alone fill the GPU
// many times over. Few: up to 4 passes the join costs more than they do (8 heads of 128, one token of 8 sequences on 1,000 keys
// 13.6 us divided, 12.7 whole; on 1,500 13.5 and 17.6), up to 8 where a tile a sequence gives every CU one (64 on 2,000 keys 48.0
// and 36.6, 64 on 0 to 2,000 31.9 and 31.5; on 0 to 4,000 56.4 and 56.4, but 32 on those 27.6 and 38.4).
Cache4Plan cache4_plan(long long T, int n, int width, int Hk, int G, int cus) {
  Cache4Plan plan{};
  const long long per = T * G / n;
  plan.rt = per <= 64 ? 1 : 2;
  const long long tiles = T * G / (16 * plan.rt) + n;
  const long long each = T * G / (16 * plan.rt) > n ? T * G / (16 * plan.rt) : n;  // tiles of a key head, about
  plan.divide = width > (each * Hk < cus ? 4 : 8) * (kPass / kCache4Page) && T * G / (16 * plan.rt) * Hk < 2LL * cus;
  plan.target = (int)((8LL * cus + Hk - 1) / Hk);
  if (plan.target > kCache4MaxChunks) plan.target = kCache4MaxChunks;
  plan.items = tiles + (plan.divide ? plan.target : 0);
  return plan;
}

template <class T, int HD, int RT>
static hipError_t launch_cache4_t(const Cache4Args& a, const Cache4Plan& plan, hipStream_t s) {
  ESM_LAUNCH((cache4_attention_kernel<T, HD, RT>), dim3((unsigned)(plan.items * a.Hk)), dim3(256), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.divide) return e;
  ESM_LAUNCH((cache4_join_kernel<T, HD>), dim3((unsigned)(a.T * a.G * a.Hk)), dim3(256), 0, s, a, 16 * RT);
  return hipGetLastError();
}
template <class T, int HD>
static hipError_t launch_cache4_hd(const Cache4Args& a, const Cache4Plan& plan, hipStream_t s) {
  switch (plan.rt) {
    case 1: return launch_cache4_t<T, HD, 1>(a, plan, s);
    default: return launch_cache4_t<T, HD, 2>(a, plan, s);
  }
}

hipError_t launch_cache4_attention(const Cache4Args& a, bool bf16, const Cache4Plan& plan, hipStream_t s) {
  if (bf16) return a.d <= 64 ? launch_cache4_hd<B16Keys, 64>(a, plan, s) : launch_cache4_hd<B16Keys, 128>(a, plan, s);
  return a.d <= 64 ? launch_cache4_hd<F16Keys, 64>(a, plan, s) : launch_cache4_hd<F16Keys, 128>(a, plan, s);
}

template <class V8, int HD>
static hipError_t launch_write_t(const Cache4Args& a, bool read, hipStream_t s) {
  const int per = 4 * EightLanes<HD>::kHeads;  // heads of a workgroup, keys' and values'
  // all heads in one workgroup where the keys alone fill the GPU, else as many workgroups as there are heads for
  const long long groups = eight_groups(a.T, a.n);
  const dim3 grid((unsigned)groups, groups >= 1024 ? 1 : (2 * a.Hk + per - 1) / per);
  if (read) {
    ESM_LAUNCH((cache4_read_kernel<V8, HD>), grid, dim3(256), 0, s, a);
  } else {
    ESM_LAUNCH((cache4_write_kernel<V8, HD>), grid, dim3(256), 0, s, a);
  }
  return hipGetLastError();
}
static hipError_t launch_rows4(const Cache4Args& a, bool bf16, bool read, hipStream_t s) {
  if (bf16) return a.d <= 64 ? launch_write_t<bf16x8, 64>(a, read, s) : launch_write_t<bf16x8, 128>(a, read, s);
  return a.d <= 64 ? launch_write_t<half8, 64>(a, read, s) : launch_write_t<half8, 128>(a, read, s);
}
hipError_t launch_cache4_write(const Cache4Args& a, bool bf16, hipStream_t s) { return launch_rows4(a, bf16, false, s); }
hipError_t launch_cache4_read(const Cache4Args& a, bool bf16, hipStream_t s) { return launch_rows4(a, bf16, true, s); }

}  // namespace esm
