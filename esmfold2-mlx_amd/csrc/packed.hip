// Attention over packed sequences of different lengths: softmax(q k^T scale) v within each sequence, query
// heads in groups of G that share a key head, both ways or causal (the last query sees the last key).
//
// The rows a workgroup takes are (query, head of the group) pairs of one sequence and key head, row = query * G +
// head: the group's heads share every key and value that is staged, and a single new token's heads fill a
// tile together. A wave holds 32 rows and takes 32 keys from LDS at a time:
//   S^T[key][row] = K Q^T       (A: K rows from LDS, B: the wave's query fragments, in registers)
//   p = 2^(S c - m c), l += p   (a lane holds one row: the maximum is over its registers and one exchange; where
//                               m c is large, 2^((S - m) c))
//   O^T[d][row] += V^T P^T      (A: V^T by the transposing LDS read, B: p in the accumulator's own key order)
// in fp32 but for p, which is rounded to the inputs' 16-bit type for the second product (an error of half a
// step of that type on each p, below the output's own rounding after the sum). m is the running maximum; it, O
// and l are rescaled only when a row's maximum has grown by more than 2^8 since (p then reaches 2^8 at most); in fp16
// 2^4, as p is kept 2^11 times as large there: fp16 loses bits below 2^-14, and thousands of keys some 2^-20 below one
// that attends to nothing (a sink) may be the whole output. Half a step holds down to 2^-25 of the row's largest, below
// that p is off by 2^-36 at most.
//
// Two kernels share that step: packed_attention_kernel (many rows: four waves of 32 rows over tiles of 64
// keys that they share, the next tile in flight) and split_attention_kernel (few rows: 32 rows, keys divided
// between the four waves and, through fp32 partials joined by a second launch, between workgroups).
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace esm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

struct Fp16 {
  typedef half8 v8;
  typedef half4 v4;
  typedef half_t elem;
  static constexpr float kGrow = 4.f, kUp = 11.f;  // (p <= 2^15, below fp16's largest)
  // exponent mask; 1, 128 and 129
  static constexpr uint16_t kExp = 0x7c00, kOne = 0x3c00, kMany = 0x5800, kBoth = 0x5808;
  static DEV f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static DEV float add(v8 v, float s) {  // s + the sum of v, two exact products with 1 at a time
    const half2v one = {(half_t)1.0f, (half_t)1.0f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2(half2v{v[i], v[i + 1]}, one, s, false);
    return s;
  }
};
struct Bf16 {
  typedef bf16x8 v8;
  typedef bf16x4 v4;
  typedef __bf16 elem;
  static constexpr float kGrow = 8.f, kUp = 0.f;  // log2: what p may reach before its row is rescaled, and all p's factor
  static constexpr uint16_t kExp = 0x7f80, kOne = 0x3f80, kMany = 0x4300, kBoth = 0x4301;
  static DEV f32x16 mfma(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static DEV float add(v8 v, float s) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    const v2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2_f32_bf16(v2{v[i], v[i + 1]}, one, s, false);
    return s;
  }
};

constexpr float kFar = 1024.f;  // least exponent of a row's maximum that its scores are made relative to

// LDS rows of HD values, 16-byte pieces swizzled so that the reads below cover the 64 banks once: K fragments
// read 16 rows at one piece; V's transposing read takes 4 rows x 4 pieces.
template <int HD>
DEV int k_piece(int n, int p) { return HD == 64 ? p ^ ((n >> 1) & 7) : p ^ (n & 15); }
template <int HD>
DEV int v_piece(int n, int p) { return HD == 64 ? p ^ (((n >> 1) & 1) << 2) : p ^ ((n & 3) << 2); }

// V^T fragment: 4 keys k0 .. k0 + 3 of column n0 + lane % 16 (common.h, ds_read_tr16x4).
template <class T, int HD>
DEV typename T::v4 v_read(const char* vs, int k0, int n0, int lane) {
  const int j = lane & 15, n = k0 + (j >> 2), d = n0 + 4 * (j & 3);
  return __builtin_bit_cast(typename T::v4, ds_read_tr16x4(vs + n * 2 * HD + 16 * v_piece<HD>(n, d >> 3) + 2 * (d & 7)));
}
template <class T, int HD>
DEV typename T::v8 v_frag(const char* vs, int j, int db, int lane) {  // keys 16 j + 4 h + {0..3, 8..11}, see p
  const int h = lane >> 5, n0 = 32 * db + 16 * ((lane >> 4) & 1);
  const typename T::v4 lo = v_read<T, HD>(vs, 16 * j + 4 * h, n0, lane), hi = v_read<T, HD>(vs, 16 * j + 8 + 4 * h, n0, lane);
  return typename T::v8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// One wave's rows: query fragments, running maximum (of the unscaled scores), sum (this lane's half of the keys)
// and output. Row r is column lane % 32 = r of every accumulator.
template <class T, int HD>
struct Rows {
  typename T::v8 q[HD / 16];
  f32x16 o[HD / 32];
  float m, l;
  int lim;  // last key this row sees, counted within the sequence

  DEV void init() {
    m = -INFINITY;
    l = 0.f;
    odd = false;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[d][i] = 0.f;
  }

  enum { kNone, kEnd, kLater };
  bool odd;  // values taken as 0 by a masked step (``add_odd`` makes up for the seen ones)

  // 32 keys key0 .. of the sequence from LDS rows ks, vs, of which some row sees only a part. kEnd: the unseen ones lie
  // behind the sequence, their rows are zeros. kLater: some are the sequence's own later keys; what they hold must
  // not count, and as a p of 0 does not silence an infinity or a NaN in V, all values that are one are taken as 0.
  // kNone: all are seen.
  template <int MASK>
  DEV void step(const char* ks, const char* vs, int key0, float c, int lane) {
    constexpr bool MASKED = MASK != kNone;
    const int r = lane & 31, h = lane >> 5;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
    for (int k = 0; k < HD / 16; k++)
      s = T::mfma(*reinterpret_cast<const typename T::v8*>(ks + r * 2 * HD + 16 * k_piece<HD>(r, 2 * k + h)), q[k], s);
    if (MASKED) {
#pragma unroll
      for (int i = 0; i < 16; i++) s[i] = key0 + acc_row32(i, lane) <= lim ? s[i] : -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__any((mx - m) * c > T::kGrow)) grow(mx, c);  // (from m = -inf at the first key a row sees)
    const float mc = reference(c, s);
    typename T::v8 p[2];
#pragma unroll
    for (int i = 0; i < 16; i++)  // (results below 2^-126 flush)
      p[i >> 3][i & 7] = (typename T::elem)__builtin_amdgcn_exp2f(fmaf(s[i], c, -mc));
#pragma unroll
    for (int j = 0; j < 2; j++) l = T::add(p[j], l);
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int d = 0; d < HD / 32; d++) {
        typename T::v8 v = v_frag<T, HD>(vs, j, d, lane);
        if (MASK == kLater) v = finite(v);
        o[d] = T::mfma(v, p[j], o[d]);
      }
  }

  // 64 keys that every row sees, in an order that the scheduler keeps: a fragment is read some matrix instructions
  // before its own (LDS answers in more than 64 cycles, one takes 32), the maximum of the first 32 keys is taken
  // between those of the next 32, and the exponentials of the second half between the value products of the first. The
  // matrix phases go before the other wave's vector work (1,100 tokens of 40 heads of 64 24.9 -> 22.6 us).
  DEV void step64(const char* ks, const char* vs, float c, int lane) {
    constexpr int NK = HD / 16, ND = HD / 32;
    typedef typename T::v8 v8;
    const int r = lane & 31, h = lane >> 5;
    const auto key = [&](int kb, int k) {
      return *reinterpret_cast<const v8*>(ks + (32 * kb + r) * 2 * HD + 16 * k_piece<HD>(r, 2 * k + h));
    };
    f32x16 s0, s1;
#pragma unroll
    for (int i = 0; i < 16; i++) s0[i] = s1[i] = 0.f;
    v8 ka[NK], kb[NK], va[ND], vb[ND];
#pragma unroll
    for (int k = 0; k < NK; k++) ka[k] = key(0, k);
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < NK; k++) {
      s0 = T::mfma(ka[k], q[k], s0);
      kb[k] = key(1, k);
      __builtin_amdgcn_sched_barrier(0);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < NK; k++) {
      s1 = T::mfma(kb[k], q[k], s1);
      if (k < ND) va[k] = v_frag<T, HD>(vs, 0, k, lane);
      if (k > 0) {  // (its results are there by then)
#pragma unroll
        for (int i = 16 * (k - 1) / (NK - 1); i < 16 * k / (NK - 1); i++) mx = fmaxf(mx, s0[i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; i++) mx = fmaxf(mx, s1[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    if (__any((mx - m) * c > T::kGrow)) grow(mx, c);
    const float mc = reference(c, s0, s1);
    v8 p[4];
    const auto prob = [&](int i) {  // probabilities 2i, 2i + 1 of 32 (results below 2^-126 flush)
      const f32x16& s = i < 8 ? s0 : s1;
      p[i >> 2][2 * (i & 3)] = (typename T::elem)__builtin_amdgcn_exp2f(fmaf(s[2 * i & 15], c, -mc));
      p[i >> 2][2 * (i & 3) + 1] = (typename T::elem)__builtin_amdgcn_exp2f(fmaf(s[(2 * i & 15) + 1], c, -mc));
    };
#pragma unroll
    for (int i = 0; i < 8; i++) prob(i);
    l = T::add(p[0], l);
    l = T::add(p[1], l);
    __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 2 * ND; u++) {  // values of keys 0 .. 31
      const int j = u / ND, d = u % ND;
      o[d] = T::mfma(j ? vb[d] : va[d], p[j], o[d]);
      (j ? va : vb)[d] = v_frag<T, HD>(vs, j + 1, d, lane);
#pragma unroll
      for (int i = 8 * u / (2 * ND); i < 8 * (u + 1) / (2 * ND); i++) prob(8 + i);
      __builtin_amdgcn_sched_barrier(0);
    }
    l = T::add(p[2], l);
    l = T::add(p[3], l);
#pragma unroll
    for (int u = 0; u < 2 * ND; u++) {  // and 32 .. 63
      const int j = u / ND, d = u % ND;
      o[d] = T::mfma(j ? vb[d] : va[d], p[2 + j], o[d]);
      if (!j) vb[d] = v_frag<T, HD>(vs, 3, d, lane);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  }

  // m c less p's own exponent, from which the exponents s c of the scores s are taken with one FMA a score. Its rounding,
  // 2^-24 of its size, goes into every p as a factor, so where it is large the scores themselves become relative to m
  // (the difference of two near scores is exact) and m c counts as 0. So too where it is not finite: c may carry m past
  // fp32's range, and a row that has seen no key, or only scores of -inf, has m = -inf; its p are 0. (1,100 tokens of
  // 40 heads of 64 22.6 -> 23.2 us with it, all else within 1%.)
  template <class... S>
  DEV float reference(float c, S&... s) {
    const float mc = m * c;
    const bool far = !(fabsf(mc) < kFar);
    if (!__any(far)) return mc - T::kUp;
    const float ref = far && m != -INFINITY ? m : 0.f;  // (m = +inf: its row becomes NaN)
    const auto relative = [&](f32x16& x) {
#pragma unroll
      for (int i = 0; i < 16; i++) x[i] -= ref;
    };
    (relative(s), ...);
    return (far ? 0.f : mc) - T::kUp;
  }

  // The row's maximum has grown to mx: everything summed so far by the new one.
  DEV void grow(float mx, float c) {
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f((m - ref) * c);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[d][i] *= alpha;
  }

  DEV typename T::v8 finite(typename T::v8 x) {
    u16x8 v = __builtin_bit_cast(u16x8, x);
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const bool bad = (v[e] & T::kExp) == T::kExp;
      odd = odd || bad;
      v[e] = bad ? 0 : v[e];
    }
    return __builtin_bit_cast(typename T::v8, v);
  }

  // What the masked steps' seen infinities and NaN bring, for keys first .. last - 1 (rows of V from `vb`, st elements
  // apart): a product of ones counts, row by row, the seen values of +inf (by 1), -inf (by 128) and NaN (by both; 16
  // of each at most, exact), and what it finds becomes that infinity (both: NaN).
  DEV void add_odd(const char* vb, long long st, int d, int first, int last, int lane) {
    typedef typename T::v8 v8;
    const int r = lane & 31, h = lane >> 5;
    for (int k0 = first; k0 < last; k0 += 16)
#pragma unroll
      for (int db = 0; db < HD / 32; db++) {
        u16x8 v, seen;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int key = k0 + 8 * h + e;
          const uint16_t x = key < last && 32 * db + r < d ? *reinterpret_cast<const uint16_t*>(vb + 2 * (st * key + 32 * db + r)) : 0;
          const bool bad = (x & T::kExp) == T::kExp, nan = (x & 0x7fff) != T::kExp;
          v[e] = !bad ? 0 : nan ? T::kBoth : x >> 15 ? T::kMany : T::kOne;
          seen[e] = key <= lim ? T::kOne : 0;
        }
        f32x16 n;
#pragma unroll
        for (int i = 0; i < 16; i++) n[i] = 0.f;
        n = T::mfma(__builtin_bit_cast(v8, v), __builtin_bit_cast(v8, seen), n);
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float down = floorf(n[i] * 0.0078125f);
          o[db][i] += n[i] - 128.f * down > 0.f ? INFINITY : 0.f;
          o[db][i] -= down > 0.f ? INFINITY : 0.f;
        }
      }
  }
};

struct Span {
  int q0, nq, k0, nk;  // first row and rows of a sequence, on the query and on the key side
};

// Sequence of a work item and the item's number within it: a sequence has as many items as tiles of `unit` rows times
// chunks of `chunk` keys (at least one; chunk 0: not counted). All lanes agree; the starts are read once, a lane a
// sequence. Starts outside 0 .. the rows there are are brought inside, so nothing a caller writes there reaches past
// the tensors.
DEV bool find_item(const PackedAttnArgs& p, int unit, int chunk, int item, int lane, Span& s, int& at) {
  for (int i0 = 0; i0 < p.n; i0 += 64) {
    const int i = min(i0 + lane, p.n - 1);
    const int a = min(max(p.cu_q[i], 0), p.Tq), b = min(max(p.cu_q[i + 1], a), p.Tq);
    const int ka = min(max(p.cu_k[i], 0), p.Tk), kb = min(max(p.cu_k[i + 1], ka), p.Tk);
    int nt = ((b - a) * p.G + unit - 1) / unit;
    if (chunk) nt *= max(1, (kb - ka + chunk - 1) / chunk);
    if (i0 + lane >= p.n) nt = 0;
    const int sum = wave_scan(nt);
    const uint64_t past = __ballot(item < sum);
    if (past) {
      const int w = __builtin_ctzll(past);
      at = item - __builtin_amdgcn_readlane(sum - nt, w);
      s.q0 = __builtin_amdgcn_readlane(a, w);
      s.nq = __builtin_amdgcn_readlane(b - a, w);
      s.k0 = __builtin_amdgcn_readlane(ka, w);
      s.nk = __builtin_amdgcn_readlane(kb - ka, w);
      return true;
    }
    item -= __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// find_item for tiles of kAttnRows rows of 2 to 64 sequences, the longest tiles first whichever sequence they are of, so
// that no long one starts last (prompts of 1 to 4,096 rows 289 -> 244 us): the keys a tile sees fall into 16 levels, and
// how many tiles of a sequence see at least so many follows from its lengths. `at` counts a sequence's tiles from the
// one that sees most.
constexpr int kAttnRows = 128;  // rows per workgroup of the many-row kernel
template <bool CAUSAL>
DEV bool find_longest(const PackedAttnArgs& p, int item, int lane, Span& s, int& at) {
  const int i = min(lane, p.n - 1);
  const int a = min(max(p.cu_q[i], 0), p.Tq), b = min(max(p.cu_q[i + 1], a), p.Tq);
  const int ka = min(max(p.cu_k[i], 0), p.Tk), kb = min(max(p.cu_k[i + 1], ka), p.Tk);
  const int nq = b - a, nk = kb - ka, tiles = lane < p.n ? (nq * p.G + kAttnRows - 1) / kAttnRows : 0;
  if (item >= wave_sum(tiles)) return false;
  const int level = wave_max(lane < p.n ? nk : 0) / 16 + 1;
  // tiles of this lane's sequence whose last row sees at least `keys` keys
  const auto seeing = [&](int keys) {
    if (keys > nk) return 0;
    if (!CAUSAL) return tiles;
    const int first = keys - 1 - nk + nq;  // the first row that does
    return first <= 0 ? tiles : max(0, tiles - (int)((long long)first * p.G / kAttnRows));
  };
  int lv = 0;  // the highest level whose tiles and those above pass the item
#pragma unroll
  for (int step = 8; step; step >>= 1)
    if (wave_sum(seeing((lv + step) * level)) > item) lv += step;
  const int above = seeing((lv + 1) * level), mine = (lv ? seeing(lv * level) : tiles) - above;
  item -= wave_sum(above);
  const int sum = wave_scan(mine);
  const int w = __builtin_ctzll(__ballot(item < sum));
  at = item - __builtin_amdgcn_readlane(sum - mine, w) + __builtin_amdgcn_readlane(above, w);
  s = Span{__builtin_amdgcn_readlane(a, w), __builtin_amdgcn_readlane(nq, w), __builtin_amdgcn_readlane(ka, w),
           __builtin_amdgcn_readlane(nk, w)};
  return true;
}

// A tile of `keys` key rows from key kt of the span on, as a buffer whose range ends with the span's last row:
// rows past it (another sequence's, or none) load zeros.
DEV dma_src_t tile_src(const char* base, long long st, int d, int first, int kt, int nk, int keys) {
  const int rows = min(keys, nk - kt);
  return dma_src(base + 2 * (st * (long long)(first + kt)), rows > 0 ? (uint32_t)(2 * ((rows - 1) * st + d)) : 0u);
}

// One wave's DMA of `count` rows (a multiple of the rows of 1 KB), from row n0 of the tile on, into LDS rows at n0.
template <int HD, bool V>
DEV void load_rows(dma_src_t src, uint32_t lds, long long st, int d, int n0, int count, int lane) {
  constexpr int kRow = 2 * HD, kPer = 1024 / kRow, kPieces = HD / 8;
#pragma unroll
  for (int i = 0; i < count / kPer; i++) {
    const int n = n0 + kPer * i + lane / kPieces, lp = lane % kPieces;
    const int piece = V ? v_piece<HD>(n, lp) : k_piece<HD>(n, lp);
    dma16(src, lds + kRow * (n0 + kPer * i), 8 * piece < d ? (uint32_t)(2 * st * n + 16 * piece) : kOOB, 0);
  }
}

// Query fragments and the limit of row `row` (of the span's nq * G).
template <class T, int HD, bool CAUSAL>
DEV void load_queries(Rows<T, HD>& w, const PackedAttnArgs& p, const Span& s, int hk, int row0, int lane) {
  const int h = lane >> 5, row = row0 + (lane & 31), i = row / p.G, g = row - i * p.G;
  const bool ok = i < s.nq;
  const char* src = (const char*)p.q + 2 * ((long long)(s.q0 + (ok ? i : 0)) * p.q_st + (long long)(hk * p.G + g) * p.q_sh);
#pragma unroll
  for (int k = 0; k < HD / 16; k++) {
    w.q[k] = typename T::v8{};
    if (ok && 16 * k + 8 * h < p.d) w.q[k] = *reinterpret_cast<const typename T::v8*>(src + 2 * (16 * k + 8 * h));
  }
  w.lim = CAUSAL && ok ? min(s.nk - 1, i + s.nk - s.nq) : s.nk - 1;
}

constexpr int kAttnKeys = 64;   // keys per tile of the many-row kernel

// Many rows: bound by the vector unit's softmax beside the matrix cores. 16,384 causal rows of 32 / 8 heads of 128
// 2.1 ms, 1.05 PFLOP/s with the matrix cores 51 % busy at 1.8 GHz; 12 proteins of 3,481 rows, 40 heads of 64, 40 us,
// 0.53 PFLOP/s. Two waves a SIMD at 256 registers: 32 rows a wave is what they hold without spills.
template <class T, int HD, bool CAUSAL>
__global__ __launch_bounds__(256, 2) void packed_attention_kernel(PackedAttnArgs p) {
  constexpr int kTile = kAttnKeys * 2 * HD;  // bytes of a K (or V) tile
  __shared__ __align__(1024) char lds[2][2 * kTile];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // key heads run fastest over the workgroups: the eight XCDs take different heads, each with its own L2, and the
  // longest tiles of every head start first
  const int hk = blockIdx.x % p.Hk, item = blockIdx.x / p.Hk;
  Span s;
  int tile;
  const bool many = p.n > 1 && p.n <= 64;
  if (many ? !find_longest<CAUSAL>(p, item, lane, s, tile) : !find_item(p, kAttnRows, 0, item, lane, s, tile)) return;
  tile = __builtin_amdgcn_readfirstlane(tile);
  const int rows = s.nq * p.G;
  tile = (rows + kAttnRows - 1) / kAttnRows - 1 - tile;  // the last see most
  const int row0 = kAttnRows * tile + 32 * wave;  // this wave's first row

  Rows<T, HD> w;
  w.init();
  load_queries<T, HD, CAUSAL>(w, p, s, hk, row0, lane);
  // keys seen by the workgroup's last row, by this wave's last row, and by its first
  const auto seen = [&](int row) { return CAUSAL ? max(min(s.nk, min(row, rows - 1) / p.G + s.nk - s.nq + 1), 0) : s.nk; };
  const int end = seen(kAttnRows * (tile + 1) - 1);
  const int wend = row0 < rows ? seen(row0 + 31) : 0;
  const char* kb = (const char*)p.k + 2 * (long long)hk * p.k_sh;
  const char* vb = (const char*)p.v + 2 * (long long)hk * p.v_sh;
  const auto load = [&](int kt, int buf) {
    constexpr int kMine = kAttnKeys / 4;
    const uint32_t at = lds_address(lds[buf]);
    load_rows<HD, false>(tile_src(kb, p.k_st, p.d, s.k0, kt, s.nk, kAttnKeys), at, p.k_st, p.d, kMine * wave, kMine, lane);
    load_rows<HD, true>(tile_src(vb, p.v_st, p.d, s.k0, kt, s.nk, kAttnKeys), at + kTile, p.v_st, p.d, kMine * wave, kMine, lane);
  };
  // whole tiles that the workgroup's first row sees, then those at the end of what its rows see
  const int whole = seen(kAttnRows * tile) / kAttnKeys * kAttnKeys;
  if (end > 0) load(0, 0);
  int kt = 0, buf = 0;
  for (; kt < whole; kt += kAttnKeys, buf ^= 1) {
    wait_vm(0);
    __syncthreads();  // this tile is in, and every wave has left the other buffer
    if (kt + kAttnKeys < end) load(kt + kAttnKeys, buf ^ 1);
    w.step64(lds[buf], lds[buf] + kTile, p.scale_log2, lane);
  }
  for (; kt < end; kt += kAttnKeys, buf ^= 1) {
    wait_vm(0);
    __syncthreads();
    if (kt + kAttnKeys < end) load(kt + kAttnKeys, buf ^ 1);
#pragma unroll 1
    for (int u = 0; u < kAttnKeys && kt + u < wend; u += 32) {
      const char *ks = lds[buf] + u * 2 * HD, *vs = ks + kTile;
      w.template step<CAUSAL ? Rows<T, HD>::kLater : Rows<T, HD>::kEnd>(ks, vs, kt + u, p.scale_log2, lane);
    }
  }
  if (CAUSAL && __any(w.odd)) w.add_odd(vb + 2 * p.v_st * s.k0, p.v_st, p.d, whole, wend, lane);

  const float l = w.l + __shfl_xor(w.l, 32);
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // a row that sees no key is 0
  const int row = row0 + (lane & 31), i = row / p.G, g = row - i * p.G;
  if (row >= rows) return;
  char* dst = (char*)p.o + 2 * ((long long)(s.q0 + i) * p.o_st + (long long)(hk * p.G + g) * p.o_sh);
#pragma unroll
  for (int d = 0; d < HD / 32; d++)
#pragma unroll
    for (int i4 = 0; i4 < 4; i4++) {
      const int col = 32 * d + acc_row32(4 * i4, lane);
      typename T::v4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = (typename T::elem)(w.o[d][4 * i4 + e] * inv);
      if (col < p.d) *reinterpret_cast<typename T::v4*>(dst + 2 * col) = y;
    }
}

// ---- few rows ---------------------------------------------------------------------------------
// 32 rows and one chunk of p.chunk keys (of every sequence the same, so that a long one has many and workgroups
// are alike) per workgroup, in passes of 4 x KW keys, KW to each wave in a private LDS tile. The waves' results are
// joined through LDS. Where sequences may have more than one chunk (p.part_o) each workgroup leaves (m, l, O) of
// its own in the workspace and attention_join_kernel sums them. Bound by the keys' and values' bytes: 8 tokens on
// 33,414 keys of 8 heads of 128 27.5 us, 5.0 TB/s, and 4.8 us for the join.
template <int HD>
constexpr int kSplitKeys = HD == 64 ? 64 : 32;  // keys per wave and pass: 64 KB of LDS, two workgroups per CU

template <class T, int HD, bool CAUSAL>
__global__ __launch_bounds__(256, 2) void split_attention_kernel(PackedAttnArgs p) {
  constexpr int KW = kSplitKeys<HD>, kTile = KW * 2 * HD, kPass = 4 * KW;
  __shared__ __align__(1024) char lds[4][2 * kTile];
  __shared__ float ml[4][2][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % p.Hk, item = blockIdx.x / p.Hk;
  Span s;
  int at;
  if (!find_item(p, 32, p.chunk, item, lane, s, at)) return;
  at = __builtin_amdgcn_readfirstlane(at);
  const int rows = s.nq * p.G, tiles = (rows + 31) / 32, chunk = at / tiles, row0 = 32 * (at - chunk * tiles);
  const int first = chunk * p.chunk;
  const auto seen = [&](int row) { return CAUSAL ? max(min(s.nk, min(row, rows - 1) / p.G + s.nk - s.nq + 1), 0) : s.nk; };
  const int last = seen(row0 + 31), end = min(last, first + min(p.chunk, s.nk - first)), wfull = seen(row0);
  if (chunk > 0 && first >= last) return;  // nothing seen: the join reads none

  Rows<T, HD> w;
  w.init();
  load_queries<T, HD, CAUSAL>(w, p, s, hk, row0, lane);
  const char* kb = (const char*)p.k + 2 * (long long)hk * p.k_sh;
  const char* vb = (const char*)p.v + 2 * (long long)hk * p.v_sh;
  char *ks = lds[wave], *vs = lds[wave] + kTile;
  const auto load = [&](int kt) {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the last pass's LDS reads are back
    __asm__ volatile("" ::: "memory");
    load_rows<HD, false>(tile_src(kb, p.k_st, p.d, s.k0, kt, s.nk, KW), lds_address(ks), p.k_st, p.d, 0, KW, lane);
    load_rows<HD, true>(tile_src(vb, p.v_st, p.d, s.k0, kt, s.nk, KW), lds_address(vs), p.v_st, p.d, 0, KW, lane);
    wait_vm(0);
  };
  int kt = first + KW * wave;
  for (; kt < end && kt + KW <= wfull; kt += kPass) {
    load(kt);
#pragma unroll
    for (int u = 0; u < KW; u += 32) w.template step<Rows<T, HD>::kNone>(ks + u * 2 * HD, vs + u * 2 * HD, kt + u, p.scale_log2, lane);
  }
  const int masked = kt;
  for (; kt < end; kt += kPass) {
    load(kt);
#pragma unroll 1
    for (int u = 0; u < KW && kt + u < end; u += 32)
      w.template step<CAUSAL ? Rows<T, HD>::kLater : Rows<T, HD>::kEnd>(ks + u * 2 * HD, vs + u * 2 * HD, kt + u, p.scale_log2,
                                                                         lane);
  }
  if (CAUSAL && __any(w.odd))
    for (kt = masked; kt < end; kt += kPass) w.add_odd(vb + 2 * p.v_st * s.k0, p.v_st, p.d, kt, min(kt + KW, end), lane);

  // (m, l, O) of the four waves through LDS; wave i then joins the d quads i, i + 4, .. of every row
  const float lsum = w.l + __shfl_xor(w.l, 32);
  if (h == 0) {
    ml[wave][0][r] = w.m;
    ml[wave][1][r] = lsum;
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __asm__ volatile("" ::: "memory");
  f32x4* ow = reinterpret_cast<f32x4*>(lds[wave]);
#pragma unroll
  for (int d = 0; d < HD / 32; d++)
#pragma unroll
    for (int i4 = 0; i4 < 4; i4++)
      ow[(4 * d + i4) * 64 + lane] = f32x4{w.o[d][4 * i4], w.o[d][4 * i4 + 1], w.o[d][4 * i4 + 2], w.o[d][4 * i4 + 3]};
  __syncthreads();
  const int row = row0 + r, i = row / p.G, g = row - i * p.G;
  if (row >= rows) return;
  float M = -INFINITY, L = 0.f, sc[4];
#pragma unroll
  for (int v = 0; v < 4; v++) M = fmaxf(M, ml[v][0][r]);
  const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int v = 0; v < 4; v++) {
    // (a wave that saw no key has m = -inf and adds 0; an infinite m gives NaN, as its row is)
    sc[v] = __builtin_amdgcn_exp2f((ml[v][0][r] - ref) * p.scale_log2);
    L += sc[v] * ml[v][1][r];
  }
  const long long q = s.q0 + i;
  const int head = hk * p.G + g;
  const bool part = p.part_o != nullptr;
  const size_t pat = ((size_t)q * (p.G * p.Hk) + head) * p.splits + chunk;
  if (part && wave == 0 && h == 0) {
    p.part_ml[2 * pat] = M;
    p.part_ml[2 * pat + 1] = L;
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  char* dst = (char*)p.o + 2 * (q * p.o_st + (long long)head * p.o_sh);
#pragma unroll
  for (int u = 0; u < HD / 32; u++) {
    const int qd = wave + 4 * u, col = 32 * (qd >> 2) + acc_row32(4 * (qd & 3), lane);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 4; v++) acc += sc[v] * reinterpret_cast<const f32x4*>(lds[v])[qd * 64 + lane];
    if (col >= p.d) continue;
    if (part) {
      *reinterpret_cast<f32x4*>(p.part_o + pat * p.d + col) = acc;
    } else {
      typename T::v4 y;
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = (typename T::elem)(acc[e] * inv);
      *reinterpret_cast<typename T::v4*>(dst + 2 * col) = y;
    }
  }
}

// The chunks of one (query, head) row, a workgroup each: a thread takes one chunk's m and l (kAttnMaxSplits of them at
// most), then groups of d / 4 lanes sum O over every 256 / (HD / 4)-th chunk, joined through LDS.
template <class T, int HD>
__global__ __launch_bounds__(256) void attention_join_kernel(PackedAttnArgs p) {
  static_assert(kAttnMaxSplits <= 256, "a chunk a thread");
  __shared__ float weight[256], red[2][4];
  __shared__ __align__(16) float sums[4][HD];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, H = p.G * p.Hk;
  const int q = blockIdx.x / H, head = blockIdx.x - q * H;
  // m and l of every chunk there may be and the first chunks' O are read before it is known which were written
  const size_t at = (size_t)blockIdx.x * p.splits;
  constexpr int kCols = HD / 4, kSide = 256 / kCols, kAhead = 4;  // lanes across a row, chunks at once, times ahead
  const int col = 4 * (t % kCols), side = t / kCols;
  const float* po = p.part_o + at * p.d;
  const bool may = t < p.splits;
  const float ml0 = may ? p.part_ml[2 * (at + t)] : 0.f, ml1 = may ? p.part_ml[2 * (at + t) + 1] : 0.f;
  f32x4 ahead[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; i++) {
    const int j = side + kSide * i;
    ahead[i] = j < p.splits && col < p.d ? *reinterpret_cast<const f32x4*>(po + (size_t)j * p.d + col) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  Span s;
  bool found = false;
  for (int i0 = 0; i0 < p.n && !found; i0 += 64) {
    const int i = min(i0 + lane, p.n - 1);
    const int a = min(max(p.cu_q[i], 0), p.Tq), b = min(max(p.cu_q[i + 1], a), p.Tq);
    const int ka = min(max(p.cu_k[i], 0), p.Tk), kb = min(max(p.cu_k[i + 1], ka), p.Tk);
    const uint64_t hit = __ballot(q >= a && q < b);
    if (hit) {
      const int w = __builtin_ctzll(hit);
      s = Span{__builtin_amdgcn_readlane(a, w), __builtin_amdgcn_readlane(b - a, w), __builtin_amdgcn_readlane(ka, w),
               __builtin_amdgcn_readlane(kb - ka, w)};
      found = true;
    }
  }
  if (!found) return;  // behind the last sequence: left as it is
  // chunks that wrote: those that the row's tile sees, or the first
  const int rows = s.nq * p.G, last = min(((q - s.q0) * p.G + head % p.G) | 31, rows - 1);
  const int seen = p.causal ? max(min(s.nk, last / p.G + s.nk - s.nq + 1), 0) : s.nk;
  const int live = max(1, (seen + p.chunk - 1) / p.chunk);
  const float m = t < live ? ml0 : -INFINITY, l = t < live ? ml1 : 0.f;
  float M = m;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
  if (lane == 0) red[0][wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float sc = __builtin_amdgcn_exp2f((m - (M == -INFINITY ? 0.f : M)) * p.scale_log2);
  weight[t] = t < live ? sc : 0.f;
  float L = t < live ? sc * l : 0.f;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) L += __shfl_xor(L, o);
  if (lane == 0) red[1][wave] = L;
  __syncthreads();
  L = red[1][0] + red[1][1] + red[1][2] + red[1][3];
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kAhead; i++)
    if (side + kSide * i < live) acc += weight[side + kSide * i] * ahead[i];
  for (int j = side + kSide * kAhead; j < live; j += kSide)
    if (col < p.d) acc += weight[j] * *reinterpret_cast<const f32x4*>(po + (size_t)j * p.d + col);
#pragma unroll
  for (int o = kCols; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], o);
  if (lane < kCols) *reinterpret_cast<f32x4*>(&sums[wave][col]) = acc;
  __syncthreads();
  if (t < kCols && col < p.d) {
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    f32x4 a = *reinterpret_cast<const f32x4*>(&sums[0][col]);
#pragma unroll
    for (int v = 1; v < 4; v++) a += *reinterpret_cast<const f32x4*>(&sums[v][col]);
    typename T::v4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = (typename T::elem)(a[e] * inv);
    *reinterpret_cast<typename T::v4*>((char*)p.o + 2 * ((long long)q * p.o_st + (long long)head * p.o_sh + col)) = y;
  }
}

template <class T, int HD, bool CAUSAL>
static hipError_t launch_attention_t(const PackedAttnArgs& a, bool many, hipStream_t s) {
  if (many) {
    const long long items = (long long)a.Tq * a.G / kAttnRows + a.n;
    ESM_LAUNCH((packed_attention_kernel<T, HD, CAUSAL>), dim3((unsigned)(items * a.Hk)), dim3(256), 0, s, a);
    return hipGetLastError();
  }
  ESM_LAUNCH((split_attention_kernel<T, HD, CAUSAL>), dim3((unsigned)(split_attention_items(a.Tq, a.Tk, a.n, a.G, a.chunk) * a.Hk)),
             dim3(256), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.part_o) return e;
  ESM_LAUNCH((attention_join_kernel<T, HD>), dim3((unsigned)(a.Tq * a.G * a.Hk)), dim3(256), 0, s, a);
  return hipGetLastError();
}

// Work items of the few-row kernel per key head, at most: (tiles, chunks) pairs of all sequences.
long long split_attention_items(long long Tq, long long Tk, int n, int G, int chunk) {
  const long long tiles = Tq * G / 32 + n, chunks = Tk / chunk + n;  // of all sequences
  const long long a = tiles * ((Tk + chunk - 1) / chunk + 1), b = ((Tq * G + 31) / 32) * chunks;  // (one may have all of either)
  return a < b ? a : b;
}

// Which kernel and which chunk of keys, from what the host knows: rows, keys, sequences and heads (the lengths are on
// the device).
AttnPlan packed_attention_plan(long long Tq, long long Tk, int n, int Hk, int G, int d, int cus) {
  AttnPlan plan{};
  // The many-row kernel where its tiles of 128 rows make some 5/8 of a workgroup per CU (us, many / few rows: 40 heads
  // of 64, 300 tokens 10.3 / 9.8, 512 tokens 12.3 / 13.6, 1,100 tokens 28 / 38; causal, 32/8 heads of 128, 512 tokens
  // 19 / 13, 1,024 tokens 29 / 30, 2,048 tokens 57 / 78; 512 new tokens on 8,192 163 / 107), or the sequences are short
  // on both sides (one of 24 tokens 4.8 / 6.0, 64 of 100 tokens 35 / 136; 64 single tokens on 100 keys 10.5 / 8.6). The
  // lengths themselves are on the device and count by their means only: a prompt of 4,096 rows beside 16 tokens on caches
  // of 16,384 takes 389 us in the many-row kernel, 148 and 198 apart.
  const long long per = Tq * G / n;
  plan.many = (Tq * G / 128 * Hk * 8 >= 5 * cus && per >= 64) || (Tk / n <= 128 && per >= 16);
  const int pass = d <= 64 ? 256 : 128;
  // as many chunks as make some four workgroups per CU, of two passes at least
  const long long rows = Tq * G / 32 + 1 < n ? n : Tq * G / 32 + 1;  // row tiles, about
  long long chunk = (Tk * Hk * ((rows + n - 1) / n) + 4 * cus - 1) / (4 * cus);
  const long long least = (Tk + kAttnMaxSplits - 1) / kAttnMaxSplits;
  chunk = chunk < least ? least : chunk;
  chunk = (chunk + pass - 1) / pass * pass;
  chunk = chunk < 2 * pass ? 2 * pass : chunk;  // (never 0: there may be no keys at all)
  plan.splits = (int)((Tk + chunk - 1) / chunk);
  plan.chunk = (int)chunk;
  // One chunk for all where the rows fill the GPU, as they do where their caches are alike (64 tokens on 64 caches of 1,760
  // keys of 8 heads of 128 86 us, 5.4 TB/s); one cache of 100,000 among 63 of 200 is then left to 8 workgroups (1.1 ms;
  // alone, in chunks, 91 us).
  if (plan.many || plan.splits <= 1 || rows * Hk >= 2 * cus) {
    plan.splits = 1;
    plan.chunk = 1 << 30;
  }
  return plan;
}

// Heads of 72 to 120 run as 128, zeros behind them (4,096 causal rows of 20 / 4 heads of 80 106 us, of 128 114, of 64 69).
template <class T>
static hipError_t launch_attention(const PackedAttnArgs& a, bool many, hipStream_t s) {
  if (a.d <= 64) return a.causal ? launch_attention_t<T, 64, true>(a, many, s) : launch_attention_t<T, 64, false>(a, many, s);
  return a.causal ? launch_attention_t<T, 128, true>(a, many, s) : launch_attention_t<T, 128, false>(a, many, s);
}

hipError_t launch_packed_attention(const PackedAttnArgs& a, bool bf16, bool many, hipStream_t s) {
  return bf16 ? launch_attention<Bf16>(a, many, s) : launch_attention<Fp16>(a, many, s);
}

}  // namespace esm
