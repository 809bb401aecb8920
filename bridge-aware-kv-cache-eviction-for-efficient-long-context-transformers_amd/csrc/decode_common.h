// What the kernels of few query rows over long caches share: the list of all sequences'
// contexts and how workgroups share it, and a wave's 32-key step (S^T = K Q^T, online softmax
// in the log2 domain, O^T += V^T P^T) with the merge of four waves.
#pragma once

#include "attn_common.h"

namespace cab {

constexpr int STEP = 32;        // keys of a wave's step
constexpr int QUAD = 4 * STEP;  // a step for each of four waves: their pieces of a context
// Pieces a workgroup of an even cut, up to which stretches begin anew with every unit (us, so
// -> running on: a tree's 256 rows, 8 units of 8128 keys 33.5 -> 40.7, of 65472 99 -> 104).
constexpr int FEW_PIECES = 32;

// The contexts of all units (a sequence's K / V head), cut into pieces, make one list, of which
// each workgroup takes an equal stretch, whatever the lengths. A: a kernel's arguments, with
// lengths (may be null: length0), most (the longest context), B, Hkv, wgs (workgroups that share the
// list) and least (the fewest pieces one takes).

__device__ __forceinline__ int context_length(const int32_t* lengths, int64_t length0, int64_t most,
                                              int b) {
  const int64_t n = lengths ? lengths[b] : length0;
  return static_cast<int>(n < 0 ? 0 : n < most ? n : most);
}

// Sums over lanes 0 .. lane of a wave (lane moves within rows of 16, then row by row).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15, 31
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// A lane's context lengths of sequences lane, lane + 64, ..; the first is kept.
template <typename A>
struct Lengths {
  const A& a;
  int first;
  __device__ __forceinline__ explicit Lengths(const A& args) : a(args), first(0) {
    if (lane_id() < a.B) first = context_length(a.lengths, a.length0, a.most, lane_id());
  }
  __device__ __forceinline__ int mine(int b0) const {  // of sequence b0 + lane, 0 past the last
    if (b0 == 0) return first;
    return b0 + lane_id() < a.B ? context_length(a.lengths, a.length0, a.most, b0 + lane_id()) : 0;
  }
  __device__ __forceinline__ int of(int b) const {  // b: the same in every lane
    return __builtin_amdgcn_readfirstlane(
        b < 64 ? __builtin_amdgcn_readlane(first, b) : context_length(a.lengths, a.length0, a.most, b));
  }
};

__device__ __forceinline__ int round_to(int x, int grain) { return (x + grain - 1) / grain * grain; }

// How the list is cut: pieces a workgroup takes, and what a unit's share of the list is
// rounded up to. An even cut takes ceil(pieces / workgroups), and its stretches run on
// from one unit into the next. Where that is only a few pieces, beginning a second part
// costs as much as the pieces: then stretches begin anew with every unit, and are as
// long as it takes for the workgroups to suffice.
struct Cut {
  int per, grain;
};
template <int KEYS>
__device__ __forceinline__ int pieces_of(int length) { return (length + KEYS - 1) / KEYS; }

template <int KEYS, typename A>
__device__ __forceinline__ Cut list_cut(const A& a, const Lengths<A>& len) {
  int all = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) all += wave_sum(pieces_of<KEYS>(len.mine(b0)));
  int per = max(a.least, (all * a.Hkv + a.wgs - 1) / a.wgs);
  if (per > FEW_PIECES || a.B * a.Hkv > a.wgs / 4) return Cut{per, 1};
  for (;; ++per) {  // (ends: one a unit suffice)
    int parts = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64)
      parts += wave_sum((pieces_of<KEYS>(len.mine(b0)) + per - 1) / per);
    if (parts * a.Hkv <= a.wgs) return Cut{per, per};
  }
}

// f(sequence, head, first piece, pieces, length) for each part of workgroup x's stretch.
template <int KEYS, typename A, typename F>
__device__ __forceinline__ void over_stretch(const A& a, int x, F f) {
  const Lengths<A> len(a);
  const Cut cut = list_cut<KEYS>(a, len);
  int at = x * cut.per;
  int before = 0, b = -1, n = 0;  // n: the sequence's pieces, rounded up
  for (int b0 = 0; b0 < a.B && b < 0; b0 += 64) {
    const int mine = round_to(pieces_of<KEYS>(len.mine(b0)), cut.grain), upto = wave_scan(mine);
    const uint64_t past = ballot64((before + upto) * a.Hkv > at);
    if (past) {
      const int i = __builtin_ctzll(past);
      b = b0 + i;
      n = __builtin_amdgcn_readlane(mine, i);
      before += __builtin_amdgcn_readlane(upto, i) - n;
    } else {
      before += __builtin_amdgcn_readlane(upto, 63);
    }
  }
  if (b < 0) return;  // past the list's end
  at -= before * a.Hkv;
  int head = at / n, piece = at - head * n;
  for (int left = cut.per; left > 0;) {
    const int length = len.of(b);
    const int take = min(left, n - piece), there = pieces_of<KEYS>(length) - piece;
    f(b, head, piece, min(take, there), length);  // (a rounded share ends in less than a stretch)
    left -= take;
    piece = 0;
    if (++head == a.Hkv) {
      head = 0;
      do {
        if (++b == a.B) return;
        n = round_to(pieces_of<KEYS>(len.of(b)), cut.grain);
      } while (n == 0);
    }
  }
}

// What weights are relative to, 2^(s c - level), for the maximum m: m c, and in fp16 15 less. There
// weights of at most 1 would lose digits from 6e-5 and be 0 from 3e-8 down, which a long
// context behind one large score adds up (140000 keys 17.4 below it: 0.4 % of the row sum
// missing in O); 2^15 more, fp16's last power of two, keeps 11 bits to 1.9e-9. Beyond 2^24 the
// level's own rounding is more than half a power of two, and nothing is added. (The factor in
// s - m instead, one operation more a score, has no such border: 4 trees of 64 over 65472 keys 346
// -> 355 us; levels formed anew in every step 334 -> 348, one token of 16 x 32768 209 -> 234.)
template <cab_dtype_t DT>
__device__ __forceinline__ float level_of(float m, float c) {
  const float mc = m * c;
  if constexpr (DT != CAB_F16) return mc;
  return __builtin_fmaf(m, c, __builtin_fabsf(mc) < 16777216.f ? -15.f : 0.f);
}
// What sums relative to the maximum m's level are multiplied by for m1's.
template <cab_dtype_t DT>
__device__ __forceinline__ float relevel(float m, float level, float m1, float level1, float c) {
  return __builtin_amdgcn_exp2f(DT == CAB_F16 ? level - level1 : (m - m1) * c);
}

// Non-temporal loads: K and V are read once, but in fp32 by every 32 rows of a unit.
template <typename T>
__device__ __forceinline__ T ld_stream(const char* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
}

// A lane's K and V values of one 32-key step (l16 = lane % 16, g = lane / 16).
// K: rows 16 tt + l16, 16 bytes at 64 j + 16 g. V: rows 16 tt + 4 g + r (number 4 tt
// + r), values (D / 16) l16 ..: output tile dt takes the dt-th of them, so that its row
// i is d = (D / 16) i + dt.
template <cab_dtype_t DT, int HD>
struct StepRegs {
  static constexpr int ES = DT == CAB_F32 ? 4 : 2;
  static constexpr int NJ = HD * ES / 64;
  static constexpr int VB = HD / 16 * ES;
  static constexpr int NV = VB / 8;
  u32x4 k[2][NJ];
  u32x2 v[8][NV];
};

// A lane's values of one key's V row.
template <int NV>
__device__ __forceinline__ void load_v(u32x2 (&v)[NV], const char* p) {
  if constexpr (NV == 1) {
    v[0] = ld_stream<u32x2>(p);
  } else {
#pragma unroll
    for (int n = 0; n < NV; n += 2) {
      const u32x4 y = ld_stream<u32x4>(p + 8 * n);
      v[n] = u32x2{y[0], y[1]};
      v[n + 1] = u32x2{y[2], y[3]};
    }
  }
}
template <int NV>
__device__ __forceinline__ void clear_v(u32x2 (&v)[NV]) {
#pragma unroll
  for (int n = 0; n < NV; ++n) v[n] = u32x2{0u, 0u};
}

template <cab_dtype_t DT, int HD, bool TAIL>
__device__ __forceinline__ void load_step(StepRegs<DT, HD>& x, const char* kp, const char* vp,
                                          uint32_t krow, uint32_t vrow, int left, int l16, int g) {
  using SR = StepRegs<DT, HD>;
#pragma unroll
  for (int tt = 0; tt < 2; ++tt) {
    const bool in = !TAIL || 16 * tt + l16 < left;
#pragma unroll
    for (int j = 0; j < SR::NJ; ++j) {
      x.k[tt][j] = u32x4{0u, 0u, 0u, 0u};
      if (in) x.k[tt][j] = ld_stream<u32x4>(kp + ((16u * tt + l16) * krow + 64u * j + 16u * g));
    }
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int key = 16 * (r >> 2) + 4 * g + (r & 3);
    const bool in = !TAIL || key < left;
    const char* p = vp + (static_cast<uint32_t>(key) * vrow + SR::VB * l16);
    if constexpr (SR::NV == 1) {
      x.v[r][0] = u32x2{0u, 0u};
      if (in) x.v[r][0] = ld_stream<u32x2>(p);
    } else {
#pragma unroll
      for (int n = 0; n < SR::NV; n += 2) {
        u32x4 y = {0u, 0u, 0u, 0u};
        if (in) y = ld_stream<u32x4>(p + 8 * n);
        x.v[r][n] = u32x2{y[0], y[1]};
        x.v[r][n + 1] = u32x2{y[2], y[3]};
      }
    }
  }
}

__device__ __forceinline__ f32x4 mfma4(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Two weights' upper 16 bits (rounded towards 0), as fp32 again, and the least operand that is no zero.
template <bool BF16>
__device__ __forceinline__ uint32_t cut2(float lo, float hi) {
  if constexpr (BF16)
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi));
}
template <bool BF16>
__device__ __forceinline__ float low_half(uint32_t x) {
  return BF16 ? __uint_as_float(x << 16) : f16_to_f32(static_cast<uint16_t>(x));
}
template <bool BF16>
__device__ __forceinline__ float high_half(uint32_t x) {
  return BF16 ? __uint_as_float(x & 0xffff0000u) : f16_to_f32(static_cast<uint16_t>(x >> 16));
}
template <bool BF16> constexpr float LEAST = BF16 ? 0x1p-126f : 0x1p-24f;
// What whole weights are multiplied by as operands (in fp16 they keep 11 bits to 1.9e-9 so, not to 6e-5).
template <bool BF16> constexpr float WEIGHT = BF16 ? 1.f : 0x1p15f;

// The maximum of no scores. WHOLE: no finite score lies below it.
template <bool WHOLE> constexpr float NO_SCORE = WHOLE ? -0x1.fffffep127f : M_EMPTY;

// QT tiles of 16 query rows and what they have seen, of one wave (l16 = lane % 16: a
// tile's row, g = lane / 16). WHOLE: weights are 2^((s - m) c) for the maximum m, with the difference
// formed first, whatever the scores' size, where else they are relative to a rounded level, which for scores
// of 2^31 and more can be more than 2^128 away from them; and the second product takes them in all their digits.
template <cab_dtype_t DT, int HD, int QT, bool WHOLE = false>
struct RowState {
  static constexpr bool F32 = DT == CAB_F32, BF16 = DT == CAB_BF16;
  static constexpr int NDT = HD / 16;
  using SR = StepRegs<DT, HD>;
  static constexpr int NJ = SR::NJ;
  f32x4 o[QT][NDT];
  float l[QT], m[QT], level[WHOLE ? 1 : QT];  // l: of this lane's keys alone

  __device__ __forceinline__ void clear(float c) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      l[qt] = 0.f;
      m[qt] = NO_SCORE<WHOLE>;
      if constexpr (!WHOLE) level[qt] = level_of<DT>(M_EMPTY, c);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[qt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // Whether a sum of this wave's is NaN (or some are infinities of both signs). By its bits: comparisons
  // may not tell.
  __device__ __forceinline__ bool not_a_number() const {
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) y += o[qt][dt];
    const float t = (y[0] + y[1]) + (y[2] + y[3]);
    uint32_t bits = __float_as_uint(t);
    asm("" : "+v"(bits));
    return __builtin_amdgcn_ballot_w64((bits & 0x7fffffffu) > 0x7f800000u) != 0;
  }

  // 32 keys; with `some`, of those alone for which in(tt, r) (key 16 tt + 4 g + r). WHOLE: 16-bit weights
  // (in fp16 times 2^15) as operands of their upper bits and of what those leave, so that only the
  // output's rounding is left: two in fp16 (22 bits, as far as they lie above 2^-24), three in bf16 (all 24. With
  // two, 16 bits, one output in 300 rounded to its other neighbour; 1 - e^-t was off by 2^-17). An operand of 0
  // times an infinite V is NaN, so weights that are not 0 have none that is: in bf16 they are 2^-126 at the
  // least. fp16's least is 2^-24, which many keys would add up: there it is with NONE_0 alone, for a second walk
  // over rows whose sums became NaN.
  template <bool NONE_0 = false, typename F>
  __device__ __forceinline__ void step(const SR& x, const u32x4 (&qr)[QT][NJ], float c, bool some, F in) {
    f32x4 sc[QT][2];  // [qt][tt][r]: key 16 tt + 4 g + r, row 16 qt + l16
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) sc[qt][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t kx = x.k[tt][j][e], qx = qr[qt][j][e];
              sc[qt][tt] = mfma4(__uint_as_float(kx), __uint_as_float(qx), sc[qt][tt]);
            }
          } else {
            sc[qt][tt] = mfma16<BF16>(x.k[tt][j], qr[qt][j], sc[qt][tt]);
          }
        }
    if (some) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!in(tt, r)) sc[qt][tt][r] = -INFINITY;
    }
    u32x4 pb[QT], rest[QT], last[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float m0 = fmaxf(fmaxf(sc[qt][0][0], sc[qt][0][1]), fmaxf(sc[qt][0][2], sc[qt][0][3]));
      const float m1 = fmaxf(fmaxf(sc[qt][1][0], sc[qt][1][1]), fmaxf(sc[qt][1][2], sc[qt][1][3]));
      float mx = fmaxf(m0, m1), mdup = mx;
      colmax2(mx, mdup);
      if (__builtin_amdgcn_ballot_w64(mx > m[qt]) != 0) {
        const float mn = fmaxf(mx, m[qt]);
        const float upto = WHOLE ? 0.f : level_of<DT>(mn, c);
        const float alpha = WHOLE ? __builtin_amdgcn_exp2f((m[qt] - mn) * c) : relevel<DT>(m[qt], level[qt], mn, upto, c);
        l[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[qt][dt] *= alpha;
        m[qt] = mn;
        if constexpr (!WHOLE) level[qt] = upto;
      }
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sc[qt][tt][r] = __builtin_amdgcn_exp2f(WHOLE ? (sc[qt][tt][r] - m[qt]) * c
                                                       : __builtin_fmaf(sc[qt][tt][r], c, -level[qt]));
      const f32x4 s2 = sc[qt][0] + sc[qt][1];
      l[qt] += (s2[0] + s2[1]) + (s2[2] + s2[3]);
      if constexpr (!F32 && WHOLE) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            const int at = 2 * tt + r / 2;
            float x[2] = {sc[qt][tt][r] * WEIGHT<BF16>, sc[qt][tt][r + 1] * WEIGHT<BF16>};
            const float least[2] = {x[0] > 0.f ? LEAST<BF16> : x[0], x[1] > 0.f ? LEAST<BF16> : x[1]};
            auto keep = [&]() {
              if constexpr (NONE_0 || BF16) {
                x[0] = fmaxf(x[0], least[0]);
                x[1] = fmaxf(x[1], least[1]);
              }
            };
            auto less = [&](uint32_t cut) {
              x[0] -= low_half<BF16>(cut);
              x[1] -= high_half<BF16>(cut);
              keep();
            };
            if constexpr (!BF16) keep();
            pb[qt][at] = cut2<BF16>(x[0], x[1]);
            less(pb[qt][at]);
            if constexpr (BF16) {
              rest[qt][at] = cut2<true>(x[0], x[1]);
              less(rest[qt][at]);
              last[qt][at] = cut2<true>(x[0], x[1]);
            } else {
              rest[qt][at] = pack2<false>(x[0], x[1]);
            }
          }
      } else if constexpr (!F32) {
        pb[qt] = u32x4{pack2<BF16>(sc[qt][0][0], sc[qt][0][1]), pack2<BF16>(sc[qt][0][2], sc[qt][0][3]),
                       pack2<BF16>(sc[qt][1][0], sc[qt][1][1]), pack2<BF16>(sc[qt][1][2], sc[qt][1][3])};
      }
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      if constexpr (F32) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const uint32_t vx = x.v[r][dt >> 1][dt & 1];
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
            o[qt][dt] = mfma4(__uint_as_float(vx), sc[qt][r >> 2][r & 3], o[qt][dt]);
        }
      } else {
        u32x4 vo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t lo = x.v[2 * e][dt >> 2][(dt >> 1) & 1];
          const uint32_t hi = x.v[2 * e + 1][dt >> 2][(dt >> 1) & 1];
          vo[e] = __builtin_amdgcn_perm(hi, lo, dt & 1 ? 0x07060302u : 0x05040100u);
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          o[qt][dt] = mfma16<BF16>(vo, pb[qt], o[qt][dt]);
          if constexpr (WHOLE) o[qt][dt] = mfma16<BF16>(vo, rest[qt], o[qt][dt]);
          if constexpr (WHOLE && BF16) o[qt][dt] = mfma16<BF16>(vo, last[qt], o[qt][dt]);
        }
      }
    }
  }
};

// Merge of four waves' rows: common maximum, then the scaled O^T and sums in wave order.
// value(qt, e, y) gets values e = 64 dt + lane of a tile's O^T, sums(qt, level, sum) a row's level
// (WHOLE: its maximum) and sum (threads 0 .. 15: the row). sum() is there for both.
template <cab_dtype_t DT, int HD, int QT, bool WHOLE = false>
struct RowMerge {
  static constexpr int NDT = HD / 16;
  f32x4 o[4][NDT * 64];  // one query tile's O^T per wave
  float m[4][QT][16], l[4][QT][16];

  __device__ __forceinline__ float sum(int qt, int row) const {
    return (l[0][qt][row] + l[1][qt][row]) + (l[2][qt][row] + l[3][qt][row]);
  }

  template <typename V, typename S>
  __device__ __forceinline__ void run(RowState<DT, HD, QT, WHOLE>& x, int w, int lane, float c, V value, S sums) {
    const int l16 = lane & 15, g = lane >> 4;
    __syncthreads();  // (the last part's merge has been read)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      x.l[qt] += shfl_xor_f32(x.l[qt], 16);
      x.l[qt] += shfl_xor_f32(x.l[qt], 32);
      if (g == 0) m[w][qt][l16] = x.m[qt];
    }
    __syncthreads();
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float mm = fmaxf(fmaxf(m[0][qt][l16], m[1][qt][l16]), fmaxf(m[2][qt][l16], m[3][qt][l16]));
      const float upto = WHOLE ? mm : level_of<DT>(mm, c);
      const float f = WHOLE ? __builtin_amdgcn_exp2f((x.m[qt] - mm) * c)
                            : relevel<DT>(x.m[qt], x.level[qt], mm, upto, c);
      const float fo = WHOLE && DT == CAB_F16 ? f * (1.f / WEIGHT<false>) : f;
      if (g == 0) l[w][qt][l16] = x.l[qt] * f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[w][dt * 64 + lane] = x.o[qt][dt] * fo;
      __syncthreads();
      for (int e = threadIdx.x; e < NDT * 64; e += 256)
        value(qt, e, (o[0][e] + o[1][e]) + (o[2][e] + o[3][e]));
      if (threadIdx.x < 16) sums(qt, upto, sum(qt, l16));
      if (qt + 1 < QT) __syncthreads();
    }
  }
};

// Eight values of a row in fp32.
template <cab_dtype_t DT>
__device__ __forceinline__ void load8(const char* p, float* x) {
  if constexpr (DT == CAB_F32) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    const u32x4 a = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = a[i >> 1];
      const uint16_t h = static_cast<uint16_t>(i & 1 ? w >> 16 : w);
      x[i] = DT == CAB_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
    }
  }
}

}  // namespace cab
