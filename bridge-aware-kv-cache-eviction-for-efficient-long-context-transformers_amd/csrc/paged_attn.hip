// Attention of one token a sequence over a cache in pages (cab_paged_attn_fwd). Sequence b's key s
// lies in page table[b][s / S] at place s % S; the query heads that share a K / V head are the
// R = group rows of one unit, and see the keys s < lengths[b] whose page is there.
//
//  1. The contexts of all units, cut into pieces of 128 keys, make one list of which each
//     workgroup takes an equal stretch. Every wave walks its own 32-key steps, K and V straight
//     from the pages into matrix operands (S^T = K Q^T, online softmax, weights 2^((s - m) c),
//     O^T += V^T P^T; maxima, sums and O in fp32; P as 16-bit operands of its upper bits and of what
//     those leave, two in fp16 and three in bf16, so that only the output is rounded; each further
//     product costs some 0.4 us of 10 at 600 keys, 1 % where pages are of 8 and nothing that shows at other
//     long contexts; fp32 on the fp32 matrix instructions). A part that is all of a unit
//     is finished there; of the others one partial (maximum, row sum, O) is left per row.
//  2. join_kernel, one wave per row, merges the partials. Where one workgroup a unit does
//     (paged_plan), there are none and it is not launched.
//
// Pages. Of sizes in whole 16 keys, a 16-key block lies in one page: a lane of the wave looks up
// one block each of the next 32 steps, and a step takes its two blocks' pages out of the lanes as
// scalars, so that no load waits for the table and addresses are a scalar base and a fixed
// offset a lane. Of other sizes the blocks are of 8, 4, 2 or 1 keys, which divide the size, and
// the lanes that load a key's parts fetch its block's page from the lane that holds it (a
// look-up of 32 keys a step, one step ahead: 100 keys in pages of 24 6.8 us, of which 5.1 are left;
// 16 sequences of up to 32768 in pages of 8 260, 248).
// Rows past the length or without a page are not read: zeros take their place, scores -inf.
//
// Bound: HBM (K and V, read once); short caches: the latency of a start, a few steps and a merge.
// Measured, D = 128: 16 sequences of up to 32768 keys, 32 heads on 8, bf16, pages of 16, 205 + 4.6 us
// (contexts + join; 6.6 TB/s of K and V; with pages in order, or of 64, the same within 4 %); one of 128000
// keys, 28 heads on 4, fp16, 46 + 5.3; one of 600, bf16, 10.7 in a graph, alone. fp32, D = 64, pages of 24: 3 x 12
// heads of up to 5003 keys 16.5 + 4.1.
#include "decode_common.h"
#include "row_layout.h"

namespace cab {
namespace {

constexpr float NO_KEY = -1.f;  // (a sum of weights is 0 or more, or NaN)

struct PagedArgs {
  const char* q;
  const char* k;
  const char* v;
  int64_t qs[2], ks[3], vs[3];  // bytes: b, h; page, h, place
  const int32_t* lengths;       // (the fields that decode_common.h asks for)
  int64_t length0, most;
  int32_t B, Hkv, wgs, least;
  const int32_t* table;
  int64_t table_ld;
  int32_t pages, size;
  int32_t shift;   // a block of 2^shift keys lies in one page
  uint64_t magic;  // 2^64 / (blocks of a page) rounded up; 0: by 1
  int32_t group, H;
  int32_t direct;  // a workgroup a unit
  float c;         // scale * log2(e)
  char* out;
  int64_t os[2];  // bytes: b, h
  float* lse;     // [B, H], may be null
  // Partials; workgroup x's of unit u is number x + u.
  float* po;  // [number][group][D]
  float* pm;  // [number][group] the maximum score
  float* pl;  // [number][group] row sums, NO_KEY where none was seen
};

// x / d for x d < 2^64.
__device__ __forceinline__ uint32_t divided(uint32_t x, uint64_t magic) {
  return magic ? static_cast<uint32_t>(__umul64hi(static_cast<uint64_t>(x), magic)) : x;
}

// The bits of a row's log-sum-exp: -inf with no key seen; NaN where keys are seen but have no
// softmax (a score of NaN or +inf, or all -inf: the sum is NaN or 0). Bits, tested and stored as
// such, because this file is compiled with -fno-honor-nans.
__device__ __forceinline__ uint32_t lse_bits(bool any, float m, float sum, float c) {
  int32_t bits = __builtin_bit_cast(int32_t, sum);
  asm("" : "+v"(bits));  // (or the test is made one of floats)
  const float x = __builtin_fmaf(m, c, __log2f(sum)) * 0.69314718055994531f;
  const uint32_t y = bits > 0 && bits <= 0x7f800000 ? __builtin_bit_cast(uint32_t, x) : 0x7fc00000u;
  return any ? y : 0xff800000u;
}

// BLOCKS: pages hold whole 16-key blocks. Grid: (workgroups or units, row tiles of 16 QT rows).
template <cab_dtype_t DT, int HD, int QT, bool BLOCKS>
__global__ __launch_bounds__(256, DT == CAB_F32 ? 1 : 2) void paged_kernel(PagedArgs a) {
  constexpr bool F32 = DT == CAB_F32, BF16 = DT == CAB_BF16;
  constexpr int NDT = HD / 16;
  using SR = StepRegs<DT, HD>;
  constexpr int NJ = SR::NJ;
  // (Two register sets spill with 32 rows of 128 in 16 bits, and gain nothing in fp32 but for 16 rows
  // of 64: 8 x 4 heads of 5000 keys 28.0 -> 26.2 us.)
  constexpr bool ONE_SET = F32 ? QT * HD > 64 : QT * HD > 128;
  __shared__ RowMerge<DT, HD, QT, true> merge;
  __shared__ int seen_by[4];

  const int row0 = blockIdx.y * (16 * QT);
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const float c = a.c;
  const uint32_t krow = static_cast<uint32_t>(a.ks[2]), vrow = static_cast<uint32_t>(a.vs[2]);

  auto part_of = [&](int b, int hk, int piece, int pieces, int len) {
    int lane = lane_id();
    asm volatile("" : "+v"(lane));  // (what follows from it is not kept over the parts)
    const int l16 = lane & 15, g = lane >> 4;
    const char* kb = a.k + hk * a.ks[1];
    const char* vb = a.v + hk * a.vs[1];
    const int32_t* table = a.table + b * a.table_ld;
    u32x4 qr[QT][NJ];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int r = row0 + 16 * qt + l16;
      const char* qp = a.q + b * a.qs[0] + (static_cast<int64_t>(hk) * a.group + r) * a.qs[1];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        qr[qt][j] = u32x4{0u, 0u, 0u, 0u};
        if (r < a.group) qr[qt][j] = *reinterpret_cast<const u32x4*>(qp + 64 * j + 16 * g);
      }
    }
    RowState<DT, HD, QT, true> rows;
    int seen = 0;

    const int end = min((len + STEP - 1) / STEP, 4 * (piece + pieces));
    const int begin = 4 * piece + w;

    // Pages of this wave's steps: lane (i << per) + j holds that of block j of step from + 4 i, and the
    // block's place in it.
    const int shift = BLOCKS ? 4 : a.shift, per = 5 - shift;
    const int kept = 64 >> per;  // steps that a look-up serves
    auto look_up = [&](int from, int& page, int& place) {
      page = -1;
      place = 0;
      const int step = from + 4 * (lane >> per);
      const int block = (step << per) + (lane & ((1 << per) - 1));
      if (step < end && block << shift < len) {
        const uint32_t col = divided(block, a.magic);
        page = table[col];
        place = (block - col * (a.size >> shift)) << shift;
      }
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) page = -1;
    };
    struct Step {
      SR x;
      uint32_t in;  // bit 4 tt + r: key 16 tt + 4 g + r is there
    };
    auto load = [&](int step, int slot, int page, int place, Step& s) __attribute__((always_inline)) {
      const int left = len - STEP * step;
      s.in = 0;
      if constexpr (BLOCKS) {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int p = __builtin_amdgcn_readlane(page, 2 * slot + tt);
          const int at = __builtin_amdgcn_readlane(place, 2 * slot + tt);
          const int rest = p < 0 ? 0 : left - 16 * tt;
          const char* kp = kb + p * a.ks[0] + at * a.ks[2];
          const char* vp = vb + p * a.vs[0] + at * a.vs[2];
          if (rest >= 16) {
            s.in |= 15u << (4 * tt);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
              s.x.k[tt][j] = ld_stream<u32x4>(kp + (l16 * krow + 64u * j + 16u * g));
#pragma unroll
            for (int r = 0; r < 4; ++r) load_v(s.x.v[4 * tt + r], vp + ((4u * g + r) * vrow + SR::VB * l16));
          } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              s.x.k[tt][j] = u32x4{0u, 0u, 0u, 0u};
              if (l16 < rest) s.x.k[tt][j] = ld_stream<u32x4>(kp + (l16 * krow + 64u * j + 16u * g));
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              clear_v(s.x.v[4 * tt + r]);
              if (4 * g + r < rest) {
                s.in |= 1u << (4 * tt + r);
                load_v(s.x.v[4 * tt + r], vp + ((4u * g + r) * vrow + SR::VB * l16));
              }
            }
          }
        }
      } else {
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const int key = 16 * tt + l16, from = (slot << per) + (key >> shift);
          const int p = __shfl(page, from, 64), at = __shfl(place, from, 64) + (key & ((1 << shift) - 1));
          const char* kp = kb + p * a.ks[0] + at * a.ks[2];
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            s.x.k[tt][j] = u32x4{0u, 0u, 0u, 0u};
            if (p >= 0 && key < left) s.x.k[tt][j] = ld_stream<u32x4>(kp + 64u * j + 16u * g);
          }
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int key = 16 * (r >> 2) + 4 * g + (r & 3);
          const int from = (slot << per) + (key >> shift);
          const int p = __shfl(page, from, 64), at = __shfl(place, from, 64) + (key & ((1 << shift) - 1));
          clear_v(s.x.v[r]);
          if (p >= 0 && key < left) {
            s.in |= 1u << r;
            load_v(s.x.v[r], vb + p * a.vs[0] + at * a.vs[2] + SR::VB * l16);
          }
        }
      }
    };
    auto compute = [&](const Step& s, auto none_0) __attribute__((always_inline)) {
      const uint64_t some = __builtin_amdgcn_ballot_w64(s.in != 255u);
      seen |= static_cast<int>(__builtin_amdgcn_ballot_w64(s.in != 0) != 0);
      rows.template step<decltype(none_0)::value>(
          s.x, qr, c, some != 0, [&](int tt, int r) { return (s.in >> (4 * tt + r) & 1u) != 0; });
    };

    auto walk = [&](auto none_0) __attribute__((always_inline)) {
      rows.clear(c);
      seen = 0;
      int page, place;
      look_up(begin, page, place);
      if constexpr (ONE_SET || decltype(none_0)::value) {
        Step x;
        int n = 0;
        for (int step = begin; step < end; step += 4) {
          load(step, n, page, place, x);
          if (++n == kept) {
            n = 0;
            look_up(step + 4, page, place);
          }
          compute(x, none_0);
        }
      } else {
        // Two register sets: a step's loads are in flight while the one before it is computed.
        Step x, y;
        int n = 1;
        if (begin < end) load(begin, 0, page, place, x);
        for (int step = begin; step < end; step += 8) {
          if (step + 4 < end) load(step + 4, n, page, place, y);
          if (++n == kept) {
            n = 0;
            look_up(step + 8, page, place);
          }
          compute(x, none_0);
          if (step + 4 < end) {
            if (step + 8 < end) load(step + 8, n, page, place, x);
            ++n;
            compute(y, none_0);
          }
        }
      }
    };
    walk(std::false_type{});
    if constexpr (DT == CAB_F16) {  // (an infinite V times an operand of 0)
      if (__builtin_expect(rows.not_a_number(), 0)) walk(std::true_type{});
    }

    if (lane == 0) seen_by[w] = seen;  // (read behind the merge's barriers, written before its first)
    const bool whole = a.direct || (piece == 0 && pieces == pieces_of<QUAD>(len));
    const int64_t part = static_cast<int64_t>(blockIdx.x) + b * a.Hkv + hk;
    merge.run(
        rows, w, lane, c,
        [&](int qt, int e, const f32x4& y) {
          const int dt = e >> 6, ll = e & 63, row = row0 + 16 * qt + (ll & 15), d0 = 4 * (ll >> 4);
          if (row >= a.group) return;
          if (!whole) {
            float* po = a.po + (part * a.group + row) * HD;
#pragma unroll
            for (int r = 0; r < 4; ++r) po[NDT * (d0 + r) + dt] = y[r];
          } else {
            const bool any = (seen_by[0] | seen_by[1] | seen_by[2] | seen_by[3]) != 0;
            const float f = 1.f / merge.sum(qt, ll & 15);  // (0 of scores that are all -inf: 0 / 0)
            char* op = a.out + b * a.os[0] + (static_cast<int64_t>(hk) * a.group + row) * a.os[1];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float z = any ? y[r] * f : 0.f;
              const int d = NDT * (d0 + r) + dt;
              if constexpr (F32) reinterpret_cast<float*>(op)[d] = z;
              else reinterpret_cast<uint16_t*>(op)[d] = static_cast<uint16_t>(pack2<BF16>(z, z));
            }
          }
        },
        [&](int qt, float m, float sum) {
          const int row = row0 + 16 * qt + static_cast<int>(threadIdx.x);
          if (row >= a.group) return;
          const bool any = (seen_by[0] | seen_by[1] | seen_by[2] | seen_by[3]) != 0;
          if (!whole) {
            a.pm[part * a.group + row] = any ? m : -INFINITY;
            a.pl[part * a.group + row] = any ? sum : NO_KEY;
          } else if (a.lse) {
            const int64_t at = static_cast<int64_t>(b) * a.H + static_cast<int64_t>(hk) * a.group + row;
            reinterpret_cast<uint32_t*>(a.lse)[at] = lse_bits(any, m, sum, c);
          }
        });
    __syncthreads();  // (seen_by and the sums have been read)
  };

  if (a.direct) {
    const int b = blockIdx.x / a.Hkv, hk = blockIdx.x - b * a.Hkv;
    const int len = context_length(a.lengths, a.length0, a.most, b);
    part_of(b, hk, 0, pieces_of<QUAD>(len), len);
  } else {
    over_stretch<QUAD>(a, blockIdx.x, part_of);
  }
}

// WAVES waves per row; groups of D / 8 lanes, each lane eight of the row's values. A group takes
// every G-th partial. (Four waves where rows are few, and so partials many: 28 rows of 64
// partials 7.5 -> 5.3 us.)
template <cab_dtype_t DT, int HD, int WAVES>
__global__ __launch_bounds__(256) void join_kernel(PagedArgs a) {
  constexpr int LG = HD / 8, ES = DT == CAB_F32 ? 4 : 2;
  constexpr int GROUPS = 64 / LG, G = GROUPS * WAVES;
  __shared__ float sums[WAVES], rows[WAVES][HD];
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = lane_id(), at = lane % LG, grp = lane / LG + (WAVES > 1 ? w * GROUPS : 0);
  const int64_t id = WAVES > 1 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + w;
  if (id >= static_cast<int64_t>(a.B) * a.H) return;
  const int b = static_cast<int>(id / a.H), h = static_cast<int>(id - static_cast<int64_t>(b) * a.H);
  const int hk = h / a.group;
  const Lengths<PagedArgs> lens(a);
  const Cut cut = list_cut<QUAD>(a, lens);
  int before = 0, len = 0;  // the sequences' shares of the list before b; b's context
  for (int b0 = 0; b0 <= b; b0 += 64) {
    const int mine = lens.mine(b0);
    before += wave_sum(b0 + lane < b ? round_to(pieces_of<QUAD>(mine), cut.grain) : 0);
    len = __builtin_amdgcn_readlane(mine, b & 63);  // (the last round's)
  }
  // The unit's partials: of the workgroups whose stretches meet its pieces.
  const int pieces = pieces_of<QUAD>(len);
  const int start = before * a.Hkv + hk * round_to(pieces, cut.grain), first = start / cut.per;
  const int parts = pieces ? (start + pieces - 1) / cut.per - first + 1 : 0;
  if (parts == 1) return;  // (finished by the workgroup that had all of it)
  const int64_t row = (static_cast<int64_t>(first) + b * a.Hkv + hk) * a.group + (h - hk * a.group);
  // (whether a key was seen goes by bits: sums may be NaN, and comparisons of those say anything)
  float m = -INFINITY;
  bool some = false;
  for (int x = lane; x < parts; x += 64) {
    const int64_t y = row + static_cast<int64_t>(x) * a.group;
    m = fmaxf(m, a.pm[y]);
    some = some || reinterpret_cast<const uint32_t*>(a.pl)[y] != __builtin_bit_cast(uint32_t, NO_KEY);
  }
  const bool any = ballot64(some) != 0;  // (the same for all waves of a row)
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, shfl_xor_f32(m, off));
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f;
  if (any) {
#pragma unroll 4
    for (int x = grp; x < parts; x += G) {
      const int64_t y = row + static_cast<int64_t>(x) * a.group;
      const float f = __builtin_amdgcn_exp2f((a.pm[y] - m) * a.c);
      l += a.pl[y] * f;
      const f32x4* po = reinterpret_cast<const f32x4*>(a.po + y * HD) + 2 * at;
      const f32x4 y0 = po[0], y1 = po[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] += y0[e] * f;
        o[4 + e] += y1[e] * f;
      }
    }
#pragma unroll
    for (int off = LG; off < 64; off <<= 1) l += shfl_xor_f32(l, off);
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int off = LG; off < 64; off <<= 1) o[e] += shfl_xor_f32(o[e], off);
    if constexpr (WAVES > 1) {
      if (lane < LG) {
#pragma unroll
        for (int e = 0; e < 8; ++e) rows[w][8 * at + e] = o[e];
        if (lane == 0) sums[w] = l;
      }
      __syncthreads();
      l = 0.f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) l += sums[v];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o[e] = 0.f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) o[e] += rows[v][8 * at + e];
      }
    }
    const float f = 1.0f / l;  // (of scores that are all -inf: 0 / 0)
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= f;
  }
  if (grp != 0) return;
  char* op = a.out + b * a.os[0] + h * a.os[1] + at * 8 * ES;
  if constexpr (DT == CAB_F32) {
    reinterpret_cast<f32x4*>(op)[0] = f32x4{o[0], o[1], o[2], o[3]};
    reinterpret_cast<f32x4*>(op)[1] = f32x4{o[4], o[5], o[6], o[7]};
  } else {
    constexpr bool BF16 = DT == CAB_BF16;
    *reinterpret_cast<u32x4*>(op) = u32x4{pack2<BF16>(o[0], o[1]), pack2<BF16>(o[2], o[3]),
                                          pack2<BF16>(o[4], o[5]), pack2<BF16>(o[6], o[7])};
  }
  if (at == 0 && a.lse) reinterpret_cast<uint32_t*>(a.lse)[id] = lse_bits(any, m, l, a.c);
}

struct PagedPlan {
  int64_t units, row_tiles, wgs;
  bool direct;
  size_t off_pm, off_pl, bytes;
};

// Workgroups that share the list: one a CU, or two where there are many units and so many parts a
// workgroup, whose beginnings and ends the other one then fills (16 bits; us, one -> two a CU: 1024
// units of up to 2048 keys 140 -> 130, 512 of up to 4096 129 -> 124, but 4 of 128000 57 -> 59), or rows are
// of 64, whose steps leave half as many bytes in flight (128 units of up to 32768 keys 150 -> 118, 8 of
// 128000 67 -> 53, of 4096 10.4 both).
constexpr int WGS = 256;
constexpr int64_t MANY_UNITS = 512;
// Places a sequence up to which a workgroup does a unit alone, without partials and join: of 16 bits,
// of fp32 (as values of a row's length, whose matrix instructions take seven times as long), and where there
// is a unit a CU (us, list -> alone: bf16, D = 128, 8 units of 608 keys 10.8 -> 10.6, 640 10.9 -> 11.0, 704 10.8 ->
// 11.7; 32 of 640 11.6 -> 15.1; 128 of 640 19.1 -> 15.8, 768 17.2 -> 18.5; D = 64, 8 units of 640 9.3 -> 8.3, 768
// 9.4 -> 9.2, 1024 9.8 -> 14.6; 32 of 640 10.1 -> 11.2; 128 of 768 14.6 -> 13.7, 1024 15.1 -> 17.2; a unit a CU,
// D = 128, 1024 28.6 -> 25.5, 1536 38.7 -> 35.6, D = 64, 1024 19.6 -> 18.3, 1536 24.5 -> 25.1; 1024 units of up to 1024 86
// -> 81, of up to 4096 256 -> 274; fp32, 8 units, D = 128, 200 keys 12.3 -> 11.2, 256 13.3 -> 13.6, 320 14.0 -> 17.5;
// D = 64, 400 11.1 -> 10.6, 512 10.9 -> 11.4; 256 units, D = 128, of 1024 56 -> 53).
constexpr int64_t BRIEF = 640, BRIEF_VALUES = 25600, BRIEF_FILLED = 1024;

PagedPlan paged_plan(cab_dtype_t dtype, int64_t B, int64_t H, int64_t Hkv, int64_t most, int64_t D) {
  PagedPlan p;
  const int64_t group = H / Hkv;
  p.units = B * Hkv;
  p.row_tiles = ceil_div(group, group <= 16 ? 16 : 32);
  p.direct = most <= (p.units >= WGS ? BRIEF_FILLED : dtype == CAB_F32 ? BRIEF_VALUES / D : BRIEF);
  const int64_t list = p.units * ceil_div(most, QUAD);
  const int64_t slots = dtype != CAB_F32 && (D == 64 || p.units >= MANY_UNITS) ? 2 * WGS : WGS;
  p.wgs = ceil_div(slots, p.row_tiles);
  if (p.wgs > list) p.wgs = list;
  if (p.wgs < 1) p.wgs = 1;
  const int64_t parts = p.direct ? 0 : (p.wgs + p.units) * group;
  p.off_pm = static_cast<size_t>(parts * D) * 4;
  p.off_pl = p.off_pm + static_cast<size_t>(round_up(parts, 4)) * 4;
  p.bytes = p.off_pl + static_cast<size_t>(round_up(parts, 4)) * 4;
  return p;
}

// Rows up to which four waves join each (us, one -> four: 32 rows, 128000 keys 46.6 -> 43.4, 256 of up to
// 16000 73 -> 65, 512 of up to 8000 63 -> 65).
constexpr int64_t FEW_JOINED = 256;

bool paged_sizes(int64_t B, int64_t H, int64_t Hkv, int64_t columns, int64_t size, int64_t D) {
  return B >= 1 && B <= 65535 && Hkv >= 1 && H >= Hkv && H % Hkv == 0 && H <= 65535 && columns >= 0 &&
         size >= 1 && size <= INT32_MAX && columns <= (INT32_MAX - 1024) / size &&
         (D == 64 || D == 128) &&
         // (the list of pieces fits 32 bits; the launches' threads are fewer than 2^32)
         B * Hkv <= INT32_MAX / 2 / (columns * size / 64 + 1) && B * H <= (int64_t{1} << 26) - 4 &&
         B * Hkv <= (int64_t{1} << 24) - 1;
}

template <cab_dtype_t DT, int HD>
void launch(const PagedPlan& pl, const PagedArgs& a, bool blocks, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(pl.direct ? pl.units : pl.wgs), static_cast<unsigned>(pl.row_tiles));
  if (pl.direct || a.most > 0) {
    if (a.group <= 16 && blocks) paged_kernel<DT, HD, 1, true><<<grid, 256, 0, s>>>(a);
    else if (a.group <= 16) paged_kernel<DT, HD, 1, false><<<grid, 256, 0, s>>>(a);
    else if (blocks) paged_kernel<DT, HD, 2, true><<<grid, 256, 0, s>>>(a);
    else paged_kernel<DT, HD, 2, false><<<grid, 256, 0, s>>>(a);
  }
  if (pl.direct) return;
  const int64_t rows = static_cast<int64_t>(a.B) * a.H;
  if (rows <= FEW_JOINED)
    join_kernel<DT, HD, 4><<<static_cast<unsigned>(rows), 256, 0, s>>>(a);
  else
    join_kernel<DT, HD, 1><<<static_cast<unsigned>(ceil_div(rows, 4)), 256, 0, s>>>(a);
}

}  // namespace
}  // namespace cab

using namespace cab;

extern "C" size_t cab_paged_attn_workspace_bytes(cab_dtype_t dtype, int64_t B, int64_t H, int64_t H_kv, int64_t columns,
                                                 int64_t page_size, int64_t D) {
  if (!valid_dtype(dtype) || !paged_sizes(B, H, H_kv, columns, page_size, D)) return 0;
  return paged_plan(dtype, B, H, H_kv, columns * page_size, D).bytes;
}

extern "C" cab_status_t cab_paged_attn_fwd(
    const void* q, const void* k_pages, const void* v_pages, cab_dtype_t dtype, int64_t B, int64_t H,
    int64_t H_kv, int64_t D, int64_t pages, int64_t page_size, const int64_t q_strides[4],
    const int64_t k_strides[4], const int64_t v_strides[4], const int64_t o_strides[4],
    const int32_t* table, int64_t table_stride, int64_t columns, const int32_t* lengths, float scale,
    void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "cab_paged_attn_fwd";
  clear_error();
  CAB_REQUIRE(valid_dtype(dtype), CAB_EDTYPE, "%s: unknown dtype %d", fn, static_cast<int>(dtype));
  CAB_REQUIRE(D == 64 || D == 128, CAB_ESHAPE, "%s: D must be 64 or 128 (got %lld)", fn, (long long)D);
  CAB_REQUIRE(B >= 0 && H >= 1 && H_kv >= 1 && H % H_kv == 0, CAB_ESHAPE,
              "%s: H must be a multiple of H_kv", fn);
  CAB_REQUIRE(pages >= 0 && page_size >= 1 && columns >= 0, CAB_ESHAPE, "%s: bad shape of the pages", fn);
  if (B == 0) return CAB_OK;
  CAB_REQUIRE(paged_sizes(B, H, H_kv, columns, page_size, D) && pages <= INT32_MAX, CAB_ESHAPE,
              "%s: problem too large", fn);
  const bool none = pages == 0 || columns == 0;  // (nobody sees a key)
  CAB_REQUIRE(q && out && q_strides && k_strides && v_strides && o_strides && lengths, CAB_EINVAL,
              "%s: null argument", fn);
  CAB_REQUIRE(none || (k_pages && v_pages && table), CAB_EINVAL, "%s: null argument", fn);
  const float c = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  CAB_REQUIRE(std::isfinite(c) && c > 0.f, CAB_EINVAL, "%s: scale must be positive, and below 2.3e38", fn);
  CAB_REQUIRE(table_stride == 0 || table_stride >= columns, CAB_ESHAPE, "%s: bad table stride", fn);
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  const void* ptrs[4] = {q, out, k_pages, v_pages};
  const int64_t* strides[4] = {q_strides, o_strides, k_strides, v_strides};
  const int64_t sizes[4][3] = {{B, H, 1}, {B, H, 1}, {pages, H_kv, page_size}, {pages, H_kv, page_size}};
  for (int t = 0; t < 4; ++t) {
    CAB_REQUIRE(strides[t][3] == 1, CAB_ESHAPE, "%s: last-dim stride must be 1", fn);
    CAB_REQUIRE(reinterpret_cast<uintptr_t>(ptrs[t]) % 16 == 0, CAB_ESHAPE,
                "%s: pointers must be 16-byte aligned", fn);
    for (int d = 0; d < 3; ++d)  // (the stride of one place has no meaning)
      CAB_REQUIRE(sizes[t][d] <= 1 || strides[t][d] * es % 16 == 0, CAB_ESHAPE,
                  "%s: rows must be 16-byte aligned", fn);
  }
  // 16 rows of K and of V are addressed by 32-bit offsets.
  const int64_t lim = int64_t{1} << 25;
  CAB_REQUIRE(page_size == 1 || (k_strides[2] >= 0 && k_strides[2] * es <= lim && v_strides[2] >= 0 &&
                                 v_strides[2] * es <= lim),
              CAB_ESHAPE, "%s: place strides of the pages must be in [0, 2^25] bytes", fn);
  const int64_t out_size[3] = {B, H, 1};
  const int64_t os3[3] = {o_strides[0], o_strides[1], 0}, qs3[3] = {q_strides[0], q_strides[1], 0};
  const RowLayout rows(os3, out_size, D);
  CAB_REQUIRE(rows.apart, CAB_ESHAPE, "%s: rows of out overlap", fn);
  const int64_t page_sizes[3] = {none ? 0 : pages, H_kv, page_size};
  // A unit's rows of out are written by the workgroup that alone reads its rows of q, after it has, or
  // by the second kernel: q itself may be written over.
  bool over_q = out == q;
  for (int d = 0; d < 2; ++d) over_q = over_q && (out_size[d] == 1 || q_strides[d] == o_strides[d]);
  CAB_REQUIRE((over_q || !rows_share(out, rows, q, RowLayout(qs3, out_size, D), es)) &&
                  !rows_share(out, rows, k_pages, RowLayout(k_strides, page_sizes, D), es) &&
                  !rows_share(out, rows, v_pages, RowLayout(v_strides, page_sizes, D), es),
              CAB_EINVAL, "%s: out shares memory with an input (only q itself may be out)", fn);
  const int64_t most = none ? 0 : columns * page_size;
  const PagedPlan pl = paged_plan(dtype, B, H, H_kv, most, D);
  CAB_REQUIRE(pl.bytes == 0 || (workspace && workspace_bytes >= pl.bytes &&
                                reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
              CAB_EWORKSPACE, "%s: workspace needs %zu bytes, 16-byte aligned", fn, pl.bytes);
  PagedArgs a;
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k_pages);
  a.v = static_cast<const char*>(v_pages);
  for (int d = 0; d < 3; ++d) {
    a.ks[d] = k_strides[d] * es;
    a.vs[d] = v_strides[d] * es;
    if (d == 2) break;
    a.qs[d] = q_strides[d] * es;
    a.os[d] = o_strides[d] * es;
  }
  a.lengths = lengths;
  a.length0 = 0;
  a.most = most;
  a.B = static_cast<int32_t>(B);
  a.Hkv = static_cast<int32_t>(H_kv);
  a.wgs = static_cast<int32_t>(pl.wgs);
  a.least = 1;
  a.table = table;
  a.table_ld = table_stride;
  a.pages = static_cast<int32_t>(pages);
  a.size = static_cast<int32_t>(page_size);
  const bool blocks = page_size % 16 == 0;
  a.shift = std::min(__builtin_ctzll(static_cast<uint64_t>(page_size)), 4);
  const uint64_t by = static_cast<uint64_t>(page_size >> a.shift);
  a.magic = by == 1 ? 0 : ~uint64_t{0} / by + 1;
  a.group = static_cast<int32_t>(H / H_kv);
  a.H = static_cast<int32_t>(H);
  a.direct = pl.direct;
  a.c = c;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  char* ws = static_cast<char*>(workspace);
  a.po = reinterpret_cast<float*>(ws);
  a.pm = reinterpret_cast<float*>(ws + pl.off_pm);
  a.pl = reinterpret_cast<float*>(ws + pl.off_pl);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    switch (dtype) {
      case CAB_F32: launch<CAB_F32, HD>(pl, a, blocks, s); break;
      case CAB_BF16: launch<CAB_BF16, HD>(pl, a, blocks, s); break;
      default: launch<CAB_F16, HD>(pl, a, blocks, s); break;
    }
  };
  if (D == 64)
    go(std::integral_constant<int, 64>{});
  else
    go(std::integral_constant<int, 128>{});
  return launch_status(fn);
}
