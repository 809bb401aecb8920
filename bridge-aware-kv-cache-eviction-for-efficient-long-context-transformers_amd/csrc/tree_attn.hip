// Attention of a tree of drafted tokens over a cache (cab_tree_attn_fwd). Sequence b
// has len_b rows of context and, behind them, the rows of its T drafts; node i sees
// the context and the drafts that are i or its ancestors. The query heads that share
// a K / V head and their T nodes are the R = group * T rows of one unit (b, K / V head).
//
//  1. The context has no mask: every row of a unit sees all of it. It is split over
//     workgroups, each leaving one partial (maximum m, row sum l, unnormalised O) per row:
//     - rows_kernel (up to 32 rows, and fp32): every wave walks its own 32-key steps, K
//       and V straight from memory into matrix operands;
//     - tile_kernel (more rows, 16 bits): 64-key tiles of K and V in LDS, read by all
//       waves, each of which holds 16 or 32 rows.
//     Both compute S^T = K Q^T, an online softmax in the log2 domain (maxima, sums and O
//     in fp32, P rounded to 16 bits as the operand of O^T += V^T P^T).
//  2. join_kernel, one wave per row, merges the row's partials and adds the drafts it
//     sees, found by walking its ancestors: a node has few of them, and no other
//     draft's K or V is touched, so nothing a row does not see can reach it.
//
// Bound: HBM (the context's K and V, read once) up to about 256 rows in 16 bits, the
// matrix cores beyond.
#include "attn_common.h"

namespace cab {
namespace {

constexpr int MAX_NODES = 256;
constexpr int MAX_SPLITS = 256;
constexpr int STEP = 32;  // keys of a wave's step in rows_kernel
constexpr int TILE = 64;  // keys of a tile in tile_kernel

struct TreeArgs {
  const char* q;
  const char* k;
  const char* v;
  int64_t qs[3], ks[3], vs[3];  // bytes: b, h, token
  const int32_t* lengths;       // may be null: length0
  int64_t length0, most;        // most: N - T, the longest context
  int32_t Hkv, group, T, R, splits, row_tiles;
  float c;    // scale * log2(e)
  float* po;  // [unit][R][splits][D]
  float* pm;  // [unit][R][splits] maxima of the scores * c
  float* pl;  // [unit][R][splits] row sums
};

__device__ __forceinline__ int context_length(const int32_t* lengths, int64_t length0, int64_t most,
                                              int b) {
  const int64_t n = lengths ? lengths[b] : length0;
  return static_cast<int>(n < 0 ? 0 : n < most ? n : most);
}

// Steps of `unit` keys a split takes of a context, and the splits that get any.
__device__ __forceinline__ int split_steps(int length, int unit, int splits, int round) {
  const int steps = (length + unit - 1) / unit;
  const int per = (steps + splits - 1) / splits;
  return (per + round - 1) / round * round;
}
__device__ __forceinline__ int live_splits(int length, int unit, int splits, int round) {
  const int per = split_steps(length, unit, splits, round);
  return per ? ((length + unit - 1) / unit + per - 1) / per : 0;
}

// K and V are read once: non-temporal loads.
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

// Grid: (splits, units, row tiles of 16 QT rows).
template <cab_dtype_t DT, int HD, int QT>
__global__ __launch_bounds__(256, DT == CAB_F32 ? 1 : 2) void rows_kernel(TreeArgs a) {
  constexpr bool F32 = DT == CAB_F32, BF16 = DT == CAB_BF16;
  constexpr int NDT = HD / 16;
  using SR = StepRegs<DT, HD>;
  constexpr int NJ = SR::NJ;
  __shared__ f32x4 merge[4][NDT * 64];  // one query tile's O^T per wave
  __shared__ float sm[4][QT][16], sl[4][QT][16];

  const int split = blockIdx.x, unit = blockIdx.y, row0 = blockIdx.z * (16 * QT);
  const int b = unit / a.Hkv, hk = unit - b * a.Hkv;
  const int len = context_length(a.lengths, a.length0, a.most, b);
  const int steps = (len + STEP - 1) / STEP;
  const int per = split_steps(len, STEP, a.splits, 4);
  if (split * per >= steps) return;
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = lane_id(), l16 = lane & 15, g = lane >> 4;
  const float c = a.c;
  const char* kb = a.k + b * a.ks[0] + hk * a.ks[1];
  const char* vb = a.v + b * a.vs[0] + hk * a.vs[1];
  const uint32_t krow = static_cast<uint32_t>(a.ks[2]), vrow = static_cast<uint32_t>(a.vs[2]);

  u32x4 qr[QT][NJ];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = row0 + 16 * qt + l16;
    const int hg = r / a.T, t = r - hg * a.T;
    const char* qp = a.q + b * a.qs[0] + (static_cast<int64_t>(hk) * a.group + hg) * a.qs[1] + t * a.qs[2];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      qr[qt][j] = u32x4{0u, 0u, 0u, 0u};
      if (r < a.R) qr[qt][j] = *reinterpret_cast<const u32x4*>(qp + 64 * j + 16 * g);
    }
  }
  f32x4 o[QT][NDT];
  float l[QT], m[QT];  // l: of this lane's keys alone
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    l[qt] = 0.f;
    m[qt] = M_EMPTY;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[qt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto load = [&](int step, SR& x) {
    const int left = len - STEP * step;
    const char* kp = kb + static_cast<int64_t>(STEP * step) * krow;
    const char* vp = vb + static_cast<int64_t>(STEP * step) * vrow;
    if (left >= STEP)
      load_step<DT, HD, false>(x, kp, vp, krow, vrow, left, l16, g);
    else
      load_step<DT, HD, true>(x, kp, vp, krow, vrow, left, l16, g);
  };
  auto compute = [&](int step, const SR& x) {
    const int left = len - STEP * step;
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
    if (left < STEP) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * tt + 4 * g + r >= left) sc[qt][tt][r] = -INFINITY;
    }
    u32x4 pb[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const float m0 = fmaxf(fmaxf(sc[qt][0][0], sc[qt][0][1]), fmaxf(sc[qt][0][2], sc[qt][0][3]));
      const float m1 = fmaxf(fmaxf(sc[qt][1][0], sc[qt][1][1]), fmaxf(sc[qt][1][2], sc[qt][1][3]));
      float mx = fmaxf(m0, m1), mdup = mx;
      colmax2(mx, mdup);
      if (__builtin_amdgcn_ballot_w64(mx > m[qt]) != 0) {
        const float mn = fmaxf(mx, m[qt]);
        const float alpha = __builtin_amdgcn_exp2f((m[qt] - mn) * c);
        l[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[qt][dt] *= alpha;
        m[qt] = mn;
      }
      const float nmc = -m[qt] * c;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sc[qt][tt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[qt][tt][r], c, nmc));
      const f32x4 s2 = sc[qt][0] + sc[qt][1];
      l[qt] += (s2[0] + s2[1]) + (s2[2] + s2[3]);
      if constexpr (!F32)
        pb[qt] = u32x4{pack2<BF16>(sc[qt][0][0], sc[qt][0][1]), pack2<BF16>(sc[qt][0][2], sc[qt][0][3]),
                       pack2<BF16>(sc[qt][1][0], sc[qt][1][1]), pack2<BF16>(sc[qt][1][2], sc[qt][1][3])};
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
        for (int qt = 0; qt < QT; ++qt) o[qt][dt] = mfma16<BF16>(vo, pb[qt], o[qt][dt]);
      }
    }
  };

  const int end = min(steps, (split + 1) * per);
  int step = split * per + w;
  if constexpr (F32 || QT * HD > 128) {  // (two register sets would spill)
    SR x;
    for (; step < end; step += 4) {
      load(step, x);
      compute(step, x);
    }
  } else {
    // Two register sets: a step's loads are in flight while the one before it is computed.
    SR x, y;
    if (step < end) load(step, x);
    for (; step < end; step += 8) {
      if (step + 4 < end) load(step + 4, y);
      compute(step, x);
      if (step + 4 < end) {
        if (step + 8 < end) load(step + 8, x);
        compute(step + 4, y);
      }
    }
  }

  // Merge of the four waves: common maximum, then the scaled O^T and sums in wave order.
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    l[qt] += shfl_xor_f32(l[qt], 16);
    l[qt] += shfl_xor_f32(l[qt], 32);
    if (g == 0) sm[w][qt][l16] = m[qt];
  }
  __syncthreads();
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const float mm = fmaxf(fmaxf(sm[0][qt][l16], sm[1][qt][l16]), fmaxf(sm[2][qt][l16], sm[3][qt][l16]));
    const float f = __builtin_amdgcn_exp2f((m[qt] - mm) * c);
    if (g == 0) sl[w][qt][l16] = l[qt] * f;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) merge[w][dt * 64 + lane] = o[qt][dt] * f;
    __syncthreads();
    for (int e = threadIdx.x; e < NDT * 64; e += 256) {
      const int dt = e >> 6, ll = e & 63, row = row0 + 16 * qt + (ll & 15);
      const f32x4 y = (merge[0][e] + merge[1][e]) + (merge[2][e] + merge[3][e]);
      if (row < a.R) {
        float* po = a.po + ((static_cast<int64_t>(unit) * a.R + row) * a.splits + split) * HD;
#pragma unroll
        for (int r = 0; r < 4; ++r) po[NDT * (4 * (ll >> 4) + r) + dt] = y[r];
      }
    }
    const int row = row0 + 16 * qt + static_cast<int>(threadIdx.x);
    if (threadIdx.x < 16 && row < a.R) {
      const int64_t x = (static_cast<int64_t>(unit) * a.R + row) * a.splits + split;
      a.pm[x] = mm * c;
      a.pl[x] = (sl[0][qt][l16] + sl[1][qt][l16]) + (sl[2][qt][l16] + sl[3][qt][l16]);
    }
    if (qt + 1 < QT) __syncthreads();
  }
}

// 64-key tiles of K and V in LDS, two of each; WAVES waves of 16 QT rows. Rows are
// stored in 16-byte chunks, chunk x of row r at x ^ swizzle(r), so that neither the
// K operand's reads (16 rows, one chunk each) nor V's transposing ones meet in a bank.
template <int HD>
__device__ __forceinline__ uint32_t tile_offset(uint32_t row, uint32_t chunk) {
  constexpr uint32_t CH = HD / 8;
  const uint32_t z = HD == 128 ? row & 15u : (row >> 1) & 7u;
  return (row * CH + (chunk ^ z)) * 16u;
}

// Grid: 1-D over (row tile fastest, split, unit), neighbours on one XCD, so that a
// split's row tiles find its K and V in one L2.
template <cab_dtype_t DT, int HD, int QT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void tile_kernel(TreeArgs a) {
  constexpr bool BF16 = DT == CAB_BF16;
  constexpr int NDT = HD / 16, NDS = HD / 32, CH = HD / 8;
  constexpr int THREADS = 64 * WAVES, LOADS = TILE * CH / THREADS;  // 16-byte pieces per thread
  constexpr uint32_t TILE_BYTES = TILE * HD * 2;
  __shared__ __align__(16) char lds[2][2][TILE_BYTES];  // [buffer][K, V]

  const int64_t id = xcd_remap(blockIdx.x, gridDim.x);
  const int rt = static_cast<int>(id % a.row_tiles);
  const int64_t us = id / a.row_tiles;
  const int split = static_cast<int>(us % a.splits), unit = static_cast<int>(us / a.splits);
  const int b = unit / a.Hkv, hk = unit - b * a.Hkv;
  const int len = context_length(a.lengths, a.length0, a.most, b);
  const int tiles = (len + TILE - 1) / TILE;
  const int per = split_steps(len, TILE, a.splits, 1);
  const int begin = split * per, end = min(tiles, begin + per);
  if (begin >= end) return;
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = lane_id(), l16 = lane & 15, g = lane >> 4;
  const int row0 = (rt * WAVES + w) * (16 * QT);
  const float c = a.c;
  const char* kb = a.k + b * a.ks[0] + hk * a.ks[1];
  const char* vb = a.v + b * a.vs[0] + hk * a.vs[1];

  u32x4 qr[QT][NDS];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    const int r = row0 + 16 * qt + l16;
    const int hg = r / a.T, t = r - hg * a.T;
    const char* qp = a.q + b * a.qs[0] + (static_cast<int64_t>(hk) * a.group + hg) * a.qs[1] + t * a.qs[2];
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      qr[qt][ds] = u32x4{0u, 0u, 0u, 0u};
      if (r < a.R) qr[qt][ds] = *reinterpret_cast<const u32x4*>(qp + 64 * ds + 16 * g);
    }
  }
  f32x4 o[QT][NDT];  // [dt][r]: d = 16 dt + 4 g + r
  float l[QT], m[QT];
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    l[qt] = 0.f;
    m[qt] = M_EMPTY;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[qt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Piece n of a thread: row and chunk of the tile. Rows past the context are zero.
  u32x4 kx[LOADS], vx[LOADS];
  auto load = [&](int tile) {
    const int left = len - tile * TILE;
    const char* kp = kb + static_cast<int64_t>(tile) * TILE * a.ks[2];
    const char* vp = vb + static_cast<int64_t>(tile) * TILE * a.vs[2];
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      const int p = n * THREADS + tid, row = p / CH, ch = p % CH;
      kx[n] = vx[n] = u32x4{0u, 0u, 0u, 0u};
      if (row < left) {
        kx[n] = *reinterpret_cast<const u32x4*>(kp + row * a.ks[2] + 16 * ch);
        vx[n] = *reinterpret_cast<const u32x4*>(vp + row * a.vs[2] + 16 * ch);
      }
    }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      const uint32_t p = n * THREADS + tid, at = tile_offset<HD>(p / CH, p % CH);
      *reinterpret_cast<u32x4*>(&lds[buf][0][at]) = kx[n];
      *reinterpret_cast<u32x4*>(&lds[buf][1][at]) = vx[n];
    }
  };

  load(begin);
  store(0);
  __syncthreads();
  for (int tile = begin; tile < end; ++tile) {
    const int buf = (tile - begin) & 1;
    if (tile + 1 < end) load(tile + 1);
    const char* kt = lds[buf][0];
    const char* vt = lds[buf][1];
    f32x4 sc[QT][4];  // [qt][tt][r]: key 16 tt + 4 g + r, row 16 qt + l16
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) sc[qt][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds)
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(kt + tile_offset<HD>(16 * tt + l16, 4 * ds + g));
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) sc[qt][tt] = mfma16<BF16>(kf, qr[qt][ds], sc[qt][tt]);
      }
    const int left = len - tile * TILE;
    if (left < TILE) {
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * tt + 4 * g + r >= left) sc[qt][tt][r] = -INFINITY;
    }
    float mx[2];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      f32x4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        y[r] = fmaxf(fmaxf(sc[qt][0][r], sc[qt][1][r]), fmaxf(sc[qt][2][r], sc[qt][3][r]));
      mx[qt] = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
    }
    if constexpr (QT == 1) mx[1] = mx[0];
    colmax2(mx[0], mx[1]);
    u32x4 pb[QT][2];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      if (__builtin_amdgcn_ballot_w64(mx[qt] > m[qt]) != 0) {
        const float mn = fmaxf(mx[qt], m[qt]);
        const float alpha = __builtin_amdgcn_exp2f((m[qt] - mn) * c);
        l[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) o[qt][dt] *= alpha;
        m[qt] = mn;
      }
      const float nmc = -m[qt] * c;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sc[qt][tt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[qt][tt][r], c, nmc));
      const f32x4 s4 = (sc[qt][0] + sc[qt][1]) + (sc[qt][2] + sc[qt][3]);
      l[qt] += (s4[0] + s4[1]) + (s4[2] + s4[3]);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
        pb[qt][hh] = u32x4{pack2<BF16>(sc[qt][2 * hh][0], sc[qt][2 * hh][1]),
                           pack2<BF16>(sc[qt][2 * hh][2], sc[qt][2 * hh][3]),
                           pack2<BF16>(sc[qt][2 * hh + 1][0], sc[qt][2 * hh + 1][1]),
                           pack2<BF16>(sc[qt][2 * hh + 1][2], sc[qt][2 * hh + 1][3])};
    }
    // V^T operand of keys 32 hh ..: k-slot 8 g + e is key 16 (e / 4) + 4 g + e % 4.
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const uint32_t row = 32 * hh + 4 * g + (l16 >> 2);
        const uint32_t ch = 2 * dt + ((l16 & 3) >> 1), in = 8 * (l16 & 1);
        const u32x2 v0 = lds_read_tr16(vt + tile_offset<HD>(row, ch) + in);
        const u32x2 v1 = lds_read_tr16(vt + tile_offset<HD>(row + 16, ch) + in);
        const u32x4 vf = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) o[qt][dt] = mfma16<BF16>(vf, pb[qt][hh], o[qt][dt]);
      }
    if (tile + 1 < end) store(buf ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int qt = 0; qt < QT; ++qt) {
    l[qt] += shfl_xor_f32(l[qt], 16);
    l[qt] += shfl_xor_f32(l[qt], 32);
    const int row = row0 + 16 * qt + l16;
    if (row >= a.R) continue;
    const int64_t x = (static_cast<int64_t>(unit) * a.R + row) * a.splits + split;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
      *reinterpret_cast<f32x4*>(a.po + x * HD + 16 * dt + 4 * g) = o[qt][dt];
    if (g == 0) {
      a.pm[x] = m[qt] * c;
      a.pl[x] = l[qt];
    }
  }
}

struct JoinArgs {
  TreeArgs t;
  const int32_t* parents;
  int64_t parents_ld;  // 0: one tree for all
  int32_t H, unit_keys, round;  // of the splits (see split_steps)
  int64_t rows;                 // B * H * T
  char* out;
  int64_t os[3];  // bytes
  float* lse;
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

// One wave per row; groups of D / 8 lanes, each lane eight of the row's values. A group
// takes every G-th partial and every G-th ancestor.
template <cab_dtype_t DT, int HD>
__global__ __launch_bounds__(256) void join_kernel(JoinArgs a) {
  constexpr int LG = HD / 8, G = 64 / LG, ES = DT == CAB_F32 ? 4 : 2;
  __shared__ int16_t list[4][MAX_NODES];
  const int w = threadIdx.x >> 6, lane = lane_id(), grp = lane / LG, at = lane % LG;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + w;
  if (id >= a.rows) return;  // (waves work apart from each other)
  const TreeArgs& ta = a.t;
  const int node = static_cast<int>(id % ta.T);
  const int64_t bh = id / ta.T;
  const int b = static_cast<int>(bh / a.H), h = static_cast<int>(bh - static_cast<int64_t>(b) * a.H);
  const int hk = h / ta.group;
  const int len = context_length(ta.lengths, ta.length0, ta.most, b);

  // The row's line: the node and its ancestors. A node that ends nowhere is absent.
  const int32_t* parents = a.parents + b * a.parents_ld;
  int n = 0, i = node;
  bool present = true;
  for (;;) {
    if (lane == 0) list[w][n] = static_cast<int16_t>(i);
    ++n;
    const int p = parents[i];
    if (p < 0 || p >= i) {
      present = p == -1;
      break;
    }
    i = p;
  }
  char* op = a.out + b * a.os[0] + h * a.os[1] + node * a.os[2] + at * 8 * ES;
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float l = 0.f, m = M_EMPTY;
  if (present) {
    const int splits = live_splits(len, a.unit_keys, ta.splits, a.round);
    const int64_t row = ((static_cast<int64_t>(b) * ta.Hkv + hk) * ta.R +
                         (h - hk * ta.group) * ta.T + node) * ta.splits;
    for (int x = lane; x < splits; x += 64) m = fmaxf(m, ta.pm[row + x]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, shfl_xor_f32(m, off));
#pragma unroll 4
    for (int x = grp; x < splits; x += G) {
      const float f = __builtin_amdgcn_exp2f(ta.pm[row + x] - m);
      l += ta.pl[row + x] * f;
      const f32x4* po = reinterpret_cast<const f32x4*>(ta.po + (row + x) * HD) + 2 * at;
      const f32x4 y0 = po[0], y1 = po[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] += y0[e] * f;
        o[4 + e] += y1[e] * f;
      }
    }
    float q[8];
    load8<DT>(ta.q + b * ta.qs[0] + h * ta.qs[1] + node * ta.qs[2] + at * 8 * ES, q);
    const char* kp = ta.k + b * ta.ks[0] + hk * ta.ks[1] + len * ta.ks[2] + at * 8 * ES;
    const char* vp = ta.v + b * ta.vs[0] + hk * ta.vs[1] + len * ta.vs[2] + at * 8 * ES;
    constexpr int U = 4;
    for (int x0 = grp; x0 < n; x0 += U * G) {
      float k[U][8], v[U][8], s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int x = x0 + u * G;
        const int64_t j = x < n ? list[w][x] : list[w][0];  // (a row it sees, not used again)
        load8<DT>(kp + j * ta.ks[2], k[u]);
        load8<DT>(vp + j * ta.vs[2], v[u]);
      }
      float hi = m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) d = __builtin_fmaf(q[e], k[u][e], d);
#pragma unroll
        for (int off = LG / 2; off >= 1; off >>= 1) d += shfl_xor_f32(d, off);
        s[u] = x0 + u * G < n ? d * ta.c : -INFINITY;
        hi = fmaxf(hi, s[u]);
      }
      const float f = __builtin_amdgcn_exp2f(m - hi);
      m = hi;
      l *= f;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (x0 + u * G >= n) continue;
        const float p = __builtin_amdgcn_exp2f(s[u] - m);
        l += p;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = __builtin_fmaf(p, v[u][e], o[e]);
      }
    }
    // The groups' states.
    float hi = m;
#pragma unroll
    for (int off = LG; off < 64; off <<= 1) hi = fmaxf(hi, shfl_xor_f32(hi, off));
    const float f = __builtin_amdgcn_exp2f(m - hi);
    m = hi;
    l *= f;
#pragma unroll
    for (int off = LG; off < 64; off <<= 1) l += shfl_xor_f32(l, off);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[e] *= f;
#pragma unroll
      for (int off = LG; off < 64; off <<= 1) o[e] += shfl_xor_f32(o[e], off);
      o[e] *= l == 0.f ? 0.f : 1.0f / l;
    }
  }
  if (grp != 0) return;
  if constexpr (DT == CAB_F32) {
    reinterpret_cast<f32x4*>(op)[0] = f32x4{o[0], o[1], o[2], o[3]};
    reinterpret_cast<f32x4*>(op)[1] = f32x4{o[4], o[5], o[6], o[7]};
  } else {
    constexpr bool BF16 = DT == CAB_BF16;
    *reinterpret_cast<u32x4*>(op) = u32x4{pack2<BF16>(o[0], o[1]), pack2<BF16>(o[2], o[3]),
                                          pack2<BF16>(o[4], o[5]), pack2<BF16>(o[6], o[7])};
  }
  if (at == 0 && a.lse)
    a.lse[id] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
}

// How a problem is cut. tile: rows of a tile_kernel workgroup (0: rows_kernel).
struct TreePlan {
  int64_t units, R, splits, row_tiles;
  int tile;
  size_t off_pm, off_pl, bytes;
};

constexpr int FEW_ROWS = 32;

TreePlan tree_plan(cab_dtype_t dtype, int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t N,
                   int64_t D) {
  TreePlan p;
  p.units = B * Hkv;
  p.R = H / Hkv * T;
  const int64_t most = N > T ? N - T : 0;
  if (p.R <= FEW_ROWS || dtype == CAB_F32) {
    p.tile = 0;
    p.row_tiles = ceil_div(p.R, p.R <= 16 ? 16 : 32);
    const int64_t want = ceil_div(1024, p.units * p.row_tiles);
    p.splits = want < MAX_SPLITS ? want : MAX_SPLITS;
    const int64_t steps = ceil_div(ceil_div(most, STEP), 4);  // four waves' steps
    if (p.splits > steps) p.splits = steps < 1 ? 1 : steps;
  } else {
    p.tile = p.R <= 64 ? 64 : p.R <= 128 ? 128 : 256;
    p.row_tiles = ceil_div(p.R, p.tile);
    const int64_t want = ceil_div(p.tile == 256 ? 256 : 512, p.units * p.row_tiles);
    p.splits = want < MAX_SPLITS ? want : MAX_SPLITS;
    const int64_t tiles = ceil_div(most, TILE);
    if (p.splits > tiles) p.splits = tiles < 1 ? 1 : tiles;
  }
  const int64_t parts = p.units * p.R * p.splits;
  p.off_pm = static_cast<size_t>(parts * D) * 4;
  p.off_pl = p.off_pm + static_cast<size_t>(round_up(parts, 4)) * 4;
  p.bytes = p.off_pl + static_cast<size_t>(round_up(parts, 4)) * 4;
  return p;
}

bool tree_sizes(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t N, int64_t D) {
  return B >= 1 && Hkv >= 1 && H >= Hkv && H % Hkv == 0 && T >= 1 && T <= MAX_NODES && N >= T &&
         N <= INT32_MAX - 1024 && (D == 64 || D == 128) && H <= 65535 && B <= 65535 &&
         B * Hkv <= 65535 && H / Hkv * T <= 65535;
}

template <cab_dtype_t DT, int HD>
void launch(const TreePlan& pl, const JoinArgs& j, hipStream_t s) {
  const TreeArgs& a = j.t;
  const unsigned units = static_cast<unsigned>(pl.units), splits = static_cast<unsigned>(pl.splits);
  if (a.most > 0) {
    const dim3 grid(splits, units, static_cast<unsigned>(pl.row_tiles));
    const unsigned wgs = static_cast<unsigned>(pl.units * pl.splits * pl.row_tiles);
    if (pl.tile == 0) {
      if (pl.R <= 16)
        rows_kernel<DT, HD, 1><<<grid, 256, 0, s>>>(a);
      else
        rows_kernel<DT, HD, 2><<<grid, 256, 0, s>>>(a);
    } else if constexpr (DT != CAB_F32) {
      if (pl.tile == 64)
        tile_kernel<DT, HD, 1, 4><<<wgs, 256, 0, s>>>(a);
      else if (pl.tile == 128)
        tile_kernel<DT, HD, 2, 4><<<wgs, 256, 0, s>>>(a);
      else
        tile_kernel<DT, HD, 2, 8><<<wgs, 512, 0, s>>>(a);
    }
  }
  join_kernel<DT, HD><<<static_cast<unsigned>(ceil_div(j.rows, 4)), 256, 0, s>>>(j);
}

}  // namespace
}  // namespace cab

using namespace cab;

extern "C" size_t cab_tree_attn_workspace_bytes(cab_dtype_t dtype, int64_t B, int64_t H,
                                                int64_t H_kv, int64_t T, int64_t N, int64_t D) {
  if (!valid_dtype(dtype) || !tree_sizes(B, H, H_kv, T, N, D)) return 0;
  return tree_plan(dtype, B, H, H_kv, T, N, D).bytes;
}

extern "C" cab_status_t cab_tree_attn_fwd(
    const void* q, const void* k, const void* v, cab_dtype_t dtype, int64_t B, int64_t H,
    int64_t H_kv, int64_t T, int64_t N, int64_t D, const int64_t q_strides[4],
    const int64_t k_strides[4], const int64_t v_strides[4], const int64_t o_strides[4],
    const int32_t* parents, int64_t parents_stride, const int32_t* lengths, int64_t length0,
    float scale, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "cab_tree_attn_fwd";
  clear_error();
  CAB_REQUIRE(valid_dtype(dtype), CAB_EDTYPE, "%s: unknown dtype %d", fn, static_cast<int>(dtype));
  CAB_REQUIRE(D == 64 || D == 128, CAB_ESHAPE, "%s: D must be 64 or 128 (got %lld)", fn, (long long)D);
  CAB_REQUIRE(B >= 0 && H >= 1 && H_kv >= 1 && H % H_kv == 0, CAB_ESHAPE,
              "%s: H must be a multiple of H_kv", fn);
  CAB_REQUIRE(T >= 1 && T <= MAX_NODES && N >= T, CAB_ESHAPE,
              "%s: a tree holds 1 to %d nodes, and the cache at least as many rows", fn, MAX_NODES);
  if (B == 0) return CAB_OK;
  CAB_REQUIRE(tree_sizes(B, H, H_kv, T, N, D), CAB_ESHAPE, "%s: problem too large", fn);
  CAB_REQUIRE(q && k && v && out && parents && q_strides && k_strides && v_strides && o_strides,
              CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(std::isfinite(scale) && scale > 0.f, CAB_EINVAL, "%s: scale must be positive", fn);
  CAB_REQUIRE(lengths || (length0 >= 0 && length0 <= N - T), CAB_EINVAL,
              "%s: the context must leave room for the drafts", fn);
  CAB_REQUIRE(parents_stride == 0 || parents_stride >= T, CAB_ESHAPE, "%s: bad parents stride", fn);
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  const void* ptrs[4] = {q, k, v, out};
  const int64_t* strides[4] = {q_strides, k_strides, v_strides, o_strides};
  for (int t = 0; t < 4; ++t) {
    CAB_REQUIRE(strides[t][3] == 1, CAB_ESHAPE, "%s: last-dim stride must be 1", fn);
    CAB_REQUIRE(reinterpret_cast<uintptr_t>(ptrs[t]) % 16 == 0, CAB_ESHAPE,
                "%s: pointers must be 16-byte aligned", fn);
    for (int d = 0; d < 3; ++d)
      CAB_REQUIRE(strides[t][d] * es % 16 == 0, CAB_ESHAPE, "%s: rows must be 16-byte aligned", fn);
  }
  // 64 rows of K and of V are addressed by 32-bit offsets.
  const int64_t lim = int64_t{1} << 25;
  CAB_REQUIRE(k_strides[2] >= 0 && k_strides[2] * es <= lim && v_strides[2] >= 0 &&
                  v_strides[2] * es <= lim,
              CAB_ESHAPE, "%s: token strides of k and v must be in [0, 2^25] bytes", fn);
  const TreePlan pl = tree_plan(dtype, B, H, H_kv, T, N, D);
  CAB_REQUIRE(workspace && workspace_bytes >= pl.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
              CAB_EWORKSPACE, "%s: workspace needs %zu bytes, 16-byte aligned", fn, pl.bytes);
  CAB_REQUIRE(pl.units * pl.splits * pl.row_tiles <= INT32_MAX, CAB_ESHAPE, "%s: problem too large", fn);
  JoinArgs j;
  TreeArgs& a = j.t;
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  for (int d = 0; d < 3; ++d) {
    a.qs[d] = q_strides[d] * es;
    a.ks[d] = k_strides[d] * es;
    a.vs[d] = v_strides[d] * es;
    j.os[d] = o_strides[d] * es;
  }
  a.lengths = lengths;
  a.length0 = length0;
  a.most = N - T;
  a.Hkv = static_cast<int32_t>(H_kv);
  a.group = static_cast<int32_t>(H / H_kv);
  a.T = static_cast<int32_t>(T);
  a.R = static_cast<int32_t>(pl.R);
  a.splits = static_cast<int32_t>(pl.splits);
  a.row_tiles = static_cast<int32_t>(pl.row_tiles);
  a.c = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  char* ws = static_cast<char*>(workspace);
  a.po = reinterpret_cast<float*>(ws);
  a.pm = reinterpret_cast<float*>(ws + pl.off_pm);
  a.pl = reinterpret_cast<float*>(ws + pl.off_pl);
  j.parents = parents;
  j.parents_ld = parents_stride;
  j.H = static_cast<int32_t>(H);
  j.unit_keys = pl.tile ? TILE : STEP;
  j.round = pl.tile ? 1 : 4;
  j.rows = B * H * T;
  j.out = static_cast<char*>(out);
  j.lse = lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    switch (dtype) {
      case CAB_F32: launch<CAB_F32, HD>(pl, j, s); break;
      case CAB_BF16: launch<CAB_BF16, HD>(pl, j, s); break;
      default: launch<CAB_F16, HD>(pl, j, s); break;
    }
  };
  if (D == 64)
    go(std::integral_constant<int, 64>{});
  else
    go(std::integral_constant<int, 128>{});
  return launch_status(fn);
}
