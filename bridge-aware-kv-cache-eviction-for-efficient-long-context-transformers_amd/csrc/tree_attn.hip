// Attention of a tree of drafted tokens over a cache (cab_tree_attn_fwd). Sequence b
// has len_b rows of context and, behind them, the rows of its T drafts; node i sees
// the context and the drafts that are i or its ancestors. The query heads that share
// a K / V head and their T nodes are the R = group * T rows of one unit (b, K / V head).
//
//  1. The context has no mask: every row of a unit sees all of it. The contexts of all
//     units, cut into pieces of as many keys as a workgroup takes at a time, make one
//     list, and each workgroup takes an equal stretch of it, whatever the lengths. Of
//     each unit that its stretch touches it leaves one partial (the maximum's level m,
//     row sum l, unnormalised O) per row:
//     - rows_kernel (few rows, and fp32, on the fp32 matrix instructions): every wave walks
//       its own 32-key steps, K and V straight from memory into matrix operands;
//     - tile_kernel (more rows, 16 bits): 64-key tiles of K and V in LDS, read by all
//       waves, each of which holds 16 or 32 rows.
//     Both compute S^T = K Q^T, an online softmax in the log2 domain (maxima, sums and O
//     in fp32, P rounded to 16 bits as the operand of O^T += V^T P^T).
//  2. join_kernel, one wave per row, merges the row's partials and adds the drafts it
//     sees, found by walking its ancestors: no other draft's K or V is touched, so nothing
//     a row does not see can reach it. A tree's node has few of them; in a chain of T
//     nodes a row has up to T, and the rows' work together grows with T^2.
//
// P goes to 16 bits because the matrix instructions take it so (fp32 ones run at a seventh of
// the rate): half a step of each weight, which with the output's own rounding is an error of
// 1.9e-3 to 2.1e-3 of the outputs in bf16 where that rounding alone is 1.65e-3 (fp16 2.5e-4,
// 2.1e-4). Nothing in a result depends on the order in which workgroups run: the same bits
// again for the same sizes and lengths.
//
// Bound: HBM (the context's K and V, read once) for few rows; for many the chain of one
// tile (operand reads, products, maxima, exponentials, products), of which two waves a
// SIMD overlap little. Measured, 32 query heads on 8, D = 128, bf16: one token of 16
// sequences of up to 32768 keys 191 + 5.6 us (contexts + join; some 6.8 TB/s of K and V); a
// tree of 64 over 65472 keys 84 + 12 us (816 TFLOP/s), over 8128 22.6 + 8.6 us, of which the
// partials of 256 workgroups (17 MB out and in) are some 5.
#include "decode_common.h"
#include "row_layout.h"

namespace cab {
namespace {

constexpr int MAX_NODES = 256;
constexpr int TILE = 64;  // tile_kernel's pieces (rows_kernel's: QUAD)

struct TreeArgs {
  const char* q;
  const char* k;
  const char* v;
  int64_t qs[3], ks[3], vs[3];  // bytes: b, h, token
  const int32_t* lengths;       // may be null: length0
  int64_t length0, most;        // most: N - T, the longest context
  int32_t B, Hkv, group, T, R, row_tiles;
  int32_t wgs, least;  // workgroups that share the list; the fewest pieces one takes
  float c;             // scale * log2(e)
  // Partials. Workgroup x's of unit u is number x + u: down the list either x or u goes
  // up by one from one partial to the next.
  float* po;  // [number][R][D]
  float* pm;  // [number][R] level_of the maximum score
  float* pl;  // [number][R] row sums
};

// Grid: (workgroups, row tiles of 16 QT rows).
template <cab_dtype_t DT, int HD, int QT>
__global__ __launch_bounds__(256, DT == CAB_F32 ? 1 : 2) void rows_kernel(TreeArgs a) {
  constexpr bool F32 = DT == CAB_F32;
  constexpr int NDT = HD / 16;
  using SR = StepRegs<DT, HD>;
  constexpr int NJ = SR::NJ;
  __shared__ RowMerge<DT, HD, QT> merge;

  const int row0 = blockIdx.y * (16 * QT);
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const float c = a.c;
  const uint32_t krow = static_cast<uint32_t>(a.ks[2]), vrow = static_cast<uint32_t>(a.vs[2]);

  over_stretch<QUAD>(a, blockIdx.x, [&](int b, int hk, int piece, int pieces, int len) {
    int lane = lane_id();
    asm volatile("" : "+v"(lane));  // (what follows from it is not kept over the parts)
    const int l16 = lane & 15, g = lane >> 4;
    const char* kb = a.k + b * a.ks[0] + hk * a.ks[1];
    const char* vb = a.v + b * a.vs[0] + hk * a.vs[1];
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
    RowState<DT, HD, QT> rows;
    rows.clear(c);

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
      rows.step(x, qr, c, left < STEP, [&](int tt, int r) { return 16 * tt + 4 * g + r < left; });
    };

    const int end = min((len + STEP - 1) / STEP, 4 * (piece + pieces));
    int step = 4 * piece + w;
    // (Two register sets spill with 32 rows of 128 in 16 bits. In fp32, one workgroup a CU,
    // they would not; one set is what the figures here are of.)
    if constexpr (F32 || QT * HD > 128) {
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

    const int64_t part = static_cast<int64_t>(blockIdx.x) + b * a.Hkv + hk;
    merge.run(
        rows, w, lane, c,
        [&](int qt, int e, const f32x4& y) {
          const int dt = e >> 6, ll = e & 63, row = row0 + 16 * qt + (ll & 15);
          if (row < a.R) {
            float* po = a.po + (part * a.R + row) * HD;
#pragma unroll
            for (int r = 0; r < 4; ++r) po[NDT * (4 * (ll >> 4) + r) + dt] = y[r];
          }
        },
        [&](int qt, float level, float sum) {
          const int row = row0 + 16 * qt + static_cast<int>(threadIdx.x);
          if (row < a.R) {
            a.pm[part * a.R + row] = level;
            a.pl[part * a.R + row] = sum;
          }
        });
  });
}

// 64-key tiles of K and V in LDS; WAVES waves of 16 QT rows. Rows are
// stored in 16-byte chunks, chunk x of row r at x ^ swizzle(r), so that neither the
// K operand's reads (16 rows, one chunk each) nor V's transposing ones meet in a bank.
template <int HD>
__device__ __forceinline__ uint32_t tile_offset(uint32_t row, uint32_t chunk) {
  constexpr uint32_t CH = HD / 8;
  const uint32_t z = HD == 128 ? row & 15u : (row >> 1) & 7u;
  return (row * CH + (chunk ^ z)) * 16u;
}

// Grid: 1-D over (row tile fastest, workgroup), neighbours on one XCD, so that a
// stretch's row tiles find its K and V in one L2.
//
// Tiles go to LDS without passing through registers, the next one in flight while one is
// computed (2 and 3 in flight measured 2 to 4 % slower). A wave waits for its own
// loads of a tile, and the workgroup's barrier makes that everybody's; the same
// barrier frees the tile before.
template <cab_dtype_t DT, int HD, int QT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void tile_kernel(TreeArgs a) {
  constexpr bool BF16 = DT == CAB_BF16;
  constexpr int NDT = HD / 16, NDS = HD / 32, CH = HD / 8;
  constexpr int ROWS = 64 / CH * WAVES;  // rows a round of the waves' loads covers (1 KB each)
  constexpr int LOADS = TILE / ROWS;     // a wave's loads of a tile of K, and of V
  static_assert(LOADS >= 1 && TILE % ROWS == 0, "a tile is whole rounds of loads");
  constexpr uint32_t TILE_BYTES = TILE * HD * 2;
  __shared__ __align__(16) char lds[2][2][TILE_BYTES];  // [slot][K, V]

  const int64_t id = xcd_remap(blockIdx.x, gridDim.x);
  const int rt = static_cast<int>(id % a.row_tiles), wg = static_cast<int>(id / a.row_tiles);
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int row0 = (rt * WAVES + w) * (16 * QT);
  const float c = a.c;

  over_stretch<TILE>(a, wg, [&](int b, int hk, int begin, int pieces, int len) {
    int lane = lane_id();
    asm volatile("" : "+v"(lane));  // (what follows from it is not kept over the parts)
    const int l16 = lane & 15, g = lane >> 4;
    const int end = begin + pieces;
    const char* kb = a.k + b * a.ks[0] + hk * a.ks[1];
    const char* vb = a.v + b * a.vs[0] + hk * a.vs[1];
    // A lane's row in a wave's first load and its place there. Lane i's 16 bytes land at
    // 16 i, so each lane fetches the chunk that tile_offset() looks for at its place.
    // (A round of loads further on the swizzle is the same.)
    const uint32_t lrow = w * (64 / CH) + lane / CH;
    const uint32_t lch = tile_offset<HD>(lrow, lane % CH) % (16 * CH);
    const uint32_t koff = lrow * static_cast<uint32_t>(a.ks[2]) + lch;
    const uint32_t voff = lrow * static_cast<uint32_t>(a.vs[2]) + lch;
    auto load = [&](int tile, int slot) {
      const int left = len - tile * TILE;
      constexpr uint32_t END = 0xffffffe0u;  // rows past the context: an offset past it, read as zero
      const sgpr_rsrc_t kr = make_sgpr_rsrc(kb + static_cast<int64_t>(tile) * TILE * a.ks[2], END);
      const sgpr_rsrc_t vr = make_sgpr_rsrc(vb + static_cast<int64_t>(tile) * TILE * a.vs[2], END);
#pragma unroll
      for (int n = 0; n < LOADS; ++n) {
        const uint32_t ks = n * ROWS * static_cast<uint32_t>(a.ks[2]);
        const uint32_t vs = n * ROWS * static_cast<uint32_t>(a.vs[2]);
        char* kt = &lds[slot][0][(n * WAVES + w) * 1024];
        char* vt = &lds[slot][1][(n * WAVES + w) * 1024];
        if (left >= TILE) {
          bdma16_untracked(kr, koff, ks, kt);
          bdma16_untracked(vr, voff, vs, vt);
        } else {
          const bool in = static_cast<int>(lrow) + n * ROWS < left;
          bdma16_untracked(kr, in ? koff + ks : END, 0, kt);
          bdma16_untracked(vr, in ? voff + vs : END, 0, vt);
        }
      }
    };
    lds_barrier();  // the last part's tiles have been read
    load(begin, 0);

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
    float l[QT], m[QT], level[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      l[qt] = 0.f;
      m[qt] = M_EMPTY;
      level[qt] = level_of<DT>(M_EMPTY, c);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[qt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // (held here, so that nothing in the loop waits for them and with them for the tiles)
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int ds = 0; ds < NDS; ++ds) asm volatile("" : "+v"(qr[qt][ds]));

    auto step = [&](int tile, const int slot) __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
      lds_barrier();
      if (tile + 1 < end) load(tile + 1, slot ^ 1);
      const char* kt = lds[slot][0];
      const char* vt = lds[slot][1];
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
          const float upto = level_of<DT>(mn, c);
          const float alpha = relevel<DT>(m[qt], level[qt], mn, upto, c);
          l[qt] *= alpha;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[qt][dt] *= alpha;
          m[qt] = mn;
          level[qt] = upto;
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            sc[qt][tt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[qt][tt][r], c, -level[qt]));
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
    };
    // (a slot's LDS addresses are constants of its own copy of the step)
    for (int tile = begin; tile < end; tile += 2) {
      step(tile, 0);
      if (tile + 1 < end) step(tile + 1, 1);
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      l[qt] += shfl_xor_f32(l[qt], 16);
      l[qt] += shfl_xor_f32(l[qt], 32);
      const int row = row0 + 16 * qt + l16;
      if (row >= a.R) continue;
      const int64_t x = (static_cast<int64_t>(wg) + b * a.Hkv + hk) * a.R + row;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
        *reinterpret_cast<f32x4*>(a.po + x * HD + 16 * dt + 4 * g) = o[qt][dt];
      if (g == 0) {
        a.pm[x] = level[qt];
        a.pl[x] = l[qt];
      }
    }
  });
}

struct JoinArgs {
  TreeArgs t;
  const int32_t* parents;
  int64_t parents_ld;  // 0: one tree for all
  int32_t H;
  int64_t rows;                 // B * H * T
  char* out;
  int64_t os[3];  // bytes
  float* lse;
};

// One wave per row; groups of D / 8 lanes, each lane eight of the row's values. A group
// takes every G-th partial and every G-th ancestor. KEYS: of the context's pieces.
template <cab_dtype_t DT, int HD, int KEYS>
__global__ __launch_bounds__(256) void join_kernel(JoinArgs a) {
  constexpr int LG = HD / 8, G = 64 / LG, ES = DT == CAB_F32 ? 4 : 2;
  __shared__ int16_t list[4][MAX_NODES];
  __shared__ int32_t above[4][MAX_NODES];
  const int w = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int lane = lane_id(), grp = lane / LG, at = lane % LG;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + w;
  if (id >= a.rows) return;  // (waves work apart from each other)
  const TreeArgs& ta = a.t;
  const int node = static_cast<int>(id % ta.T);
  const int64_t bh = id / ta.T;
  const int b = static_cast<int>(bh / a.H), h = static_cast<int>(bh - static_cast<int64_t>(b) * a.H);
  const int hk = h / ta.group;
  // The row's line: the node and its ancestors. A node that ends nowhere is absent.
  const Lengths<TreeArgs> lens(ta);
  float q[8];
  load8<DT>(ta.q + b * ta.qs[0] + h * ta.qs[1] + node * ta.qs[2] + at * 8 * ES, q);
  const int32_t* parents = a.parents + b * a.parents_ld;
  for (int x = lane; x <= node; x += 64) above[w][x] = parents[x];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  int n = 0, i = node;
  bool present = true;
  for (;;) {
    if (lane == 0) list[w][n] = static_cast<int16_t>(i);
    ++n;
    const int p = above[w][i];
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
    const Cut cut = list_cut<KEYS>(ta, lens);
    int before = 0, len = 0;  // the sequences' shares of the list before b; b's context
    for (int b0 = 0; b0 <= b; b0 += 64) {
      const int mine = lens.mine(b0);
      before += wave_sum(b0 + lane < b ? round_to(pieces_of<KEYS>(mine), cut.grain) : 0);
      len = __builtin_amdgcn_readlane(mine, b & 63);  // (the last round's)
    }
    // The unit's partials: of the workgroups whose stretches meet its pieces.
    const int pieces = pieces_of<KEYS>(len);
    const int start = before * ta.Hkv + hk * round_to(pieces, cut.grain), first = start / cut.per;
    const int parts = pieces ? (start + pieces - 1) / cut.per - first + 1 : 0;
    const int64_t row = (static_cast<int64_t>(first) + b * ta.Hkv + hk) * ta.R +
                        (h - hk * ta.group) * ta.T + node;
    for (int x = lane; x < parts; x += 64) m = fmaxf(m, ta.pm[row + static_cast<int64_t>(x) * ta.R]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, shfl_xor_f32(m, off));
#pragma unroll 4
    for (int x = grp; x < parts; x += G) {
      const int64_t y = row + static_cast<int64_t>(x) * ta.R;
      const float f = __builtin_amdgcn_exp2f(ta.pm[y] - m);
      l += ta.pl[y] * f;
      const f32x4* po = reinterpret_cast<const f32x4*>(ta.po + y * HD) + 2 * at;
      const f32x4 y0 = po[0], y1 = po[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] += y0[e] * f;
        o[4 + e] += y1[e] * f;
      }
    }
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
      o[e] *= 1.0f / l;  // (l 0, all scores -inf: 0 / 0)
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
  // -inf is for absent nodes alone: a node that is there and has no softmax (a score of NaN or
  // +inf, or all of them -inf: l is NaN or 0) has NaN for both results. l's bits are tested
  // because this file is compiled with -fno-honor-nans.
  if (at == 0 && a.lse) {
    int32_t bits = __builtin_bit_cast(int32_t, l);
    asm("" : "+v"(bits));  // (or the test is made one of floats)
    const float sum = (m + __log2f(l)) * 0.69314718055994531f;
    uint32_t x = bits > 0 && bits <= 0x7f800000 ? __builtin_bit_cast(uint32_t, sum) : 0x7fc00000u;
    if (!present) x = 0xff800000u;
    reinterpret_cast<uint32_t*>(a.lse)[id] = x;
  }
}

// How a problem is cut. tile: rows of a tile_kernel workgroup (0: rows_kernel).
struct TreePlan {
  int64_t units, R, row_tiles, wgs, least;
  int tile;
  size_t off_pm, off_pl, bytes;
};

// Rows per unit up to which rows_kernel runs, and those beyond which it does for long
// lists only (keys of all units' longest contexts). 32 heads on 8, D = 128, bf16, us, here ->
// tile_kernel: 4 rows, 16 sequences of 32768 keys 198 -> 228; 32 rows, 8184 keys 22.9 ->
// 19.7, but 16 sequences of 32768 keys 208 -> 238, and 20 rows, 8 of 16384 65 -> 72.
constexpr int FEW_ROWS = 32, FEWER_ROWS = 16;
constexpr int64_t LONG_LIST = int64_t{1} << 18;
// Lists up to which 129 to 256 rows go in two tiles of 128 with stretches twice as long, which
// halves the partials (us, one tile of 256 -> so: 8 units of 500 keys 21.5 -> 18.4, of 8128
// 33.6 -> 30.5, 16 of up to 5936 32.1 -> 28.5; 8 of 65472 97 -> 119).
constexpr int64_t BRIEF_LIST = int64_t{1} << 17;
// Workgroups that share the list: one a CU (rows_kernel; 512: 4 rows, 16 x 32768 keys 202 us
// against 198, fp32, 256 rows of 4032 keys 84 against 70), or as many as the registers
// allow: one of 8 waves, two of 4 (256: 64 rows, 8 x 8192 keys 54 us against 49).
constexpr int WGS = 256, SMALL_TILE_WGS = 512;

TreePlan tree_plan(cab_dtype_t dtype, int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t N,
                   int64_t D) {
  TreePlan p;
  p.units = B * Hkv;
  p.R = H / Hkv * T;
  const int64_t most = N > T ? N - T : 0;
  int64_t slots = WGS;
  int keys;
  if (dtype == CAB_F32 || p.R <= FEWER_ROWS || (p.R <= FEW_ROWS && p.units * most > LONG_LIST)) {
    p.tile = 0;
    p.row_tiles = ceil_div(p.R, p.R <= 16 ? 16 : 32);
    p.least = 1;
    keys = QUAD;
  } else {
    const bool halves = p.R > 128 && p.R <= 256 && p.units * most <= BRIEF_LIST;
    p.tile = p.R <= 64 ? 64 : p.R <= 128 || halves ? 128 : 256;
    p.row_tiles = ceil_div(p.R, p.tile);
    // (two tiles a workgroup at least; four of the small ones at D = 128 in all but short
    // lists: 64 rows of 8 x 8176 keys 19.9 us against 22.1, 20 of 8 x 595 15.1 against 12.9)
    p.least = p.tile < 256 && D == 128 && p.units * most > 512 * TILE ? 4 : 2;
    if (p.tile < 256 && !halves) slots = SMALL_TILE_WGS;
    keys = TILE;
  }
  // No more workgroups than the longest contexts have stretches.
  const int64_t list = p.units * ceil_div(most, keys);
  p.wgs = ceil_div(slots, p.row_tiles);
  if (p.wgs > ceil_div(list, p.least)) p.wgs = ceil_div(list, p.least);
  if (p.wgs < 1) p.wgs = 1;
  const int64_t parts = (p.wgs + p.units) * p.R;
  p.off_pm = static_cast<size_t>(parts * D) * 4;
  p.off_pl = p.off_pm + static_cast<size_t>(round_up(parts, 4)) * 4;
  p.bytes = p.off_pl + static_cast<size_t>(round_up(parts, 4)) * 4;
  return p;
}

bool tree_sizes(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t N, int64_t D) {
  // (the list of pieces, and where a stretch begins, fit 32 bits)
  return B >= 1 && Hkv >= 1 && H >= Hkv && H % Hkv == 0 && T >= 1 && T <= MAX_NODES && N >= T &&
         N <= INT32_MAX - 1024 && (D == 64 || D == 128) && H <= 65535 && B <= 65535 &&
         B * Hkv <= INT32_MAX / 2 / ceil_div(N, TILE) && H / Hkv * T <= 65535 &&
         // (join_kernel's threads, 64 a row in workgroups of four: fewer than 2^32)
         H * T <= ((int64_t{1} << 26) - 4) / B;
}

template <cab_dtype_t DT, int HD>
void launch(const TreePlan& pl, const JoinArgs& j, hipStream_t s) {
  const TreeArgs& a = j.t;
  const unsigned wgs = static_cast<unsigned>(pl.wgs), tiles = static_cast<unsigned>(pl.row_tiles);
  const unsigned join = static_cast<unsigned>(ceil_div(j.rows, 4));
  if (pl.tile == 0) {
    if (a.most > 0) {
      if (pl.R <= 16)
        rows_kernel<DT, HD, 1><<<dim3(wgs, tiles), 256, 0, s>>>(a);
      else
        rows_kernel<DT, HD, 2><<<dim3(wgs, tiles), 256, 0, s>>>(a);
    }
    join_kernel<DT, HD, QUAD><<<join, 256, 0, s>>>(j);
  } else if constexpr (DT != CAB_F32) {
    if (a.most > 0) {
      if (pl.tile == 64)
        tile_kernel<DT, HD, 1, 4><<<wgs * tiles, 256, 0, s>>>(a);
      else if (pl.tile == 128)
        tile_kernel<DT, HD, 2, 4><<<wgs * tiles, 256, 0, s>>>(a);
      else
        tile_kernel<DT, HD, 2, 8><<<wgs * tiles, 512, 0, s>>>(a);
    }
    join_kernel<DT, HD, TILE><<<join, 256, 0, s>>>(j);
  }
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
  const int64_t out_size[3] = {B, H, T};
  const RowLayout rows(o_strides, out_size, D);
  CAB_REQUIRE(rows.apart, CAB_ESHAPE, "%s: rows of out overlap", fn);
  // 64 rows of K and of V are addressed by 32-bit offsets.
  const int64_t lim = int64_t{1} << 25;
  CAB_REQUIRE(k_strides[2] >= 0 && k_strides[2] * es <= lim && v_strides[2] >= 0 &&
                  v_strides[2] * es <= lim,
              CAB_ESHAPE, "%s: token strides of k and v must be in [0, 2^25] bytes", fn);
  const TreePlan pl = tree_plan(dtype, B, H, H_kv, T, N, D);
  CAB_REQUIRE(workspace && workspace_bytes >= pl.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
              CAB_EWORKSPACE, "%s: workspace needs %zu bytes, 16-byte aligned", fn, pl.bytes);
  // join_kernel reads q's rows and the drafts' of k and v while it writes: q's own rows alone may
  // be written over.
  const int64_t kv_size[3] = {B, H_kv, N};
  bool over_q = out == q;
  for (int d = 0; d < 3; ++d) over_q = over_q && (out_size[d] == 1 || q_strides[d] == o_strides[d]);
  CAB_REQUIRE((over_q || !rows_share(out, rows, q, RowLayout(q_strides, out_size, D), es)) &&
                  !rows_share(out, rows, k, RowLayout(k_strides, kv_size, D), es) &&
                  !rows_share(out, rows, v, RowLayout(v_strides, kv_size, D), es),
              CAB_EINVAL, "%s: out shares memory with an input (only q itself may be out)", fn);
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
  a.B = static_cast<int32_t>(B);
  a.wgs = static_cast<int32_t>(pl.wgs);
  a.least = static_cast<int32_t>(pl.least);
  a.row_tiles = static_cast<int32_t>(pl.row_tiles);
  a.c = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  char* ws = static_cast<char*>(workspace);
  a.po = reinterpret_cast<float*>(ws);
  a.pm = reinterpret_cast<float*>(ws + pl.off_pm);
  a.pl = reinterpret_cast<float*>(ws + pl.off_pl);
  j.parents = parents;
  j.parents_ld = parents_stride;
  j.H = static_cast<int32_t>(H);
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
