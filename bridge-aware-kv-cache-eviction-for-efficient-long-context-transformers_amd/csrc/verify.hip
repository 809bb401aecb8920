// Verification of drafted tokens against the target's logits, from given random
// numbers (cab_verify_drafts). Node 0 of a sequence's tree is the token the model
// has taken already; the walk goes from it to the first child that is accepted, and
// so on. With p = softmax(logits[node] / temperature), and r the child's own uniform
// number:
//   greedy (temperature 0): the child whose token is the row's argmax;
//   point (no draft logits): a child x is accepted if r Z < p(x), where Z is what the
//     siblings rejected before it have left of p (their tokens' weights become 0): the row's
//     sum less theirs, or, where that is little of it, the sum of the others;
//   draft, with q = softmax(draft_logits[node] / temperature): each rejection leaves
//     max(p - q, 0) / c of p. As max(max(y, 0) - z, 0) = max(y - z, 0) for z >= 0, the
//     residual after any number of rejections is max(p - a q, 0) / c with two numbers:
//     a' = a + c, c' = sum max(p - a' q, 0), from a = 0, c = 1. A child is accepted if
//     r c q(x) < max(p(x) - a q(x), 0).
// At the node with no accepted child the next token is argmax_x w(x) / noise(x) over
// the residual w; with noise ~ Exp(1) that is a sample of w / sum w. It needs no
// cumulative sum (whose order would decide between tokens) and no normaliser.
//
// One walk needs the rows of the accepted nodes, one after another. Two ways:
//  - walk_kernel<.., false>: one workgroup of 16 waves a sequence reads just those
//    rows. A row takes a CU about 8 us per 100000 values (the exponentials), whatever
//    the batch up to the chip's 256 CUs.
//  - where the logits are few enough, stats_kernel first takes the maximum and sum (or the
//    argmax) of every row that has children, spread over the chip; walk_kernel<.., true>
//    then decides from these alone.
// Either way pick_kernel draws the next token, several workgroups a sequence.
//
// Bound: launches and latency (a tree of 64 over 128000 tokens, bf16: 6.9 + 8.6 + 6.7 us for
// statistics, walk and pick), for a batch the rows' bytes (32 trees of 32: 131 of 262 MB
// read in 37 us, 3.5 TB/s; then 9.8 + 10.8 us).
#include "cab_internal.h"

namespace cab {
namespace {

constexpr int MAX_NODES = 256;
constexpr int WALK_THREADS = 1024;
constexpr int SLICE_THREADS = 256;  // of stats_kernel and pick_kernel
enum { GREEDY = 0, POINT = 1, DRAFT = 2 };

// 16 bytes at any element's alignment (global loads need none on gfx950).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

struct VerifyArgs {
  const char* logits;
  const char* drafts;
  int64_t ls[2], ds[2];  // bytes: b, node
  const int64_t* tokens;
  const int32_t* parents;
  const float* uniforms;
  const float* noise;
  int64_t parents_ld;  // 0: one tree for all
  int32_t T, V;
  float c_hi, c_lo, d_min;  // log2(e) / temperature in two parts; the least exponent
  int32_t* path;
  int32_t* counts;
  int64_t* next;
  // With rows' statistics (see VerifyPlan):
  struct RowStats* stats;    // [logits, drafts][row][slices]
  struct WalkEnd* ends;      // [B]
  struct Candidate* picks;   // [B][picks of a row]
  int32_t slices, slice;     // slices of a row in stats_kernel, their values
  int32_t picks_a_row, pick;  // in pick_kernel
  int64_t rows;              // B * T
};

// A slice of a row: its maximum (at least the lowest float) and sum of weights, or
// (greedy) the order_key of its argmax.
struct RowStats {
  union {
    double s;
    unsigned long long key;
  };
  float m, unused;
};

// Where a sequence's walk ended, for pick_kernel.
struct WalkEnd {
  double ip, iq, used;  // 1 / sums of weights; a
  float m, mq;
  int32_t node, n_gone;
  uint32_t done;  // pick_kernel's workgroups that are through
  uint32_t unused;
  int32_t gone[MAX_NODES];
};

// The best of a slice, from the residual, and from the whole row for when nothing is left
// of it: score (relative to m), and the logit and 1 / noise it comes from.
struct Candidate {
  float m, score[2], x[2], y[2];
  int32_t index[2];
  int32_t unused[3];
};
// What one workgroup leaves for another of the same launch goes past the L2 caches, which
// the XCDs do not share; a release fence would write a whole L2 back (512 workgroups of
// pick_kernel: 28 us with fences, 12 so).
template <typename T>
__device__ __forceinline__ void put(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T get(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <cab_dtype_t DT>
__device__ __forceinline__ float value_at(const char* row, int i) {
  if constexpr (DT == CAB_F32)
    return reinterpret_cast<const float*>(row)[i];
  else if constexpr (DT == CAB_BF16)
    return bf16_to_f32(reinterpret_cast<const uint16_t*>(row)[i]);
  else
    return f16_to_f32(reinterpret_cast<const uint16_t*>(row)[i]);
}

template <cab_dtype_t DT>
struct Chunk {
  static constexpr int N = DT == CAB_F32 ? 4 : 8;
  u32x4_any raw;
  __device__ __forceinline__ void load(const char* row, int c) {
    raw = reinterpret_cast<const u32x4_any*>(row)[c];
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (DT == CAB_F32) {
      return __uint_as_float(raw[i]);
    } else {
      const uint32_t w = raw[i >> 1];
      const uint16_t h = static_cast<uint16_t>(i & 1 ? w >> 16 : w);
      return DT == CAB_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
    }
  }
};

// exp((x - m) / temperature): the exponent's integer and fractional parts apart, so
// that the error stays at 1e-7 however far x is below m. m is the row's maximum, at
// least the lowest float. A NaN, and -inf, weigh 0; +inf is its own maximum.
__device__ __forceinline__ float weight(float x, float m, const VerifyArgs& a) {
  const float d = x == m ? 0.f : fmaxf(x - m, a.d_min);
  const float i = __builtin_rintf(d * a.c_hi);
  const float f = __builtin_fmaf(d, a.c_lo, __builtin_fmaf(d, a.c_hi, -i));
  return __builtin_ldexpf(__builtin_amdgcn_exp2f(f), static_cast<int>(i));
}

// max(p - a q, 0) with p = ep * ip, a q = eq * uq. Both products are rounded before the
// difference (no contraction), so that equal ones leave nothing.
__device__ __forceinline__ double residual(float ep, double ip, float eq, double uq) {
#pragma clang fp contract(off)
  const double p = ep * ip, q = eq * uq;
  return fmax(p - q, 0.0);
}

// The same in 32 bits, for sums of many.
__device__ __forceinline__ float residual32(float ep, float ip, float eq, float uq) {
#pragma clang fp contract(off)
  const float p = ep * ip, q = eq * uq;
  return fmaxf(p - q, 0.f);
}

template <int THREADS>
struct Scratch {
  static constexpr int WAVES = THREADS / 64;
  float m[WAVES];
  double s[WAVES];
  unsigned long long key[WAVES], key2[WAVES];
};

template <int THREADS>
__device__ __forceinline__ double block_sum(double v, Scratch<THREADS>& sh) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += shfl_xor_f64(v, off);
  __syncthreads();
  if (lane_id() == 0) sh.s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) v += sh.s[w];
  return v;
}

// The largest of each of two keys, over a wave and over the workgroup.
__device__ __forceinline__ void wave_max2(unsigned long long (&k)[2]) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned long long o = __shfl_xor(k[i], off, 64);
      k[i] = o > k[i] ? o : k[i];
    }
}
template <int THREADS>
__device__ __forceinline__ void block_max2(unsigned long long (&k)[2], Scratch<THREADS>& sh) {
  wave_max2(k);
  __syncthreads();
  if (lane_id() == 0) {
    sh.key[threadIdx.x >> 6] = k[0];
    sh.key2[threadIdx.x >> 6] = k[1];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    k[0] = sh.key[w] > k[0] ? sh.key[w] : k[0];
    k[1] = sh.key2[w] > k[1] ? sh.key2[w] : k[1];
  }
}

template <int THREADS>
__device__ __forceinline__ unsigned long long block_max(unsigned long long k, Scratch<THREADS>& sh) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const unsigned long long o = __shfl_xor(k, off, 64);
    k = o > k ? o : k;
  }
  __syncthreads();
  if (lane_id() == 0) sh.key[threadIdx.x >> 6] = k;
  __syncthreads();
  k = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) k = sh.key[w] > k ? sh.key[w] : k;
  return k;
}

// Which of N values from `at` on are among n indexes.
template <int N>
__device__ __forceinline__ uint32_t gone_mask(const int32_t* gone, int n, int at) {
  uint32_t mask = 0;
  for (int k = 0; k < n; ++k) {
    const uint32_t d = static_cast<uint32_t>(gone[k] - at);
    if (d < static_cast<uint32_t>(N)) mask |= 1u << d;
  }
  return mask;
}

// Order of floats as unsigned numbers, and the lower of equal ones' indexes first.
__device__ __forceinline__ unsigned long long order_key(float x, int i) {
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<unsigned long long>(o) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int key_index(unsigned long long k) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k));
}

// f(first index, values, other row's values, how many) over the 16-byte chunks of V values,
// U of them loaded at a time, then the last values one by one. TWO: of two rows alike.
template <cab_dtype_t DT, int U, int THREADS, bool TWO, typename F>
__device__ __forceinline__ void over_rows(const char* row, const char* other, int V, F f) {
  constexpr int N = Chunk<DT>::N;
  const int n = V / N;
  for (int c0 = threadIdx.x; c0 < n; c0 += U * THREADS) {
    Chunk<DT> x[U], y[TWO ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * THREADS < n) {
        x[u].load(row, c0 + u * THREADS);
        if constexpr (TWO) y[u].load(other, c0 + u * THREADS);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * THREADS < n) {
        float v[N], v2[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          v[i] = x[u].get(i);
          v2[i] = TWO ? y[TWO ? u : 0].get(i) : 0.f;
        }
        f((c0 + u * THREADS) * N, v, v2, std::integral_constant<int, N>{});
      }
  }
  const int i = n * N + static_cast<int>(threadIdx.x);
  if (i < V) {
    const float v[1] = {value_at<DT>(row, i)}, v2[1] = {TWO ? value_at<DT>(other, i) : 0.f};
    f(i, v, v2, std::integral_constant<int, 1>{});
  }
}
template <cab_dtype_t DT, int U, int THREADS, typename F>
__device__ __forceinline__ void over_row(const char* row, int V, F f) {
  over_rows<DT, U, THREADS, false>(row, nullptr, V,
                                   [&](int at, const float* v, const float*, auto n) { f(at, v, n); });
}

// weight() with the exponent in one product: off by 2^-24 of the exponent, which is as
// exact for the values near the maximum that sums are made of.
__device__ __forceinline__ float near_weight(float x, float m, const VerifyArgs& a) {
  return x == m ? 1.f : __builtin_amdgcn_exp2f(fmaxf(x - m, a.d_min) * a.c_hi);
}

// Maximum (at least the lowest float) and sum of weights of a row.
template <cab_dtype_t DT, int THREADS>
__device__ void row_softmax(const char* row, int V, const VerifyArgs& a, Scratch<THREADS>& sh, float& m,
                            double& s) {
  float mt = -__FLT_MAX__;
  double st = 0.0;
  over_row<DT, 4, THREADS>(row, V, [&](int, const float* v, auto n) {
    constexpr int N = decltype(n)::value;
    float hi = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) hi = fmaxf(hi, v[i]);
    if (hi > mt) {
      st *= weight(mt, hi, a);
      mt = hi;
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += near_weight(v[i], mt, a);
    st += sum;
  });
  float mw = mt;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) mw = fmaxf(mw, shfl_xor_f32(mw, off));
  __syncthreads();
  if (lane_id() == 0) sh.m[threadIdx.x >> 6] = mw;
  __syncthreads();
  m = sh.m[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) m = fmaxf(m, sh.m[w]);
  s = block_sum<THREADS>(st * weight(mt, m, a), sh);
}

// order_key of the largest value (NaN below all) and its lowest index; 0 if there is none.
template <cab_dtype_t DT, int THREADS>
__device__ unsigned long long row_argmax(const char* row, int V, Scratch<THREADS>& sh) {
  float best = -INFINITY;
  int index = -1;
  over_row<DT, 4, THREADS>(row, V, [&](int at, const float* v, auto n) {
#pragma unroll
    for (int i = 0; i < decltype(n)::value; ++i)
      if (v[i] > best) {  // (indexes ascend within a thread)
        best = v[i];
        index = at + i;
      }
  });
  return block_max<THREADS>(index >= 0 ? order_key(best, index) : 0, sh);
}

// Grid: slices of rows, row-major; blockIdx.y: logits, or the drafts'.
template <cab_dtype_t DT, int MODE>
__global__ __launch_bounds__(SLICE_THREADS) void stats_kernel(VerifyArgs a) {
  __shared__ Scratch<SLICE_THREADS> sh;
  const int64_t row = blockIdx.x / a.slices;
  const int slice = static_cast<int>(blockIdx.x - row * a.slices);
  const int b = static_cast<int>(row / a.T), node = static_cast<int>(row - static_cast<int64_t>(b) * a.T);
  // Rows without children decide nothing (greedy: any row may give the next token).
  if constexpr (MODE != GREEDY) {
    const int i = threadIdx.x;  // (as many threads as a tree has nodes at most)
    const int mine = i > node && i < a.T && a.parents[b * a.parents_ld + i] == node;
    if (!__syncthreads_or(mine)) return;
  }
  constexpr int ES = DT == CAB_F32 ? 4 : 2;
  const char* p = blockIdx.y ? a.drafts + b * a.ds[0] + node * a.ds[1] : a.logits + b * a.ls[0] + node * a.ls[1];
  const int from = slice * a.slice, n = min(a.slice, a.V - from);
  p += static_cast<int64_t>(from) * ES;
  RowStats r;
  if constexpr (MODE == GREEDY) {
    r.key = row_argmax<DT, SLICE_THREADS>(p, n, sh);
    if (r.key) r.key -= static_cast<uint32_t>(from);  // (indexes are stored downwards)
    r.m = 0.f;
  } else {
    row_softmax<DT, SLICE_THREADS>(p, n, a, sh, r.m, r.s);
  }
  r.unused = 0.f;
  if (threadIdx.x == 0) a.stats[(blockIdx.y * a.rows + row) * a.slices + slice] = r;
}

// A row's statistics from its slices', in the `width` lanes that hold one each (a power of
// two; st null: none).
__device__ __forceinline__ void merge_softmax(const RowStats* st, int width, const VerifyArgs& a, float& m,
                                              double& s) {
  const float ml = st ? st->m : -__FLT_MAX__;
  const double sl = st ? st->s : 0.0;
  m = ml;
  for (int off = width >> 1; off >= 1; off >>= 1) m = fmaxf(m, shfl_xor_f32(m, off));
  s = sl * weight(ml, m, a);
  for (int off = width >> 1; off >= 1; off >>= 1) s += shfl_xor_f64(s, off);
}
__device__ __forceinline__ unsigned long long merge_argmax(const RowStats* st, int width) {
  unsigned long long key = st ? st->key : 0;
  for (int off = width >> 1; off >= 1; off >>= 1) {
    const unsigned long long o = __shfl_xor(key, off, 64);
    key = o > key ? o : key;
  }
  return key;
}

// Sums and weights are off by 1e-7 of the row's, so what is left after rejections, by
// subtraction, by up to that over its share: below this share it is summed anew (a pass over
// the row, which one node in 16 needs at most).
constexpr double LEAST_LEFT = 1.0 / 16;

// STATS: rows' statistics are there. Where the walk ended is left for pick_kernel.
template <cab_dtype_t DT, int MODE, bool STATS>
__global__ __launch_bounds__(WALK_THREADS) void walk_kernel(VerifyArgs a) {
  constexpr int THREADS = WALK_THREADS;
  // gone: rejected tokens at the end; greedy with STATS: the rows' argmax.
  __shared__ int32_t parent[MAX_NODES], token[MAX_NODES], out[MAX_NODES], gone[MAX_NODES];
  // Each draft's uniform number, and its logit in its parent's row (and the draft's).
  __shared__ float uniform[MAX_NODES], value[MAX_NODES], drawn[MODE == DRAFT ? MAX_NODES : 1];
  // STATS: rows' maxima and sums (of nodes without children, whatever the workspace held).
  constexpr int SIDES = MODE == DRAFT ? 2 : 1;
  __shared__ float high[STATS ? SIDES : 1][MAX_NODES];
  __shared__ double total[STATS ? SIDES : 1][MAX_NODES];
  __shared__ Scratch<THREADS> sh;
  const int b = blockIdx.x, tid = threadIdx.x, lane = lane_id();
  const char* logits = a.logits + b * a.ls[0];
  const char* drafts = MODE == DRAFT ? a.drafts + b * a.ds[0] : nullptr;
  for (int i = tid; i < MAX_NODES; i += THREADS) {
    out[i] = -1;
    parent[i] = -1;  // (nodes 0 and past T are nobody's children)
    if (i > 0 && i < a.T) {
      const int32_t p = a.parents[b * a.parents_ld + i];
      const int64_t x = a.tokens[static_cast<int64_t>(b) * a.T + i];
      const bool in = x >= 0 && x < a.V;
      parent[i] = p < i ? p : -1;
      token[i] = in ? static_cast<int32_t>(x) : -1;  // -1: passed over
      if constexpr (MODE != GREEDY) {
        uniform[i] = a.uniforms[static_cast<int64_t>(b) * a.T + i];
        if (in && p >= 0 && p < i) {
          value[i] = value_at<DT>(logits + p * a.ls[1], static_cast<int>(x));
          if constexpr (MODE == DRAFT) drawn[i] = value_at<DT>(drafts + p * a.ds[1], static_cast<int>(x));
        }
      }
    }
  }
  if constexpr (STATS) {
    // All at once: the walk itself then waits for no memory.
    const RowStats* stats = a.stats + static_cast<int64_t>(b) * a.T * a.slices;
    int width = 1;  // lanes a row
    while (width < a.slices) width <<= 1;
    const int at = tid & (width - 1);
    for (int x = tid / width; x - tid / width < SIDES * a.T; x += THREADS / width) {
      const int side = x >= a.T, i = x - side * a.T;
      const bool in = x < SIDES * a.T;
      const RowStats* st = in && at < a.slices ? stats + (side * a.rows + i) * a.slices + at : nullptr;
      if constexpr (MODE == GREEDY) {
        const unsigned long long key = merge_argmax(st, width);
        if (in && at == 0) gone[i] = key ? key_index(key) : -1;
      } else {
        float m;
        double s;
        merge_softmax(st, width, a, m, s);
        if (in && at == 0) {
          high[side][i] = m;
          total[side][i] = s;
        }
      }
    }
  }
  __syncthreads();
  // (every wave scans and decides alike; only row passes meet at barriers)
  auto next_child = [&](int node, int after) {
    for (int i0 = (after + 1) & ~63; i0 < a.T; i0 += 64) {
      const int i = i0 + lane;
      const uint64_t m = ballot64(i > after && parent[i] == node);
      if (m) return i0 + __builtin_ctzll(m);
    }
    return -1;
  };
  auto softmax_of = [&](int side, int node, const char* row, float& m, double& s) {
    if constexpr (STATS) {
      m = high[side][node];
      s = total[side][node];
    } else {
      row_softmax<DT, THREADS>(row, a.V, a, sh, m, s);
    }
  };
  const char* lrow;
  const char* qrow = nullptr;
  float m = 0.f, mq = 0.f;
  double s = 0.0, ip = 0.0, iq = 0.0, left = 0.0, used = 0.0;
  int node = 0, count = 0, best = -1;
  for (;;) {
    if (tid == 0) out[count] = node;
    ++count;
    lrow = logits + node * a.ls[1];
    int taken = -1;
    const int first = next_child(node, node);
    if constexpr (MODE == GREEDY) {
      if constexpr (STATS) {
        best = gone[node];
      } else {
        const unsigned long long key = row_argmax<DT, THREADS>(lrow, a.V, sh);
        best = key ? key_index(key) : -1;
      }
      for (int i = first; i >= 0 && taken < 0; i = next_child(node, i))
        if (token[i] >= 0 && token[i] == best) taken = i;
    } else if constexpr (MODE == POINT) {
      if (first >= 0) softmax_of(0, node, lrow, m, s);
      left = s;
      double base = s;     // what the row's last pass gave
      int rejected = 0;    // tokens in gone
      for (int i = first; i >= 0 && taken < 0; i = next_child(node, i)) {
        const int x = token[i];
        if (x < 0) continue;
        bool before = false;  // an earlier sibling's token: its weight is gone
        for (int j0 = 0; j0 < i; j0 += 64) {
          const int j = j0 + lane;
          before = before || ballot64(j < i && parent[j] == node && token[j] == x) != 0;
        }
        if (before) continue;
        if (left < base * LEAST_LEFT) {
          __syncthreads();  // (gone is there)
          double c = 0.0;
          over_row<DT, 4, THREADS>(lrow, a.V, [&](int at, const float* v, auto n) {
            const uint32_t out_of = gone_mask<decltype(n)::value>(gone, rejected, at);
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < decltype(n)::value; ++k) sum += out_of >> k & 1 ? 0.f : weight(v[k], m, a);
            c += sum;
          });
          base = left = block_sum<THREADS>(c, sh);
        }
        const float e = weight(value[i], m, a);
        if (static_cast<double>(uniform[i]) * left < static_cast<double>(e)) {
          taken = i;
        } else {
          left = fmax(left - static_cast<double>(e), 0.0);
          if (tid == 0) gone[rejected] = x;
          ++rejected;
        }
      }
    } else {
      qrow = drafts + node * a.ds[1];
      left = 1.0;
      used = 0.0;
      if (first >= 0) {
        double sq;
        softmax_of(0, node, lrow, m, s);
        softmax_of(1, node, qrow, mq, sq);
        ip = s > 0.0 ? 1.0 / s : 0.0;
        iq = sq > 0.0 ? 1.0 / sq : 0.0;
      }
      bool known = true;  // left is the residual's sum
      for (int i = first; i >= 0 && taken < 0; i = next_child(node, i)) {
        if (token[i] < 0) continue;
        if (!known) {
          double c = 0.0;
          const double uq = used * iq;
          const float fp = static_cast<float>(ip), fq = static_cast<float>(uq);
          over_rows<DT, 4, THREADS, true>(lrow, qrow, a.V, [&](int, const float* v, const float* v2, auto n) {
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < decltype(n)::value; ++k)
              sum += residual32(near_weight(v[k], m, a), fp, near_weight(v2[k], mq, a), fq);
            c += sum;
          });
          left = block_sum<THREADS>(c, sh);
          known = true;
        }
        const float ep = weight(value[i], m, a);
        const float eq = weight(drawn[i], mq, a);
        if (static_cast<double>(uniform[i]) * left * (eq * iq) < residual(ep, ip, eq, used * iq)) {
          taken = i;
        } else {
          used += left;
          known = false;
        }
      }
    }
    if (taken < 0) break;
    node = taken;
  }

  // The rejected tokens: all the children's.
  int n_gone = 0;
  if constexpr (MODE == POINT)
    for (int i = next_child(node, node); i >= 0; i = next_child(node, i)) {
      if (tid == 0) gone[n_gone] = token[i];
      ++n_gone;
    }
  __syncthreads();
  for (int i = tid; i < a.T; i += THREADS) a.path[static_cast<int64_t>(b) * a.T + i] = out[i];
  if (tid == 0) a.counts[b] = count;
  if constexpr (MODE == GREEDY) {
    if (tid == 0) a.next[b] = best;
  } else {
    WalkEnd& e = a.ends[b];
    for (int i = tid; i < n_gone; i += THREADS) e.gone[i] = gone[i];
    if (tid == 0) {
      e.ip = ip;
      e.iq = iq;
      e.used = used;
      e.m = m;
      e.mq = mq;
      e.node = node;
      e.n_gone = n_gone;
      e.done = 0;
    }
  }
}

// Grid: slices of a row, by sequence. A thread compares its values relative to the
// largest it has seen (a leaf's row has no statistics, and none are needed: the
// argmax is the same whatever all weights are relative to), or, where the residual takes
// the draft's weights off, to the row's. The sequence's last workgroup compares the slices'.
template <cab_dtype_t DT, int MODE>
__global__ __launch_bounds__(SLICE_THREADS) void pick_kernel(VerifyArgs a) {
  constexpr int ES = DT == CAB_F32 ? 4 : 2;
  __shared__ Scratch<SLICE_THREADS> sh;
  __shared__ int32_t gone[MAX_NODES];
  __shared__ bool last;
  const int b = blockIdx.x / a.picks_a_row, at_slice = blockIdx.x - b * a.picks_a_row, tid = threadIdx.x;
  WalkEnd& e = a.ends[b];
  const int n_gone = MODE == POINT ? e.n_gone : 0;
  const int from = at_slice * a.pick, n = min(a.pick, a.V - from);
  const char* lrow = a.logits + b * a.ls[0] + e.node * a.ls[1] + static_cast<int64_t>(from) * ES;
  const float* noise = a.noise + static_cast<int64_t>(b) * a.V + from;
  if constexpr (MODE == POINT) {
    gone[tid] = e.gone[tid] - from;  // (behind n_gone: whatever the workspace held)
    __syncthreads();
  }
  // top[0]: of the residual; top[1]: of the row, for when nothing is left of that.
  const bool whole = MODE == POINT || e.used == 0.0;
  struct Top {
    float score, x, y;  // x, y: the logit and 1 / noise it comes from
    int32_t at;
  };
  Top top[2] = {{-1.f, 0.f, 0.f, -1}, {-1.f, 0.f, 0.f, -1}};
  float m = -__FLT_MAX__;
  auto score_of = [&](float x, float iy, float to) {
    const float w = weight(x, to, a);
    return w > 0.f ? w * iy : -1.f;
  };
  auto beat = [](Top& t, float score, float x, float y, int at) {
    if (score > t.score) t = Top{score, x, y, at};  // (indexes ascend within a thread; NaN beats nothing)
  };
  // Scores of another reference are formed anew from logit and noise: equal ones stay equal.
  auto refer = [&](Top& t, float to) {
    t.score = t.at >= 0 ? score_of(t.x, t.y, to) : -1.f;
    if (!(t.score >= 0.f)) t = Top{-1.f, 0.f, 0.f, -1};
  };
  if (whole) {
    over_row<DT, 1, SLICE_THREADS>(lrow, n, [&](int at, const float* v, auto nn) {
      constexpr int N = decltype(nn)::value;
      float y[N], hi = m;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        y[k] = noise[at + k];
        hi = fmaxf(hi, v[k]);
      }
      if (hi > m) {
        m = hi;
        refer(top[0], m);
        refer(top[1], m);
      }
      const uint32_t out_of = gone_mask<N>(gone, n_gone, at);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float iy = __builtin_amdgcn_rcpf(y[k]), score = score_of(v[k], iy, m);
        const bool out = out_of >> k & 1;
        beat(top[0], out ? -1.f : score, v[k], iy, from + at + k);
        if (out_of) beat(top[1], out ? score : -1.f, v[k], iy, from + at + k);
      }
    });
  } else {
    const char* qrow = a.drafts + b * a.ds[0] + e.node * a.ds[1] + static_cast<int64_t>(from) * ES;
    const double ip = e.ip, uq = e.used * e.iq;
    const float mq = e.mq;
    m = e.m;
    over_rows<DT, 1, SLICE_THREADS, true>(lrow, qrow, n, [&](int at, const float* v, const float* v2, auto nn) {
#pragma unroll
      for (int k = 0; k < decltype(nn)::value; ++k) {
        const float w = weight(v[k], m, a), iy = __builtin_amdgcn_rcpf(noise[at + k]);
        const float r = static_cast<float>(residual(w, ip, weight(v2[k], mq, a), uq));
        beat(top[0], r > 0.f ? r * iy : -1.f, v[k], iy, from + at + k);
        beat(top[1], w > 0.f ? w * iy : -1.f, v[k], iy, from + at + k);
      }
    });
  }
  // The workgroup's candidates.
  if (whole) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = fmaxf(m, shfl_xor_f32(m, off));
    if (lane_id() == 0) sh.m[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sh.m[0], sh.m[1]), fmaxf(sh.m[2], sh.m[3]));
    refer(top[0], m);
    refer(top[1], m);
  }
  unsigned long long mine[2], most[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) most[i] = mine[i] = top[i].at >= 0 ? order_key(top[i].score, top[i].at) : 0;
  block_max2<SLICE_THREADS>(most, sh);
  Candidate* const c = a.picks + blockIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (most[i] ? mine[i] == most[i] : tid == 0) {  // (keys of two threads differ: their indexes do)
      put(&c->index[i], top[i].at);
      put(&c->score[i], top[i].score);
      put(&c->x[i], top[i].x);
      put(&c->y[i], top[i].y);
    }
  if (tid == 0) put(&c->m, m);
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // (what was put has arrived)
  __syncthreads();
  if (tid == 0)
    last = __hip_atomic_fetch_add(&e.done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 ==
           static_cast<uint32_t>(a.picks_a_row);
  __syncthreads();
  if (!last || tid >= 64) return;
  const bool in = tid < a.picks_a_row;  // (at most 64)
  const Candidate* all = a.picks + static_cast<int64_t>(b) * a.picks_a_row + (in ? tid : 0);
  float hi = get(&all->m);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    top[i] = Top{get(&all->score[i]), get(&all->x[i]), get(&all->y[i]), get(&all->index[i])};
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) hi = fmaxf(hi, shfl_xor_f32(hi, off));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (whole) refer(top[i], hi);
    most[i] = in && top[i].at >= 0 ? order_key(top[i].score, top[i].at) : 0;
  }
  wave_max2(most);
  if (tid == 0) a.next[b] = most[0] ? key_index(most[0]) : most[1] ? key_index(most[1]) : -1;
}

// How a call is run: a row's slices, and the workspace.
struct VerifyPlan {
  bool stats;
  int64_t slices, slice, picks, pick;
  size_t off_ends, off_picks, bytes;
};

// Bytes of logits up to which all rows' statistics are taken (us, bf16, so -> rows one after
// another: 1 tree of 64, 128000 tokens 22 -> 43, 32 of 5 29 -> 55, 4 drafted ones of 26,
// fp32, 50001 30 -> 87; 32 of 32, 128000, 262 MB 58 -> 56; 64 of 64, 64000, 524 MB 96 -> 47).
constexpr int64_t STATS_BYTES = int64_t{1} << 28;

VerifyPlan verify_plan(cab_dtype_t dtype, int mode, int64_t B, int64_t T, int64_t V) {
  VerifyPlan p = {};
  const int64_t es = static_cast<int64_t>(dtype_size(dtype)), rows = B * T, sides = mode == DRAFT ? 2 : 1;
  // (stats_kernel's threads: 256 a slice, within 32 bits)
  p.stats = rows * sides <= STATS_BYTES / (V * es) && rows <= (int64_t{1} << 23);
  // Slices of up to `loads` 16-byte loads a thread (rows just past a whole number of them are
  // cut evenly: half as many in the worst case), longer ones where that were more than 64 a
  // row (one wave merges them) or more than fill the chip. (32 trees of 32 rows: 2048 workgroups
  // of statistics 68 us the call, 4096 60, 16384 62; 512 that pick 60, 1024 58, 2048 59.)
  auto cut = [&](int64_t loads, int64_t units, int64_t fill, int64_t& n, int64_t& size) {
    n = ceil_div(V, SLICE_THREADS * loads * 16 / es);
    if (n > ceil_div(fill, units)) n = ceil_div(fill, units);
    if (n > 64) n = 64;
    size = round_up(ceil_div(V, n), 16 / es);
    n = ceil_div(V, size);
  };
  cut(4, rows * sides, 4096, p.slices, p.slice);
  cut(1, B, 1024, p.picks, p.pick);
  p.off_ends = p.stats ? static_cast<size_t>(sides * rows * p.slices) * sizeof(RowStats) : 0;
  p.off_picks = p.off_ends + (mode == GREEDY ? 0 : static_cast<size_t>(B) * sizeof(WalkEnd));
  p.bytes = p.off_picks + (mode == GREEDY ? 0 : static_cast<size_t>(B * p.picks) * sizeof(Candidate));
  return p;
}

bool verify_sizes(int64_t B, int64_t T, int64_t V) {
  // (walk_kernel's threads: 1024 a sequence, within 32 bits)
  return T >= 1 && T <= MAX_NODES && B >= 1 && B <= (int64_t{1} << 21) && V >= 1 && V <= INT32_MAX / 2;
}

template <cab_dtype_t DT, int MODE>
void run(const VerifyPlan& p, const VerifyArgs& a, unsigned B, hipStream_t s) {
  if (!p.stats) {
    walk_kernel<DT, MODE, false><<<B, WALK_THREADS, 0, s>>>(a);
  } else {
    const dim3 grid(static_cast<unsigned>(a.rows * p.slices), MODE == DRAFT ? 2 : 1);
    stats_kernel<DT, MODE><<<grid, SLICE_THREADS, 0, s>>>(a);
    walk_kernel<DT, MODE, true><<<B, WALK_THREADS, 0, s>>>(a);
  }
  if constexpr (MODE != GREEDY)
    pick_kernel<DT, MODE><<<static_cast<unsigned>(p.picks) * B, SLICE_THREADS, 0, s>>>(a);
}

template <cab_dtype_t DT>
void launch(const VerifyPlan& p, const VerifyArgs& a, int mode, unsigned B, hipStream_t s) {
  switch (mode) {
    case GREEDY: run<DT, GREEDY>(p, a, B, s); break;
    case POINT: run<DT, POINT>(p, a, B, s); break;
    default: run<DT, DRAFT>(p, a, B, s); break;
  }
}

}  // namespace
}  // namespace cab

using namespace cab;

extern "C" size_t cab_verify_drafts_workspace_bytes(cab_dtype_t dtype, int64_t B, int64_t T,
                                                     int64_t V, int greedy, int drafted) {
  if (!valid_dtype(dtype) || !verify_sizes(B, T, V)) return 0;
  return verify_plan(dtype, greedy ? GREEDY : drafted ? DRAFT : POINT, B, T, V).bytes;
}

extern "C" cab_status_t cab_verify_drafts(const void* logits, const void* draft_logits,
                                          cab_dtype_t dtype, int64_t B, int64_t T, int64_t V,
                                          const int64_t logit_strides[2],
                                          const int64_t draft_strides[2], const int64_t* tokens,
                                          const int32_t* parents, int64_t parents_stride,
                                          const float* uniforms, const float* noise,
                                          float temperature, int32_t* path, int32_t* counts,
                                          int64_t* next_tokens, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  const char* fn = "cab_verify_drafts";
  clear_error();
  CAB_REQUIRE(valid_dtype(dtype), CAB_EDTYPE, "%s: unknown dtype %d", fn, static_cast<int>(dtype));
  CAB_REQUIRE(B >= 0 && T >= 1 && V >= 1, CAB_ESHAPE, "%s: bad shape", fn);
  CAB_REQUIRE(T <= MAX_NODES, CAB_ESHAPE, "%s: a tree holds at most %d nodes", fn, MAX_NODES);
  // (1 / temperature and the exponents it scales stay ordinary floats)
  CAB_REQUIRE(temperature == 0.f || (temperature >= 1e-6f && temperature <= 1e6f), CAB_EINVAL,
              "%s: temperature must be 0 (greedy) or in [1e-6, 1e6]", fn);
  if (B == 0) return CAB_OK;
  CAB_REQUIRE(verify_sizes(B, T, V), CAB_ESHAPE, "%s: problem too large", fn);
  const bool greedy = temperature == 0.f;
  CAB_REQUIRE(logits && logit_strides && tokens && parents && path && counts && next_tokens,
              CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(greedy || (uniforms && noise), CAB_EINVAL, "%s: sampling needs uniforms and noise", fn);
  CAB_REQUIRE(!draft_logits || draft_strides, CAB_EINVAL, "%s: null draft strides", fn);
  CAB_REQUIRE(parents_stride == 0 || parents_stride >= T, CAB_ESHAPE, "%s: bad parents stride", fn);
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  CAB_REQUIRE(reinterpret_cast<uintptr_t>(logits) % es == 0 &&
                  reinterpret_cast<uintptr_t>(draft_logits) % es == 0,
              CAB_ESHAPE, "%s: logits not aligned to their elements", fn);
  VerifyArgs a;
  a.logits = static_cast<const char*>(logits);
  a.drafts = static_cast<const char*>(draft_logits);
  for (int d = 0; d < 2; ++d) {
    a.ls[d] = logit_strides[d] * es;
    a.ds[d] = draft_logits ? draft_strides[d] * es : 0;
  }
  a.tokens = tokens;
  a.parents = parents;
  a.uniforms = uniforms;
  a.noise = noise;
  a.parents_ld = parents_stride;
  a.T = static_cast<int32_t>(T);
  a.V = static_cast<int32_t>(V);
  const double c = greedy ? 0.0 : 1.4426950408889634 / static_cast<double>(temperature);
  a.c_hi = static_cast<float>(c);
  a.c_lo = static_cast<float>(c - static_cast<double>(a.c_hi));
  a.d_min = greedy ? 0.f : static_cast<float>(-200.0 / c);  // 2^-200 is 0 in fp32
  a.path = path;
  a.counts = counts;
  a.next = next_tokens;
  const int mode = greedy ? GREEDY : draft_logits ? DRAFT : POINT;
  const VerifyPlan p = verify_plan(dtype, mode, B, T, V);
  CAB_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes &&
                               reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
              CAB_EWORKSPACE, "%s: workspace needs %zu bytes, 16-byte aligned", fn, p.bytes);
  char* ws = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<RowStats*>(ws);
  a.ends = reinterpret_cast<WalkEnd*>(ws + p.off_ends);
  a.picks = reinterpret_cast<Candidate*>(ws + p.off_picks);
  a.slices = static_cast<int32_t>(p.slices);
  a.slice = static_cast<int32_t>(p.slice);
  a.picks_a_row = static_cast<int32_t>(p.picks);
  a.pick = static_cast<int32_t>(p.pick);
  a.rows = B * T;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case CAB_F32: launch<CAB_F32>(p, a, mode, static_cast<unsigned>(B), s); break;
    case CAB_BF16: launch<CAB_BF16>(p, a, mode, static_cast<unsigned>(B), s); break;
    default: launch<CAB_F16>(p, a, mode, static_cast<unsigned>(B), s); break;
  }
  return launch_status(fn);
}
