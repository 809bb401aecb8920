// Verification of drafted tokens against the target's logits, from given random
// numbers (cab_verify_drafts). Node 0 of a sequence's tree is the token the model
// has taken already; the walk goes from it to the first child that is accepted, and
// so on. With p = softmax(logits[node] / temperature), and r the child's own uniform
// number:
//   greedy (temperature 0): the child whose token is the row's argmax;
//   point (no draft logits): a child x is accepted if r Z < p(x), where Z is what the
//     siblings rejected before it have left of p (their tokens' weights become 0);
//   draft, with q = softmax(draft_logits[node] / temperature): each rejection leaves
//     max(p - q, 0) / c of p. As max(max(y, 0) - z, 0) = max(y - z, 0) for z >= 0, the
//     residual after any number of rejections is max(p - a q, 0) / c with two numbers:
//     a' = a + c, c' = sum max(p - a' q, 0), from a = 0, c = 1. A child is accepted if
//     r c q(x) < max(p(x) - a q(x), 0).
// At the node with no accepted child the next token is argmax_x w(x) / noise(x) over
// the residual w; with noise ~ Exp(1) that is a sample of w / sum w. It needs no
// cumulative sum (whose order would decide between tokens) and no normaliser.
//
// Only the rows of accepted nodes are read. One workgroup of 16 waves walks a
// sequence's tree.
#include "cab_internal.h"

namespace cab {
namespace {

constexpr int MAX_NODES = 256;
constexpr int THREADS = 1024, WAVES = THREADS / 64;
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
};

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

struct Scratch {
  float m[WAVES];
  double s[WAVES];
  unsigned long long key[WAVES];
};

__device__ __forceinline__ double block_sum(double v, Scratch& sh) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += shfl_xor_f64(v, off);
  __syncthreads();
  if (lane_id() == 0) sh.s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) v += sh.s[w];
  return v;
}

__device__ __forceinline__ unsigned long long block_max(unsigned long long k, Scratch& sh) {
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
  for (int w = 0; w < WAVES; ++w) k = sh.key[w] > k ? sh.key[w] : k;
  return k;
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

// f(first index, number, values...) over a row's 16-byte chunks, U of them loaded at
// a time, then its last values one by one.
template <cab_dtype_t DT, int U, typename F>
__device__ __forceinline__ void over_row(const char* row, int V, F f) {
  constexpr int N = Chunk<DT>::N;
  const int n = V / N;
  for (int c0 = threadIdx.x; c0 < n; c0 += U * THREADS) {
    Chunk<DT> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * THREADS < n) x[u].load(row, c0 + u * THREADS);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * THREADS < n) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = x[u].get(i);
        f((c0 + u * THREADS) * N, v, std::integral_constant<int, N>{});
      }
  }
  const int i = n * N + static_cast<int>(threadIdx.x);
  if (i < V) {
    float v[1] = {value_at<DT>(row, i)};
    f(i, v, std::integral_constant<int, 1>{});
  }
}

// Maximum (at least the lowest float) and sum of weights of a row.
template <cab_dtype_t DT>
__device__ void row_softmax(const char* row, const VerifyArgs& a, Scratch& sh, float& m, double& s) {
  float mt = -__FLT_MAX__;
  double st = 0.0;
  over_row<DT, 4>(row, a.V, [&](int, const float* v, auto n) {
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
    for (int i = 0; i < N; ++i) sum += weight(v[i], mt, a);
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
  for (int w = 1; w < WAVES; ++w) m = fmaxf(m, sh.m[w]);
  s = block_sum(st * weight(mt, m, a), sh);
}

// The row's largest value (NaN below all) and its lowest index; -1 if there is none.
template <cab_dtype_t DT>
__device__ int row_argmax(const char* row, const VerifyArgs& a, Scratch& sh) {
  unsigned long long key = 0;
  over_row<DT, 4>(row, a.V, [&](int at, const float* v, auto n) {
#pragma unroll
    for (int i = 0; i < decltype(n)::value; ++i) {
      const unsigned long long k = order_key(v[i], at + i);
      if (v[i] > -INFINITY && k > key) key = k;
    }
  });
  key = block_max(key, sh);
  return key ? key_index(key) : -1;
}

template <cab_dtype_t DT, int MODE>
__global__ __launch_bounds__(THREADS) void verify_kernel(VerifyArgs a) {
  __shared__ int32_t parent[MAX_NODES], token[MAX_NODES], out[MAX_NODES], gone[MAX_NODES];
  __shared__ float uniform[MODE == GREEDY ? 1 : MAX_NODES];
  __shared__ Scratch sh;
  const int b = blockIdx.x, tid = threadIdx.x, lane = lane_id();
  for (int i = tid; i < MAX_NODES; i += THREADS) {
    out[i] = -1;
    parent[i] = -1;  // (nodes 0 and past T are nobody's children)
    if (i > 0 && i < a.T) {
      const int32_t p = a.parents[b * a.parents_ld + i];
      const int64_t x = a.tokens[static_cast<int64_t>(b) * a.T + i];
      parent[i] = p < i ? p : -1;
      token[i] = x >= 0 && x < a.V ? static_cast<int32_t>(x) : -1;  // -1: never accepted
      if constexpr (MODE != GREEDY) uniform[i] = a.uniforms[static_cast<int64_t>(b) * a.T + i];
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
  const char* lrow;
  const char* qrow = nullptr;
  float m = 0.f, mq = 0.f;
  double s = 0.0, ip = 0.0, iq = 0.0, left = 0.0, used = 0.0;
  int node = 0, count = 0, best = -1;
  for (;;) {
    if (tid == 0) out[count] = node;
    ++count;
    lrow = a.logits + b * a.ls[0] + node * a.ls[1];
    int taken = -1;
    if constexpr (MODE == GREEDY) {
      best = row_argmax<DT>(lrow, a, sh);
      for (int i = next_child(node, node); i >= 0 && taken < 0; i = next_child(node, i))
        if (token[i] >= 0 && token[i] == best) taken = i;
    } else if constexpr (MODE == POINT) {
      row_softmax<DT>(lrow, a, sh, m, s);
      left = s;
      for (int i = next_child(node, node); i >= 0 && taken < 0; i = next_child(node, i)) {
        const int x = token[i];
        if (x < 0) continue;
        bool before = false;  // an earlier sibling's token: its weight is gone
        for (int j0 = 0; j0 < i; j0 += 64) {
          const int j = j0 + lane;
          before = before || ballot64(j < i && parent[j] == node && token[j] == x) != 0;
        }
        if (before) continue;
        const float e = weight(value_at<DT>(lrow, x), m, a);
        if (static_cast<double>(uniform[i]) * left < static_cast<double>(e))
          taken = i;
        else
          left = fmax(left - static_cast<double>(e), 0.0);
      }
    } else {
      double sq;
      qrow = a.drafts + b * a.ds[0] + node * a.ds[1];
      row_softmax<DT>(lrow, a, sh, m, s);
      row_softmax<DT>(qrow, a, sh, mq, sq);
      ip = s > 0.0 ? 1.0 / s : 0.0;
      iq = sq > 0.0 ? 1.0 / sq : 0.0;
      left = 1.0;
      used = 0.0;
      bool known = true;  // left is the residual's sum
      for (int i = next_child(node, node); i >= 0 && taken < 0; i = next_child(node, i)) {
        if (!known) {
          double c = 0.0;
          const double uq = used * iq;
          over_row<DT, 2>(lrow, a.V, [&](int at, const float* v, auto n) {
#pragma unroll
            for (int k = 0; k < decltype(n)::value; ++k) {
              const float ep = weight(v[k], m, a);
              const float eq = weight(value_at<DT>(qrow, at + k), mq, a);
              c += residual(ep, ip, eq, uq);
            }
          });
          left = block_sum(c, sh);
          known = true;
        }
        const int x = token[i];
        if (x < 0) continue;
        const float ep = weight(value_at<DT>(lrow, x), m, a);
        const float eq = weight(value_at<DT>(qrow, x), mq, a);
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

  int64_t chosen = best;
  if constexpr (MODE != GREEDY) {
    // The rejected tokens: all the children's.
    int n_gone = 0;
    for (int i = next_child(node, node); MODE == POINT && i >= 0; i = next_child(node, i)) {
      if (tid == 0) gone[n_gone] = token[i];
      ++n_gone;
    }
    __syncthreads();
    const float* noise = a.noise + static_cast<int64_t>(b) * a.V;
    double uq = used * iq;
    unsigned long long key = 0;
    // The second time over the whole row's weights, if nothing is left of them.
    for (int pass = 0; pass < 2 && key == 0; ++pass) {
      over_row<DT, 2>(lrow, a.V, [&](int at, const float* v, auto n) {
        constexpr int N = decltype(n)::value;
        uint32_t out_of = 0;
        for (int k = 0; k < n_gone; ++k) {
          const uint32_t d = static_cast<uint32_t>(gone[k] - at);
          if (d < static_cast<uint32_t>(N)) out_of |= 1u << d;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          float w = weight(v[k], m, a);
          if constexpr (MODE == DRAFT)
            w = static_cast<float>(residual(w, ip, weight(value_at<DT>(qrow, at + k), mq, a), uq));
          const float score = w * __builtin_amdgcn_rcpf(noise[at + k]);
          const unsigned long long o = order_key(score, at + k);
          if (w > 0.f && score >= 0.f && !(out_of >> k & 1) && o > key) key = o;
        }
      });
      key = block_max(key, sh);
      uq = 0.0;
      n_gone = 0;
    }
    chosen = key ? key_index(key) : -1;
  }
  __syncthreads();
  for (int i = tid; i < a.T; i += THREADS) a.path[static_cast<int64_t>(b) * a.T + i] = out[i];
  if (tid == 0) {
    a.counts[b] = count;
    a.next[b] = chosen;
  }
}

template <cab_dtype_t DT>
void launch(const VerifyArgs& a, int mode, unsigned B, hipStream_t s) {
  switch (mode) {
    case GREEDY: verify_kernel<DT, GREEDY><<<B, THREADS, 0, s>>>(a); break;
    case POINT: verify_kernel<DT, POINT><<<B, THREADS, 0, s>>>(a); break;
    default: verify_kernel<DT, DRAFT><<<B, THREADS, 0, s>>>(a); break;
  }
}

}  // namespace
}  // namespace cab

using namespace cab;

extern "C" cab_status_t cab_verify_drafts(const void* logits, const void* draft_logits,
                                          cab_dtype_t dtype, int64_t B, int64_t T, int64_t V,
                                          const int64_t logit_strides[2],
                                          const int64_t draft_strides[2], const int64_t* tokens,
                                          const int32_t* parents, int64_t parents_stride,
                                          const float* uniforms, const float* noise,
                                          float temperature, int32_t* path, int32_t* counts,
                                          int64_t* next_tokens, void* stream) {
  const char* fn = "cab_verify_drafts";
  clear_error();
  CAB_REQUIRE(valid_dtype(dtype), CAB_EDTYPE, "%s: unknown dtype %d", fn, static_cast<int>(dtype));
  CAB_REQUIRE(B >= 0 && T >= 1 && V >= 1, CAB_ESHAPE, "%s: bad shape", fn);
  CAB_REQUIRE(T <= MAX_NODES, CAB_ESHAPE, "%s: a tree holds at most %d nodes", fn, MAX_NODES);
  CAB_REQUIRE(V <= INT32_MAX / 2 && B <= INT32_MAX, CAB_ESHAPE, "%s: problem too large", fn);
  // (1 / temperature and the exponents it scales stay ordinary floats)
  CAB_REQUIRE(temperature == 0.f || (temperature >= 1e-6f && temperature <= 1e6f), CAB_EINVAL,
              "%s: temperature must be 0 (greedy) or in [1e-6, 1e6]", fn);
  if (B == 0) return CAB_OK;
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case CAB_F32: launch<CAB_F32>(a, mode, static_cast<unsigned>(B), s); break;
    case CAB_BF16: launch<CAB_BF16>(a, mode, static_cast<unsigned>(B), s); break;
    default: launch<CAB_F16>(a, mode, static_cast<unsigned>(B), s); break;
  }
  return launch_status(fn);
}
