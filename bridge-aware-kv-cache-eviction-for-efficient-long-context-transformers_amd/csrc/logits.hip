// Logits before the next token is chosen (cab_adjust_logits): penalties for repeated tokens,
// biases, and the tokens that a grammar allows, in one pass.
//
//   x = logits[b, t, v];  c = times v was generated, counted from the history behind the prompt
//   and (a tree of drafts) from node t's line;  seen = c > 0 or v is in the prompt
//   x = seen ? (x > 0 ? x / r : x r) : x;  x -= f c + p [c > 0];  x += bias;  not allowed: -inf
//
// Bound: HBM, each row read and written once. A workgroup takes a stretch of the vocabulary of
// one sequence and counts the history's tokens that fall into it in LDS (whole numbers: the order
// of the atomics does not show). A bit per token says which have a count or a bias at all,
// so that almost all values pass with two LDS reads a 16 bytes. In a tree the counts stay as they
// are from node to node, and only the tokens of a node's line are added and taken off again.
// The history is read again for each stretch, from L2: stretches are long where rows are many.
#include "attn_common.h"
#include "row_layout.h"

namespace cab {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_NODES = 256;
constexpr uint32_t GIVEN = 0x80000000u;  // in the prompt; below it the count

struct AdjustArgs {
  const char* x;
  char* out;
  int64_t xs[2], os[2];  // bytes: b, t
  int32_t B, T, V, stretch, stretches, nodes;  // nodes: of a workgroup
  const int32_t* history;
  int64_t history_ld;
  int32_t L;
  const int32_t* lengths;  // may be null: L
  const int32_t* prompts;  // may be null: 0
  const float *repetition, *presence, *frequency;  // [B], may be null: the values below
  float r, p, f;
  const int32_t* bias_tokens;
  const float* bias;
  int64_t bias_ld;
  int32_t biases;
  const uint32_t* allowed;
  int64_t as[2];  // words: b, t
  const int64_t* drafts;  // [B, T], may be null
  const int32_t* parents;
  int64_t parents_ld;
};

template <cab_dtype_t DT> __device__ __forceinline__ float load1(const char* p) {
  if constexpr (DT == CAB_F32) return *reinterpret_cast<const float*>(p);
  const uint16_t h = *reinterpret_cast<const uint16_t*>(p);
  return DT == CAB_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
}
template <cab_dtype_t DT> __device__ __forceinline__ void store1(char* p, float x) {
  if constexpr (DT == CAB_F32) *reinterpret_cast<float*>(p) = x;
  else *reinterpret_cast<uint16_t*>(p) = DT == CAB_BF16 ? f32_to_bf16(x) : f32_to_f16(x);
}

// LDS: counts [stretch], places in the list of biases [stretch] (with biases), bits, lines.
template <cab_dtype_t DT, bool BIAS, bool TREE>
__global__ __launch_bounds__(THREADS) void adjust_kernel(AdjustArgs a) {
  constexpr int ES = DT == CAB_F32 ? 4 : 2, P = 16 / ES;
  extern __shared__ uint32_t lds[];
  uint32_t* count = lds;
  uint32_t* place = count + a.stretch;  // 1 + the place; 0: none
  uint32_t* bits = place + (BIAS ? a.stretch : 0);
  uint32_t* line = bits + a.stretch / 32 + 1;  // [T][8]
  const int id = blockIdx.x;
  const int part = id % a.stretches, rest = id / a.stretches;
  const int groups = (a.T + a.nodes - 1) / a.nodes;
  const int group = rest % groups, b = rest / groups;
  const int v0 = part * a.stretch, v1 = min(a.V, v0 + a.stretch);
  const uint32_t span = v1 - v0;
  for (int i = threadIdx.x; i < a.stretch; i += THREADS) {
    count[i] = 0;
    if (BIAS) place[i] = 0;
  }
  for (int i = threadIdx.x; i < a.stretch / 32 + 1; i += THREADS) bits[i] = 0;
  __syncthreads();
  auto mark = [&](uint32_t at) { atomicOr(&bits[at >> 5], 1u << (at & 31)); };
  if (a.history) {
    const int32_t* h = a.history + b * a.history_ld;
    const int len = min(a.lengths ? a.lengths[b] : a.L, a.L);
    const int given = a.prompts ? a.prompts[b] : 0;
    auto tell = [&](int i, int32_t token) {
      const uint32_t at = static_cast<uint32_t>(token) - static_cast<uint32_t>(v0);
      if (at >= span || token < 0 || i >= len) return;
      if (i < given) atomicOr(&count[at], GIVEN);
      else atomicAdd(&count[at], 1u);
      mark(at);
    };
    if ((reinterpret_cast<uintptr_t>(h) & 15) == 0) {
      for (int i = 4 * threadIdx.x; i < len; i += 4 * THREADS) {
        if (i + 4 <= a.L) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(h + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t token = w[e];
            tell(i + e, static_cast<int32_t>(token));
          }
        } else {
          for (int e = i; e < len; ++e) tell(e, h[e]);
        }
      }
    } else {
      for (int i = threadIdx.x; i < len; i += THREADS) tell(i, h[i]);
    }
  }
  if constexpr (BIAS) {
    for (int i = threadIdx.x; i < a.biases; i += THREADS) {
      const int32_t token = a.bias_tokens[b * a.bias_ld + i];
      const uint32_t at = static_cast<uint32_t>(token) - static_cast<uint32_t>(v0);
      if (at >= span || token < 0) continue;
      atomicMax(&place[at], static_cast<uint32_t>(i) + 1);  // (listed twice: the last one)
      mark(at);
    }
  }
  const int32_t* parents = a.parents + b * a.parents_ld;
  int64_t draft = -1;  // thread j: node j's token
  if constexpr (TREE) {
    const int j = threadIdx.x;
    if (j < a.T) {
      draft = a.drafts[static_cast<int64_t>(b) * a.T + j];
      uint32_t* mine = line + 8 * j;
      for (int w = 0; w < 8; ++w) mine[w] = 0;
      for (int i = j;;) {
        mine[i >> 5] |= 1u << (i & 31);
        const int up = parents[i];
        if (up < 0 || up >= i) break;
        i = up;
      }
    }
  }
  const bool here = TREE && draft >= v0 && draft < v1;
  const uint32_t draft_at = here ? static_cast<uint32_t>(draft - v0) : 0;
  if constexpr (TREE)
    if (here) mark(draft_at);
  __syncthreads();

  const float r = a.repetition ? a.repetition[b] : a.r;
  const float p = a.presence ? a.presence[b] : a.p;
  const float f = a.frequency ? a.frequency[b] : a.f;
  auto adjusted = [&](float x, uint32_t at) {
    const uint32_t c = count[at], n = c & ~GIVEN;
    if (c) x = x > 0.f ? x / r : x * r;
    if (n) x = x - f * static_cast<float>(n) - p;
    if constexpr (BIAS) {
      const uint32_t i = place[at];
      if (i) x += a.bias[b * a.bias_ld + i - 1];
    }
    return x;
  };
  const int t1 = min(a.T, (group + 1) * a.nodes);
  for (int t = group * a.nodes; t < t1; ++t) {
    bool mine = false;
    if constexpr (TREE) {
      mine = here && (line[8 * t + (threadIdx.x >> 5)] >> (threadIdx.x & 31) & 1u);
      if (mine) atomicAdd(&count[draft_at], 1u);
      __syncthreads();
    }
    const char* x = a.x + b * a.xs[0] + t * a.xs[1];
    char* out = a.out + b * a.os[0] + t * a.os[1];
    const uint32_t* allowed = a.allowed ? a.allowed + b * a.as[0] + t * a.as[1] : nullptr;
    auto single = [&](int v) {
      const uint32_t at = v - v0;
      float y = load1<DT>(x + static_cast<int64_t>(v) * ES);
      if (bits[at >> 5] >> (at & 31) & 1u) y = adjusted(y, at);
      if (allowed && !(allowed[v >> 5] >> (v & 31) & 1u)) y = -INFINITY;
      store1<DT>(out + static_cast<int64_t>(v) * ES, y);
    };
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) & 15);
    if (off == (reinterpret_cast<uintptr_t>(out) & 15)) {
      // Whole 16 bytes, and what is before and behind them one by one.
      const int lead = (P - (v0 + static_cast<int>(off) / ES) % P) % P;
      const int from = min(v1, v0 + lead), units = (v1 - from) / P;
      for (int u = threadIdx.x; u < units; u += THREADS) {
        const int v = from + u * P;
        const uint32_t at = v - v0;
        u32x4 w = *reinterpret_cast<const u32x4*>(x + static_cast<int64_t>(v) * ES);
        const uint64_t two = bits[at >> 5] | static_cast<uint64_t>(bits[(at >> 5) + 1]) << 32;
        const uint32_t hit = static_cast<uint32_t>(two >> (at & 31)) & ((1u << P) - 1);
        uint32_t keep = (1u << P) - 1;
        if (allowed) {
          const uint32_t lo = allowed[v >> 5], hi = allowed[(v + P - 1) >> 5];
          keep &= static_cast<uint32_t>((lo | static_cast<uint64_t>(hi) << 32) >> (v & 31));
        }
        if (hit) {
#pragma unroll
          for (int e = 0; e < P; ++e) {
            if (!(hit >> e & 1u)) continue;
            if constexpr (DT == CAB_F32) {
              const uint32_t y = w[e];
              w[e] = __float_as_uint(adjusted(__uint_as_float(y), at + e));
            } else {
              const uint32_t y = w[e >> 1];
              const uint16_t old = static_cast<uint16_t>(e & 1 ? y >> 16 : y);
              const float z = adjusted(DT == CAB_BF16 ? bf16_to_f32(old) : f16_to_f32(old), at + e);
              const uint32_t now = DT == CAB_BF16 ? f32_to_bf16(z) : f32_to_f16(z);
              w[e >> 1] = e & 1 ? (y & 0xffffu) | now << 16 : (y & 0xffff0000u) | now;
            }
          }
        }
        if (keep != (1u << P) - 1) {
          constexpr uint32_t LOW = DT == CAB_F32 ? 0xff800000u : DT == CAB_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
          for (int e = 0; e < P; ++e) {
            if (keep >> e & 1u) continue;
            if constexpr (DT == CAB_F32) w[e] = LOW;
            else w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | LOW << 16 : (w[e >> 1] & 0xffff0000u) | LOW;
          }
        }
        *reinterpret_cast<u32x4*>(out + static_cast<int64_t>(v) * ES) = w;
      }
      for (int v = v0 + threadIdx.x; v < from; v += THREADS) single(v);
      for (int v = from + units * P + threadIdx.x; v < v1; v += THREADS) single(v);
    } else {
      for (int v = v0 + threadIdx.x; v < v1; v += THREADS) single(v);
    }
    if constexpr (TREE) {
      __syncthreads();  // (this node's counts have been read)
      if (mine) atomicSub(&count[draft_at], 1u);
    }
  }
}

}  // namespace
}  // namespace cab

using namespace cab;

extern "C" cab_status_t cab_adjust_logits(
    const void* logits, void* out, cab_dtype_t dtype, int64_t B, int64_t T, int64_t V,
    const int64_t logit_strides[2], const int64_t out_strides[2], const int32_t* history,
    int64_t history_len, int64_t history_stride, const int32_t* lengths,
    const int32_t* prompt_lengths, const float* repetition, float repetition0,
    const float* presence, float presence0, const float* frequency, float frequency0,
    const int32_t* bias_tokens, const float* bias, int64_t biases, int64_t bias_stride,
    const int32_t* allowed, const int64_t allowed_strides[2], const int64_t* drafts,
    const int32_t* parents, int64_t parents_stride, void* stream) {
  const char* fn = "cab_adjust_logits";
  clear_error();
  CAB_REQUIRE(valid_dtype(dtype), CAB_EDTYPE, "%s: unknown dtype %d", fn, static_cast<int>(dtype));
  CAB_REQUIRE(B >= 0 && T >= 0 && V >= 0 && history_len >= 0 && biases >= 0, CAB_ESHAPE,
              "%s: negative size", fn);
  CAB_REQUIRE(drafts == nullptr || T <= MAX_NODES, CAB_ESHAPE, "%s: a tree holds up to %d nodes", fn,
              MAX_NODES);
  if (B == 0 || T == 0 || V == 0) return CAB_OK;
  CAB_REQUIRE(logits && out && logit_strides && out_strides, CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(V <= INT32_MAX / 2 && history_len <= INT32_MAX / 2 && biases <= INT32_MAX / 2 &&
                  T <= INT32_MAX / 2,
              CAB_ESHAPE, "%s: problem too large", fn);
  const bool tree = drafts != nullptr, with_bias = biases > 0;
  // The longest stretch that leaves some four workgroups a CU.
  int64_t stretch = with_bias ? 4096 : 8192;  // (64 KB of LDS)
  while (stretch > 1024 && ceil_div(V, stretch) * T < ceil_div(1024, B)) stretch /= 2;
  const int64_t stretches = ceil_div(V, stretch);
  int64_t groups = ceil_div(1024, B);
  groups = ceil_div(groups, stretches);
  if (groups > T) groups = T;
  const int64_t nodes = ceil_div(T, groups);
  groups = ceil_div(T, nodes);
  // (threads of the launch: fewer than 2^32)
  CAB_REQUIRE(groups * stretches < (int64_t{1} << 24) && B < (int64_t{1} << 24) / (groups * stretches),
              CAB_ESHAPE, "%s: problem too large", fn);
  CAB_REQUIRE(history_len == 0 || (history && (history_stride == 0 || history_stride >= history_len)),
              CAB_EINVAL, "%s: no history, or a bad stride of it", fn);
  CAB_REQUIRE(biases == 0 || (bias_tokens && bias && (bias_stride == 0 || bias_stride >= biases)),
              CAB_EINVAL, "%s: no biases, or a bad stride of them", fn);
  CAB_REQUIRE(allowed == nullptr || allowed_strides, CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(drafts == nullptr || parents, CAB_EINVAL, "%s: drafts need parents", fn);
  CAB_REQUIRE(drafts == nullptr || parents_stride == 0 || parents_stride >= T, CAB_ESHAPE,
              "%s: bad parents stride", fn);
  CAB_REQUIRE(repetition || (std::isfinite(repetition0) && repetition0 > 0.f), CAB_EINVAL,
              "%s: the repetition penalty must be positive", fn);
  CAB_REQUIRE((presence || std::isfinite(presence0)) && (frequency || std::isfinite(frequency0)),
              CAB_EINVAL, "%s: penalties must be finite", fn);
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  CAB_REQUIRE((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) % es == 0,
              CAB_ESHAPE, "%s: pointers not aligned to their elements", fn);
  const int64_t size[3] = {B, T, 1};
  const int64_t xs[3] = {logit_strides[0], logit_strides[1], 0};
  const int64_t os[3] = {out_strides[0], out_strides[1], 0};
  const RowLayout to(os, size, V);
  CAB_REQUIRE(to.apart, CAB_ESHAPE, "%s: rows of out overlap", fn);
  const bool same = out == logits && (B == 1 || xs[0] == os[0]) && (T == 1 || xs[1] == os[1]);
  CAB_REQUIRE(same || !rows_share(out, to, logits, RowLayout(xs, size, V), es), CAB_EINVAL,
              "%s: out shares memory with the logits (only they themselves may be out)", fn);
  AdjustArgs a;
  a.x = static_cast<const char*>(logits);
  a.out = static_cast<char*>(out);
  for (int d = 0; d < 2; ++d) {
    a.xs[d] = xs[d] * es;
    a.os[d] = os[d] * es;
    a.as[d] = allowed ? allowed_strides[d] : 0;
  }
  a.B = static_cast<int32_t>(B);
  a.T = static_cast<int32_t>(T);
  a.V = static_cast<int32_t>(V);
  a.history = history_len ? history : nullptr;
  a.history_ld = history_stride;
  a.L = static_cast<int32_t>(history_len);
  a.lengths = lengths;
  a.prompts = prompt_lengths;
  a.repetition = repetition;
  a.presence = presence;
  a.frequency = frequency;
  a.r = repetition0;
  a.p = presence0;
  a.f = frequency0;
  a.bias_tokens = bias_tokens;
  a.bias = bias;
  a.bias_ld = bias_stride;
  a.biases = static_cast<int32_t>(biases);
  a.allowed = reinterpret_cast<const uint32_t*>(allowed);
  a.drafts = drafts;
  a.parents = parents;
  a.parents_ld = parents_stride;
  a.stretch = static_cast<int32_t>(stretch);
  a.stretches = static_cast<int32_t>(stretches);
  a.nodes = static_cast<int32_t>(nodes);
  const unsigned grid = static_cast<unsigned>(B * groups * stretches);
  const unsigned bytes =
      static_cast<unsigned>(stretch * (with_bias ? 2 : 1) + stretch / 32 + 1 + (tree ? 8 * T : 0)) * 4;
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto dt) {
    constexpr cab_dtype_t DT = decltype(dt)::value;
    if (with_bias && tree) adjust_kernel<DT, true, true><<<grid, THREADS, bytes, s>>>(a);
    else if (with_bias) adjust_kernel<DT, true, false><<<grid, THREADS, bytes, s>>>(a);
    else if (tree) adjust_kernel<DT, false, true><<<grid, THREADS, bytes, s>>>(a);
    else adjust_kernel<DT, false, false><<<grid, THREADS, bytes, s>>>(a);
  };
  switch (dtype) {
    case CAB_F32: go(std::integral_constant<cab_dtype_t, CAB_F32>{}); break;
    case CAB_F16: go(std::integral_constant<cab_dtype_t, CAB_F16>{}); break;
    default: go(std::integral_constant<cab_dtype_t, CAB_BF16>{}); break;
  }
  return launch_status(fn);
}
