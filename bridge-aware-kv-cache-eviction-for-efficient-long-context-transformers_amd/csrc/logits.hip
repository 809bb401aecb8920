// Logits before the next token is chosen (cab_adjust_logits): penalties for repeated tokens,
// biases, and the tokens that a grammar allows, in one pass.
//
//   x = logits[b, t, v];  c = times v was generated, counted from the history behind the prompt
//   and (a tree of drafts) from node t's line;  seen = c > 0 or v is in the prompt
//   x = seen ? (x > 0 ? x / r : x r) : x;  x -= f c + p [c > 0];  x += bias;  not allowed: -inf
//
// Bound: HBM, each row read and written once, and beside it the vector instructions of counting
// and of the values that are asked something (64 sequences of 128000 tokens, bf16, histories of
// 8192, new logits in every call: 13.0 us in a graph of calls, 13.7 in a trace; over the same logits 12.5, of which
// 11.1 without biases and mask, 6.4 with nothing to do; a copy's rate: 6.9; four trees of 26 x 50001, fp32, 12.7,
// bf16 12.3). A workgroup takes a stretch of the vocabulary of
// one sequence and counts the history's tokens that fall into it in LDS (whole numbers: the order
// of the atomics does not show). In a tree the counts stay as they are from node to node,
// and only the tokens of a node's line are added and taken off again. The history is read again
// for each stretch, from L2: stretches are long where rows are many.
#include "attn_common.h"
#include "row_layout.h"

namespace cab {
namespace {

constexpr int THREADS = 512;
constexpr int MAX_NODES = 256;

// Where a token's place in the list of biases is kept (1 + the place; 0: it has none): nowhere, in
// the upper half of its count's word, or in a word of its own. Halves suffice for histories and
// lists below 2^15, and leave room for stretches twice as long, which read the history half as
// often (64 sequences of 128000 tokens, histories of 8192: 23.8 -> 18.0 us).
enum { NO_PLACES, HALVES, WORDS };
constexpr int64_t HALF = 1 << 15;
template <int PLACES> constexpr uint32_t GIVEN = PLACES == HALVES ? 0x8000u : 0x80000000u;  // in the prompt

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
  const uint8_t* allowed;
  int64_t as[2];  // bytes: b, t
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

// What a workgroup keeps in LDS, in words: a count (and place) for every token of its window, and
// the lines of a tree. A row's 16-byte units may begin up to a unit before the stretch, so the
// window does.
struct Window {
  int tokens;  // rounded up to 16 bytes
  __host__ __device__ Window(int stretch, int unit) : tokens((stretch + unit + 3) & ~3) {}
  __host__ __device__ int words(int places, int nodes) const {
    return tokens * (places == WORDS ? 2 : 1) + 8 * nodes;
  }
};

template <cab_dtype_t DT, int PLACES, bool TREE>
__global__ __launch_bounds__(THREADS) void adjust_kernel(AdjustArgs a) {
  constexpr int ES = DT == CAB_F32 ? 4 : 2, P = 16 / ES;
  extern __shared__ __align__(16) uint32_t lds[];
  const Window size(a.stretch, P);
  uint32_t* count = lds;
  uint32_t* place = count + size.tokens;  // (WORDS)
  uint32_t* line = place + (PLACES == WORDS ? size.tokens : 0);  // [T][8]
  const int b = blockIdx.x, part = blockIdx.y, group = blockIdx.z;
  const int v0 = part * a.stretch, v1 = min(a.V, v0 + a.stretch);
  const int base = v0 - P;

  // Row t, and the units of it that are this workgroup's: [from, from + P units) of tokens.
  struct Row {
    const char* x;
    char* out;
    const uint8_t* allowed;
    int lo, hi, from, units;  // tokens lo .. hi are this workgroup's
  };
  auto row_of = [&](int t) {
    Row r;
    r.x = a.x + b * a.xs[0] + t * a.xs[1];
    r.out = a.out + b * a.os[0] + t * a.os[1];
    r.allowed = a.allowed ? a.allowed + b * a.as[0] + t * a.as[1] : nullptr;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(r.x) & 15);
    r.lo = v0;
    r.hi = v1;
    r.from = v1;
    r.units = 0;  // (in and out at different places in 16 bytes: value by value)
    if (off == static_cast<int>(reinterpret_cast<uintptr_t>(r.out) & 15)) {
      const int k = off / ES;
      r.lo = part ? v0 - k : 0;
      r.hi = v1 == a.V ? v1 : v1 - k;
      r.from = min(r.hi, part ? r.lo : (P - k) % P);
      r.units = (r.hi - r.from) / P;
    }
    return r;
  };
  struct Loaded {
    u32x4 w;
    uint32_t lo, hi;  // bytes of `allowed`
  };
  auto load = [&](const Row& r, int u) {
    Loaded x;
    const int v = r.from + u * P;
    x.w = *reinterpret_cast<const u32x4*>(r.x + static_cast<int64_t>(v) * ES);
    x.lo = x.hi = 255u;
    if (r.allowed) {
      x.lo = r.allowed[v >> 3];
      x.hi = r.allowed[(v + P - 1) >> 3];
    }
    return x;
  };
  const int t0 = group * a.nodes, t1 = min(a.T, t0 + a.nodes);
  Row row = row_of(t0);
  // What is read first is asked for before LDS is cleared: a thread's first unit of the first
  // row, its part of the history (whose length is looked at when it is there).
  Loaded ahead = {};
  if (static_cast<int>(threadIdx.x) < row.units) ahead = load(row, threadIdx.x);
  const int32_t* h = a.history ? a.history + b * a.history_ld : nullptr;
  const int whole = (reinterpret_cast<uintptr_t>(h) & 15) == 0 ? a.L & ~3 : 0;  // in 16 bytes
  auto read = [&](int i) {
    return i < whole ? *reinterpret_cast<const u32x4*>(h + i) : u32x4{~0u, ~0u, ~0u, ~0u};
  };
  u32x4 words = read(4 * threadIdx.x);
  int32_t biased = -1;  // a thread's first token of the list of biases
  if (PLACES != NO_PLACES && static_cast<int>(threadIdx.x) < a.biases)
    biased = a.bias_tokens[b * a.bias_ld + threadIdx.x];
  const int len = h ? min(a.lengths ? a.lengths[b] : a.L, a.L) : 0;
  const int given = a.prompts ? a.prompts[b] : 0;
  const float r = a.repetition ? a.repetition[b] : a.r;
  const float p = a.presence ? a.presence[b] : a.p;
  const float f = a.frequency ? a.frequency[b] : a.f;

  for (int i = 4 * threadIdx.x; i < size.words(PLACES, 0); i += 4 * THREADS)
    *reinterpret_cast<u32x4*>(lds + i) = u32x4{0u, 0u, 0u, 0u};
  lds_barrier();
  // (as unsigned numbers, negative tokens lie past every window: 0 is its first one at the least)
  const uint32_t first = max(base, 0), shift = first - static_cast<uint32_t>(base), here_to = v1 - first;
  if constexpr (PLACES != NO_PLACES) {
    for (int i = threadIdx.x; i < a.biases; i += THREADS) {
      const int32_t token = i < THREADS ? biased : a.bias_tokens[b * a.bias_ld + i];
      uint32_t at = static_cast<uint32_t>(token) - first;
      if (at >= here_to) continue;
      at += shift;
      // (listed twice: the last one. Halves: the counts are still 0)
      if (PLACES == HALVES) atomicMax(&count[at], (static_cast<uint32_t>(i) + 1) << 16);
      else atomicMax(&place[at], static_cast<uint32_t>(i) + 1);
    }
    if (PLACES == HALVES) lds_barrier();
  }
  auto tell = [&](int i, int32_t token) {
    const uint32_t at = static_cast<uint32_t>(token) - first;
    if (at >= here_to || i >= len) return;
    if (i < given) atomicOr(&count[at + shift], GIVEN<PLACES>);
    else atomicAdd(&count[at + shift], 1u);
  };
  // (Rolled, the next 16 bytes on their way: unrolled loops here and below were slower, by their
  // instructions' way into the cache.)
#pragma unroll 1
  for (int i = 4 * threadIdx.x; i < min(len, whole); i += 4 * THREADS) {
    const u32x4 now = words;
    words = read(i + 4 * THREADS);
    // (of a wave, nearly always all of the prompt or all generated: a subtraction, a comparison
    // and an addition a token)
    const bool made = i >= given && i + 4 <= len;
    if (ballot64(!made) == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t at = now[e] - first;
        if (at < here_to) atomicAdd(&count[at + shift], 1u);
      }
    } else if (ballot64(i + 4 > given || i + 4 > len) == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t at = now[e] - first;
        if (at < here_to) atomicOr(&count[at + shift], GIVEN<PLACES>);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t token = now[e];
        tell(i + e, static_cast<int32_t>(token));
      }
    }
  }
  for (int i = whole + threadIdx.x; i < len; i += THREADS) tell(i, h[i]);
  bool here = false;  // thread j: whether node j's token lies in the window, and where
  uint32_t draft_at = 0;
  if constexpr (TREE) {
    const int32_t* parents = a.parents + b * a.parents_ld;
    const int j = threadIdx.x;
    if (j < a.T) {
      const int64_t draft = a.drafts[static_cast<int64_t>(b) * a.T + j];
      here = draft >= 0 && draft >= base && draft < v1;
      if (here) draft_at = static_cast<uint32_t>(draft - base);
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
  lds_barrier();

  // x / r as x times 1 / r in two parts, the first one rounded down: so the quotient is rounded once, and in 16
  // bits it is the fp32 one's value, where x times a rounded 1 / r was the neighbour's for a 60th of all x at
  // r = 1.2. Where nothing is divided the second part is the least number, which no sum shows, since an
  // infinity times 0 is none. Penalties whose inverse is of no use: divided.
  constexpr float NEXT_TO_0 = 0x1p-149f;
  const bool usual = r > 1e-30f && r < 1e30f;
  float inverse = 1.f / r, rest = __builtin_fmaf(-r, inverse, 1.f);
  if (rest < 0.f) {
    inverse = __uint_as_float(__float_as_uint(inverse) - 1);
    rest = __builtin_fmaf(-r, inverse, 1.f);
  }
  rest = fmaxf(rest * inverse, NEXT_TO_0);
  auto penalised = [&](float x, uint32_t word) {
    const uint32_t c = PLACES == HALVES ? word & 0xffffu : word, n = c & (GIVEN<PLACES> - 1);
    const float factor = c ? (x > 0.f ? inverse : r) : 1.f;
    float y = __builtin_fmaf(x, factor, x * (c && x > 0.f ? rest : NEXT_TO_0));
    if (!usual && c) y = x > 0.f ? x / r : x * r;
    const float off = f * static_cast<float>(n) + p;
    return y - (n ? off : 0.f);
  };
  auto single = [&](int v) {
    const uint32_t at = v - base, word = count[at];
    float y = penalised(load1<DT>(row.x + static_cast<int64_t>(v) * ES), word);
    if constexpr (PLACES != NO_PLACES) {
      const uint32_t i = PLACES == HALVES ? word >> 16 : place[at];
      if (i) y += a.bias[b * a.bias_ld + i - 1];
    }
    const bool keep = !row.allowed || (row.allowed[v >> 3] >> (v & 7) & 1u);
    store1<DT>(row.out + static_cast<int64_t>(v) * ES, keep ? y : -INFINITY);
  };
  auto unit = [&](Loaded x, int u) {
    constexpr uint32_t ALL = (1u << P) - 1;
    const int v = row.from + u * P;
    const uint32_t at = v - base;
    uint32_t word[P], at_place[P] = {}, some = 0;
    auto fetch = [&](const uint32_t* from, uint32_t* to) {
      if ((at & 3) == 0) {  // (all of a row's units or none)
#pragma unroll
        for (int e = 0; e < P; e += 4) {
          const u32x4 y = *reinterpret_cast<const u32x4*>(from + at + e);
#pragma unroll
          for (int i = 0; i < 4; ++i) to[e + i] = y[i];
        }
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) to[e] = from[at + e];
      }
#pragma unroll
      for (int e = 0; e < P; ++e) some |= to[e];
    };
    fetch(count, word);
    if constexpr (PLACES == WORDS) fetch(place, at_place);
    const uint32_t keep = (x.lo | x.hi << 8) >> (v & 7) & ALL;
    // All ones in the values' bits whose bit of `which` is set.
    auto mask = [&](uint32_t which, int i) {
      const auto ones = [&](int e) { return static_cast<uint32_t>(static_cast<int32_t>(which << (31 - e)) >> 31); };
      if constexpr (DT == CAB_F32) return ones(i);
      else return (ones(2 * i) & 0xffffu) | (ones(2 * i + 1) & 0xffff0000u);
    };
    if (some) {
      float z[P];
      uint32_t listed = 0;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const uint32_t y = x.w[DT == CAB_F32 ? e : e >> 1];
        const uint16_t h = static_cast<uint16_t>(e & 1 ? y >> 16 : y);
        z[e] = penalised(DT == CAB_F32 ? __uint_as_float(y) : DT == CAB_BF16 ? bf16_to_f32(h) : f16_to_f32(h),
                         word[e]);
        const uint32_t i = PLACES == HALVES ? word[e] >> 16 : PLACES == WORDS ? at_place[e] : 0;
        listed |= i;
      }
      if (PLACES != NO_PLACES && listed) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const uint32_t i = PLACES == HALVES ? word[e] >> 16 : at_place[e];
          if (i) z[e] += a.bias[b * a.bias_ld + i - 1];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (values of which nothing is asked are x 1 - 0: themselves)
        if constexpr (DT == CAB_F32) x.w[i] = __float_as_uint(z[i]);
        else x.w[i] = pack2<DT == CAB_BF16>(z[2 * i], z[2 * i + 1]);
      }
    }
    if (keep != ALL) {
      constexpr uint32_t LOW = DT == CAB_F32 ? 0xff800000u : DT == CAB_BF16 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t m = mask(keep, i);
        x.w[i] = (x.w[i] & m) | (LOW & ~m);
      }
    }
    *reinterpret_cast<u32x4*>(row.out + static_cast<int64_t>(v) * ES) = x.w;
  };
  for (int t = t0; t < t1; ++t) {
    bool mine = false;
    if constexpr (TREE) {
      mine = here && (line[8 * t + (threadIdx.x >> 5)] >> (threadIdx.x & 31) & 1u);
      if (mine) atomicAdd(&count[draft_at], 1u);
      lds_barrier();
    }
#pragma unroll 1
    for (int u = threadIdx.x; u < row.units; u += THREADS) {
      const Loaded now = ahead;
      if (u + THREADS < row.units) ahead = load(row, u + THREADS);
      unit(now, u);
    }
    // (what is before the first unit and behind the last)
    for (int v = row.lo + threadIdx.x; v < row.from; v += THREADS) single(v);
    for (int v = row.from + row.units * P + threadIdx.x; v < row.hi; v += THREADS) single(v);
    if (t + 1 < t1) {
      row = row_of(t + 1);
      if (static_cast<int>(threadIdx.x) < row.units) ahead = load(row, threadIdx.x);
      if constexpr (TREE) {
        lds_barrier();  // (this node's counts have been read)
        if (mine) atomicSub(&count[draft_at], 1u);
      }
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
  // The longest stretch that leaves a workgroup a CU, and as many groups of a tree's nodes, each of
  // which counts the history anew, as make three of them. (us, with 4 for both -> so: 8 rows of
  // 128000, histories of 8000, bf16, 7.9 -> 5.3; a tree of 26 x 50001, fp32, 8.3 -> 6.7, four 13.5 -> 12.6; four of
  // 64 x 32000, fp32, 15.2 -> 15.7, bf16 13.6 -> 13.7; eight of 32 x 128000, bf16, 30.5 -> 33.5. Two groups: four of
  // 26 x 50001 14.3, the last 34.4; four on these stretches: 12.7, 30.4.)
  // (in a tree the T nodes of a line are counted too)
  const int places = !with_bias ? NO_PLACES
                     : history_len + (tree ? T : 0) < HALF && biases < HALF ? HALVES : WORDS;
  int64_t stretch = places == WORDS ? 4096 : 8192;  // (at most 64 KB of LDS)
  while (stretch > 1024 && ceil_div(V, stretch) * T < ceil_div(256, B)) stretch /= 2;
  const int64_t stretches = ceil_div(V, stretch);
  int64_t groups = ceil_div(768, B);
  groups = ceil_div(groups, stretches);
  if (groups > T) groups = T;
  const int64_t nodes = ceil_div(T, groups);
  groups = ceil_div(T, nodes);
  // (a launch's dims; threads along x: fewer than 2^32)
  CAB_REQUIRE(B <= (1 << 22) && stretches <= 65535 && groups <= 65535, CAB_ESHAPE,
              "%s: problem too large", fn);
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
    a.as[d] = allowed ? 4 * allowed_strides[d] : 0;
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
  a.allowed = reinterpret_cast<const uint8_t*>(allowed);
  a.drafts = drafts;
  a.parents = parents;
  a.parents_ld = parents_stride;
  a.stretch = static_cast<int32_t>(stretch);
  a.stretches = static_cast<int32_t>(stretches);
  a.nodes = static_cast<int32_t>(nodes);
  // (sequences next to each other: their workgroups lie on one XCD, whose L2 then holds the history
  // once, and the stretches of common tokens on all of them)
  const dim3 grid(static_cast<unsigned>(B), static_cast<unsigned>(stretches), static_cast<unsigned>(groups));
  const unsigned bytes = 4 * static_cast<unsigned>(Window(a.stretch, static_cast<int>(16 / es))
                                                       .words(places, tree ? a.T : 0));
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto go = [&](auto dt) {
    constexpr cab_dtype_t DT = decltype(dt)::value;
    auto run = [&](auto kept) {
      constexpr int PLACES = decltype(kept)::value;
      if (tree) adjust_kernel<DT, PLACES, true><<<grid, THREADS, bytes, s>>>(a);
      else adjust_kernel<DT, PLACES, false><<<grid, THREADS, bytes, s>>>(a);
    };
    if (places == NO_PLACES) run(std::integral_constant<int, NO_PLACES>{});
    else if (places == HALVES) run(std::integral_constant<int, HALVES>{});
    else run(std::integral_constant<int, WORDS>{});
  };
  switch (dtype) {
    case CAB_F32: go(std::integral_constant<cab_dtype_t, CAB_F32>{}); break;
    case CAB_F16: go(std::integral_constant<cab_dtype_t, CAB_F16>{}); break;
    default: go(std::integral_constant<cab_dtype_t, CAB_BF16>{}); break;
  }
  return launch_status(fn);
}
