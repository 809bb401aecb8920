// Rotary positions (cab_rotary), and new K and V rows into the pages of a cache with K and the
// queries rotated on the way (cab_paged_append).
//
// Pair i of a row at position p is turned by p f_i radians: (x, y) -> A (x cos - y sin,
// x sin + y cos), A the amplitude. The backward pass is the transpose: the same with -sin.
//
// Angles. f_i / 2 pi, the pair's turns a position, comes as a 64-bit fixed-point fraction, so
// that p times it modulo 2^64 is the angle's fraction of a turn, to p 2^-65 of one: far positions
// lose nothing (4e-10 rad at 2^31; an fp32 product would be 0.06 rad off at 10^6), and no table
// of cosines is read. The top 32 bits (1.5e-9 rad) give the nearest quarter turn and a remainder
// of at most an eighth, which is held in fp32 (three roundings: 1.4e-7 rad at the most; 7.4e-8 seen), and whose
// sine and cosine are Taylor polynomials to fp32's rounding.
//
// Bound: HBM, each row read and written once. A workgroup takes 2 tokens (1 where there are few),
// forms their angles once for all heads (through LDS) and streams the heads: 16 bytes of
// both of a pair's halves a lane, neighbouring lanes along the row, then tokens, then heads; one
// head in flight a thread, many waves. Measured, bf16, D = 128: 40 heads of 16384 tokens 62 us, 5.4 TB/s (4 tokens
// and 4 heads in flight 75, 4 and 2 70, 2 and 1 67, so with non-temporal stores 63, loads too 62);
// 8000 tokens into pages, 32 + 8 + 8 heads, 43 us (51); one token of 16 sequences 3.6 us in a graph.
#include "attn_common.h"
#include "row_layout.h"

namespace cab {
namespace {

constexpr int MAX_DIM = 512, MAX_PAIRS = MAX_DIM / 2;
constexpr int TOKENS = 2;  // of a workgroup, at most
constexpr int64_t MAX_ROWS = (1 << 24) - 1;  // a launch of up to 256 threads a token: below 2^32

struct TurnTensor {
  const char* src;
  char* dst;
  int64_t ss[3], ds[3];  // bytes: b, h, token; of pages: page, h, place
};

struct TurnArgs {
  TurnTensor t[3];  // queries; keys; values
  int32_t upto[3];  // heads of the tensors up to each one's end
  int32_t turned;   // heads before this one are turned, the others copied
  int32_t paged;    // heads from this one on go into pages
  int32_t N, half, chunks, tokens;
  int32_t last;     // units of a row
  int64_t rows;     // B * N
  const int32_t* positions;  // may be null: lengths[b] + n, or n
  int64_t positions_ld;
  const int32_t* lengths;    // may be null
  const int32_t* counts;     // may be null
  const int32_t* table;
  int64_t table_ld;
  int32_t columns, pages, size;
  const uint64_t* turns;
  float amplitude, sign;
};

// Sine and cosine of t / 2^32 turns.
__device__ __forceinline__ void turn_sincos(uint32_t t, float& sine, float& cosine) {
  const uint32_t quarter = (t + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(t - (quarter << 30))) *
                  static_cast<float>(6.283185307179586 / 4294967296.0);
  const float y = x * x;
  // (next terms at pi / 4: 1.8e-9 and 1.1e-10)
  float s = __builtin_fmaf(y, 1.f / 362880.f, -1.f / 5040.f);
  s = __builtin_fmaf(y, s, 1.f / 120.f);
  s = __builtin_fmaf(y, s, -1.f / 6.f);
  s = __builtin_fmaf(x * y, s, x);
  float c = __builtin_fmaf(y, -1.f / 3628800.f, 1.f / 40320.f);
  c = __builtin_fmaf(y, c, -1.f / 720.f);
  c = __builtin_fmaf(y, c, 1.f / 24.f);
  c = __builtin_fmaf(y, c, -0.5f);
  c = __builtin_fmaf(y, c, 1.f);
  const float a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
  sine = quarter & 2 ? -a : a;
  cosine = (quarter + 1) & 2 ? -b : b;
}

// P values as they lie in memory: 16 bytes, or one value.
template <cab_dtype_t DT, int P> struct Unit { typedef u32x4 T; };
template <> struct Unit<CAB_F32, 1> { typedef uint32_t T; };
template <> struct Unit<CAB_F16, 1> { typedef uint16_t T; };
template <> struct Unit<CAB_BF16, 1> { typedef uint16_t T; };

template <cab_dtype_t DT, int P>
__device__ __forceinline__ void unpack(const typename Unit<DT, P>::T& u, float* x) {
  if constexpr (P == 1) {
    if constexpr (DT == CAB_F32) x[0] = __uint_as_float(u);
    else x[0] = DT == CAB_BF16 ? bf16_to_f32(u) : f16_to_f32(u);
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint32_t w = u[DT == CAB_F32 ? i : i >> 1];
      if constexpr (DT == CAB_F32) {
        x[i] = __uint_as_float(w);
      } else {
        const uint16_t h = static_cast<uint16_t>(i & 1 ? w >> 16 : w);
        x[i] = DT == CAB_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
      }
    }
  }
}

template <cab_dtype_t DT, int P>
__device__ __forceinline__ typename Unit<DT, P>::T pack(const float* x) {
  if constexpr (P == 1) {
    if constexpr (DT == CAB_F32) return __float_as_uint(x[0]);
    else return DT == CAB_BF16 ? f32_to_bf16(x[0]) : f32_to_f16(x[0]);
  } else if constexpr (DT == CAB_F32) {
    return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                 __float_as_uint(x[3])};
  } else {
    constexpr bool BF16 = DT == CAB_BF16;
    return u32x4{pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]),
                 pack2<BF16>(x[6], x[7])};
  }
}

// A thread's chunk of a row is two units of P values: pairs i .. i + P of the part that turns
// (its two halves, or 2 P values side by side), or two units of the rest.
// Grid: (tokens, groups of heads).
template <cab_dtype_t DT, int P, bool INTERLEAVED>
__global__ __launch_bounds__(256) void turn_kernel(TurnArgs a) {
  using U = typename Unit<DT, P>::T;
  __shared__ float cosines[TOKENS * MAX_PAIRS], sines[TOKENS * MAX_PAIRS];
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.tokens;
  const int chunk = threadIdx.x % a.chunks, slot = threadIdx.x / a.chunks;
  const int lanes = 256 / a.chunks / a.tokens;  // heads side by side
  const int r = slot % a.tokens, lane = slot / a.tokens;
  const int64_t row = row0 + r;
  const bool active = lane < lanes && row < a.rows;
  const int64_t b = active ? row / a.N : 0;
  const int32_t n = active ? static_cast<int32_t>(row - b * a.N) : 0;
  // The chunk's units.
  const int turning = a.half / P;
  int u0, u1;
  if (chunk < turning) {
    u0 = INTERLEAVED ? 2 * chunk : chunk;
    u1 = INTERLEAVED ? u0 + 1 : chunk + turning;
  } else {
    u0 = 2 * chunk;
    u1 = u0 + 1 < a.last ? u0 + 1 : u0;
  }
  const int step = lanes * gridDim.y;
  const int end = active ? a.upto[2] : 0;
  auto tensor_of = [&](int h) { return h < a.upto[0] ? 0 : h < a.upto[1] ? 1 : 2; };
  auto head_of = [&](int h, int t) { return t == 0 ? h : h - a.upto[t - 1]; };
  U x, y;
  auto fetch = [&](int h) {
    if (h >= end) return;
    const int t = tensor_of(h);
    const TurnTensor& tt = a.t[t];
    const char* from = tt.src + b * tt.ss[0] + head_of(h, t) * tt.ss[1] + n * tt.ss[2];
    x = *reinterpret_cast<const U*>(from + u0 * static_cast<int>(sizeof(U)));
    y = *reinterpret_cast<const U*>(from + u1 * static_cast<int>(sizeof(U)));
  };
  // The first head is asked for before the angles are formed.
  int h = blockIdx.y * lanes + lane;
  fetch(h);

  for (int i = threadIdx.x; i < a.tokens * a.half; i += 256) {
    const int q = i / a.half, j = i - q * a.half;
    const int64_t other = row0 + q;
    if (other >= a.rows) break;
    const int64_t ob = other / a.N;
    const int32_t on = static_cast<int32_t>(other - ob * a.N);
    const int64_t p = a.positions ? a.positions[ob * a.positions_ld + on]
                                  : (a.lengths ? static_cast<int64_t>(a.lengths[ob]) : 0) + on;
    float s, c;
    turn_sincos(static_cast<uint32_t>((static_cast<uint64_t>(p) * a.turns[j]) >> 32), s, c);
    cosines[i] = c * a.amplitude;
    sines[i] = s * (a.amplitude * a.sign);
  }
  // Where the row goes in the pages.
  bool there = false;
  int64_t page = 0, place = 0;
  if (a.table && active) {
    const int64_t len = a.lengths[b], to = len + n;
    if (len >= 0 && to < static_cast<int64_t>(a.columns) * a.size && (!a.counts || n < a.counts[b])) {
      const uint32_t col = static_cast<uint32_t>(to) / static_cast<uint32_t>(a.size);
      page = a.table[b * a.table_ld + col];
      place = to - static_cast<int64_t>(col) * a.size;
      there = page >= 0 && page < a.pages;
    }
  }
  lds_barrier();
  float cs[P], sn[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    cs[i] = chunk < turning ? cosines[r * a.half + chunk * P + i] : 1.f;
    sn[i] = chunk < turning ? sines[r * a.half + chunk * P + i] : 0.f;
  }
  for (; h < end; h += step, fetch(h)) {
    const bool in_pages = h >= a.paged;
    if (in_pages && !there) continue;
    if (chunk < turning && h < a.turned) {
      float p[P], q[P], z[2 * P];
      unpack<DT, P>(x, p);
      unpack<DT, P>(y, q);
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < P; ++e) z[e] = p[e], z[P + e] = q[e];
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const float u = z[2 * e], v = z[2 * e + 1];
          z[2 * e] = __builtin_fmaf(u, cs[e], -(v * sn[e]));
          z[2 * e + 1] = __builtin_fmaf(u, sn[e], v * cs[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          z[e] = __builtin_fmaf(p[e], cs[e], -(q[e] * sn[e]));
          z[P + e] = __builtin_fmaf(p[e], sn[e], q[e] * cs[e]);
        }
      }
      x = pack<DT, P>(z);
      y = pack<DT, P>(z + P);
    }
    const int t = tensor_of(h);
    const TurnTensor& tt = a.t[t];
    char* to = tt.dst + (in_pages ? page : b) * tt.ds[0] + head_of(h, t) * tt.ds[1] +
               (in_pages ? place : n) * tt.ds[2];
    __builtin_nontemporal_store(x, reinterpret_cast<U*>(to + u0 * static_cast<int>(sizeof(U))));
    __builtin_nontemporal_store(y, reinterpret_cast<U*>(to + u1 * static_cast<int>(sizeof(U))));
  }
}

// Fills sizes and launches. wide: all rows may be read and written 16 bytes at a time.
cab_status_t launch(const char* fn, TurnArgs& a, cab_dtype_t dtype, int64_t D, int64_t R, bool wide,
                    bool interleaved, hipStream_t s) {
  const int64_t per = 16 / static_cast<int64_t>(dtype_size(dtype));
  wide = wide && R % (2 * per) == 0 && D % per == 0;
  const int64_t P = wide ? per : 1;
  a.half = static_cast<int32_t>(R / 2);
  a.last = static_cast<int32_t>(D / P);
  a.chunks = static_cast<int32_t>(ceil_div(a.last, 2));
  // One token a workgroup where there are too few to go round, or a row takes all threads (us, one -> two:
  // 40 heads of 128, 16 tokens 3.7 -> 5.0, 1023 6.2 -> 6.8, 4000 16.4 -> 15.0; 8 of 64, 4000 7.9 -> 5.4).
  a.tokens = a.rows < 1024 || a.chunks > 256 / TOKENS ? 1 : TOKENS;
  const int64_t lanes = 256 / a.chunks / a.tokens;
  const int64_t blocks = ceil_div(a.rows, a.tokens);
  // As many groups of heads as it takes for some four workgroups a CU (one -> four: 40 heads of 16 tokens
  // 4.5 -> 3.7, of 1023 7.5 -> 6.2, of 2000 10.5 -> 9.2).
  int64_t groups = ceil_div(1024, blocks);
  if (groups > ceil_div(a.upto[2], lanes)) groups = ceil_div(a.upto[2], lanes);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups));
  auto go = [&](auto dt) {
    constexpr cab_dtype_t DT = decltype(dt)::value;
    constexpr int W = DT == CAB_F32 ? 4 : 8;
    if (wide && interleaved) turn_kernel<DT, W, true><<<grid, 256, 0, s>>>(a);
    else if (wide) turn_kernel<DT, W, false><<<grid, 256, 0, s>>>(a);
    else if (interleaved) turn_kernel<DT, 1, true><<<grid, 256, 0, s>>>(a);
    else turn_kernel<DT, 1, false><<<grid, 256, 0, s>>>(a);
  };
  switch (dtype) {
    case CAB_F32: go(std::integral_constant<cab_dtype_t, CAB_F32>{}); break;
    case CAB_F16: go(std::integral_constant<cab_dtype_t, CAB_F16>{}); break;
    default: go(std::integral_constant<cab_dtype_t, CAB_BF16>{}); break;
  }
  return launch_status(fn);
}

// Strides in bytes; whether rows there start on 16-byte boundaries.
bool in_bytes(const void* p, const int64_t* strides, int64_t es, int64_t* bytes) {
  bool wide = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int d = 0; d < 3; ++d) {
    bytes[d] = strides[d] * es;
    wide = wide && bytes[d] % 16 == 0;
  }
  return wide;
}

}  // namespace
}  // namespace cab

using namespace cab;

extern "C" cab_status_t cab_rotary(int32_t n_tensors, const void* const* x, void* const* out,
                                   cab_dtype_t dtype, int64_t B, const int64_t* heads, int64_t N,
                                   int64_t D, const int64_t* x_strides, const int64_t* out_strides,
                                   const int32_t* positions, int64_t positions_stride,
                                   const uint64_t* turns, int64_t rotary_dim, int interleaved,
                                   float amplitude, int inverse, void* stream) {
  const char* fn = "cab_rotary";
  clear_error();
  CAB_REQUIRE(valid_dtype(dtype), CAB_EDTYPE, "%s: unknown dtype %d", fn, static_cast<int>(dtype));
  CAB_REQUIRE(n_tensors >= 1 && n_tensors <= 2 && B >= 0 && N >= 0, CAB_ESHAPE,
              "%s: bad shape (one or two tensors)", fn);
  CAB_REQUIRE(D >= 2 && D <= MAX_DIM && rotary_dim >= 2 && rotary_dim <= D && rotary_dim % 2 == 0,
              CAB_ESHAPE, "%s: rotary_dim must be even, in [2, D], and D at most %d", fn, MAX_DIM);
  CAB_REQUIRE(x && out && heads && x_strides && out_strides && turns, CAB_EINVAL,
              "%s: null argument", fn);
  CAB_REQUIRE(std::isfinite(amplitude), CAB_EINVAL, "%s: amplitude must be finite", fn);
  CAB_REQUIRE(positions == nullptr || positions_stride == 0 || positions_stride >= N, CAB_ESHAPE,
              "%s: bad positions stride", fn);
  int64_t all = 0;
  for (int t = 0; t < n_tensors; ++t) {
    CAB_REQUIRE(heads[t] >= 0 && heads[t] <= 65535, CAB_ESHAPE, "%s: bad number of heads", fn);
    all += heads[t];
  }
  if (B == 0 || N == 0 || all == 0) return CAB_OK;
  CAB_REQUIRE(N <= MAX_ROWS && B <= MAX_ROWS / N, CAB_ESHAPE, "%s: more than 2^24 - 1 tokens", fn);
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  TurnArgs a = {};
  bool wide = true;
  int32_t upto = 0;
  const void* outs[2];
  for (int t = 0; t < 2; ++t) {
    if (t < n_tensors && heads[t] > 0) {
      const int64_t *xs = x_strides + 4 * t, *os = out_strides + 4 * t;
      CAB_REQUIRE(x[t] && out[t], CAB_EINVAL, "%s: null argument", fn);
      CAB_REQUIRE((reinterpret_cast<uintptr_t>(x[t]) | reinterpret_cast<uintptr_t>(out[t])) % es == 0,
                  CAB_ESHAPE, "%s: pointers not aligned to their elements", fn);
      CAB_REQUIRE(xs[3] == 1 && os[3] == 1, CAB_ESHAPE, "%s: last-dim stride must be 1", fn);
      const int64_t size[3] = {B, heads[t], N};
      const RowLayout to(os, size, D);
      CAB_REQUIRE(to.apart, CAB_ESHAPE, "%s: rows of out overlap", fn);
      // (a thread reads what it writes over before it does: x itself may be out)
      for (int o = 0; o < n_tensors; ++o) {
        const int64_t* s = x_strides + 4 * o;
        const int64_t from[3] = {B, heads[o], N};
        bool same = o == t && out[t] == x[t];
        for (int d = 0; d < 3; ++d) same = same && (size[d] == 1 || s[d] == os[d]);
        CAB_REQUIRE(same || heads[o] == 0 || !rows_share(out[t], to, x[o], RowLayout(s, from, D), es),
                    CAB_EINVAL, "%s: out shares memory with an input (only x itself may be out)", fn);
      }
      if (t == 1 && heads[0] > 0) {
        const int64_t first[3] = {B, heads[0], N};
        CAB_REQUIRE(!rows_share(out[1], to, out[0], RowLayout(out_strides, first, D), es), CAB_EINVAL,
                    "%s: the outputs share memory", fn);
      }
      a.t[t].src = static_cast<const char*>(x[t]);
      a.t[t].dst = static_cast<char*>(out[t]);
      const bool from_wide = in_bytes(x[t], xs, es, a.t[t].ss);
      const bool to_wide = in_bytes(out[t], os, es, a.t[t].ds);
      wide = wide && from_wide && to_wide;
      upto += static_cast<int32_t>(heads[t]);
    }
    a.upto[t] = upto;
  }
  a.upto[2] = a.turned = a.paged = upto;
  a.N = static_cast<int32_t>(N);
  a.rows = B * N;
  a.positions = positions;
  a.positions_ld = positions_stride;
  a.turns = turns;
  a.amplitude = amplitude;
  a.sign = inverse ? -1.f : 1.f;
  return launch(fn, a, dtype, D, rotary_dim, wide, interleaved != 0, static_cast<hipStream_t>(stream));
}

extern "C" cab_status_t cab_paged_append(
    const void* k, const void* v, void* k_pages, void* v_pages, const void* q, void* q_out,
    cab_dtype_t dtype, int64_t B, int64_t H, int64_t H_kv, int64_t n, int64_t D, int64_t pages,
    int64_t page_size, const int64_t k_strides[4], const int64_t v_strides[4],
    const int64_t k_page_strides[4], const int64_t v_page_strides[4], const int64_t q_strides[4],
    const int64_t q_out_strides[4], const int32_t* table, int64_t table_stride, int64_t columns,
    const int32_t* lengths, const int32_t* counts, const int32_t* positions,
    int64_t positions_stride, const uint64_t* turns, int64_t rotary_dim, int interleaved,
    float amplitude, void* stream) {
  const char* fn = "cab_paged_append";
  clear_error();
  CAB_REQUIRE(valid_dtype(dtype), CAB_EDTYPE, "%s: unknown dtype %d", fn, static_cast<int>(dtype));
  CAB_REQUIRE(B >= 0 && n >= 0 && H >= 0 && H <= 65535 && H_kv >= 1 && H_kv <= 65535 && pages >= 0 &&
                  page_size >= 1 && columns >= 0,
              CAB_ESHAPE, "%s: bad shape", fn);
  CAB_REQUIRE(D >= 1 && D <= MAX_DIM, CAB_ESHAPE, "%s: D must be in [1, %d]", fn, MAX_DIM);
  CAB_REQUIRE(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 2 == 0, CAB_ESHAPE,
              "%s: rotary_dim must be even and at most D", fn);
  if (B == 0 || n == 0) return CAB_OK;
  CAB_REQUIRE(n <= MAX_ROWS && B <= MAX_ROWS / n, CAB_ESHAPE, "%s: more than 2^24 - 1 tokens", fn);
  CAB_REQUIRE(pages <= INT32_MAX && page_size <= INT32_MAX &&
                  columns <= (INT32_MAX - 1024) / page_size,
              CAB_ESHAPE, "%s: more than 2^31 places a sequence", fn);
  CAB_REQUIRE(k && v && k_strides && v_strides && k_page_strides && v_page_strides && lengths,
              CAB_EINVAL, "%s: null argument", fn);
  const bool none = pages == 0 || columns == 0;  // (nothing is appended, q is still rotated)
  CAB_REQUIRE(none || (k_pages && v_pages && table), CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(rotary_dim == 0 || turns, CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(H == 0 || (q && q_out && q_strides && q_out_strides), CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(std::isfinite(amplitude), CAB_EINVAL, "%s: amplitude must be finite", fn);
  CAB_REQUIRE(table_stride == 0 || table_stride >= columns, CAB_ESHAPE, "%s: bad table stride", fn);
  CAB_REQUIRE(positions == nullptr || positions_stride == 0 || positions_stride >= n, CAB_ESHAPE,
              "%s: bad positions stride", fn);
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  const void* src[3] = {q, k, v};
  void* dst[3] = {q_out, k_pages, v_pages};
  const int64_t* ss[3] = {q_strides, k_strides, v_strides};
  const int64_t* ds[3] = {q_out_strides, k_page_strides, v_page_strides};
  const int64_t from_size[3] = {B, H_kv, n}, q_size[3] = {B, H, n};
  const int64_t page_sizes[3] = {none ? 0 : pages, H_kv, page_size};
  TurnArgs a = {};
  bool wide = true;
  for (int t = H == 0 ? 1 : 0; t < 3; ++t) {
    CAB_REQUIRE((reinterpret_cast<uintptr_t>(src[t]) | reinterpret_cast<uintptr_t>(dst[t])) % es == 0,
                CAB_ESHAPE, "%s: pointers not aligned to their elements", fn);
    CAB_REQUIRE(D == 1 || (ss[t][3] == 1 && ds[t][3] == 1), CAB_ESHAPE, "%s: last-dim stride must be 1", fn);
    CAB_REQUIRE(RowLayout(ds[t], t == 0 ? q_size : page_sizes, D).apart, CAB_ESHAPE,
                "%s: rows of %s overlap", fn, t == 0 ? "q_out" : "the pages");
    a.t[t].src = static_cast<const char*>(src[t]);
    a.t[t].dst = static_cast<char*>(dst[t]);
    const bool from_wide = in_bytes(src[t], ss[t], es, a.t[t].ss);
    const bool to_wide = in_bytes(dst[t], ds[t], es, a.t[t].ds);
    wide = wide && from_wide && to_wide;
  }
  // Nothing that is written may be read or written elsewhere in the call.
  for (int t = H == 0 ? 1 : 0; t < 3; ++t) {
    const RowLayout to(ds[t], t == 0 ? q_size : page_sizes, D);
    for (int o = H == 0 ? 1 : 0; o < 3; ++o) {
      bool same = t == 0 && o == 0 && q == q_out;
      for (int d = 0; d < 3; ++d) same = same && (q_size[d] == 1 || ss[0][d] == ds[0][d]);
      CAB_REQUIRE(same || !rows_share(dst[t], to, src[o],
                                      RowLayout(ss[o], o == 0 ? q_size : from_size, D), es),
                  CAB_EINVAL, "%s: the new rows share memory with what is written", fn);
      CAB_REQUIRE(o >= t || !rows_share(dst[t], to, dst[o],
                                        RowLayout(ds[o], o == 0 ? q_size : page_sizes, D), es),
                  CAB_EINVAL, "%s: %s share memory", fn,
                  o == 0 ? "q_out and the pages" : "the pages of K and V");
    }
  }
  a.upto[0] = static_cast<int32_t>(H);
  a.upto[1] = static_cast<int32_t>(H + H_kv);
  a.upto[2] = static_cast<int32_t>(H + 2 * H_kv);
  a.turned = a.upto[1];
  a.paged = a.upto[0];
  a.N = static_cast<int32_t>(n);
  a.rows = B * n;
  a.positions = positions;
  a.positions_ld = positions_stride;
  a.lengths = lengths;
  a.counts = counts;
  a.table = none ? nullptr : table;
  a.table_ld = table_stride;
  a.columns = static_cast<int32_t>(columns);
  a.pages = static_cast<int32_t>(pages);
  a.size = static_cast<int32_t>(page_size);
  a.turns = turns;
  a.amplitude = amplitude;
  a.sign = 1.f;
  return launch(fn, a, dtype, D, rotary_dim, wide, interleaved != 0, static_cast<hipStream_t>(stream));
}
