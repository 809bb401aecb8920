// Caches whose sequences have lengths of their own, and drafted tokens in them:
// new K and V rows behind each sequence's length (cab_kv_append_at), and, once the
// drafts are verified, the accepted rows moved to the front of the drafted ones in
// every layer (cab_kv_commit). lengths, counts and paths are read on the device, so
// a decode loop needs no read-back and can be captured.
//
// A step moves little: 4 sequences, 8 heads, D = 128, bf16, 64 drafts, up to 6 accepted: 1 MB a
// layer in, at most 0.1 MB a layer moved. What counts is launches: one per layer for
// K and V together (3.4 us there, 2.3 for 5 drafts of one sequence), one per 64 tensors for the
// compaction (4.9 us for 32 layers, 3.6 for 28).
#include "cab_internal.h"
#include "row_layout.h"

#include <algorithm>

namespace cab {
namespace {

struct AppendAtArgs {
  const char* src[2];  // K, V
  char* dst[2];
  int64_t ss[2][4];    // source strides in bytes: b, h, row, unit
  int64_t ds[2][3];    // destination strides in bytes: b, h, row
  const int32_t* lengths;
  const int32_t* counts;  // may be null: n rows of every sequence
  uint32_t H, n, units, rows;  // units: copies of U bytes per row; rows: of the buffers
  uint32_t total;              // B * H * n * units
};

// U bytes per thread and step; blockIdx.y: K or V. Sequence b's new row r goes to
// row lengths[b] + r; rows at or past counts[b], and rows outside the buffer, nowhere.
template <typename U>
__global__ __launch_bounds__(256) void kv_append_at_kernel(AppendAtArgs a) {
  const int t = blockIdx.y;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * 256;
  for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < a.total; i += step) {
    const uint32_t x = static_cast<uint32_t>(i);
    const uint32_t row = x / a.units, u = x - row * a.units;
    const uint32_t bh = row / a.n, r = row - bh * a.n;
    const uint32_t b = bh / a.H, h = bh - b * a.H;
    const int64_t to = static_cast<int64_t>(a.lengths[b]) + r;
    if (to < r || to >= a.rows) continue;  // (a negative length appends nothing)
    if (a.counts && static_cast<int32_t>(r) >= a.counts[b]) continue;
    *reinterpret_cast<U*>(a.dst[t] + b * a.ds[t][0] + h * a.ds[t][1] + to * a.ds[t][2] +
                          static_cast<int64_t>(u) * sizeof(U)) =
        *reinterpret_cast<const U*>(a.src[t] + b * a.ss[t][0] + h * a.ss[t][1] + r * a.ss[t][2] +
                                    u * a.ss[t][3]);
  }
}

constexpr int COMMIT_TENSORS = 64;  // per launch (their pointers travel as arguments)
constexpr int COMMIT_THREADS = 128;
constexpr int COMMIT_AHEAD = 8;     // rows loaded before the first of them is stored

struct CommitArgs {
  char* t[COMMIT_TENSORS];
  int64_t st[3];            // strides in bytes: b, h, row
  const int32_t* lengths;   // may be null: length0
  const int32_t* path;      // [B, path_ld]
  const int32_t* counts;    // may be null: count0
  int32_t* new_lengths;     // may be null
  int64_t length0, path_ld;
  int32_t count0, nodes;    // nodes: entries of a path
  uint32_t columns, units;  // columns: H * units copies of U bytes a row
  int64_t rows;
};

// A path entry j holds the draft row that becomes row j. Entries strictly ascend, so
// path[j] >= j: going up j, a row is read before it is written to. An entry that does
// not, or that lies outside the drafts or the buffer, ends the path.
template <typename U>
__global__ __launch_bounds__(COMMIT_THREADS) void kv_commit_kernel(CommitArgs a) {
  const int b = blockIdx.y;
  const int64_t len = a.lengths ? a.lengths[b] : a.length0;
  const int32_t want = a.counts ? a.counts[b] : a.count0;
  const int32_t most = len < 0 ? 0 : want < a.nodes ? want : a.nodes;
  const int32_t* path = a.path + b * a.path_ld;
  const uint32_t c = blockIdx.x * COMMIT_THREADS + threadIdx.x;
  const bool in = c < a.columns;
  const uint32_t h = c / a.units, u = c - h * a.units;
  char* p = a.t[blockIdx.z] + b * a.st[0] + len * a.st[2];
  if (in) p += h * a.st[1] + static_cast<int64_t>(u) * sizeof(U);
  int32_t last = -1, j = 0;
  bool open = true;
  while (open && j < most) {
    int32_t from[COMMIT_AHEAD];
    U x[COMMIT_AHEAD];
#pragma unroll
    for (int i = 0; i < COMMIT_AHEAD; ++i) {
      from[i] = -1;
      if (open && j + i < most) {
        const int32_t f = path[j + i];
        open = f > last && f < a.nodes && len + f < a.rows;
        if (open) {
          last = from[i] = f;
          if (in && f != j + i) x[i] = *reinterpret_cast<const U*>(p + f * a.st[2]);
        }
      }
    }
    int32_t done = 0;
#pragma unroll
    for (int i = 0; i < COMMIT_AHEAD; ++i) {
      if (from[i] < 0) continue;
      ++done;
      if (in && from[i] != j + i) *reinterpret_cast<U*>(p + (j + i) * a.st[2]) = x[i];
    }
    j += done;
    open = open && done == COMMIT_AHEAD;
  }
  if (a.new_lengths && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0)
    a.new_lengths[b] = static_cast<int32_t>(len + j);
}

constexpr int MOST_TENSORS = 4096;

// 1: a tensor is there twice, 2: two of them share a row, 0: neither. By rising address
// neighbours decide, unless tensors lie in one another's gaps: there all pairs that reach each
// other do, or, where all lie within the smallest stride and the others are multiples of it
// (layers side by side in each row), neighbours' rows.
int tensors_share(void* const* tensors, int n, const RowLayout& layout, int64_t es) {
  const char* t[MOST_TENSORS];
  for (int i = 0; i < n; ++i) t[i] = static_cast<const char*>(tensors[i]);
  std::sort(t, t + n);
  for (int i = 1; i < n; ++i)
    if (t[i] == t[i - 1]) return 1;
  if (layout.empty) return 0;
  const int64_t step = layout.dims ? layout.st[layout.dims - 1] : INT64_MAX / es;
  bool side_by_side = t[n - 1] - t[0] <= (step - layout.row) * es;
  for (int d = 0; d < layout.dims; ++d) side_by_side = side_by_side && layout.st[d] % step == 0;
  for (int i = 0; i < n; ++i)
    for (int j = i + 1; j < n && t[j] - t[i] < layout.extent * es; ++j) {
      if (side_by_side ? t[j] - t[i] < layout.row * es : layout.meets((t[j] - t[i]) / es)) return 2;
      if (side_by_side) break;
    }
  return 0;
}

}  // namespace
}  // namespace cab

using namespace cab;

extern "C" cab_status_t cab_kv_append_at(const void* k, const void* v, void* k_dst, void* v_dst,
                                         int32_t element_bytes, int64_t B, int64_t H, int64_t n,
                                         int64_t D, int64_t rows, const int64_t k_strides[4],
                                         const int64_t v_strides[4],
                                         const int64_t k_dst_strides[4],
                                         const int64_t v_dst_strides[4], const int32_t* lengths,
                                         const int32_t* counts, void* stream) {
  const char* fn = "cab_kv_append_at";
  clear_error();
  CAB_REQUIRE(element_bytes == 2 || element_bytes == 4, CAB_EDTYPE,
              "%s: element size %d unsupported (2 or 4)", fn, (int)element_bytes);
  CAB_REQUIRE(B >= 0 && H >= 0 && n >= 0 && D >= 0 && rows >= 0, CAB_ESHAPE, "%s: negative size", fn);
  if (B == 0 || H == 0 || n == 0 || D == 0 || rows == 0) return CAB_OK;
  CAB_REQUIRE(k && v && k_dst && v_dst && k_strides && v_strides && k_dst_strides && v_dst_strides &&
                  lengths,
              CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(k_dst_strides[3] == 1 && v_dst_strides[3] == 1, CAB_ESHAPE,
              "%s: the buffers' last-dim stride must be 1", fn);
  CAB_REQUIRE(rows <= INT32_MAX && B <= INT32_MAX / H && n <= INT32_MAX / (B * H) &&
                  D <= INT32_MAX / (B * H * n),
              CAB_ESHAPE, "%s: more than 2^31 values", fn);
  const int64_t es = element_bytes;
  AppendAtArgs a;
  const void* src[2] = {k, v};
  void* dst[2] = {k_dst, v_dst};
  const int64_t* ss[2] = {k_strides, v_strides};
  const int64_t* ds[2] = {k_dst_strides, v_dst_strides};
  const int64_t size[3] = {B, H, rows};
  const RowLayout layout[2] = {RowLayout(k_dst_strides, size, D), RowLayout(v_dst_strides, size, D)};
  bool wide = D * es % 16 == 0;
  for (int t = 0; t < 2; ++t) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(src[t]) | reinterpret_cast<uintptr_t>(dst[t]);
    CAB_REQUIRE(at % es == 0, CAB_ESHAPE, "%s: pointers not aligned to their elements", fn);
    CAB_REQUIRE(layout[t].apart, CAB_ESHAPE, "%s: rows of a buffer overlap", fn);
    a.src[t] = static_cast<const char*>(src[t]);
    a.dst[t] = static_cast<char*>(dst[t]);
    wide = wide && ss[t][3] == 1 && at % 16 == 0;
    for (int d = 0; d < 4; ++d) a.ss[t][d] = ss[t][d] * es;
    for (int d = 0; d < 3; ++d) {
      a.ds[t][d] = ds[t][d] * es;
      wide = wide && a.ss[t][d] % 16 == 0 && a.ds[t][d] % 16 == 0;
    }
  }
  // (one tensor as K and V of one buffer is written twice alike)
  bool one = k == v && k_dst == v_dst;
  for (int d = 0; d < 4; ++d)
    one = one && k_strides[d] == v_strides[d] && k_dst_strides[d] == v_dst_strides[d];
  CAB_REQUIRE(one || !rows_share(k_dst, layout[0], v_dst, layout[1], es), CAB_EINVAL,
              "%s: the buffers of K and V share memory", fn);
  if (wide) a.ss[0][3] = a.ss[1][3] = 16;
  const int64_t units = wide ? D * es / 16 : D;
  a.lengths = lengths;
  a.counts = counts;
  a.H = static_cast<uint32_t>(H);
  a.n = static_cast<uint32_t>(n);
  a.units = static_cast<uint32_t>(units);
  a.rows = static_cast<uint32_t>(rows);
  a.total = static_cast<uint32_t>(B * H * n * units);
  const int64_t blocks = ceil_div(a.total, 256);
  const dim3 grid(static_cast<unsigned>(blocks < 4096 ? blocks : 4096), 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (wide)
    kv_append_at_kernel<u32x4><<<grid, 256, 0, s>>>(a);
  else if (es == 4)
    kv_append_at_kernel<uint32_t><<<grid, 256, 0, s>>>(a);
  else
    kv_append_at_kernel<uint16_t><<<grid, 256, 0, s>>>(a);
  return launch_status(fn);
}

extern "C" cab_status_t cab_kv_commit(void* const* tensors, int32_t n_tensors,
                                      int32_t element_bytes, int64_t B, int64_t H, int64_t rows,
                                      int64_t D, const int64_t strides[4], const int32_t* lengths,
                                      int64_t length0, const int32_t* path, int64_t nodes,
                                      int64_t path_stride, const int32_t* counts, int32_t count0,
                                      int32_t* new_lengths, void* stream) {
  const char* fn = "cab_kv_commit";
  clear_error();
  CAB_REQUIRE(element_bytes == 2 || element_bytes == 4, CAB_EDTYPE,
              "%s: element size %d unsupported (2 or 4)", fn, (int)element_bytes);
  CAB_REQUIRE(n_tensors >= 1 && n_tensors <= MOST_TENSORS && B >= 0 && H >= 1 && rows >= 0 && D >= 1 &&
                  nodes >= 0,
              CAB_ESHAPE, "%s: bad shape", fn);
  CAB_REQUIRE(length0 >= 0 && count0 >= 0, CAB_EINVAL, "%s: negative length or count", fn);
  if (B == 0) return CAB_OK;
  CAB_REQUIRE(tensors && strides && (nodes == 0 || path), CAB_EINVAL, "%s: null argument", fn);
  CAB_REQUIRE(rows <= INT32_MAX && nodes <= INT32_MAX && B <= 65535 && H <= INT32_MAX / D &&
                  length0 <= rows,
              CAB_ESHAPE, "%s: problem too large", fn);
  CAB_REQUIRE(strides[3] == 1, CAB_ESHAPE, "%s: the last-dim stride must be 1", fn);
  CAB_REQUIRE(path_stride == 0 || path_stride >= nodes, CAB_ESHAPE, "%s: bad path stride", fn);
  CAB_REQUIRE(new_lengths == nullptr || new_lengths != lengths, CAB_EINVAL,
              "%s: the new lengths cannot be written over the old ones", fn);
  const int64_t es = element_bytes;
  const int64_t size[3] = {B, H, rows};
  const RowLayout layout(strides, size, D);
  CAB_REQUIRE(layout.apart, CAB_ESHAPE, "%s: rows of a tensor overlap", fn);
  CommitArgs a;
  bool wide = D * es % 16 == 0;
  for (int d = 0; d < 3; ++d) {
    a.st[d] = strides[d] * es;
    wide = wide && a.st[d] % 16 == 0;
  }
  for (int t = 0; t < n_tensors; ++t) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(tensors[t]);
    CAB_REQUIRE(at != 0, CAB_EINVAL, "%s: null tensor", fn);
    CAB_REQUIRE(at % es == 0, CAB_ESHAPE, "%s: pointers not aligned to their elements", fn);
    wide = wide && at % 16 == 0;
  }
  // (moved twice, a row would be moved from where it went)
  switch (tensors_share(tensors, n_tensors, layout, es)) {
    case 0: break;
    case 1: CAB_REQUIRE(false, CAB_EINVAL, "%s: a tensor is listed twice", fn);
    default: CAB_REQUIRE(false, CAB_EINVAL, "%s: two tensors share memory", fn);
  }
  const int64_t units = wide ? D * es / 16 : D;
  a.lengths = lengths;
  a.path = path;
  a.counts = counts;
  a.length0 = length0;
  a.path_ld = path_stride;
  a.count0 = count0;
  a.nodes = static_cast<int32_t>(nodes);
  a.columns = static_cast<uint32_t>(H * units);
  a.units = static_cast<uint32_t>(units);
  a.rows = rows;
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int32_t t0 = 0; t0 < n_tensors; t0 += COMMIT_TENSORS) {
    const int32_t m = n_tensors - t0 < COMMIT_TENSORS ? n_tensors - t0 : COMMIT_TENSORS;
    for (int32_t i = 0; i < m; ++i) a.t[i] = static_cast<char*>(tensors[t0 + i]);
    a.new_lengths = t0 == 0 ? new_lengths : nullptr;
    const dim3 grid(static_cast<unsigned>(ceil_div(a.columns, COMMIT_THREADS)),
                    static_cast<unsigned>(B), static_cast<unsigned>(m));
    if (wide)
      kv_commit_kernel<u32x4><<<grid, COMMIT_THREADS, 0, s>>>(a);
    else if (es == 4)
      kv_commit_kernel<uint32_t><<<grid, COMMIT_THREADS, 0, s>>>(a);
    else
      kv_commit_kernel<uint16_t><<<grid, COMMIT_THREADS, 0, s>>>(a);
    const cab_status_t r = launch_status(fn);
    if (r != CAB_OK) return r;
  }
  return CAB_OK;
}
