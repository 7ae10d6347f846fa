// What the packed and the stepwise selective scan share: operands, the step transform, a lane's slice of a state.
#pragma once

#include "packed.cuh"

#include "../../include/ossm_b200.h"

namespace ossm_b200 {
namespace packed {

constexpr int kStates = 16;      // states in a lane's registers
constexpr int kTile = 16;        // rows staged at a time

struct ScanPacked {
  Sequences q;
  const void *u, *dt, *B, *C, *z;            // [rows, D] (u, dt, z) and [rows, N] (B, C), pitches below; z may be null
  const float *A, *skip, *bias;              // [D, N]; [D] or null; [D] or null
  const float* start;                        // [entries, D, N] or null
  float* end;                                // [entries, D, N] or null; may be `start`
  void* out;                                 // [rows, D]
  float* kept;                               // [ceil(rows / keep), D, N] states for the backward, or null
  long long ldu, lddt, ldb, ldc, ldz, ldo;
  int D, N, softplus, zero_rest;
  int by_u, by_dt, by_z, by_b, by_c;         // bytes copied at a time, by alignment
  int keep;                                  // rows between kept states, a divisor of kTile
  int vec;                                   // states may be read 16 bytes at a time
  // time segments: see scan_packed_kernel
  int segments, segment_rows;
  int pieces;                                // of a segment in the summary passes: 1, 2 or 4
  float* seg_state;                          // [segments * pieces, D, N]
  float* seg_first;                          // [segments, D, N]
  float* seg_dt;                             // [segments * pieces, D]
  int* seg_kind;                             // [segments * pieces]
};

#ifdef __CUDACC__
// log(1 + exp(x)), the identity above 20.  With y = exp(-|x|) in (0, 1] it is max(x, 0) + log(1 + y), and
// log(1 + y) = 2 atanh(r), r = y / (2 + y) <= 1/3: the series to r^13 leaves less than 2e-8 of the value, so that small
// steps keep their relative accuracy.
__device__ __forceinline__ float softplus_f(float x) {
  const float y = ex2f(-fabsf(x) * kLog2eF);
  const float r = y * rcpf(2.0f + y), s = r * r;
  float p = fmaf(s, 1.0f / 13, 1.0f / 11);
  p = fmaf(s, p, 1.0f / 9);
  p = fmaf(s, p, 1.0f / 7);
  p = fmaf(s, p, 1.0f / 5);
  p = fmaf(s, p, 1.0f / 3);
  p = fmaf(s, p, 1.0f);
  return x > 20.0f ? x : fmaf(2.0f * r, p, fmaxf(x, 0.0f));
}
// exp(x) / (1 + exp(x)) from dt = softplus(x): 1 - exp(-dt), by its series where that would cancel.
__device__ __forceinline__ float softplus_slope(float dt) {
  const float series = dt * fmaf(dt, fmaf(dt, fmaf(dt, -1.0f / 24, 1.0f / 6), -0.5f), 1.0f);
  return dt < 0.05f ? series : 1.0f - ex2f(-dt * kLog2eF);
}

// Two states at a time: a packed instruction takes one issue slot for two results (both read the same register ports).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 ex2f2(float2 a) { return make_float2(ex2f(a.x), ex2f(a.y)); }

// A state (or its adjoint) carried over the rows between two seams, whose decays multiply to 2^e, and what these rows add.
// States may grow: a zero stays zero where 2^e is no float32 number.
__device__ __forceinline__ float carried(float h, float e, float own) { return h == 0.0f ? own : fmaf(ex2f(e), h, own); }

// 16 consecutive states of a channel, zeros past the state size.
__device__ __forceinline__ void load_states(const float* p, int left, bool vec, float (&v)[kStates]) {
  if (vec) {
#pragma unroll
    for (int j = 0; j < kStates; j += 4) {
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j < left) q = *reinterpret_cast<const float4*>(p + j);
      v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kStates; ++j) v[j] = j < left ? p[j] : 0.0f;
  }
}
__device__ __forceinline__ void store_states(float* p, int left, bool vec, const float (&v)[kStates]) {
  if (vec) {
#pragma unroll
    for (int j = 0; j < kStates; j += 4)
      if (j < left) *reinterpret_cast<float4*>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < kStates; ++j)
      if (j < left) p[j] = v[j];
  }
}
// ---- tiles: rows of an operand on their way into shared memory ----------------------------------------
// kBytes at a time, asynchronously for 16 and 4 (the alignment that base and pitch share decides), 2 with a plain load;
// what lies past the operand's width becomes zero.
template <int kBytes>
__device__ __forceinline__ void copy_piece(void* dst, const void* src, int valid) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid) : "memory");
  else if constexpr (kBytes == 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(valid) : "memory");
  else
    *static_cast<uint16_t*>(dst) = valid > 0 ? *static_cast<const uint16_t*>(src) : (uint16_t)0;
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// A thread's share of a tile of `cols` columns: one column piece, every `step`-th row.  The CTA's threads are a multiple
// of the pieces of a row: cols is 16 per warp that shares the states, or 32 per channel group.
struct TileLane {
  int row, col, step, valid;     // col in elements; valid: bytes of the piece that exist
};
template <typename T>
__device__ __forceinline__ TileLane tile_lane(int bytes, int cols, int exist) {
  const int each = bytes / (int)sizeof(T), pieces = cols / each;
  TileLane l;
  l.row = threadIdx.x / pieces;
  l.col = (threadIdx.x % pieces) * each;
  l.step = blockDim.x / pieces;
  l.valid = min(max(exist - l.col, 0), each) * (int)sizeof(T);
  return l;
}
template <typename T, int kBytes>
__device__ __forceinline__ void tile_rows(T* dst, int cols, const T* src, long long ld, int rows, const TileLane& l) {
  // a piece without a column reads nothing: its address stays inside the row
  const T* at = src + (l.valid > 0 ? l.col : 0);
  for (int r = l.row; r < rows; r += l.step) copy_piece<kBytes>(dst + r * cols + l.col, at + r * ld, l.valid);
}
template <typename T>
__device__ __forceinline__ void tile_load(T* dst, int cols, const T* src, long long ld, int rows, int bytes, const TileLane& l) {
  if (bytes == 16) tile_rows<T, 16>(dst, cols, src, ld, rows, l);
  else if (bytes == 4) tile_rows<T, 4>(dst, cols, src, ld, rows, l);
  else if constexpr (sizeof(T) == 2) tile_rows<T, 2>(dst, cols, src, ld, rows, l);
}
#endif  // __CUDACC__

// How many bytes at a time the rows of an operand may be copied.
inline int piece_bytes(const void* p, long long ld, size_t element) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * (long long)element);
  return (a & 15u) == 0 ? 16 : ((a & 3u) == 0 ? 4 : 2);
}

// CTA of the packed kernels: a warp holds 32 channels x 16 states; `splits` warps share the states of a channel block,
// `groups` channel blocks lie side by side.
struct ScanShape {
  int splits, groups, threads, channels;
  unsigned column_blocks;
};
inline ScanShape scan_shape(int64_t D, int64_t N) {
  ScanShape s;
  s.splits = (int)((N + kStates - 1) / kStates);
  s.groups = s.splits == 1 ? 4 : (s.splits == 2 ? 2 : 1);
  s.threads = 32 * s.splits * s.groups;
  s.channels = 32 * s.groups;
  s.column_blocks = (unsigned)((D + s.channels - 1) / s.channels);
  return s;
}

// How the rows are cut: segments that fill the GPU once (`resident` CTAs at a time: one more would wait for another to end),
// none shorter than 32 rows and no more than 2 sqrt(rows), since a seam costs about what 8 rows do and they follow one
// another (one sequence x 64 channels x 16 states, forward: 2000 rows 28 us, 49 with segments of at least 128 rows; 8000 rows
// 42 us, 58).  Segments that are long because the GPU is full are summarised in pieces.  Two segments where there is no room
// for more: 8192 rows x 2048 channels x 256 states, backward 8.1 ms, 15.9 in one; one sequence 8.8 and 15.9, since its
// summary is cheaper than the walk itself.  The forward's is not by as much: there from `two_from` rows on (one sequence x
// 2048 x 256: 128 rows 60 us in one, 70 in two; 512 rows 220 and 174 us).
struct ScanCut {
  int segments, segment_rows, pieces;
};
inline ScanCut scan_cut(int64_t rows, int64_t resident, int64_t column_blocks, int multiple, int64_t two_from) {
  int64_t g = resident / column_blocks;
  if (g > rows / 32) g = rows / 32;
  while (g > 1 && g * g > 4 * rows) g = g - g / 8 - 1;
  if (g < 1 || (g == 2 && rows < two_from)) g = 1;
  const int64_t each = ((rows + g - 1) / g + multiple - 1) / multiple * multiple;
  ScanCut c;
  c.segment_rows = (int)each;
  c.segments = rows ? (int)((rows + each - 1) / each) : 1;
  c.pieces = each >= 256 && multiple % 4 == 0 ? 4 : (each >= 128 && multiple % 2 == 0 ? 2 : 1);
  return c;
}

int check_scan(const char* fn, int64_t rows, int64_t D, int64_t N, int64_t count, int64_t entries, int io, int dt);

}  // namespace packed
}  // namespace ossm_b200
