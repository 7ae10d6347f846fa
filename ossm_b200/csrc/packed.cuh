// Packed batches: sequences of different lengths back to back in one [tokens, channels] tensor.
//
// offsets[i] .. offsets[i + 1] are the rows of sequence i.  They live on the device, so no host check can see them:
// every kernel clamps what it reads into the tensor, and records kStatusPackedOffsets / kStatusPackedSlot in its device
// status word where an offset runs backwards or past the rows, or a slot past the cache (such a sequence is treated
// like one without a slot).  Rows outside every sequence (before offsets[0], from offsets[S] on) are never read into a
// result.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace ossm_b200 {
namespace packed {

struct Sequences {
  const int* offsets;            // [count + 1]
  const int* slots;              // [count] cache entry of each sequence, negative for none; null: entry i for sequence i
  const unsigned char* resume;   // [count] sequence continues from its entry (else from zeros); null: resume_all
  int resume_all;
  int count;
  int rows;                      // rows of the packed tensors
  long long entries;             // entries of the cache
};

#ifdef __CUDACC__
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements as floats: 16 bytes (one vector load), or the element itself (V = 1).  Raw is what a
// load leaves in registers until its values are needed.
template <typename T, int V>
struct Vec;
template <typename T>
struct Vec<T, 1> {
  using Raw = T;
  static __device__ __forceinline__ Raw fetch(const T* p) { return *p; }
  static __device__ __forceinline__ void unpack(Raw r, float (&v)[1]) { v[0] = to_float(r); }
  static __device__ __forceinline__ void load(const T* p, float (&v)[1]) { v[0] = to_float(*p); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[1]) { *p = from_float<T>(v[0]); }
};
template <>
struct Vec<float, 4> {
  using Raw = float4;
  static __device__ __forceinline__ Raw fetch(const float* p) { return *reinterpret_cast<const float4*>(p); }
  static __device__ __forceinline__ void unpack(Raw q, float (&v)[4]) { v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) { unpack(fetch(p), v); }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct Vec<__nv_bfloat16, 8> {
  using Raw = uint4;
  static __device__ __forceinline__ Raw fetch(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ void unpack(Raw q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[8]) { unpack(fetch(p), v); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&two);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ void report(int code) { atomicCAS(&g_device_status, 0, code); }

// offsets[i], held inside the rows.
__device__ __forceinline__ int offset_at(const Sequences& q, int i) {
  const int v = __ldg(q.offsets + i);
  if (v < 0 || v > q.rows) report(kStatusPackedOffsets);
  return v < 0 ? 0 : (v > q.rows ? q.rows : v);
}

// End of sequence i, which begins at `begin`.
__device__ __forceinline__ int end_of(const Sequences& q, int i, int begin) {
  const int v = offset_at(q, i + 1);
  if (v < begin) report(kStatusPackedOffsets);
  return v < begin ? begin : v;
}

// First sequence that is not over before row t: the number of sequences with begin < t and end <= t.  (A sequence
// without rows that lies at t is still to come.)  Bisection by one thread.
__device__ __forceinline__ int first_sequence(const Sequences& q, int t) {
  int lo = 0, hi = q.count;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    const bool over = __ldg(q.offsets + mid) < t && __ldg(q.offsets + mid + 1) <= t;
    if (over) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// The same by the 32 lanes of a warp, 32 probes a round.
__device__ __forceinline__ int first_sequence_warp(const Sequences& q, int t, int lane) {
  int lo = 0, n = q.count;
  while (n > 0) {
    const int stride = (n + 31) >> 5;
    const int i = lo + lane * stride + stride - 1;
    const bool over = i < lo + n && __ldg(q.offsets + i) < t && __ldg(q.offsets + i + 1) <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, over));
    const int past = lo + n;
    lo += c * stride;
    n = min(stride - 1, past - lo);
  }
  return min(lo, q.count);
}

// Cache entry of sequence i, or -1.
__device__ __forceinline__ long long entry_of(const Sequences& q, int i) {
  if (q.slots == nullptr) return i < q.entries ? i : -1;
  const int v = __ldg(q.slots + i);
  if (v >= q.entries) { report(kStatusPackedSlot); return -1; }
  return v < 0 ? -1 : v;
}
__device__ __forceinline__ bool resumes(const Sequences& q, int i) {
  return q.resume != nullptr ? __ldg(q.resume + i) != 0 : q.resume_all != 0;
}

constexpr float kLog2eF = 1.4426950408889634f;
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcpf(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / (1 + exp(-x)): 0 where exp(-x) overflows
__device__ __forceinline__ float sigmoid(float x) { return rcpf(1.0f + ex2f(-kLog2eF * x)); }
#endif  // __CUDACC__

}  // namespace packed
}  // namespace ossm_b200
