// Mamba selective scan over a packed batch: gradients (sm_100a).
//
// With p_t = exp(dt_t A) h_{t-1} (so h_t = p_t + dt_t u_t B_t), dy = dout silu(z), and the adjoint of the state
//   g_t = C_t dy_t + exp(dt_{t+1} A) g_{t+1}            (the gradient of the state behind a sequence's last row)
// the gradients are sums of products:
//   dB_t = sum_d g_t dt_t u_t      dC_t = sum_d dy_t h_t        d(dt u)_t = sum_n g_t B_t      dA = sum_t dt_t g_t p_t
//   d(dt)_t = sum_n A g_t p_t + u_t d(dt u)_t                   du_t = dt_t d(dt u)_t + skip dy_t
//   dz_t = dout y_t silu'(z_t)     draw = d(dt) (1 - exp(-dt))  dskip = sum_t dy u              dbias = sum_t draw
#include "scan_packed.cuh"

#include <type_traits>

namespace ossm_b200 {
OSSM_B200_STATUS_ACCESSOR(status_packed_scan_backward)
namespace packed {

struct ScanPackedGrad {
  ScanPacked f;
  const void* grad;                          // dout [rows, D]
  const float* grad_end;                     // [count, D, N] or null
  void *du, *ddt, *dB, *dC, *dz;             // dense; dz may be null
  float *dA, *dskip, *dbias, *dstart;        // [D, N], [D] or null, [D] or null, [count, D, N] or null
  long long ldg;
  float *part_bc;                            // [column blocks, rows, 2 N]
  float *part_A;                             // [segments, D, N]
  float *part_d;                             // [segments, 2, D] sums for skip and bias
  int column_blocks, by_g;
  int even;                                  // every operand may be copied 16 bytes at a time, and N is a multiple of 16
  int vec_rows, vec_bc;                      // du, ddt, dz, and dB, dC, may be written four elements at a time
};

// Four adjacent elements of a row, in shared or global memory; `vec` where the address allows it at once.
template <typename T>
__device__ __forceinline__ void get4(const T* p, float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(q.x << 16); v[1] = __uint_as_float(q.x & 0xffff0000u);
    v[2] = __uint_as_float(q.y << 16); v[3] = __uint_as_float(q.y & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ void put4(T* p, const float (&v)[4], bool vec, int exist) {
  if (vec && exist >= 4) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < exist) p[i] = from_float<T>(v[i]);
  }
}

// Elements 2n and 2n + 1 of an array in registers.
__device__ __forceinline__ float2 pair(const float (&v)[4], int n) { return make_float2(v[2 * n], v[2 * n + 1]); }
__device__ __forceinline__ void set(float (&v)[4], int n, float2 a) { v[2 * n] = a.x; v[2 * n + 1] = a.y; }

// Adjoint at the seams of the time segments, the mirror image of the forward's summary: the rows of each segment that
// belong to the sequence crossing its beginning, from the right, starting from zero or from that sequence's grad_end; in
// pieces, like there.  seg_state of a segment's first piece becomes the gradient of the state entering the segment.
template <typename IO, typename DT, int kGroups>
__global__ void __launch_bounds__(kGroups == 1 ? 512 : 128, kGroups == 1 ? 1 : 4) scan_packed_adjoint_kernel(const ScanPackedGrad pg, int splits) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  constexpr int kCols = 32 * kGroups;
  constexpr bool kWiden = sizeof(IO) == 2, kOne = kGroups == 4;     // kOne: one warp has all the states of its channels
  const ScanPacked& p = pg.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = warp % splits, group = warp / splits;
  const int NP = splits * kStates;
  const int raw_bytes = kTile * (kCols * (2 * (int)sizeof(IO) + (int)sizeof(DT)) + NP * (int)sizeof(IO));
  const int o_g = kTile * kCols * (int)sizeof(DT), o_z = o_g + kTile * kCols * (int)sizeof(IO),
            o_c = o_z + kTile * kCols * (int)sizeof(IO);
  float* s_c = reinterpret_cast<float*>(smem_raw + 2 * raw_bytes);      // [kTile][NP] (kWiden)
  float2* s_dt = reinterpret_cast<float2*>(s_c + (kWiden ? kTile * NP : 0));   // [kTile][kCols] (dt, dy) (not kOne)
  const Sequences& q = p.q;
  const int piece = blockIdx.y + p.pieces, seg = piece / p.pieces;  // nobody asks the first segment
  const int seam = seg * p.segment_rows;                            // where the segment begins
  const int t0 = piece * (p.segment_rows / p.pieces);
  const int t1 = min(seg == p.segments - 1 ? q.rows : seam + p.segment_rows, t0 + p.segment_rows / p.pieces);
  const int d0 = blockIdx.x * kCols, col = group * 32 + lane, d = d0 + col, n0 = split * kStates;
  const int left = d < p.D ? p.N - n0 : 0;
  const bool vec = p.vec != 0;
  const long long at = (long long)d * p.N + n0, DN = (long long)p.D * p.N;
  const IO *grad = static_cast<const IO*>(pg.grad) + d0, *Cm = static_cast<const IO*>(p.C),
           *z = p.z ? static_cast<const IO*>(p.z) + d0 : nullptr;
  const DT* dt = static_cast<const DT*>(p.dt) + d0;

  const int s = first_sequence_warp(q, seam, lane);
  const int begin = s < q.count ? offset_at(q, s) : seam;
  const int end = begin < seam ? end_of(q, s, begin) : 0;
  const bool here = begin < seam && end > t0 && t0 < t1;            // rows of a sequence that crosses the seam
  if (blockIdx.x == 0 && tid == 0) p.seg_kind[piece] = !here ? 0 : (end <= t1 ? 1 : 2);
  if (!here) return;
  const TileLane l_g = tile_lane<IO>(pg.by_g, kCols, p.D - d0), l_z = tile_lane<IO>(p.by_z, kCols, p.D - d0),
                 l_dt = tile_lane<DT>(p.by_dt, kCols, p.D - d0), l_c = tile_lane<IO>(p.by_c, NP, p.N);
  auto fetch = [&](int lo, int rows, int buffer) {
    unsigned char* raw = smem_raw + buffer * raw_bytes;
    const long long row = lo;
    tile_load(reinterpret_cast<DT*>(raw), kCols, dt + row * p.lddt, p.lddt, rows, p.by_dt, l_dt);
    tile_load(reinterpret_cast<IO*>(raw + o_g), kCols, grad + row * pg.ldg, pg.ldg, rows, pg.by_g, l_g);
    if (z) tile_load(reinterpret_cast<IO*>(raw + o_z), kCols, z + row * p.ldz, p.ldz, rows, p.by_z, l_z);
    tile_load(reinterpret_cast<IO*>(raw + o_c), NP, Cm + row * p.ldc, p.ldc, rows, p.by_c, l_c);
    copies_commit();
  };
  int hi = min(end, t1), buffer = 0;
  if (hi > t0) fetch(max(t0, hi - kTile), min(kTile, hi - t0), 0);
  float A[kStates], g[kStates];
  load_states(p.A + at, left, vec, A);
#pragma unroll
  for (int j = 0; j < kStates; ++j) { A[j] *= kLog2eF; g[j] = 0.0f; }
  if (end <= t1 && pg.grad_end) load_states(pg.grad_end + (long long)s * DN + at, left, vec, g);
  float dt_sum = 0.0f;
  const int c = kOne ? col : tid % kCols;
  const float bias = p.bias && d0 + c < p.D ? p.bias[d0 + c] : 0.0f;
  auto step_and_dy = [&](DT raw, IO up, IO gate) {
    float x = to_float(raw) + bias, dy = to_float(up);
    if (p.softplus) x = softplus_f(x);
    if (z) { const float w = to_float(gate); dy *= w * sigmoid(w); }
    return make_float2(x, dy);
  };
  auto row_back = [&](float2 x, const float* cr) {
    const float2 x2 = both(x.x), dy2 = both(x.y);
#pragma unroll
    for (int j = 0; j < kStates; j += 4) {
      const float4 cv = *reinterpret_cast<const float4*>(cr + j);
      const float2 g0 = mul2(ex2f2(mul2(x2, make_float2(A[j], A[j + 1]))), fma2(make_float2(cv.x, cv.y), dy2, make_float2(g[j], g[j + 1])));
      const float2 g1 = mul2(ex2f2(mul2(x2, make_float2(A[j + 2], A[j + 3]))), fma2(make_float2(cv.z, cv.w), dy2, make_float2(g[j + 2], g[j + 3])));
      g[j] = g0.x; g[j + 1] = g0.y; g[j + 2] = g1.x; g[j + 3] = g1.y;
    }
    dt_sum += x.x;
  };
  for (; hi > t0; buffer ^= 1) {
    const int lo = max(t0, hi - kTile), rows = hi - lo;
    unsigned char* raw = smem_raw + buffer * raw_bytes;
    const DT* r_dt = reinterpret_cast<const DT*>(raw);
    const IO *r_g = reinterpret_cast<const IO*>(raw + o_g), *r_z = reinterpret_cast<const IO*>(raw + o_z),
             *r_c = reinterpret_cast<const IO*>(raw + o_c);
    copies_wait();
    __syncthreads();
    if (lo > t0) fetch(max(t0, lo - kTile), min(kTile, lo - t0), buffer ^ 1);
    const float* ct;
    if constexpr (kWiden) {
      for (int i = tid * 4; i < rows * NP; i += blockDim.x * 4) {
        float v[4];
        get4(r_c + i, v);
        put4(s_c + i, v, true, 4);
      }
      ct = s_c;
    } else {
      ct = reinterpret_cast<const float*>(r_c);
    }
    if constexpr (!kOne) {
#pragma unroll 2
      for (int i = tid; i < rows * kCols; i += blockDim.x) s_dt[i] = step_and_dy(r_dt[i], r_g[i], r_z[i]);
    }
    if constexpr (kWiden || !kOne) __syncthreads();
    if constexpr (kOne) {
      int r = rows - 1;
      for (; r >= 3; r -= 4) {
        float2 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = step_and_dy(r_dt[(r - j) * kCols + col], r_g[(r - j) * kCols + col], r_z[(r - j) * kCols + col]);
#pragma unroll
        for (int j = 0; j < 4; ++j) row_back(x[j], ct + (r - j) * NP);
      }
      for (; r >= 0; --r) row_back(step_and_dy(r_dt[r * kCols + col], r_g[r * kCols + col], r_z[r * kCols + col]), ct + r * NP);
    } else {
      for (int r = rows - 1; r >= 0; --r) row_back(s_dt[r * kCols + col], ct + r * NP + n0);
    }
    hi = lo;
  }
  store_states(p.seg_state + piece * DN + at, left, vec, g);
  if (split == 0 && d < p.D) p.seg_dt[(long long)piece * p.D + d] = dt_sum;
}

__global__ void __launch_bounds__(128) scan_adjoint_seams_kernel(const ScanPacked p) {
  const long long DN = (long long)p.D * p.N, i = (long long)blockIdx.x * 128 + threadIdx.x;
  if (i >= DN) return;
  const long long d = i / p.N;
  const float a = p.A[i] * kLog2eF;
  float g = 0.0f;
  constexpr int kBatch = 16;
  const int first = p.pieces;
  for (int k0 = p.segments * p.pieces - 1; k0 >= first; k0 -= kBatch) {
    int kind[kBatch];
    float own[kBatch], sum[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int k = max(k0 - j, first);
      kind[j] = p.seg_kind[k]; own[j] = p.seg_state[k * DN + i]; sum[j] = p.seg_dt[(long long)k * p.D + d];
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (k0 - j < first || kind[j] == 0) continue;
      g = kind[j] == 1 ? own[j] : carried(g, a * sum[j], own[j]);
      if (((k0 - j) & (p.pieces - 1)) == 0) p.seg_state[(k0 - j) * DN + i] = g;
    }
  }
}

// A lane holds 4 channels x 4 states: the sums over channels (dB, dC) and over states (y, d(dt u), d(dt)) are then
// mostly sums within a lane.  A warp is 8 lanes of channels x 4 lanes of states = 32 x 16 pairs.  The rows go right to
// left in windows of W, copied asynchronously one window ahead: a forward walk from the kept state entering the window
// leaves p in shared memory, the backward walk reads it, evaluates the decay a second time and leaves the lanes' sums in
// the row that it has just read; then the CTA adds them up and finishes the rows.  Nothing is added by atomics: what CTAs
// share goes to partial sums.  32768 rows x 2048 channels x 16 states (bf16): 1.73 ms, 0.62e12 pairs a second; 12800 rows x
// 128 channels x 256 states (float32): 0.69 ms.  Neither the issue slots (45 and 51 %) nor the special functions (33 and 28 %)
// nor memory (1 TB/s) are near their limit: at 16 states p and 240 registers leave eight warps an SM, two a scheduler, which
// do not cover the latencies; at 256 the 16 warps are one CTA that meets at three barriers a window (1.9 of 8.2 issue slots
// between a warp's instructions).  Windows of 4, 5 or 6 rows and 10 to 14 warps an SM, 16 states: 1.82 to 2.08 ms.
constexpr int kRowFloats = 512;   // of a warp and row: p; after the row: 4 x 32 sums of dB | dC, then 4 x 3 x 32 of y | d(dt u) | d(dt)
constexpr int kFlushWindows = 16; // windows after which a lane's sums for dA go to memory: a second level that keeps them exact

template <typename IO, typename DT, int W, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == 1 ? 8 : (kWarps == 2 ? 4 : 1)) scan_packed_backward_kernel(const ScanPackedGrad pg, int splits) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  constexpr int kCols = 32;
  constexpr bool kWiden = sizeof(IO) == 2;
  constexpr bool kRoom = kWarps <= 8;             // 255 registers a thread
  const ScanPacked& p = pg.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x / 32;
  const int split = warp;
  const int cg = lane >> 2, sg = lane & 3;
  const int NP = splits * kStates;
  const int raw_bytes = W * (kCols * (3 * (int)sizeof(IO) + (int)sizeof(DT)) + 2 * NP * (int)sizeof(IO));
  const int o_u = W * kCols * (int)sizeof(DT), o_z = o_u + W * kCols * (int)sizeof(IO), o_g = o_z + W * kCols * (int)sizeof(IO),
            o_b = o_g + W * kCols * (int)sizeof(IO), o_c = o_b + W * NP * (int)sizeof(IO);
  float* s_rows = reinterpret_cast<float*>(smem_raw + 2 * raw_bytes);   // [warps][W][kRowFloats]
  float* s_dt = s_rows + warps * W * kRowFloats;                    // [W][kCols]
  float* s_dtu = s_dt + W * kCols;                                  // [W][kCols]
  float* s_dy = s_dtu + W * kCols;                                  // [W][kCols]
  float* s_bc = s_dy + W * kCols;                                   // [2][W][NP] (kWiden)
  int* s_seq = reinterpret_cast<int*>(s_bc + (kWiden ? 2 * W * NP : 0)); // [2][W] the sequence whose first / last row this is
  float* mine = s_rows + warp * W * kRowFloats;
  const Sequences& q = p.q;
  const int seg = blockIdx.y;
  const int t0 = seg * p.segment_rows, t1 = seg == p.segments - 1 ? q.rows : t0 + p.segment_rows;
  const int d0 = blockIdx.x * kCols, n0 = split * kStates + 4 * sg, dw = d0 + 4 * cg;
  const long long DN = (long long)p.D * p.N;
  const IO *u = static_cast<const IO*>(p.u) + d0, *Bm = static_cast<const IO*>(p.B), *Cm = static_cast<const IO*>(p.C),
           *z = p.z ? static_cast<const IO*>(p.z) + d0 : nullptr, *grad = static_cast<const IO*>(pg.grad) + d0;
  const DT* dt = static_cast<const DT*>(p.dt) + d0;
  const bool vec = p.vec != 0;
  auto fetch = [&](int w0, int buffer) {
    const TileLane l_u = tile_lane<IO>(p.by_u, kCols, p.D - d0), l_z = tile_lane<IO>(p.by_z, kCols, p.D - d0),
                   l_g = tile_lane<IO>(pg.by_g, kCols, p.D - d0), l_dt = tile_lane<DT>(p.by_dt, kCols, p.D - d0),
                   l_b = tile_lane<IO>(p.by_b, NP, p.N), l_c = tile_lane<IO>(p.by_c, NP, p.N);
    unsigned char* raw = smem_raw + buffer * raw_bytes;
    const int rows = min(W, t1 - w0);
    const long long row = w0;
    tile_load(reinterpret_cast<DT*>(raw), kCols, dt + row * p.lddt, p.lddt, rows, p.by_dt, l_dt);
    tile_load(reinterpret_cast<IO*>(raw + o_u), kCols, u + row * p.ldu, p.ldu, rows, p.by_u, l_u);
    if (z) tile_load(reinterpret_cast<IO*>(raw + o_z), kCols, z + row * p.ldz, p.ldz, rows, p.by_z, l_z);
    tile_load(reinterpret_cast<IO*>(raw + o_g), kCols, grad + row * pg.ldg, pg.ldg, rows, pg.by_g, l_g);
    tile_load(reinterpret_cast<IO*>(raw + o_b), NP, Bm + row * p.ldb, p.ldb, rows, p.by_b, l_b);
    tile_load(reinterpret_cast<IO*>(raw + o_c), NP, Cm + row * p.ldc, p.ldc, rows, p.by_c, l_c);
    copies_commit();
  };
  // Whole windows of operands that lie on 16 bytes: the pieces of all operands are dealt out to the threads once, and a
  // window further left is the same places `move` bytes before.
  constexpr int kLeast = kWarps == 8 ? 3 : (kWarps == 16 ? 9 : kWarps);   // warps of the smallest state size that comes here
  constexpr int kMostPieces = (W * 2 * (3 * (int)sizeof(IO) + (int)sizeof(DT)) + 2 * W * kLeast * (int)sizeof(IO) + 32 * kLeast - 1) / (32 * kLeast);
  const bool even = pg.even && d0 + kCols <= p.D;
  const char* piece_src[kMostPieces];
  int piece_dst[kMostPieces], piece_move[kMostPieces];
  auto deal = [&](int w0) {                      // for the window at w0
    const int wide = kCols * (int)sizeof(IO) / 16, wide_dt = kCols * (int)sizeof(DT) / 16, states = NP * (int)sizeof(IO) / 16;
    const int ends[6] = {W * wide_dt, W * (wide_dt + wide), W * (wide_dt + 2 * wide), W * (wide_dt + 3 * wide),
                         W * (wide_dt + 3 * wide + states), W * (wide_dt + 3 * wide + 2 * states)};
#pragma unroll
    for (int k = 0; k < kMostPieces; ++k) {
      int i = tid + k * blockDim.x;
      piece_src[k] = nullptr;
      piece_dst[k] = i * 16;                     // the operands' tiles follow one another in this order
      piece_move[k] = 0;
      if (i >= ends[5]) continue;
      const char* base;
      long long ld;
      int per;
      if (i < ends[0]) { base = reinterpret_cast<const char*>(dt); ld = p.lddt * (int)sizeof(DT); per = wide_dt; }
      else if (i < ends[1]) { base = reinterpret_cast<const char*>(u); ld = p.ldu * (int)sizeof(IO); per = wide; i -= ends[0]; }
      else if (i < ends[2]) { base = reinterpret_cast<const char*>(z); ld = p.ldz * (int)sizeof(IO); per = wide; i -= ends[1]; }
      else if (i < ends[3]) { base = reinterpret_cast<const char*>(grad); ld = pg.ldg * (int)sizeof(IO); per = wide; i -= ends[2]; }
      else if (i < ends[4]) { base = reinterpret_cast<const char*>(Bm); ld = p.ldb * (int)sizeof(IO); per = states; i -= ends[3]; }
      else { base = reinterpret_cast<const char*>(Cm); ld = p.ldc * (int)sizeof(IO); per = states; i -= ends[4]; }
      if (base == nullptr) continue;             // no gate
      const int r = i / per;
      piece_src[k] = base + (w0 + r) * ld + (i - r * per) * 16;
      piece_move[k] = (int)(W * ld);
    }
  };
  auto fetch_even = [&](int buffer) {            // the window before the last one asked for
#pragma unroll
    for (int k = 0; k < kMostPieces; ++k)
      if (piece_src[k] != nullptr) {
        piece_src[k] -= piece_move[k];
        copy_piece<16>(smem_raw + buffer * raw_bytes + piece_dst[k], piece_src[k], 16);
      }
    copies_commit();
  };

  float A[4][4], g[4][4], dA[4][4], h[4][4];
  auto zero = [&](float (&v)[4][4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int n = 0; n < 4; ++n) v[c][n] = 0.0f;
  };
  auto load = [&](const float* base, float (&v)[4][4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float* r = base + (long long)(dw + c) * p.N + n0;
      if (vec) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (dw + c < p.D && n0 < p.N) x = *reinterpret_cast<const float4*>(r);
        v[c][0] = x.x; v[c][1] = x.y; v[c][2] = x.z; v[c][3] = x.w;
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n) v[c][n] = dw + c < p.D && n0 + n < p.N ? r[n] : 0.0f;
      }
    }
  };
  auto store = [&](float* base, const float (&v)[4][4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float* r = base + (long long)(dw + c) * p.N + n0;
      if (dw + c >= p.D) continue;
#pragma unroll
      for (int n = 0; n < 4; ++n)
        if (n0 + n < p.N) r[n] = v[c][n];
    }
  };
  const int real0 = q.count ? offset_at(q, 0) : 0, real1 = q.count ? max(real0, offset_at(q, q.count)) : 0;
  // The state entering a window is asked for a window ahead: into h, which is free on the walk back, or, where 16 warps
  // leave a thread 128 registers, into the lane's own place in shared memory.
  constexpr bool kKeptInSmem = kWarps == 16;
  float* s_kept = reinterpret_cast<float*>(s_seq + 2 * W) + (kRoom ? 0 : (2 + 2 * splits) * kCols) + warp * 512;   // [4][32][4]
  auto kept = [&](int w0) {
    const bool real = w0 >= real0 && w0 < real1;
    const float* base = p.kept + (real ? (long long)(w0 / W) * DN : 0);
    if constexpr (kKeptInSmem) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool here = real && dw + c < p.D;
        const float* r = base + (here ? (long long)(dw + c) * p.N : 0);
        float* o = s_kept + (c * 32 + lane) * 4;
        if (vec) {
          const bool some = here && n0 < p.N;
          copy_piece<16>(o, r + (some ? n0 : 0), some ? 16 : 0);
        } else {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const bool some = here && n0 + n < p.N;
            copy_piece<4>(o + n, r + (some ? n0 + n : 0), some ? 4 : 0);
          }
        }
      }
    } else if (real) {
      load(base, h);
    } else {
      zero(h);
    }
  };
  const int w_last = t0 + (t1 - t0 - 1) / W * W;
  if constexpr (kKeptInSmem) kept(w_last);
  fetch(w_last, 0);
  if (even) deal(w_last);
  load(p.A, A);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) A[c][n] *= kLog2eF;
  zero(g); zero(dA);

  // the last sequence with a row before t1
  int s = first_sequence_warp(q, t1, lane);
  int begin = s < q.count ? offset_at(q, s) : q.rows, end = begin;
  if (s < q.count && begin < t1) {
    end = end_of(q, s, begin);                   // it goes on in the next segment
    if (seg + 1 < p.segments) load(p.seg_state + (seg + 1) * p.pieces * DN, g);
  } else {
    --s;
    if (s >= 0) { begin = offset_at(q, s); end = end_of(q, s, begin); }
  }
  if constexpr (!kKeptInSmem) kept(w_last);
  // the transform takes (row, four channels) an item; the finish the same, its sums over many states in four parts
  constexpr int kItems = kWarps <= 2 ? 2 : 1;
  constexpr int kQuads = kCols / 4, kParts = kWarps > 2 ? 4 : 1;
  const int quad = tid % kQuads, my_d = d0 + 4 * quad, in_row = tid / kQuads, in_step = blockDim.x / kQuads;
  const int part = kParts == 1 ? 0 : in_row % kParts, out_row = in_row / kParts, out_step = in_step / kParts;
  // skip, bias and their gradients' sums stay in registers up to 8 warps; where 16 share the
  // register file they lie in shared memory, each thread's sums in a place of its own
  float* s_own = reinterpret_cast<float*>(s_seq + 2 * W);           // [2][kCols] skip | bias, [out_step][2][kCols] sums (not kRoom)
  float* s_sum = s_own + 2 * kCols + out_row * 2 * kCols + 4 * quad;
  float skip[4], bias[4], sum_skip[4] = {}, sum_bias[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    skip[i] = p.skip && my_d + i < p.D ? p.skip[my_d + i] : 0.0f;
    bias[i] = p.bias && my_d + i < p.D ? p.bias[my_d + i] : 0.0f;
  }
  if constexpr (!kRoom) {
    if (in_row == 0) {
      *reinterpret_cast<float4*>(s_own + 4 * quad) = make_float4(skip[0], skip[1], skip[2], skip[3]);
      *reinterpret_cast<float4*>(s_own + kCols + 4 * quad) = make_float4(bias[0], bias[1], bias[2], bias[3]);
    }
    if (part == 0) *reinterpret_cast<float4*>(s_sum) = *reinterpret_cast<float4*>(s_sum + kCols) = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const bool vec_out = pg.vec_rows != 0;
  bool flushed = false;
  auto flush = [&]() {
    float* base = pg.part_A + seg * DN;
    if (flushed) {
      float old[4][4];
      load(base, old);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n) dA[c][n] += old[c][n];
    }
    store(base, dA);
    zero(dA);
    flushed = true;
  };

  int buffer = 0, windows = 0;
  for (int w0 = w_last; w0 >= t0; w0 -= W, buffer ^= 1) {
    const int rows = min(W, t1 - w0);
    unsigned char* raw = smem_raw + buffer * raw_bytes;
    const DT* r_dt = reinterpret_cast<const DT*>(raw);
    const IO *r_u = reinterpret_cast<const IO*>(raw + o_u), *r_z = reinterpret_cast<const IO*>(raw + o_z),
             *r_g = reinterpret_cast<const IO*>(raw + o_g);
    IO *r_b = reinterpret_cast<IO*>(raw + o_b), *r_c = reinterpret_cast<IO*>(raw + o_c);
    if (tid < 2 * W) s_seq[tid] = -1;
    copies_wait();
    __syncthreads();                             // the window has landed, and the one behind it is done with
    if (w0 > t0) {
      if (even) fetch_even(buffer ^ 1);
      else fetch(w0 - W, buffer ^ 1);
    }
    // who begins and ends in the window (the same walk in every thread)
    unsigned firsts = 0, lasts = 0;
    while (s >= 0 && end > w0) {
      if (end > begin) {
        if (end <= w0 + rows) { lasts |= 1u << (end - 1 - w0); if (tid == 0) s_seq[W + end - 1 - w0] = s; }
        if (begin >= w0 && begin < w0 + rows) { firsts |= 1u << (begin - w0); if (tid == 0) s_seq[begin - w0] = s; }
      }
      if (begin < w0) break;                     // began before: the next window meets it again
      --s;
      if (s >= 0) {
        const int e = begin;
        begin = min(offset_at(q, s), e);
        end = e;
      }
    }
    const bool whole = w0 >= real0 && w0 + rows <= real1;
#pragma unroll(kItems)
    for (int r = in_row; r < rows; r += in_step) {
      const int i = r * kCols + 4 * quad;
      float x[4] = {}, xu[4] = {}, dy[4] = {};
      if (whole || (w0 + r >= real0 && w0 + r < real1)) {
        float uv[4], zv[4];
        if constexpr (!kRoom) get4(s_own + kCols + 4 * quad, bias);
        get4(r_dt + i, x); get4(r_u + i, uv); get4(r_g + i, dy);
        if (z) get4(r_z + i, zv);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] += bias[k];
          if (p.softplus) x[k] = softplus_f(x[k]);
          xu[k] = x[k] * uv[k];
          if (z) dy[k] *= zv[k] * sigmoid(zv[k]);
        }
      }
      *reinterpret_cast<float4*>(s_dt + i) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(s_dtu + i) = make_float4(xu[0], xu[1], xu[2], xu[3]);
      *reinterpret_cast<float4*>(s_dy + i) = make_float4(dy[0], dy[1], dy[2], dy[3]);
    }
    if (kWiden || !whole) {
      for (int i = tid * 4; i < rows * NP; i += blockDim.x * 4) {
        float bv[4], cv[4];
        get4(r_b + i, bv); get4(r_c + i, cv);
        if (!whole && (w0 + i / NP < real0 || w0 + i / NP >= real1))
#pragma unroll
          for (int k = 0; k < 4; ++k) bv[k] = cv[k] = 0.0f;
        if constexpr (kWiden) { put4(s_bc + i, bv, true, 4); put4(s_bc + W * NP + i, cv, true, 4); }
        else { put4(r_b + i, bv, true, 4); put4(r_c + i, cv, true, 4); }
      }
    }
    const float* bt = kWiden ? s_bc : reinterpret_cast<const float*>(r_b);
    const float* ct = kWiden ? s_bc + W * NP : reinterpret_cast<const float*>(r_c);
    __syncthreads();
    const int own = 4 * cg, st = split * kStates + 4 * sg;
    if constexpr (kKeptInSmem) {
#pragma unroll
      for (int c = 0; c < 4; ++c) get4(s_kept + (c * 32 + lane) * 4, h[c]);
    }
    for (int r = 0; r < rows; ++r) {
      if (r > 0 && (firsts >> r & 1)) {          // at r = 0 the kept state is the sequence's own
        if (p.start) load(p.start + (long long)s_seq[r] * DN, h);
        else zero(h);
      }
      float x[4], xu[4], bv[4];
      get4(s_dt + r * kCols + own, x); get4(s_dtu + r * kCols + own, xu); get4(bt + r * NP + st, bv);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 x2 = both(x[c]), xu2 = both(xu[c]);
        float2 v[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          v[n] = mul2(ex2f2(mul2(x2, pair(A[c], n))), pair(h[c], n));
          set(h[c], n, fma2(xu2, pair(bv, n), v[n]));
        }
        *reinterpret_cast<float4*>(mine + r * kRowFloats + (c * 32 + lane) * 4) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
      }
    }
    if (w0 > t0) {
      kept(w0 - W);                              // for the next window: it arrives during the walk back
      if constexpr (kKeptInSmem) copies_commit();
    }
    // (Asking for the next row's operands, p and decays while a row's products are formed made this slower, 1.83 -> 2.0
    // .. 2.3 ms at the first size above: the registers and the code it takes cost more than the latencies.)
    for (int r = rows - 1; r >= 0; --r) {
      if (lasts >> r & 1) {
        if (pg.grad_end) load(pg.grad_end + (long long)s_seq[W + r] * DN, g);
        else zero(g);
      }
      float x[4], xu[4], dy[4], bv[4], cv[4], pv[4][4];
      get4(s_dt + r * kCols + own, x); get4(s_dtu + r * kCols + own, xu); get4(s_dy + r * kCols + own, dy);
      get4(bt + r * NP + st, bv); get4(ct + r * NP + st, cv);
#pragma unroll
      for (int c = 0; c < 4; ++c) get4(mine + r * kRowFloats + (c * 32 + lane) * 4, pv[c]);
      float sb[4] = {}, sc[4] = {}, sy[4], s1[4], s2[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 x2 = both(x[c]), xu2 = both(xu[c]), dy2 = both(dy[c]);
        float2 ty = both(0.0f), t1 = both(0.0f), t2 = both(0.0f);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float2 b2 = pair(bv, n), c2 = pair(cv, n), p2 = pair(pv[c], n), a2 = pair(A[c], n);
          const float2 hv = fma2(xu2, b2, p2), gv = fma2(c2, dy2, pair(g[c], n));
          set(sc, n, fma2(dy2, hv, pair(sc, n)));
          set(sb, n, fma2(xu2, gv, pair(sb, n)));
          ty = fma2(c2, hv, ty);
          t1 = fma2(b2, gv, t1);
          const float2 qv = mul2(gv, p2);
          t2 = fma2(a2, qv, t2);
          set(dA[c], n, fma2(x2, qv, pair(dA[c], n)));
          set(g[c], n, mul2(ex2f2(mul2(x2, a2)), gv));
        }
        sy[c] = ty.x + ty.y; s1[c] = t1.x + t1.y; s2[c] = t2.x + t2.y;
      }
      // lanes of channels 0..3 take dB, 4..7 dC, each for the two; the sums' writes then fit where p was
      const bool upper = lane & 16;
      float bc[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) bc[n] = (upper ? sc[n] : sb[n]) + __shfl_xor_sync(0xffffffffu, upper ? sb[n] : sc[n], 16);
      __syncwarp();                              // the row's p has been read by all
      float* to = mine + r * kRowFloats;
      // odd lanes of channels swap the halves: no bank conflict
      put4(to + (cg & 3) * 32 + (((upper ? 16 : 0) + sg * 4) ^ ((cg & 1) << 4)), bc, true, 4);
      to += 128 + sg * 96 + ((cg + 2 * sg) & 7) * 4;
      put4(to, sy, true, 4); put4(to + 32, s1, true, 4); put4(to + 64, s2, true, 4);
      if ((firsts >> r & 1) && pg.dstart) store(pg.dstart + (long long)s_seq[r] * DN, g);
    }
    if (++windows == kFlushWindows) { flush(); windows = 0; }
    __syncthreads();
    // dB and dC of the window: over the channels of the CTA, four states an item
    for (int i = tid; i < rows * splits * 8; i += blockDim.x) {
      const int v = (i & 7) * 4, kr = i >> 3, r = kr / splits, k = kr - r * splits;
      float a[4] = {};
      const float* o = s_rows + (k * W + r) * kRowFloats;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 e = *reinterpret_cast<const float4*>(o + j * 32 + (v ^ ((j & 1) << 4)));
        a[0] += e.x; a[1] += e.y; a[2] += e.z; a[3] += e.w;
      }
      const int n = k * kStates + (v & 15);
      const long long row = w0 + r;
      if (!whole && (row < real0 || row >= real1))   // 0 * inf: what a sequence's last states or first adjoints left behind
        a[0] = a[1] = a[2] = a[3] = 0.0f;
      if (pg.column_blocks > 1)
        put4(pg.part_bc + ((long long)blockIdx.x * q.rows + row) * 2 * p.N + (v < 16 ? 0 : p.N) + n, a, p.N % 4 == 0, p.N - n);
      else
        put4(static_cast<IO*>(v < 16 ? pg.dB : pg.dC) + row * p.N + n, a, pg.vec_bc != 0, p.N - n);
    }
    // the rows' own gradients: over the states
#pragma unroll(kItems)
    for (int r = out_row; r < rows; r += out_step) {
      const long long row = w0 + r;
      float y[4] = {}, s1[4] = {}, s2[4] = {};
      for (int k = part; k < splits; k += kParts) {
        const float* o = s_rows + (k * W + r) * kRowFloats + 128;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float* e = o + j * 96 + ((quad + 2 * j) & 7) * 4;
          const float4 e0 = *reinterpret_cast<const float4*>(e), e1 = *reinterpret_cast<const float4*>(e + 32),
                       e2 = *reinterpret_cast<const float4*>(e + 64);
          y[0] += e0.x; y[1] += e0.y; y[2] += e0.z; y[3] += e0.w;
          s1[0] += e1.x; s1[1] += e1.y; s1[2] += e1.z; s1[3] += e1.w;
          s2[0] += e2.x; s2[1] += e2.y; s2[2] += e2.z; s2[3] += e2.w;
        }
      }
      if constexpr (kParts > 1) {                // a warp has one row: 8 quads x 4 parts
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[i] += __shfl_xor_sync(0xffffffffu, y[i], 8); y[i] += __shfl_xor_sync(0xffffffffu, y[i], 16);
          s1[i] += __shfl_xor_sync(0xffffffffu, s1[i], 8); s1[i] += __shfl_xor_sync(0xffffffffu, s1[i], 16);
          s2[i] += __shfl_xor_sync(0xffffffffu, s2[i], 8); s2[i] += __shfl_xor_sync(0xffffffffu, s2[i], 16);
        }
        if (part != 0) continue;
      }
      float du[4] = {}, draw[4] = {}, dzv[4] = {};
      if (whole || (row >= real0 && row < real1)) {
        const int i = r * kCols + 4 * quad;
        float x[4], dy[4], uv[4], zv[4], gv[4];
        if constexpr (!kRoom) { get4(s_own + 4 * quad, skip); get4(s_sum, sum_skip); get4(s_sum + kCols, sum_bias); }
        get4(s_dt + i, x); get4(s_dy + i, dy); get4(r_u + i, uv);
        if (z) { get4(r_z + i, zv); get4(r_g + i, gv); }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          du[k] = fmaf(s1[k], x[k], dy[k] * skip[k]);
          draw[k] = fmaf(s1[k], uv[k], s2[k] * 0.6931471805599453f);
          if (p.softplus) draw[k] *= softplus_slope(x[k]);
          if (z) {
            const float sig = sigmoid(zv[k]);
            dzv[k] = gv[k] * fmaf(skip[k], uv[k], y[k]) * sig * fmaf(zv[k], 1.0f - sig, 1.0f);
          }
          sum_skip[k] = fmaf(dy[k], uv[k], sum_skip[k]);
          sum_bias[k] += draw[k];
        }
        if constexpr (!kRoom) { put4(s_sum, sum_skip, true, 4); put4(s_sum + kCols, sum_bias, true, 4); }
      }
      const long long to = row * p.D + my_d;
      put4(static_cast<IO*>(pg.du) + to, du, vec_out, p.D - my_d);
      put4(static_cast<DT*>(pg.ddt) + to, draw, vec_out, p.D - my_d);
      if (pg.dz) put4(static_cast<IO*>(pg.dz) + to, dzv, vec_out, p.D - my_d);
    }
  }
  flush();
  __syncthreads();
  // over the threads that took rows of the same channels
  const float* s_all = kRoom ? s_rows : s_own + 2 * kCols;
  if (kRoom && part == 0) {
    put4(s_rows + out_row * 2 * kCols + 4 * quad, sum_skip, true, 4);
    put4(s_rows + (out_row * 2 + 1) * kCols + 4 * quad, sum_bias, true, 4);
  }
  __syncthreads();
  for (int i = tid; i < 2 * kCols; i += blockDim.x) {
    const int c = i % kCols, which = i / kCols;
    if (d0 + c >= p.D) continue;
    float a = 0.0f;
    for (int k = 0; k < out_step; ++k) a += s_all[(k * 2 + which) * kCols + c];
    pg.part_d[((long long)seg * 2 + which) * p.D + d0 + c] = a;
  }
}

// dB, dC from the column blocks' sums, dA, dskip, dbias from the segments' sums, in a fixed order.  Four states at a time
// where N allows it (kFour): the sums of dB | dC are the bulk, 8 bytes a state, row and column block, once.
template <typename IO, bool kFour>
__global__ void __launch_bounds__(256) scan_backward_sums_kernel(const ScanPackedGrad pg) {
  constexpr int V = kFour ? 4 : 1;
  const ScanPacked& p = pg.f;
  const long long DN = (long long)p.D * p.N, wide = (long long)p.q.rows * 2 * p.N, bc = pg.column_blocks > 1 ? wide / V : 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < bc + DN + 2ll * p.D; i += (long long)gridDim.x * 256) {
    if (i < bc) {
      float a[4] = {};
#pragma unroll 4
      for (int k = 0; k < pg.column_blocks; ++k) {
        const float* from = pg.part_bc + k * wide + i * V;
        if constexpr (kFour) {
          const float4 v = *reinterpret_cast<const float4*>(from);
          a[0] += v.x; a[1] += v.y; a[2] += v.z; a[3] += v.w;
        } else {
          a[0] += *from;
        }
      }
      const long long row = i * V / (2 * p.N);
      const int n = (int)(i * V - row * 2 * p.N);
      put4(static_cast<IO*>(n < p.N ? pg.dB : pg.dC) + row * p.N + (n < p.N ? n : n - p.N), a, kFour && pg.vec_bc, V);
      continue;
    }
    float a = 0.0f;
    if (i < bc + DN) {
#pragma unroll 4
      for (int k = 0; k < p.segments; ++k) a += pg.part_A[k * DN + i - bc];
      pg.dA[i - bc] = a;
    } else {
      const long long j = i - bc - DN;
#pragma unroll 4
      for (int k = 0; k < p.segments; ++k) a += pg.part_d[k * 2ll * p.D + j];
      float* to = j < p.D ? pg.dskip : pg.dbias;
      if (to) to[j < p.D ? j : j - p.D] = a;
    }
  }
}

// A sequence without rows hands the gradient of its state on.
__global__ void __launch_bounds__(256) scan_empty_starts_kernel(const ScanPackedGrad pg) {
  const ScanPacked& p = pg.f;
  const long long DN = (long long)p.D * p.N;
  for (int s = blockIdx.x; s < p.q.count; s += gridDim.x) {
    const int begin = offset_at(p.q, s);
    if (end_of(p.q, s, begin) > begin) continue;
    for (long long i = threadIdx.x; i < DN; i += 256) pg.dstart[s * DN + i] = pg.grad_end ? pg.grad_end[s * DN + i] : 0.0f;
  }
}

// CTA of the backward: 32 channels, a warp for every 16 states.
static ScanShape backward_shape(int64_t D, int64_t N) {
  ScanShape s;
  s.splits = (int)((N + kStates - 1) / kStates);
  s.groups = 1;
  s.threads = 32 * s.splits;
  s.channels = 32;
  s.column_blocks = (unsigned)((D + 31) / 32);
  return s;
}
template <typename IO, typename DT>
static const void* backward_kernel_of(int splits) {
  if (splits == 1) return (const void*)scan_packed_backward_kernel<IO, DT, 8, 1>;
  return splits <= 2 ? (const void*)scan_packed_backward_kernel<IO, DT, 8, 2>
                     : (splits <= 8 ? (const void*)scan_packed_backward_kernel<IO, DT, 8, 8> : (const void*)scan_packed_backward_kernel<IO, DT, 4, 16>);
}
static size_t backward_smem(const ScanShape& s, size_t W, size_t io, size_t dt) {
  const size_t NP = s.splits * kStates, cols = s.channels;
  return 2 * W * (cols * (3 * io + dt) + 2 * NP * io) +
         ((size_t)s.splits * W * kRowFloats + 3 * W * cols + (io == 2 ? 2 * W * NP : 0) + 2 * W +
          (s.splits > 8 ? 2 * cols + 2 * s.splits * cols + s.threads * 16 : 0)) * sizeof(float);
}
static ScanCut backward_cut(int64_t rows, int64_t D, int64_t N, int io, int dt) {
  const ScanShape s = backward_shape(D, N);
  const int W = ossm_b200_selective_scan_packed_tile(N);
  const size_t ib = io == OSSM_B200_DTYPE_BF16 ? 2 : 4, db = dt == OSSM_B200_DTYPE_BF16 ? 2 : 4;
  const void* kernel = ib == 4 ? backward_kernel_of<float, float>(s.splits)
                               : (db == 4 ? backward_kernel_of<__nv_bfloat16, float>(s.splits) : backward_kernel_of<__nv_bfloat16, __nv_bfloat16>(s.splits));
  return scan_cut(rows, resident_ctas(kernel, s.threads, backward_smem(s, W, ib, db), 1), s.column_blocks, W, 0);
}
static size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

struct BackwardPlan {
  ScanCut cut;
  size_t dts, kinds, part_A, part_d, part_bc, total;   // offsets into the workspace
};
static BackwardPlan backward_plan(int64_t rows, int64_t D, int64_t N, int io, int dt) {
  BackwardPlan b{};
  b.cut = backward_cut(rows, D, N, io, dt);
  const ScanShape s = backward_shape(D, N);
  const size_t states = up256((size_t)b.cut.segments * D * N * 4), pieces = (size_t)b.cut.segments * b.cut.pieces;
  b.dts = up256(pieces * D * N * 4);
  b.kinds = b.dts + up256(pieces * D * 4);
  b.part_A = b.kinds + up256(pieces * 4);
  b.part_d = b.part_A + states;
  b.part_bc = b.part_d + up256((size_t)b.cut.segments * 2 * D * 4);
  b.total = b.part_bc + (s.column_blocks > 1 ? (size_t)s.column_blocks * rows * 2 * N * 4 : 0);
  return b;
}

template <typename IO, typename DT, int kGroups>
static int launch_adjoint(const ScanPackedGrad& pg, const ScanShape& s, cudaStream_t stream) {
  const size_t NP = s.splits * kStates, io = sizeof(IO), cols = s.channels;
  const size_t bytes = 2 * kTile * (cols * (2 * io + sizeof(DT)) + NP * io) + (io == 2 ? kTile * NP * sizeof(float) : 0) +
                       (kGroups == 4 ? 0 : kTile * cols * sizeof(float2));
  if (int rc = ensure_dynamic_smem((const void*)scan_packed_adjoint_kernel<IO, DT, kGroups>, bytes)) return rc;
  scan_packed_adjoint_kernel<IO, DT, kGroups><<<dim3(s.column_blocks, (pg.f.segments - 1) * pg.f.pieces), s.threads, bytes, stream>>>(pg, s.splits);
  return kOk;
}

template <typename IO, typename DT, int W, int kWarps>
static int launch_backward_w(const ScanPackedGrad& pg, cudaStream_t stream) {
  const ScanPacked& p = pg.f;
  const ScanShape s = backward_shape(p.D, p.N);
  const size_t bytes = backward_smem(s, W, sizeof(IO), sizeof(DT));
  if (int rc = ensure_dynamic_smem((const void*)scan_packed_backward_kernel<IO, DT, W, kWarps>, bytes)) return rc;
  if (p.segments > 1) {
    const ScanShape a = scan_shape(p.D, p.N);
    if (int rc = a.groups == 4 ? launch_adjoint<IO, DT, 4>(pg, a, stream)
                               : (a.groups == 2 ? launch_adjoint<IO, DT, 2>(pg, a, stream) : launch_adjoint<IO, DT, 1>(pg, a, stream)))
      return rc;
    scan_adjoint_seams_kernel<<<(unsigned)(((long long)p.D * p.N + 127) / 128), 128, 0, stream>>>(p);
  }
  if (pg.dstart && p.q.count) scan_empty_starts_kernel<<<p.q.count < 1024 ? p.q.count : 1024, 256, 0, stream>>>(pg);
  scan_packed_backward_kernel<IO, DT, W, kWarps><<<dim3(s.column_blocks, p.segments), s.threads, bytes, stream>>>(pg, s.splits);
  const bool four = p.N % 4 == 0;
  const long long items = (pg.column_blocks > 1 ? (long long)p.q.rows * 2 * p.N / (four ? 4 : 1) : 0) + (long long)p.D * (p.N + 2);
  const long long blocks = (items + 255) / 256, most = (long long)sm_count() * 16;
  const unsigned grid = (unsigned)(blocks < most ? blocks : most);
  if (four) scan_backward_sums_kernel<IO, true><<<grid, 256, 0, stream>>>(pg);
  else scan_backward_sums_kernel<IO, false><<<grid, 256, 0, stream>>>(pg);
  return check_cuda(cudaGetLastError(), "scan_packed_backward_kernel launch");
}

template <typename IO, typename DT>
static int launch_backward(ScanPackedGrad pg, cudaStream_t stream) {
  ScanPacked& p = pg.f;
  p.by_u = piece_bytes(p.u, p.ldu, sizeof(IO)); p.by_z = piece_bytes(p.z, p.ldz, sizeof(IO));
  pg.by_g = piece_bytes(pg.grad, pg.ldg, sizeof(IO)); p.by_dt = piece_bytes(p.dt, p.lddt, sizeof(DT));
  p.by_b = piece_bytes(p.B, p.ldb, sizeof(IO)); p.by_c = piece_bytes(p.C, p.ldc, sizeof(IO));
  const long long widest = 1 << 24;   // a window's move fits 32 bits
  const bool narrow = p.ldu < widest && p.lddt < widest && p.ldz < widest && pg.ldg < widest && p.ldb < widest && p.ldc < widest;
  // the gradients lie wherever the caller puts them: four at a time only where every row and pointer allows it
  const auto at = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  pg.vec_rows = p.D % 4 == 0 && ((at(pg.du) | at(pg.dz)) & (4 * sizeof(IO) - 1)) == 0 && (at(pg.ddt) & (4 * sizeof(DT) - 1)) == 0;
  pg.vec_bc = p.N % 4 == 0 && ((at(pg.dB) | at(pg.dC)) & (4 * sizeof(IO) - 1)) == 0;
  pg.even = narrow && p.N % kStates == 0 && p.by_u == 16 && p.by_z == 16 && pg.by_g == 16 && p.by_dt == 16 && p.by_b == 16 && p.by_c == 16;
  if (p.N <= kStates) return launch_backward_w<IO, DT, 8, 1>(pg, stream);
  if (p.N <= 2 * kStates) return launch_backward_w<IO, DT, 8, 2>(pg, stream);
  return p.N <= 8 * kStates ? launch_backward_w<IO, DT, 8, 8>(pg, stream) : launch_backward_w<IO, DT, 4, 16>(pg, stream);
}

}  // namespace packed
}  // namespace ossm_b200

extern "C" {

using namespace ossm_b200;

size_t ossm_b200_selective_scan_packed_backward_workspace_bytes(int64_t rows, int64_t D, int64_t N, int io_dtype,
                                                                int dt_dtype) {
  if (rows <= 0 || D <= 0 || N <= 0 || N > 256) return 0;
  return packed::backward_plan(rows, D, N, io_dtype, dt_dtype).total;
}

int ossm_b200_selective_scan_packed_backward(const void* dout, int64_t ldg, const void* u, int64_t ldu, const void* dt,
                                             int64_t lddt, const float* A, const void* Bm, int64_t ldb, const void* Cm,
                                             int64_t ldc, const void* z, int64_t ldz, const float* Dskip,
                                             const float* delta_bias, int delta_softplus, const int* offsets,
                                             const float* start, const float* grad_end, const float* kept, void* du,
                                             void* ddt, float* dA, void* dB, void* dC, void* dz, float* dD,
                                             float* ddelta_bias, float* grad_start, void* workspace,
                                             size_t workspace_bytes, int64_t rows, int64_t count, int64_t D, int64_t N,
                                             int io_dtype, int dt_dtype, ossm_b200_stream_t stream) {
  const char* fn = "selective_scan_packed_backward";
  if (int rc = packed::check_scan(fn, rows, D, N, count, count, io_dtype, dt_dtype)) return rc;
  if (D == 0) return kOk;
  if (rows == 0) { set_last_error("%s: no rows", fn); return kErrInvalidArgument; }
  if (!dout || !u || !dt || !A || !Bm || !Cm || !offsets || !kept || !du || !ddt || !dA || !dB || !dC || (z && !dz)) {
    set_last_error("%s: null pointer", fn);
    return kErrInvalidArgument;
  }
  if (ldg < D || ldu < D || lddt < D || ldb < N || ldc < N || (z && ldz < D)) { set_last_error("%s: row pitch smaller than the row", fn); return kErrInvalidArgument; }
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0 ||
      workspace_bytes < ossm_b200_selective_scan_packed_backward_workspace_bytes(rows, D, N, io_dtype, dt_dtype)) {
    set_last_error("%s: workspace too small or not on a 16-byte boundary", fn);
    return kErrWorkspace;
  }
  const packed::BackwardPlan b = packed::backward_plan(rows, D, N, io_dtype, dt_dtype);
  char* w = static_cast<char*>(workspace);
  packed::ScanPackedGrad pg{};
  packed::ScanPacked& p = pg.f;
  p.q = {offsets, nullptr, nullptr, 1, (int)count, (int)rows, count};
  p.u = u; p.dt = dt; p.B = Bm; p.C = Cm; p.z = z; p.A = A; p.skip = Dskip; p.bias = delta_bias; p.start = start;
  p.kept = const_cast<float*>(kept);
  p.ldu = ldu; p.lddt = lddt; p.ldb = ldb; p.ldc = ldc; p.ldz = ldz;
  p.D = (int)D; p.N = (int)N; p.softplus = delta_softplus;
  p.vec = N % 4 == 0 && ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(start) | reinterpret_cast<uintptr_t>(grad_end) |
                          reinterpret_cast<uintptr_t>(kept)) & 15u) == 0;
  p.segments = b.cut.segments; p.segment_rows = b.cut.segment_rows; p.pieces = b.cut.pieces;
  p.seg_state = reinterpret_cast<float*>(w);
  p.seg_dt = reinterpret_cast<float*>(w + b.dts);
  p.seg_kind = reinterpret_cast<int*>(w + b.kinds);
  pg.grad = dout; pg.grad_end = grad_end; pg.ldg = ldg;
  pg.du = du; pg.ddt = ddt; pg.dB = dB; pg.dC = dC; pg.dz = z ? dz : nullptr;
  pg.dA = dA; pg.dskip = dD; pg.dbias = ddelta_bias; pg.dstart = grad_start;
  pg.part_A = reinterpret_cast<float*>(w + b.part_A);
  pg.part_d = reinterpret_cast<float*>(w + b.part_d);
  pg.part_bc = reinterpret_cast<float*>(w + b.part_bc);
  pg.column_blocks = (int)packed::backward_shape(D, N).column_blocks;
  if (io_dtype == OSSM_B200_DTYPE_F32) return packed::launch_backward<float, float>(pg, stream);
  if (dt_dtype == OSSM_B200_DTYPE_F32) return packed::launch_backward<__nv_bfloat16, float>(pg, stream);
  return packed::launch_backward<__nv_bfloat16, __nv_bfloat16>(pg, stream);
}

}  // extern "C"
