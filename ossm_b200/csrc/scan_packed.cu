// Mamba selective scan over a packed batch (forward) and over single tokens (sm_100a).
//
//   dt = softplus(raw + bias[d])         h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t         y_t = C_t . h_t + skip[d] u_t
//   out_t = y_t silu(z_t)
//
// The state before a sequence's first row is its cache entry (or zeros), the state behind its last row goes back there.
#include "scan_packed.cuh"

#include <type_traits>

namespace ossm_b200 {
OSSM_B200_STATUS_ACCESSOR(status_packed_scan)
namespace packed {

// A lane holds one channel and 16 of its states in registers and walks the rows in order: per state and row one
// exponential, two products and two fused sums, two states an instruction.  The exponentials bound it: 16 + 4 a row and
// lane (the step transform and the gate take two each) at 16 an SM and cycle; the read ports of the register file, which
// give three operands in 1.5 cycles, come close behind.  Rows come in tiles of 16 through shared memory, copied
// asynchronously one tile ahead; B and C are widened to float32 there, since every lane reads all of them.  With up to 16
// states a lane also does its channel's step transform and gate; above, `splits` warps share a channel, so the transform
// is evaluated once into shared memory and the warps' partial outputs meet there.  Sixteen warps an SM at 128 registers
// beat twenty at 96 (24576 rows x 2048 channels x 16 states: 0.314 against 0.345 ms) and thirty-two at 64 (12800 rows x 128
// channels x 256 states: 0.253 against 0.277 ms).  The special functions run at 0.69 of their rate at 16 states, at 0.39 at
// 256, where an SM has one CTA of 16 warps that meet at three barriers a tile.  65536 rows of one sequence, 2048 channels x 16 states: 0.81 ms, 2.6e12
// states a second, and 0.61 ms for the summary of the seams.
//
// Time segments: the rows are cut into `segments` stretches, one CTA each, so that a long sequence fills the GPU as well
// as many short ones do.  A sequence that crosses a seam needs the state there: the summary pass (kSummary) runs only the
// rows of each segment's last, crossing sequence and leaves the state they reach from zero and the sum of their steps (the
// decay over them is exp(A sum dt)); scan_seams_kernel chains those into the state entering each segment; the scan
// proper starts from it.  These rows are few in one segment and all of them in the next, so the summary takes a segment
// in `pieces`, a CTA each: more CTAs than fit even the load out.  seg_kind of a piece: 0 it has no such rows, 1 the
// sequence begins in it (its summary is the state itself), 2 the sequence came from before.  The piece where it begins
// also copies its entry state to seg_first, since another CTA of the scan proper may already have written the cache.
template <typename IO, typename DT, int kGroups, bool kSummary>
__global__ void __launch_bounds__(kGroups == 1 ? 512 : 128, kGroups == 1 ? 1 : 4) scan_packed_kernel(const ScanPacked p, int splits) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  constexpr int kCols = 32 * kGroups;
  constexpr bool kWiden = sizeof(IO) == 2, kOne = kGroups == 4;     // kOne: one warp has all the states of its channels
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = warp % splits, group = warp / splits;
  const int NP = splits * kStates;
  // two tiles of raw operands, then what is shared in float32
  const int raw_bytes = kTile * (kCols * (2 * (int)sizeof(IO) + (int)sizeof(DT)) + 2 * NP * (int)sizeof(IO));
  const int o_u = kTile * kCols * (int)sizeof(DT), o_z = o_u + kTile * kCols * (int)sizeof(IO),
            o_b = o_z + kTile * kCols * (int)sizeof(IO), o_c = o_b + kTile * NP * (int)sizeof(IO);
  float* s_bc = reinterpret_cast<float*>(smem_raw + 2 * raw_bytes);             // [2][kTile][NP] (kWiden)
  float2* s_dt = reinterpret_cast<float2*>(s_bc + (kWiden ? 2 * kTile * NP : 0)); // [kTile][kCols] (dt, dt u) (not kOne)
  float* s_y = reinterpret_cast<float*>(s_dt + (kOne ? 0 : kTile * kCols));     // [splits][kTile][kCols] (not kOne)
  const Sequences& q = p.q;
  const int seg = kSummary ? blockIdx.y / p.pieces : blockIdx.y;
  const bool last = seg == p.segments - 1;
  const int seam = last ? q.rows : min(q.rows, (seg + 1) * p.segment_rows);   // where the segment ends
  const int t0 = kSummary ? blockIdx.y * (p.segment_rows / p.pieces) : seg * p.segment_rows;
  const int t1 = kSummary ? min(seam, t0 + p.segment_rows / p.pieces) : seam;
  const int d0 = blockIdx.x * kCols, col = group * 32 + lane, d = d0 + col, n0 = split * kStates;
  const int left = d < p.D ? p.N - n0 : 0;                          // states of this lane that exist
  const bool vec = p.vec != 0;
  const long long at = (long long)d * p.N + n0, DN = (long long)p.D * p.N;
  const IO *u = static_cast<const IO*>(p.u) + d0, *Bm = static_cast<const IO*>(p.B), *Cm = static_cast<const IO*>(p.C),
           *z = p.z ? static_cast<const IO*>(p.z) + d0 : nullptr;
  const DT* dt = static_cast<const DT*>(p.dt) + d0;
  const TileLane l_u = tile_lane<IO>(p.by_u, kCols, p.D - d0), l_z = tile_lane<IO>(p.by_z, kCols, p.D - d0),
                 l_dt = tile_lane<DT>(p.by_dt, kCols, p.D - d0), l_b = tile_lane<IO>(p.by_b, NP, p.N),
                 l_c = tile_lane<IO>(p.by_c, NP, p.N);
  auto fetch = [&](int tile, int end, int buffer) {
    unsigned char* raw = smem_raw + buffer * raw_bytes;
    const int rows = min(kTile, end - tile);
    const long long row = tile;
    tile_load(reinterpret_cast<DT*>(raw), kCols, dt + row * p.lddt, p.lddt, rows, p.by_dt, l_dt);
    tile_load(reinterpret_cast<IO*>(raw + o_u), kCols, u + row * p.ldu, p.ldu, rows, p.by_u, l_u);
    tile_load(reinterpret_cast<IO*>(raw + o_b), NP, Bm + row * p.ldb, p.ldb, rows, p.by_b, l_b);
    if constexpr (!kSummary) {
      if (z) tile_load(reinterpret_cast<IO*>(raw + o_z), kCols, z + row * p.ldz, p.ldz, rows, p.by_z, l_z);
      tile_load(reinterpret_cast<IO*>(raw + o_c), NP, Cm + row * p.ldc, p.ldc, rows, p.by_c, l_c);
    }
    copies_commit();
  };

  float A[kStates], h[kStates];
  load_states(p.A + at, left, vec, A);
#pragma unroll
  for (int j = 0; j < kStates; ++j) { A[j] *= kLog2eF; h[j] = 0.0f; }
  const float bias = p.bias && d < p.D ? p.bias[d] : 0.0f, skip = p.skip && d < p.D ? p.skip[d] : 0.0f;
  float dt_sum = 0.0f;

  int from = t0, s, stop;
  bool active;
  if constexpr (kSummary) {
    s = first_sequence_warp(q, seam, lane);      // the sequence that may cross the seam
    const int begin = s < q.count ? offset_at(q, s) : seam;
    const bool here = begin < t1;                // rows of it in this piece
    if (blockIdx.x == 0 && tid == 0) p.seg_kind[blockIdx.y] = !here ? 0 : (begin >= t0 ? 1 : 2);
    if (!here) return;
    from = max(t0, begin);
    fetch(from, t1, 0);
    if (begin >= t0) {
      const long long entry = entry_of(q, s);
      if (p.start != nullptr && entry >= 0 && resumes(q, s)) load_states(p.start + entry * DN + at, left, vec, h);
      store_states(p.seg_first + seg * DN + at, left, vec, h);
    }
    active = true;
    stop = t1;
  } else {
    fetch(from, t1, 0);
    s = first_sequence_warp(q, t0, lane);
    const int begin = s < q.count ? offset_at(q, s) : q.rows;
    active = begin < t0;
    stop = max(t0, active ? end_of(q, s, begin) : begin);   // t0 only where offsets run backwards
    if (active) load_states(p.seg_state + (seg * p.pieces - 1) * DN + at, left, vec, h);
  }
  const int real0 = q.count ? offset_at(q, 0) : 0, real1 = q.count ? offset_at(q, q.count) : 0;

  // leaves the current sequence and enters the one with rows that begins at `stop`, if any
  auto finish = [&]() {
    const long long entry = entry_of(q, s);
    if (p.end != nullptr && entry >= 0) store_states(p.end + entry * DN + at, left, vec, h);
    ++s;
  };
  auto enter = [&]() {
    if (active) finish();
    active = false;
    const int begin = stop;
    while (s < q.count) {
      const int end = end_of(q, s, begin);
      const long long entry = entry_of(q, s);
      const bool cont = p.start != nullptr && entry >= 0 && resumes(q, s);
#pragma unroll
      for (int j = 0; j < kStates; ++j) h[j] = 0.0f;
      if (!last && end > t1) load_states(p.seg_first + seg * DN + at, left, vec, h);
      else if (cont) load_states(p.start + entry * DN + at, left, vec, h);
      if (end > begin) { active = true; stop = end; return; }
      finish();                                  // a sequence without rows hands its state on
    }
    stop = 0x7fffffff;
  };
  // one row: the states move on by (dt, dt u); returns the lane's part of C . h
  auto row_step = [&](float x, float xu, const float* b, const float* c) {
    const float2 x2 = both(x), xu2 = both(xu);
    float2 y0 = both(0.0f), y1 = both(0.0f);
#pragma unroll
    for (int j = 0; j < kStates; j += 4) {
      const float4 bv = *reinterpret_cast<const float4*>(b + j);
      float2 h0 = make_float2(h[j], h[j + 1]), h1 = make_float2(h[j + 2], h[j + 3]);
      h0 = fma2(ex2f2(mul2(x2, make_float2(A[j], A[j + 1]))), h0, mul2(xu2, make_float2(bv.x, bv.y)));
      h1 = fma2(ex2f2(mul2(x2, make_float2(A[j + 2], A[j + 3]))), h1, mul2(xu2, make_float2(bv.z, bv.w)));
      h[j] = h0.x; h[j + 1] = h0.y; h[j + 2] = h1.x; h[j + 3] = h1.y;
      if constexpr (!kSummary) {
        const float4 cv = *reinterpret_cast<const float4*>(c + j);
        y0 = fma2(h0, make_float2(cv.x, cv.y), y0);
        y1 = fma2(h1, make_float2(cv.z, cv.w), y1);
      }
    }
    y0 = add2(y0, y1);
    return y0.x + y0.y;
  };
  auto step_of = [&](float raw, float add) {
    const float x = raw + add;
    return p.softplus ? softplus_f(x) : x;
  };

  int buffer = 0;
  for (int tile = from; tile < t1; tile += kTile, buffer ^= 1) {
    const int rows = min(kTile, t1 - tile), tend = tile + rows;
    unsigned char* raw = smem_raw + buffer * raw_bytes;
    const DT* r_dt = reinterpret_cast<const DT*>(raw);
    const IO *r_u = reinterpret_cast<const IO*>(raw + o_u), *r_z = reinterpret_cast<const IO*>(raw + o_z),
             *r_b = reinterpret_cast<const IO*>(raw + o_b), *r_c = reinterpret_cast<const IO*>(raw + o_c);
    copies_wait();
    __syncthreads();                             // this tile has landed, and the last one is done with
    if (tend < t1) fetch(tend, t1, buffer ^ 1);
    const float *bt, *ct;
    if constexpr (kWiden) {
      for (int i = tid * 2; i < rows * NP; i += blockDim.x * 2) {
        const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(r_b + i));
        *reinterpret_cast<float2*>(s_bc + i) = v;
        if constexpr (!kSummary) {
          const float2 w = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(r_c + i));
          *reinterpret_cast<float2*>(s_bc + kTile * NP + i) = w;
        }
      }
      bt = s_bc; ct = s_bc + kTile * NP;
    } else {
      bt = reinterpret_cast<const float*>(r_b); ct = reinterpret_cast<const float*>(r_c);
    }
    if constexpr (!kOne) {
#pragma unroll 2
      for (int i = tid; i < rows * kCols; i += blockDim.x) {
        const int c = i % kCols;
        const float x = step_of(to_float(r_dt[i]), p.bias && d0 + c < p.D ? p.bias[d0 + c] : 0.0f);
        s_dt[i] = make_float2(x, x * to_float(r_u[i]));
      }
    }
    if constexpr (kWiden || !kOne) __syncthreads();
    int t = tile;
    while (t < tend) {
      int upto = tend;
      if constexpr (!kSummary) {
        if (t == stop) enter();
        upto = min(stop, tend);
        if (p.kept != nullptr) {
          if (active && t % p.keep == 0) store_states(p.kept + (t / p.keep) * DN + at, left, vec, h);
          upto = min(upto, (t / p.keep + 1) * p.keep);
        }
        if (!active) {                           // rows of no sequence
          if (kOne && p.zero_rest && d < p.D)
            for (int row = t; row < upto; ++row) static_cast<IO*>(p.out)[(long long)row * p.ldo + d] = from_float<IO>(0.0f);
          t = upto;
          continue;
        }
      }
      int r = t - tile;
      const int r_end = upto - tile;
      t = upto;
      if constexpr (!kOne) {
        for (; r < r_end; ++r) {
          const float2 x = s_dt[r * kCols + col];
          const float y = row_step(x.x, x.y, bt + r * NP + n0, ct + r * NP + n0);
          if constexpr (kSummary) dt_sum += x.x;
          else s_y[(split * kTile + r) * kCols + col] = y;
        }
      } else {
        auto rows_of = [&](auto count) {
          constexpr int k = decltype(count)::value;
          float x[k], uv[k], y[k];
#pragma unroll
          for (int j = 0; j < k; ++j) {
            x[j] = step_of(to_float(r_dt[(r + j) * kCols + col]), bias);
            uv[j] = to_float(r_u[(r + j) * kCols + col]);
          }
#pragma unroll
          for (int j = 0; j < k; ++j) {
            y[j] = row_step(x[j], x[j] * uv[j], bt + (r + j) * NP, ct + (r + j) * NP);
            if constexpr (kSummary) dt_sum += x[j];
          }
          if constexpr (!kSummary) {
            IO* out = static_cast<IO*>(p.out) + (long long)(tile + r) * p.ldo + d;
#pragma unroll
            for (int j = 0; j < k; ++j) {
              float v = fmaf(skip, uv[j], y[j]);
              if (z) { const float g = to_float(r_z[(r + j) * kCols + col]); v *= g * sigmoid(g); }
              if (d < p.D) out[j * p.ldo] = from_float<IO>(v);
            }
          }
          r += k;
        };
        while (r + 4 <= r_end) rows_of(std::integral_constant<int, 4>());
        while (r < r_end) rows_of(std::integral_constant<int, 1>());
      }
    }
    if constexpr (!kSummary && !kOne) {
      __syncthreads();
#pragma unroll 2
      for (int i = tid; i < rows * kCols; i += blockDim.x) {
        const int r = i / kCols, c = i % kCols;
        const long long row = tile + r;
        if (d0 + c >= p.D) continue;
        const bool real = row >= real0 && row < real1;
        if (!real && !p.zero_rest) continue;
        float y = 0.0f;
        if (real) {
          for (int k = 0; k < splits; ++k) y += s_y[(k * kTile + r) * kCols + c];
          if (p.skip) y = fmaf(p.skip[d0 + c], to_float(r_u[i]), y);
          if (z) { const float g = to_float(r_z[i]); y *= g * sigmoid(g); }
        }
        static_cast<IO*>(p.out)[row * p.ldo + d0 + c] = from_float<IO>(y);
      }
    }
  }
  if constexpr (kSummary) {
    store_states(p.seg_state + blockIdx.y * DN + at, left, vec, h);
    if (split == 0 && d < p.D) p.seg_dt[(long long)blockIdx.y * p.D + d] = dt_sum;
  } else {
    if (last) { stop = q.rows; enter(); }        // sequences without rows at the very end too
    else if (active && stop == t1) finish();
  }
}

// State behind each segment, in place of its last piece's summary.  The loads of sixteen pieces go out together: only the chain itself is
// serial.
__global__ void __launch_bounds__(128) scan_seams_kernel(const ScanPacked p) {
  constexpr int kBatch = 16;
  const long long DN = (long long)p.D * p.N, i = (long long)blockIdx.x * 128 + threadIdx.x;
  if (i >= DN) return;
  const long long d = i / p.N;
  const float a = p.A[i] * kLog2eF;
  const int count = (p.segments - 1) * p.pieces;
  float h = 0.0f;
  for (int g0 = 0; g0 < count; g0 += kBatch) {
    int kind[kBatch];
    float own[kBatch], sum[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int g = min(g0 + k, count - 1);
      kind[k] = p.seg_kind[g]; own[k] = p.seg_state[g * DN + i]; sum[k] = p.seg_dt[(long long)g * p.D + d];
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (g0 + k >= count || kind[k] == 0) continue;
      h = kind[k] == 1 ? own[k] : carried(h, a * sum[k], own[k]);
      if (((g0 + k + 1) & (p.pieces - 1)) == 0) p.seg_state[(g0 + k) * DN + i] = h;
    }
  }
}

constexpr int kStepRows = 512;     // most sequences of a CTA of the bulk kernel

struct ScanStep {
  const void *u, *dt, *B, *C, *z;
  const float *A, *skip, *bias;
  const int* slots;
  float* cache;                  // [entries, D, N], updated in place
  void* out;
  long long ldu, lddt, ldb, ldc, ldz, ldo, entries;
  int D, N, count, softplus, per;   // per: sequences of a thread
  int vec_a, vec_bc;                // A, and B and C, may be read four states at a time
};

// N elements at p as floats: 16 or 8 bytes at once (`vec`), or one by one.
template <typename T, int V>
__device__ __forceinline__ void get_states(const T* p, bool vec, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_float(p[0]);
  } else if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 q = *reinterpret_cast<const float4*>(p);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      v[0] = __uint_as_float(q.x << 16); v[1] = __uint_as_float(q.x & 0xffff0000u);
      v[2] = __uint_as_float(q.y << 16); v[3] = __uint_as_float(q.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_float(p[j]);
  }
}

// The same left as it was loaded, so that a load asked for early is not waited for before its values are needed.
template <typename T>
struct Raw4;
template <>
struct Raw4<float> {
  float v[4];
  __device__ __forceinline__ void load(const float* p, bool vec) { get_states<float, 4>(p, vec, v); }
  __device__ __forceinline__ void unpack(float (&o)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = v[j];
  }
};
template <>
struct Raw4<__nv_bfloat16> {
  uint32_t v[2];
  __device__ __forceinline__ void load(const __nv_bfloat16* p, bool vec) {
    if (vec) {
      const uint2 q = *reinterpret_cast<const uint2*>(p);
      v[0] = q.x; v[1] = q.y;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
      v[0] = h[0] | (uint32_t)h[1] << 16;
      v[1] = h[2] | (uint32_t)h[3] << 16;
    }
  }
  __device__ __forceinline__ void unpack(float (&o)[4]) const {
    o[0] = __uint_as_float(v[0] << 16); o[1] = __uint_as_float(v[0] & 0xffff0000u);
    o[2] = __uint_as_float(v[1] << 16); o[3] = __uint_as_float(v[1] & 0xffff0000u);
  }
};

// One token of each sequence, for state sizes that are no power of two.  The whole state is read and written once, 8 bytes
// a state, but a thread's few plain loads under way stay far from the HBM rate: 512 sequences x 4096 channels x 20 states
// (bf16) 314 us, 1.1 TB/s; x 1024 x 100 330 us, 1.3 TB/s.  LPC lanes share a channel and take V adjacent states each, kBlocks
// times over for larger states; a thread keeps its place in (channel, state) over `per` sequences, so that A is read once
// for them, kSeqs of them at a time.
template <typename IO, typename DT, int V, int LPC, int kBlocks>
__global__ void __launch_bounds__(256) scan_step_kernel(const ScanStep p) {
  constexpr int kSeqs = kBlocks == 1 ? 4 : 2;
  const int n0 = (threadIdx.x % LPC) * V;
  const long long d = ((long long)blockIdx.x * 256 + threadIdx.x) / LPC;
  if (d >= p.D) return;                          // a channel's lanes leave together
  const unsigned mask = __activemask();
  Sequences q{};
  q.slots = p.slots; q.entries = p.entries;
  const IO *u = static_cast<const IO*>(p.u), *Bm = static_cast<const IO*>(p.B), *Cm = static_cast<const IO*>(p.C), *z = static_cast<const IO*>(p.z);
  const DT* dt = static_cast<const DT*>(p.dt);
  const float skip = p.skip ? p.skip[d] : 0.0f, bias = p.bias ? p.bias[d] : 0.0f;
  float A[kBlocks][V];
#pragma unroll
  for (int k = 0; k < kBlocks; ++k) {
    const int n = n0 + k * LPC * V;
#pragma unroll
    for (int j = 0; j < V; ++j) A[k][j] = 0.0f;
    if (n < p.N) get_states<float, V>(p.A + d * p.N + n, p.vec_a, A[k]);
#pragma unroll
    for (int j = 0; j < V; ++j) A[k][j] *= kLog2eF;
  }
  const int b1 = min((int)((blockIdx.y + 1) * p.per), p.count);
  for (int b0 = blockIdx.y * p.per; b0 < b1; b0 += kSeqs) {
    long long entry[kSeqs];
    float h[kSeqs][kBlocks][V], Bv[kSeqs][kBlocks][V], Cv[kSeqs][kBlocks][V], x[kSeqs], uv[kSeqs], gate[kSeqs];
#pragma unroll
    for (int i = 0; i < kSeqs; ++i) entry[i] = b0 + i < b1 ? entry_of(q, b0 + i) : -1;
#pragma unroll
    for (int i = 0; i < kSeqs; ++i) {
      const long long b = b0 + i;
      const bool here = b < b1;
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
        const int n = n0 + k * LPC * V;
#pragma unroll
        for (int j = 0; j < V; ++j) h[i][k][j] = Bv[i][k][j] = Cv[i][k][j] = 0.0f;
        if (n >= p.N) continue;
        if (entry[i] >= 0) get_states<float, V>(p.cache + (entry[i] * p.D + d) * p.N + n, true, h[i][k]);
        if (here) {
          get_states<IO, V>(Bm + b * p.ldb + n, p.vec_bc, Bv[i][k]);
          get_states<IO, V>(Cm + b * p.ldc + n, p.vec_bc, Cv[i][k]);
        }
      }
      x[i] = uv[i] = gate[i] = 0.0f;
      if (here) {
        x[i] = to_float(dt[b * p.lddt + d]);
        uv[i] = to_float(u[b * p.ldu + d]);
        if (z) gate[i] = to_float(z[b * p.ldz + d]);
      }
    }
#pragma unroll
    for (int i = 0; i < kSeqs; ++i) {
      x[i] += bias;
      if (p.softplus) x[i] = softplus_f(x[i]);
      const float xu = x[i] * uv[i];
      float y = 0.0f;
#pragma unroll
      for (int k = 0; k < kBlocks; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          h[i][k][j] = fmaf(ex2f(x[i] * A[k][j]), h[i][k][j], xu * Bv[i][k][j]);
          y = fmaf(h[i][k][j], Cv[i][k][j], y);
        }
        const int n = n0 + k * LPC * V;
        if (entry[i] >= 0 && n < p.N) {
          float* to = p.cache + (entry[i] * p.D + d) * p.N + n;
          if constexpr (V == 4) *reinterpret_cast<float4*>(to) = make_float4(h[i][k][0], h[i][k][1], h[i][k][2], h[i][k][3]);
          else *to = h[i][k][0];
        }
      }
#pragma unroll
      for (int o = LPC / 2; o > 0; o >>= 1) y += __shfl_xor_sync(mask, y, o);
      if (threadIdx.x % LPC == 0 && b0 + i < b1) {
        y = fmaf(skip, uv[i], y);
        if (z) y *= gate[i] * sigmoid(gate[i]);
        static_cast<IO*>(p.out)[(b0 + i) * p.ldo + d] = from_float<IO>(y);
      }
    }
  }
}

// The same for many sequences, whose states are the traffic: a CTA has 1024 adjacent states of every entry it visits (4 KB:
// 64 channels of 16 states) and moves them with bulk copies, six entries ahead, in place through a ring in shared memory.
// 512 sequences x 4096 channels x 16 states (bf16): 55 us for the 285 MB of states and operands, 0.80 of the measured HBM
// rate, with one cache as with four in turn (537 MB: nothing left in the L2); plain loads, four entries a thread, leave too
// few bytes under way (176 us).  A single sequence takes 3.5 us either way, so that this kernel runs whenever the state size
// allows it.  LPC lanes share a channel (N = 4 LPC, or 256 with two pieces a lane).
constexpr int kRing = 8, kPiece = 1024;

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
}

template <typename IO, typename DT, int LPC, bool kWide>
__global__ void __launch_bounds__(128) scan_step_bulk_kernel(const ScanStep p) {
  __shared__ __align__(128) float ring[kRing][kPiece];
  __shared__ uint64_t full[kRing];
  __shared__ int s_slot[kStepRows];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long DN = (long long)p.D * p.N, at = (long long)blockIdx.x * kPiece;
  const int floats = (int)(DN - at < kPiece ? DN - at : kPiece);
  const int b0 = blockIdx.y * p.per, count = min(p.per, p.count - b0);
  Sequences q{};
  q.slots = p.slots; q.entries = p.entries;
  for (int i = tid; i < count; i += 128) s_slot[i] = (int)entry_of(q, b0 + i);
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncthreads();
  auto request = [&](int i) {                    // by thread 0
    uint64_t* bar = &full[i % kRing];
    if (s_slot[i] < 0) { mbar_arrive(bar); return; }
    mbar_expect_tx(bar, floats * 4);
    bulk_load(ring[i % kRing], p.cache + s_slot[i] * DN + at, floats * 4, bar);
  };
  if (tid == 0)
    for (int i = 0; i < min(count, kRing - 2); ++i) request(i);

  const IO *u = static_cast<const IO*>(p.u), *Bm = static_cast<const IO*>(p.B), *Cm = static_cast<const IO*>(p.C), *z = static_cast<const IO*>(p.z);
  const DT* dt = static_cast<const DT*>(p.dt);
  // piece k of a lane: four states of one channel; the second piece lies 128 states on, kStepD channels or in the same one
  constexpr int kStepD = kWide ? 0 : 32 / LPC, kStepN = kWide ? 128 : 0;
  const int off = (warp * 64 + lane) * 4;
  const bool here[2] = {off < floats, off + 128 < floats};
  const long long first = at + (here[0] ? off : 0), d = first / p.N;
  const int n = (int)(first - d * p.N);
  float A[2][4], skip[2], bias[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    get_states<float, 4>(p.A + first + (here[k] ? 128 * k : 0), p.vec_a, A[k]);
#pragma unroll
    for (int j = 0; j < 4; ++j) A[k][j] *= kLog2eF;
    const long long dk = d + (here[k] ? kStepD * k : 0);
    skip[k] = p.skip ? p.skip[dk] : 0.0f;
    bias[k] = p.bias ? p.bias[dk] : 0.0f;
  }
  constexpr int kBC = kWide ? 2 : 1, kScalars = kWide ? 1 : 2;     // pieces whose B and C, whose channel differ
  Raw4<IO> Bv[kBC], Cv[kBC];
  DT x[kScalars];
  IO uv[kScalars], gate[kScalars];
#pragma unroll
  for (int k = 0; k < kScalars; ++k) { x[k] = from_float<DT>(0.0f); uv[k] = gate[k] = from_float<IO>(0.0f); }
  // where the next sequence's operands lie: the pointers move on by a row each time
  const IO *pB = Bm + b0 * p.ldb + n, *pC = Cm + b0 * p.ldc + n, *pu = u + b0 * p.ldu + d, *pz = z ? z + b0 * p.ldz + d : nullptr;
  const DT* pt = dt + b0 * p.lddt + d;
  IO* out = static_cast<IO*>(p.out) + b0 * p.ldo + d;
  auto operands = [&]() {
#pragma unroll
    for (int k = 0; k < kBC; ++k) { Bv[k].load(pB + kStepN * k, p.vec_bc); Cv[k].load(pC + kStepN * k, p.vec_bc); }
#pragma unroll
    for (int k = 0; k < kScalars; ++k)
      if (here[k]) {
        x[k] = pt[kStepD * k];
        uv[k] = pu[kStepD * k];
        if (z) gate[k] = pz[kStepD * k];
      }
    pB += p.ldb; pC += p.ldc; pu += p.ldu; pt += p.lddt;
    if (z) pz += p.ldz;
  };
  operands();
  int i = 0;
  for (; i < count; ++i) {
    float* stage = ring[i % kRing];
    const bool kept = s_slot[i] >= 0;
    float step[kScalars], us[kScalars], gs[kScalars], bs[kBC][4], cs[kBC][4];
#pragma unroll
    for (int k = 0; k < kScalars; ++k) { step[k] = to_float(x[k]) + bias[k]; us[k] = to_float(uv[k]); gs[k] = to_float(gate[k]); }
#pragma unroll
    for (int k = 0; k < kBC; ++k) { Bv[k].unpack(bs[k]); Cv[k].unpack(cs[k]); }
    if (i + 1 < count) operands();               // the next sequence's, while this one's are used
    if (p.softplus)
#pragma unroll
      for (int k = 0; k < kScalars; ++k) step[k] = softplus_f(step[k]);
    const bool ok = mbar_wait(&full[i % kRing], (i / kRing) & 1);
    float y[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float4* at4 = reinterpret_cast<float4*>(stage + off + 128 * k);
      const float4 v = kept && here[k] ? *at4 : make_float4(0.f, 0.f, 0.f, 0.f);
      float h[4] = {v.x, v.y, v.z, v.w};
      const float s = step[kScalars == 1 ? 0 : k], xu = s * us[kScalars == 1 ? 0 : k];
      y[k] = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[j] = fmaf(ex2f(s * A[k][j]), h[j], xu * bs[kBC == 1 ? 0 : k][j]);
        y[k] = fmaf(h[j], cs[kBC == 1 ? 0 : k][j], y[k]);
      }
      if (kept && here[k] && ok) *at4 = make_float4(h[0], h[1], h[2], h[3]);
    }
    if (kWide) y[0] += y[1];
#pragma unroll
    for (int k = 0; k < kScalars; ++k) {
#pragma unroll
      for (int o = LPC / 2; o > 0; o >>= 1) y[k] += __shfl_xor_sync(0xffffffffu, y[k], o);
      if (lane % LPC == 0 && here[k] && ok) {
        float v = fmaf(skip[k], us[k], y[k]);
        if (z) v *= gs[k] * sigmoid(gs[k]);
        out[kStepD * k] = from_float<IO>(v);
      }
    }
    out += p.ldo;
    fence_proxy_async();                         // the states written above, before the copy that reads them
    if (__syncthreads_or(!ok)) break;            // a copy that never came: reported by the wait
    if (tid == 0) {
      if (kept) bulk_store(p.cache + s_slot[i] * DN + at, stage, floats * 4);
      bulk_commit_group();
      if (i + kRing - 2 < count) {               // the place of entry i - 2, whose copy out has been read by now
        asm volatile("cp.async.bulk.wait_group.read 2;" ::: "memory");
        request(i + kRing - 2);
      }
    }
  }
  if (tid == 0) {
    for (int j = i + 1; j < min(count, i + kRing - 2); ++j) mbar_wait(&full[j % kRing], (j / kRing) & 1);   // after a break only
    bulk_wait_all();
  }
}

static size_t scan_smem(const ScanShape& s, size_t io, size_t dt) {
  const size_t NP = s.splits * kStates;
  size_t bytes = 2 * kTile * (s.channels * (2 * io + dt) + 2 * NP * io);
  if (io == 2) bytes += 2 * kTile * NP * sizeof(float);
  if (s.groups != 4) bytes += kTile * s.channels * sizeof(float2) + s.splits * kTile * s.channels * sizeof(float);
  return bytes;
}

template <typename IO, typename DT>
static const void* scan_kernel_of(int groups) {
  return groups == 4 ? (const void*)scan_packed_kernel<IO, DT, 4, false>
                     : (groups == 2 ? (const void*)scan_packed_kernel<IO, DT, 2, false> : (const void*)scan_packed_kernel<IO, DT, 1, false>);
}
static ScanCut forward_cut(int64_t rows, int64_t D, int64_t N, int io, int dt) {
  const ScanShape s = scan_shape(D, N);
  const size_t ib = io == OSSM_B200_DTYPE_BF16 ? 2 : 4, db = dt == OSSM_B200_DTYPE_BF16 ? 2 : 4;
  const void* kernel = ib == 4 ? scan_kernel_of<float, float>(s.groups)
                               : (db == 4 ? scan_kernel_of<__nv_bfloat16, float>(s.groups) : scan_kernel_of<__nv_bfloat16, __nv_bfloat16>(s.groups));
  return scan_cut(rows, resident_ctas(kernel, s.threads, scan_smem(s, ib, db), 4), s.column_blocks, kTile, 256);
}
static size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

template <typename IO, typename DT, int kGroups>
static int launch_scan_g(const ScanPacked& p, const ScanShape& s, cudaStream_t stream) {
  const size_t bytes = scan_smem(s, sizeof(IO), sizeof(DT));
  if (int rc = ensure_dynamic_smem((const void*)scan_packed_kernel<IO, DT, kGroups, false>, bytes)) return rc;
  if (p.segments > 1) {
    if (int rc = ensure_dynamic_smem((const void*)scan_packed_kernel<IO, DT, kGroups, true>, bytes)) return rc;
    scan_packed_kernel<IO, DT, kGroups, true><<<dim3(s.column_blocks, (p.segments - 1) * p.pieces), s.threads, bytes, stream>>>(p, s.splits);
    scan_seams_kernel<<<(unsigned)(((long long)p.D * p.N + 127) / 128), 128, 0, stream>>>(p);
  }
  scan_packed_kernel<IO, DT, kGroups, false><<<dim3(s.column_blocks, p.segments), s.threads, bytes, stream>>>(p, s.splits);
  return check_cuda(cudaGetLastError(), "scan_packed_kernel launch");
}
template <typename IO, typename DT>
static int launch_scan(ScanPacked p, cudaStream_t stream) {
  const ScanShape s = scan_shape(p.D, p.N);
  p.by_u = piece_bytes(p.u, p.ldu, sizeof(IO)); p.by_z = piece_bytes(p.z, p.ldz, sizeof(IO));
  p.by_dt = piece_bytes(p.dt, p.lddt, sizeof(DT));
  p.by_b = piece_bytes(p.B, p.ldb, sizeof(IO)); p.by_c = piece_bytes(p.C, p.ldc, sizeof(IO));
  if (s.groups == 4) return launch_scan_g<IO, DT, 4>(p, s, stream);
  if (s.groups == 2) return launch_scan_g<IO, DT, 2>(p, s, stream);
  return launch_scan_g<IO, DT, 1>(p, s, stream);
}

template <typename IO, typename DT, int V, int LPC, int kBlocks>
static void launch_step_at(ScanStep p, cudaStream_t stream) {
  const long long blocks = ((long long)p.D * LPC + 255) / 256;
  // sequences of a thread: as many as leave every SM eight CTAs, up to 16
  long long per = blocks * p.count / ((long long)sm_count() * 8);
  p.per = (int)(per < 1 ? 1 : (per > 16 ? 16 : per));
  if ((p.count - 1) / 65535 + 1 > p.per) p.per = (p.count - 1) / 65535 + 1;   // the grid's limit
  scan_step_kernel<IO, DT, V, LPC, kBlocks><<<dim3((unsigned)blocks, (unsigned)((p.count + p.per - 1) / p.per)), 256, 0, stream>>>(p);
}

template <typename IO, typename DT, int LPC, bool kWide>
static void launch_step_bulk(ScanStep p, cudaStream_t stream) {
  const long long pieces = ((long long)p.D * p.N + kPiece - 1) / kPiece;
  const int held = resident_ctas((const void*)scan_step_bulk_kernel<IO, DT, LPC, kWide>, 128, 0, 6);
  long long y = held / pieces;                   // CTAs that run together, each with its share of the sequences
  if (y < 1) y = 1;
  long long per = (p.count + y - 1) / y;
  p.per = (int)(per > kStepRows ? kStepRows : per);
  scan_step_bulk_kernel<IO, DT, LPC, kWide><<<dim3((unsigned)pieces, (unsigned)((p.count + p.per - 1) / p.per)), 128, 0, stream>>>(p);
}

template <typename IO, typename DT>
static int launch_step(ScanStep p, cudaStream_t stream) {
  const uintptr_t bc = reinterpret_cast<uintptr_t>(p.B) | reinterpret_cast<uintptr_t>(p.C) | (uintptr_t)((p.ldb | p.ldc) * (long long)sizeof(IO));
  p.vec_a = (reinterpret_cast<uintptr_t>(p.A) & 15u) == 0;
  p.vec_bc = (bc & (4 * sizeof(IO) - 1)) == 0;
  const bool vec = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(p.cache) & 15u) == 0;
  if (vec && (p.N & (p.N - 1)) == 0 && p.entries < 0x7fffffff && p.count <= 65535 * 32) {
    switch (p.N) {
      case 4: launch_step_bulk<IO, DT, 1, false>(p, stream); break;
      case 8: launch_step_bulk<IO, DT, 2, false>(p, stream); break;
      case 16: launch_step_bulk<IO, DT, 4, false>(p, stream); break;
      case 32: launch_step_bulk<IO, DT, 8, false>(p, stream); break;
      case 64: launch_step_bulk<IO, DT, 16, false>(p, stream); break;
      case 128: launch_step_bulk<IO, DT, 32, false>(p, stream); break;
      default: launch_step_bulk<IO, DT, 32, true>(p, stream); break;   // 256
    }
  } else if (vec) {
    if (p.N <= 16) launch_step_at<IO, DT, 4, 4, 1>(p, stream);
    else if (p.N <= 32) launch_step_at<IO, DT, 4, 8, 1>(p, stream);
    else if (p.N <= 64) launch_step_at<IO, DT, 4, 16, 1>(p, stream);
    else if (p.N <= 128) launch_step_at<IO, DT, 4, 32, 1>(p, stream);
    else launch_step_at<IO, DT, 4, 32, 2>(p, stream);
  } else if (p.N <= 8) {
    launch_step_at<IO, DT, 1, 8, 1>(p, stream);
  } else if (p.N <= 64) {
    launch_step_at<IO, DT, 1, 32, 2>(p, stream);
  } else {
    launch_step_at<IO, DT, 1, 32, 8>(p, stream);
  }
  return check_cuda(cudaGetLastError(), "scan_step_kernel launch");
}

int check_scan(const char* fn, int64_t rows, int64_t D, int64_t N, int64_t count, int64_t entries, int io, int dt) {
  if (rows < 0 || D < 0 || count < 0 || entries < 0) { set_last_error("%s: negative extent", fn); return kErrInvalidArgument; }
  if (N < 1 || N > 256) { set_last_error("%s: state size must be 1..256", fn); return kErrUnsupported; }
  if (rows > 0x7ffffff0ll || count > 0x7ffffff0ll || D > (1 << 22)) { set_last_error("%s: too many rows, sequences or channels", fn); return kErrUnsupported; }
  if ((io != OSSM_B200_DTYPE_F32 && io != OSSM_B200_DTYPE_BF16) || (dt != io && dt != OSSM_B200_DTYPE_F32)) {
    set_last_error("%s: element types must be float32, or bfloat16 with bfloat16 or float32 steps", fn);
    return kErrInvalidArgument;
  }
  return kOk;
}

}  // namespace packed
}  // namespace ossm_b200

extern "C" {

using namespace ossm_b200;

// The backward keeps a window of rows in shared memory, 2.5 KB a row for every 16 states of a channel block.
int ossm_b200_selective_scan_packed_tile(int64_t N) { return N <= 128 ? 8 : 4; }

size_t ossm_b200_selective_scan_packed_workspace_bytes(int64_t rows, int64_t D, int64_t N, int io_dtype, int dt_dtype) {
  if (rows <= 0 || D <= 0 || N <= 0 || N > 256) return 0;
  const packed::ScanCut c = packed::forward_cut(rows, D, N, io_dtype, dt_dtype);
  if (c.segments == 1) return 0;
  const size_t g = c.segments, pieces = g * c.pieces;
  return packed::align256(pieces * D * N * 4) + packed::align256(g * D * N * 4) + packed::align256(pieces * D * 4) +
         packed::align256(pieces * 4);
}

int ossm_b200_selective_scan_packed_forward(const void* u, int64_t ldu, const void* dt, int64_t lddt, const float* A,
                                            const void* Bm, int64_t ldb, const void* Cm, int64_t ldc, const void* z,
                                            int64_t ldz, const float* Dskip, const float* delta_bias, int delta_softplus,
                                            const int* offsets, const int* slots, const void* resume, int resume_all,
                                            const float* start, float* end, int64_t entries, void* out, int64_t ldo,
                                            int zero_rest, float* kept, void* workspace, size_t workspace_bytes,
                                            int64_t rows, int64_t count, int64_t D, int64_t N, int io_dtype,
                                            int dt_dtype, ossm_b200_stream_t stream) {
  const char* fn = "selective_scan_packed_forward";
  if (int rc = packed::check_scan(fn, rows, D, N, count, entries, io_dtype, dt_dtype)) return rc;
  if (D == 0 || (rows == 0 && count == 0)) return kOk;
  if (!A || !offsets || (rows > 0 && (!u || !dt || !Bm || !Cm || !out))) { set_last_error("%s: null pointer", fn); return kErrInvalidArgument; }
  if (ldu < D || lddt < D || ldb < N || ldc < N || ldo < D || (z && ldz < D)) { set_last_error("%s: row pitch smaller than the row", fn); return kErrInvalidArgument; }
  if ((start || end) && !slots && entries < count) { set_last_error("%s: fewer entries than sequences, and no slots", fn); return kErrInvalidArgument; }
  packed::ScanPacked p{};
  p.q = {offsets, slots, static_cast<const unsigned char*>(resume), resume_all, (int)count, (int)rows, entries};
  p.u = u; p.dt = dt; p.B = Bm; p.C = Cm; p.z = z; p.A = A; p.skip = Dskip; p.bias = delta_bias;
  p.start = start; p.end = end; p.out = out; p.kept = kept;
  p.ldu = ldu; p.lddt = lddt; p.ldb = ldb; p.ldc = ldc; p.ldz = ldz; p.ldo = ldo;
  p.D = (int)D; p.N = (int)N; p.softplus = delta_softplus; p.zero_rest = zero_rest;
  p.keep = ossm_b200_selective_scan_packed_tile(N);
  p.vec = N % 4 == 0 && ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(start) | reinterpret_cast<uintptr_t>(end) |
                          reinterpret_cast<uintptr_t>(kept)) & 15u) == 0;
  const packed::ScanCut cut = packed::forward_cut(rows, D, N, io_dtype, dt_dtype);
  p.segments = cut.segments; p.segment_rows = cut.segment_rows; p.pieces = cut.pieces;
  if (p.segments > 1) {
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0 ||
        workspace_bytes < ossm_b200_selective_scan_packed_workspace_bytes(rows, D, N, io_dtype, dt_dtype)) {
      set_last_error("%s: workspace too small or not on a 16-byte boundary", fn);
      return kErrWorkspace;
    }
    const size_t pieces = (size_t)p.segments * p.pieces;
    char* w = static_cast<char*>(workspace);
    p.seg_state = reinterpret_cast<float*>(w); w += packed::align256(pieces * D * N * 4);
    p.seg_first = reinterpret_cast<float*>(w); w += packed::align256((size_t)p.segments * D * N * 4);
    p.seg_dt = reinterpret_cast<float*>(w); w += packed::align256(pieces * D * 4);
    p.seg_kind = reinterpret_cast<int*>(w);
  }
  if (io_dtype == OSSM_B200_DTYPE_F32) return packed::launch_scan<float, float>(p, stream);
  if (dt_dtype == OSSM_B200_DTYPE_F32) return packed::launch_scan<__nv_bfloat16, float>(p, stream);
  return packed::launch_scan<__nv_bfloat16, __nv_bfloat16>(p, stream);
}

int ossm_b200_selective_scan_step(const void* u, int64_t ldu, const void* dt, int64_t lddt, const float* A,
                                  const void* Bm, int64_t ldb, const void* Cm, int64_t ldc, const void* z, int64_t ldz,
                                  const float* Dskip, const float* delta_bias, int delta_softplus, const int* slots,
                                  float* cache, int64_t entries, void* out, int64_t ldo, int64_t count, int64_t D,
                                  int64_t N, int io_dtype, int dt_dtype, ossm_b200_stream_t stream) {
  const char* fn = "selective_scan_step";
  if (int rc = packed::check_scan(fn, 0, D, N, count, entries, io_dtype, dt_dtype)) return rc;
  if (D == 0 || count == 0) return kOk;
  if (!u || !dt || !A || !Bm || !Cm || !out || (!cache && entries > 0)) { set_last_error("%s: null pointer", fn); return kErrInvalidArgument; }
  if (ldu < D || lddt < D || ldb < N || ldc < N || ldo < D || (z && ldz < D)) { set_last_error("%s: row pitch smaller than the row", fn); return kErrInvalidArgument; }
  if (cache && !slots && entries < count) { set_last_error("%s: fewer entries than sequences, and no slots", fn); return kErrInvalidArgument; }
  packed::ScanStep p{};
  p.u = u; p.dt = dt; p.B = Bm; p.C = Cm; p.z = z; p.A = A; p.skip = Dskip; p.bias = delta_bias; p.slots = slots;
  p.cache = cache; p.out = out; p.entries = entries;
  p.ldu = ldu; p.lddt = lddt; p.ldb = ldb; p.ldc = ldc; p.ldz = ldz; p.ldo = ldo;
  p.D = (int)D; p.N = (int)N; p.count = (int)count; p.softplus = delta_softplus;
  if (io_dtype == OSSM_B200_DTYPE_F32) return packed::launch_step<float, float>(p, stream);
  if (dt_dtype == OSSM_B200_DTYPE_F32) return packed::launch_step<__nv_bfloat16, float>(p, stream);
  return packed::launch_step<__nv_bfloat16, __nv_bfloat16>(p, stream);
}

}  // extern "C"
