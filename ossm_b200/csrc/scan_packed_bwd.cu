// Mamba selective scan over a packed batch: gradients (sm_100a).
//
// With p_t = exp(dt_t A) h_{t-1} (so h_t = p_t + dt_t u_t B_t), dy = dout silu(z), and the adjoint of the state
//   g_t = C_t dy_t + exp(dt_{t+1} A) g_{t+1}            (the gradient of the state behind a sequence's last row)
// the gradients are sums of products:
//   dB_t = sum_d g_t dt_t u_t      dC_t = sum_d dy_t h_t        d(dt u)_t = sum_n g_t B_t      dA = sum_t dt_t g_t p_t
//   d(dt)_t = sum_n A g_t p_t + u_t d(dt u)_t                   du_t = dt_t d(dt u)_t + skip dy_t
//   dz_t = dout y_t silu'(z_t)     draw = d(dt) (1 - exp(-dt))  dskip = sum_t dy u              dbias = sum_t draw
#include "scan_packed.cuh"

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
  int column_blocks, window;
};

// Adjoint at the seams of the time segments, the mirror image of the forward's summary: the rows of each segment that
// belong to the sequence crossing its beginning, from the right, starting from zero or from that sequence's grad_end.
// seg_state[g] becomes the gradient of the state entering segment g.
template <typename IO, typename DT>
__global__ void __launch_bounds__(512, 2) scan_packed_adjoint_kernel(const ScanPackedGrad pg, int splits) {
  extern __shared__ __align__(16) float smem[];
  const ScanPacked& p = pg.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int groups = blockDim.x / 32 / splits, channels = 32 * groups;
  const int split = warp % splits, group = warp / splits;
  const int NP = splits * kStates;
  float2* s_dt = reinterpret_cast<float2*>(smem);                   // [kTile][channels] (dt, dy)
  float* s_c = smem + 2 * kTile * channels;                         // [kTile][NP]
  const Sequences& q = p.q;
  const int seg = blockIdx.y + 1;
  const int t0 = seg * p.segment_rows, t1 = seg == p.segments - 1 ? q.rows : t0 + p.segment_rows;
  const int d0 = blockIdx.x * channels, col = group * 32 + lane, d = d0 + col, n0 = split * kStates;
  const int left = d < p.D ? p.N - n0 : 0;
  const bool vec = p.vec != 0;
  const long long at = (long long)d * p.N + n0, DN = (long long)p.D * p.N;
  const IO *grad = static_cast<const IO*>(pg.grad), *Cm = static_cast<const IO*>(p.C), *z = static_cast<const IO*>(p.z);
  const DT* dt = static_cast<const DT*>(p.dt);

  const int s = first_sequence_warp(q, t0, lane);
  const int begin = s < q.count ? offset_at(q, s) : t0;
  const bool crosses = begin < t0;
  const int end = crosses ? end_of(q, s, begin) : t0;
  if (blockIdx.x == 0 && tid == 0) p.seg_kind[seg] = !crosses ? 0 : (end <= t1 ? 1 : 2);
  if (!crosses) return;
  float A[kStates], g[kStates];
  load_states(p.A + at, left, vec, A);
#pragma unroll
  for (int j = 0; j < kStates; ++j) { A[j] *= kLog2eF; g[j] = 0.0f; }
  if (end <= t1 && pg.grad_end) load_states(pg.grad_end + (long long)s * DN + at, left, vec, g);
  float dt_sum = 0.0f;
  int hi = min(end, t1);
  while (hi > t0) {
    const int lo = max(t0, hi - kTile), rows = hi - lo;
    for (int i = tid; i < rows * channels; i += blockDim.x) {
      const int r = i / channels, c = i - r * channels;
      float2 v = make_float2(0.f, 0.f);
      if (d0 + c < p.D) {
        const long long row = lo + r;
        float x = to_float(dt[row * p.lddt + d0 + c]);
        if (p.bias) x += p.bias[d0 + c];
        if (p.softplus) x = softplus_f(x);
        float dy = to_float(grad[row * pg.ldg + d0 + c]);
        if (z) { const float w = to_float(z[row * p.ldz + d0 + c]); dy *= w * sigmoid(w); }
        v = make_float2(x, dy);
      }
      s_dt[i] = v;
    }
    for (int i = tid; i < rows * NP; i += blockDim.x) {
      const int r = i / NP, n = i - r * NP;
      s_c[i] = n < p.N ? to_float(Cm[(long long)(lo + r) * p.ldc + n]) : 0.0f;
    }
    __syncthreads();
    for (int r = rows - 1; r >= 0; --r) {
      const float2 x = s_dt[r * channels + col];
      const float* c = s_c + r * NP + n0;
#pragma unroll
      for (int j = 0; j < kStates; j += 4) {
        const float4 cv = *reinterpret_cast<const float4*>(c + j);
        g[j] = ex2f(x.x * A[j]) * fmaf(cv.x, x.y, g[j]);
        g[j + 1] = ex2f(x.x * A[j + 1]) * fmaf(cv.y, x.y, g[j + 1]);
        g[j + 2] = ex2f(x.x * A[j + 2]) * fmaf(cv.z, x.y, g[j + 2]);
        g[j + 3] = ex2f(x.x * A[j + 3]) * fmaf(cv.w, x.y, g[j + 3]);
      }
      dt_sum += x.x;
    }
    __syncthreads();
    hi = lo;
  }
  store_states(p.seg_state + seg * DN + at, left, vec, g);
  if (split == 0 && d < p.D) p.seg_dt[(long long)seg * p.D + d] = dt_sum;
}

__global__ void __launch_bounds__(128) scan_adjoint_seams_kernel(const ScanPacked p) {
  const long long DN = (long long)p.D * p.N, i = (long long)blockIdx.x * 128 + threadIdx.x;
  if (i >= DN) return;
  const long long d = i / p.N;
  const float a = p.A[i] * kLog2eF;
  float g = 0.0f;
  for (int k = p.segments - 1; k > 0; --k) {
    const int kind = p.seg_kind[k];
    if (kind == 0) continue;
    const float own = p.seg_state[k * DN + i];
    g = kind == 1 ? own : fmaf(ex2f(a * p.seg_dt[(long long)k * p.D + d]), g, own);
    p.seg_state[k * DN + i] = g;
  }
}

// A lane holds 4 channels x 4 states: the sums over channels (dB, dC) and over states (y, d(dt u), d(dt)) are then
// mostly sums within a lane.  A warp is 8 lanes of channels x 4 lanes of states = 32 x 16 pairs.  The rows go right to
// left in windows of W: a forward walk from the kept state entering the window leaves p in shared memory, the backward
// walk reads it, evaluates the decay a second time and leaves the lanes' sums in the row that it has just read; then
// the CTA adds them up and finishes the rows.  Nothing is added by atomics: what CTAs share goes to partial sums.
constexpr int kRowFloats = 640;   // of a warp and row: p (512); after the row: 8 x 32 sums of dB | dC, then 4 x 3 x 32 of y | d(dt u) | d(dt)

template <typename IO, typename DT, int W>
__global__ void __launch_bounds__(512, 1) scan_packed_backward_kernel(const ScanPackedGrad pg, int splits) {
  extern __shared__ __align__(16) float smem[];
  const ScanPacked& p = pg.f;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int warps = blockDim.x / 32, groups = warps / splits, channels = 32 * groups;
  const int split = warp % splits, group = warp / splits;
  const int cg = lane >> 2, sg = lane & 3;
  const int NP = splits * kStates;
  float* s_rows = smem;                                             // [warps][W][kRowFloats]
  float* s_dt = s_rows + warps * W * kRowFloats;                    // [W][channels]
  float* s_dtu = s_dt + W * channels;                               // [W][channels]
  float* s_dy = s_dtu + W * channels;                               // [W][channels]
  float* s_b = s_dy + W * channels;                                 // [W][NP]
  float* s_c = s_b + W * NP;                                        // [W][NP]
  int* s_seq = reinterpret_cast<int*>(s_c + W * NP);                // [2][W] the sequence whose first / last row this is
  float* mine = s_rows + warp * W * kRowFloats;
  const Sequences& q = p.q;
  const int seg = blockIdx.y;
  const int t0 = seg * p.segment_rows, t1 = seg == p.segments - 1 ? q.rows : t0 + p.segment_rows;
  const int d0 = blockIdx.x * channels, n0 = split * kStates + 4 * sg, dw = d0 + group * 32 + 4 * cg;
  const long long DN = (long long)p.D * p.N;
  const IO *u = static_cast<const IO*>(p.u), *Bm = static_cast<const IO*>(p.B), *Cm = static_cast<const IO*>(p.C),
           *z = static_cast<const IO*>(p.z), *grad = static_cast<const IO*>(pg.grad);
  const DT* dt = static_cast<const DT*>(p.dt);
  const bool vec = p.vec != 0;

  float A[4][4], g[4][4], dA[4][4], h[4][4];
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
  load(p.A, A);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int n = 0; n < 4; ++n) { A[c][n] *= kLog2eF; g[c][n] = dA[c][n] = 0.0f; }

  const int real0 = q.count ? offset_at(q, 0) : 0, real1 = q.count ? max(real0, offset_at(q, q.count)) : 0;
  // the last sequence with a row before t1
  int s = first_sequence_warp(q, t1, lane);
  int begin = s < q.count ? offset_at(q, s) : q.rows, end = begin;
  if (s < q.count && begin < t1) {
    end = end_of(q, s, begin);                   // it goes on in the next segment
    if (seg + 1 < p.segments) load(p.seg_state + (seg + 1) * DN, g);
  } else {
    --s;
    if (s >= 0) { begin = offset_at(q, s); end = end_of(q, s, begin); }
  }
  const int my_c = tid % channels, my_d = d0 + my_c, my_r = tid / channels, row_step = blockDim.x / channels;
  const float skip = p.skip && my_d < p.D ? p.skip[my_d] : 0.0f;
  float sum_skip = 0.0f, sum_bias = 0.0f;

  for (int w0 = t0 + (t1 - t0 - 1) / W * W; w0 >= t0; w0 -= W) {
    const int rows = min(W, t1 - w0);
    // who begins and ends in the window (the same walk in every thread)
    unsigned firsts = 0, lasts = 0;
    int inside = s;                              // the sequence of the window's first row, once the walk is done
    if (tid < 2 * W) s_seq[tid] = -1;
    __syncthreads();                             // ... and the previous window is done with shared memory
    while (inside >= 0 && end > w0) {
      if (end > begin) {
        if (end <= w0 + rows) { lasts |= 1u << (end - 1 - w0); if (tid == 0) s_seq[W + end - 1 - w0] = inside; }
        if (begin >= w0 && begin < w0 + rows) { firsts |= 1u << (begin - w0); if (tid == 0) s_seq[begin - w0] = inside; }
      }
      if (begin < w0) break;                     // began before: the next window meets it again
      --inside;
      if (inside >= 0) {
        const int e = begin;
        begin = min(offset_at(q, inside), e);
        end = e;
      }
    }
    s = inside;
    for (int i = tid; i < W * channels; i += blockDim.x) {
      const int r = i / channels, c = i - r * channels;
      const long long row = w0 + r;
      float x = 0.0f, xu = 0.0f, dy = 0.0f;
      if (row < t1 && row >= real0 && row < real1 && d0 + c < p.D) {
        x = to_float(dt[row * p.lddt + d0 + c]);
        if (p.bias) x += p.bias[d0 + c];
        if (p.softplus) x = softplus_f(x);
        xu = x * to_float(u[row * p.ldu + d0 + c]);
        dy = to_float(grad[row * pg.ldg + d0 + c]);
        if (z) { const float w = to_float(z[row * p.ldz + d0 + c]); dy *= w * sigmoid(w); }
      }
      s_dt[i] = x; s_dtu[i] = xu; s_dy[i] = dy;
    }
    for (int i = tid; i < W * NP; i += blockDim.x) {
      const int r = i / NP, n = i - r * NP;
      const long long row = w0 + r;
      const bool ok = row < t1 && row >= real0 && row < real1 && n < p.N;
      s_b[i] = ok ? to_float(Bm[row * p.ldb + n]) : 0.0f;
      s_c[i] = ok ? to_float(Cm[row * p.ldc + n]) : 0.0f;
    }
    if (w0 >= real0 && w0 < real1) {
      load(p.kept + (long long)(w0 / W) * DN, h);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int n = 0; n < 4; ++n) h[c][n] = 0.0f;
    }
    __syncthreads();
    const int own = group * 32 + 4 * cg, st = split * kStates + 4 * sg;
    for (int r = 0; r < rows; ++r) {
      if (r > 0 && (firsts >> r & 1)) {          // at r = 0 the kept state is the sequence's own
        if (p.start) load(p.start + (long long)s_seq[r] * DN, h);
        else
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int n = 0; n < 4; ++n) h[c][n] = 0.0f;
      }
      const float4 x4 = *reinterpret_cast<const float4*>(s_dt + r * channels + own);
      const float4 xu4 = *reinterpret_cast<const float4*>(s_dtu + r * channels + own);
      const float4 b4 = *reinterpret_cast<const float4*>(s_b + r * NP + st);
      const float x[4] = {x4.x, x4.y, x4.z, x4.w}, xu[4] = {xu4.x, xu4.y, xu4.z, xu4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float4 v;
        v.x = ex2f(x[c] * A[c][0]) * h[c][0];
        v.y = ex2f(x[c] * A[c][1]) * h[c][1];
        v.z = ex2f(x[c] * A[c][2]) * h[c][2];
        v.w = ex2f(x[c] * A[c][3]) * h[c][3];
        *reinterpret_cast<float4*>(mine + r * kRowFloats + (c * 32 + lane) * 4) = v;
        h[c][0] = fmaf(xu[c], b[0], v.x); h[c][1] = fmaf(xu[c], b[1], v.y);
        h[c][2] = fmaf(xu[c], b[2], v.z); h[c][3] = fmaf(xu[c], b[3], v.w);
      }
    }
    for (int r = rows - 1; r >= 0; --r) {
      if (lasts >> r & 1) {
        if (pg.grad_end) load(pg.grad_end + (long long)s_seq[W + r] * DN, g);
        else
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int n = 0; n < 4; ++n) g[c][n] = 0.0f;
      }
      const float4 x4 = *reinterpret_cast<const float4*>(s_dt + r * channels + own);
      const float4 xu4 = *reinterpret_cast<const float4*>(s_dtu + r * channels + own);
      const float4 dy4 = *reinterpret_cast<const float4*>(s_dy + r * channels + own);
      const float4 b4 = *reinterpret_cast<const float4*>(s_b + r * NP + st);
      const float4 c4 = *reinterpret_cast<const float4*>(s_c + r * NP + st);
      const float x[4] = {x4.x, x4.y, x4.z, x4.w}, xu[4] = {xu4.x, xu4.y, xu4.z, xu4.w}, dy[4] = {dy4.x, dy4.y, dy4.z, dy4.w};
      const float b[4] = {b4.x, b4.y, b4.z, b4.w}, cc[4] = {c4.x, c4.y, c4.z, c4.w};
      float sb[4] = {}, sc[4] = {}, sy[4], s1[4], s2[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 v = *reinterpret_cast<const float4*>(mine + r * kRowFloats + (c * 32 + lane) * 4);
        const float pv[4] = {v.x, v.y, v.z, v.w};
        sy[c] = s1[c] = s2[c] = 0.0f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float hv = fmaf(xu[c], b[n], pv[n]);
          const float gv = fmaf(cc[n], dy[c], g[c][n]);
          sc[n] = fmaf(dy[c], hv, sc[n]);
          sb[n] = fmaf(xu[c], gv, sb[n]);
          sy[c] = fmaf(cc[n], hv, sy[c]);
          s1[c] = fmaf(b[n], gv, s1[c]);
          const float qv = gv * pv[n];
          s2[c] = fmaf(A[c][n], qv, s2[c]);
          dA[c][n] = fmaf(x[c], qv, dA[c][n]);
          g[c][n] = ex2f(x[c] * A[c][n]) * gv;
        }
      }
      __syncwarp();                              // the row's p has been read: its place takes the sums
      float* o = mine + r * kRowFloats;
      const int half = (cg & 1) << 4;            // odd lanes of channels swap dB and dC: no bank conflict
      *reinterpret_cast<float4*>(o + cg * 32 + (sg * 4 ^ half)) = make_float4(sb[0], sb[1], sb[2], sb[3]);
      *reinterpret_cast<float4*>(o + cg * 32 + ((16 + sg * 4) ^ half)) = make_float4(sc[0], sc[1], sc[2], sc[3]);
      o += 256 + sg * 96 + ((cg + 2 * sg) & 7) * 4;
      *reinterpret_cast<float4*>(o) = make_float4(sy[0], sy[1], sy[2], sy[3]);
      *reinterpret_cast<float4*>(o + 32) = make_float4(s1[0], s1[1], s1[2], s1[3]);
      *reinterpret_cast<float4*>(o + 64) = make_float4(s2[0], s2[1], s2[2], s2[3]);
      if ((firsts >> r & 1) && pg.dstart) store(pg.dstart + (long long)s_seq[r] * DN, g);
    }
    __syncthreads();
    // dB and dC of the window: over the channels of the CTA
    for (int i = tid; i < rows * splits * 32; i += blockDim.x) {
      const int v = i & 31, k = (i >> 5) % splits, r = (i >> 5) / splits;
      float a = 0.0f;
      for (int gr = 0; gr < groups; ++gr) {
        const float* o = s_rows + ((gr * splits + k) * W + r) * kRowFloats;
#pragma unroll
        for (int j = 0; j < 8; ++j) a += o[j * 32 + (v ^ ((j & 1) << 4))];
      }
      const int n = k * kStates + (v & 15);
      if (n < p.N) {
        const long long row = w0 + r;
        if (pg.column_blocks > 1)
          pg.part_bc[((long long)blockIdx.x * q.rows + row) * 2 * p.N + (v < 16 ? 0 : p.N) + n] = a;
        else
          static_cast<IO*>(v < 16 ? pg.dB : pg.dC)[row * p.N + n] = from_float<IO>(a);
      }
    }
    // the rows' own gradients: over the states
    for (int r = my_r; r < rows; r += row_step) {
      const long long row = w0 + r;
      if (my_d >= p.D) continue;
      float du = 0.0f, draw = 0.0f, dzv = 0.0f;
      if (row >= real0 && row < real1) {
        float y = 0.0f, s1 = 0.0f, s2 = 0.0f;
        const int c = my_c & 31;
        for (int k = 0; k < splits; ++k) {
          const float* o = s_rows + (((my_c >> 5) * splits + k) * W + r) * kRowFloats + 256;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float* e = o + j * 96 + (((c >> 2) + 2 * j) & 7) * 4 + (c & 3);
            y += e[0]; s1 += e[32]; s2 += e[64];
          }
        }
        const float x = s_dt[r * channels + my_c], dy = s_dy[r * channels + my_c];
        const float uv = to_float(u[row * p.ldu + my_d]);
        du = fmaf(s1, x, dy * skip);
        const float ddt = fmaf(s1, uv, s2 * 0.6931471805599453f);
        draw = p.softplus ? ddt * softplus_slope(x) : ddt;
        if (z) {
          const float w = to_float(z[row * p.ldz + my_d]), sig = sigmoid(w);
          dzv = to_float(grad[row * pg.ldg + my_d]) * fmaf(skip, uv, y) * sig * fmaf(w, 1.0f - sig, 1.0f);
        }
        sum_skip = fmaf(dy, uv, sum_skip);
        sum_bias += draw;
      }
      static_cast<IO*>(pg.du)[row * p.D + my_d] = from_float<IO>(du);
      static_cast<DT*>(pg.ddt)[row * p.D + my_d] = from_float<DT>(draw);
      if (pg.dz) static_cast<IO*>(pg.dz)[row * p.D + my_d] = from_float<IO>(dzv);
    }
  }
  store(pg.part_A + seg * DN, dA);
  __syncthreads();
  s_rows[tid] = sum_skip;
  s_rows[blockDim.x + tid] = sum_bias;
  __syncthreads();
  if (tid < channels && my_d < p.D) {
    for (int k = 1; k < row_step; ++k) { sum_skip += s_rows[k * channels + tid]; sum_bias += s_rows[blockDim.x + k * channels + tid]; }
    pg.part_d[((long long)seg * 2) * p.D + my_d] = sum_skip;
    pg.part_d[((long long)seg * 2 + 1) * p.D + my_d] = sum_bias;
  }
}

// dB, dC from the column blocks' sums, dA, dskip, dbias from the segments' sums, in a fixed order.
template <typename IO>
__global__ void __launch_bounds__(256) scan_backward_sums_kernel(const ScanPackedGrad pg) {
  const ScanPacked& p = pg.f;
  const long long DN = (long long)p.D * p.N, bc = pg.column_blocks > 1 ? (long long)p.q.rows * 2 * p.N : 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < bc + DN + 2ll * p.D; i += (long long)gridDim.x * 256) {
    float a = 0.0f;
    if (i < bc) {
      for (int k = 0; k < pg.column_blocks; ++k) a += pg.part_bc[k * bc + i];
      const long long row = i / (2 * p.N);
      const int n = (int)(i - row * 2 * p.N);
      static_cast<IO*>(n < p.N ? pg.dB : pg.dC)[row * p.N + (n < p.N ? n : n - p.N)] = from_float<IO>(a);
    } else if (i < bc + DN) {
      for (int k = 0; k < p.segments; ++k) a += pg.part_A[k * DN + i - bc];
      pg.dA[i - bc] = a;
    } else {
      const long long j = i - bc - DN;
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

static int backward_segments(int64_t rows, int64_t D, int64_t N) {
  const ScanShape s = scan_shape(D, N);
  const int64_t warps = (int64_t)s.column_blocks * s.threads / 32;
  int64_t g = ((int64_t)sm_count() * 8 + warps - 1) / warps;
  if (g > rows / 128) g = rows / 128;
  return (int)(g < 1 ? 1 : (g > 4096 ? 4096 : g));
}
static size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

struct BackwardPlan {
  int segments, segment_rows;
  size_t state, dts, kinds, part_A, part_d, part_bc, total;   // offsets into the workspace
};
static BackwardPlan backward_plan(int64_t rows, int64_t D, int64_t N) {
  BackwardPlan b{};
  b.segments = backward_segments(rows, D, N);
  b.segment_rows = (int)((rows + b.segments - 1) / b.segments + kTile - 1) / kTile * kTile;
  b.segments = (int)((rows + b.segment_rows - 1) / b.segment_rows);
  const ScanShape s = scan_shape(D, N);
  const size_t states = up256((size_t)b.segments * D * N * 4);
  b.dts = states;
  b.kinds = b.dts + up256((size_t)b.segments * D * 4);
  b.part_A = b.kinds + up256((size_t)b.segments * 4);
  b.part_d = b.part_A + states;
  b.part_bc = b.part_d + up256((size_t)b.segments * 2 * D * 4);
  b.total = b.part_bc + (s.column_blocks > 1 ? (size_t)s.column_blocks * rows * 2 * N * 4 : 0);
  return b;
}

template <typename IO, typename DT, int W>
static int launch_backward_w(const ScanPackedGrad& pg, const ScanShape& s, cudaStream_t stream) {
  const ScanPacked& p = pg.f;
  const int warps = s.threads / 32;
  const size_t bytes = ((size_t)warps * W * kRowFloats + 3 * W * s.channels + 2 * W * s.splits * kStates + 2 * W) * sizeof(float);
  if (int rc = ensure_dynamic_smem((const void*)scan_packed_backward_kernel<IO, DT, W>, bytes)) return rc;
  if (p.segments > 1) {
    const size_t small = (size_t)(2 * kTile * s.channels + kTile * s.splits * kStates) * sizeof(float);
    if (int rc = ensure_dynamic_smem((const void*)scan_packed_adjoint_kernel<IO, DT>, small)) return rc;
    scan_packed_adjoint_kernel<IO, DT><<<dim3(s.column_blocks, p.segments - 1), s.threads, small, stream>>>(pg, s.splits);
    scan_adjoint_seams_kernel<<<(unsigned)(((long long)p.D * p.N + 127) / 128), 128, 0, stream>>>(p);
  }
  if (pg.dstart && p.q.count) scan_empty_starts_kernel<<<p.q.count < 1024 ? p.q.count : 1024, 256, 0, stream>>>(pg);
  scan_packed_backward_kernel<IO, DT, W><<<dim3(s.column_blocks, p.segments), s.threads, bytes, stream>>>(pg, s.splits);
  const long long items = (pg.column_blocks > 1 ? (long long)p.q.rows * 2 * p.N : 0) + (long long)p.D * (p.N + 2);
  const long long blocks = (items + 255) / 256, most = (long long)sm_count() * 16;
  scan_backward_sums_kernel<IO><<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(pg);
  return check_cuda(cudaGetLastError(), "scan_packed_backward_kernel launch");
}

template <typename IO, typename DT>
static int launch_backward(const ScanPackedGrad& pg, cudaStream_t stream) {
  const ScanShape s = scan_shape(pg.f.D, pg.f.N);
  return pg.window == 8 ? launch_backward_w<IO, DT, 8>(pg, s, stream) : launch_backward_w<IO, DT, 4>(pg, s, stream);
}

}  // namespace packed
}  // namespace ossm_b200

extern "C" {

using namespace ossm_b200;

size_t ossm_b200_selective_scan_packed_backward_workspace_bytes(int64_t rows, int64_t D, int64_t N) {
  if (rows <= 0 || D <= 0 || N <= 0) return 0;
  return packed::backward_plan(rows, D, N).total;
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
      workspace_bytes < ossm_b200_selective_scan_packed_backward_workspace_bytes(rows, D, N)) {
    set_last_error("%s: workspace too small or not on a 16-byte boundary", fn);
    return kErrWorkspace;
  }
  const packed::BackwardPlan b = packed::backward_plan(rows, D, N);
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
  p.segments = b.segments; p.segment_rows = b.segment_rows;
  p.seg_state = reinterpret_cast<float*>(w);
  p.seg_dt = reinterpret_cast<float*>(w + b.dts);
  p.seg_kind = reinterpret_cast<int*>(w + b.kinds);
  pg.grad = dout; pg.grad_end = grad_end; pg.ldg = ldg;
  pg.du = du; pg.ddt = ddt; pg.dB = dB; pg.dC = dC; pg.dz = z ? dz : nullptr;
  pg.dA = dA; pg.dskip = dD; pg.dbias = ddelta_bias; pg.dstart = grad_start;
  pg.part_A = reinterpret_cast<float*>(w + b.part_A);
  pg.part_d = reinterpret_cast<float*>(w + b.part_d);
  pg.part_bc = reinterpret_cast<float*>(w + b.part_bc);
  pg.column_blocks = (int)packed::scan_shape(D, N).column_blocks;
  pg.window = ossm_b200_selective_scan_packed_tile(N);
  if (io_dtype == OSSM_B200_DTYPE_F32) return packed::launch_backward<float, float>(pg, stream);
  if (dt_dtype == OSSM_B200_DTYPE_F32) return packed::launch_backward<__nv_bfloat16, float>(pg, stream);
  return packed::launch_backward<__nv_bfloat16, __nv_bfloat16>(pg, stream);
}

}  // extern "C"
