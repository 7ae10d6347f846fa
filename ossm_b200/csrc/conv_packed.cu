// Causal depthwise conv1d + bias + SiLU over a packed batch and over single tokens, with its gradients (sm_100a).
//
//   pre[t, d] = bias[d] + sum_k w[d, k] x[t - (K - 1) + k, d]        out = pre * sigmoid(pre)
//
// A tap that reaches before the first row of its sequence reads the sequence's window: the K - 1 inputs that came
// before it (zeros for a fresh sequence).  The window left behind a sequence is its last K - 1 inputs, its own window
// included.  HBM-bound: x is read and out written once; everything else is small.
//
// Work is cut into runs of consecutive rows.  A thread takes V adjacent channels (16 bytes of them where bases, pitches
// and D allow) through one run and keeps the window in registers.  The run that holds the FIRST row of a sequence
// computes the sequence's first K - 1 rows even where they reach into the next run, and writes the window left behind
// it: so the cache entry of a sequence is read and written by one thread only, and a call may update it in place.
#include "packed.cuh"

#include "../../include/ossm_b200.h"

namespace ossm_b200 {
OSSM_B200_STATUS_ACCESSOR(status_packed_conv)
namespace packed {

struct ConvPacked {
  Sequences q;
  const void* x;                 // [rows, D], pitch ldx
  const void* w;                 // [D, K]
  const void* bias;              // [D] or null
  const void* start;             // [entries, K - 1, D] or null
  void* end;                     // [entries, K - 1, D] or null; may be `start`
  void* out;                     // [rows, D], pitch ldo
  int zero_rest;                 // rows outside every sequence become zero (else they are left as they are)
  // backward
  const void* grad;              // [rows, D], pitch ldg
  const void* grad_end;          // [count, K - 1, D] or null
  void* grad_x;                  // [rows, D], dense
  void* grad_start;              // [count, K - 1, D] or null
  float* partial;                // [runs, K + 1, D]
  long long ldx, ldo, ldg;
  int D, run, runs;
};

template <typename WT, int V, int K>
__device__ __forceinline__ void load_taps(const ConvPacked& p, int d, float (&w)[K][V], float (&bias)[V]) {
  const WT* wp = static_cast<const WT*>(p.w) + (long long)d * K;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][v] = to_float(wp[v * K + k]);
    bias[v] = p.bias ? to_float(static_cast<const WT*>(p.bias)[d + v]) : 0.0f;
  }
}

template <typename IO, int V>
__device__ __forceinline__ void zero_rows(IO* out, long long ld, int from, int to) {
  const float zero[V] = {};
  for (int t = from; t < to; ++t) Vec<IO, V>::store(out + t * ld, zero);
}

template <typename IO, typename WT, int V, int K>
__global__ void __launch_bounds__(128) conv_packed_forward_kernel(const ConvPacked p) {
  constexpr int H = K - 1;
  const int d = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  const long long at = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (d >= p.D || at >= p.runs) return;
  const Sequences& q = p.q;
  const int r0 = (int)(at * p.run);
  const bool last = at == p.runs - 1;
  const int r1 = last ? q.rows : r0 + p.run;
  const IO* x = static_cast<const IO*>(p.x) + d;
  IO* out = static_cast<IO*>(p.out) + d;
  float w[K][V], bias[V];
  load_taps<WT, V, K>(p, d, w, bias);

  int s = first_sequence(q, r0);
  int begin = s < q.count ? offset_at(q, s) : (q.count ? offset_at(q, q.count) : 0);
  if (p.zero_rest && s == 0) zero_rows<IO, V>(out, p.ldo, r0, min(begin, r1));
  while (s < q.count && (begin < r1 || last)) {
    const int end = end_of(q, s, begin);
    const bool first = begin >= r0;
    const long long entry = first ? entry_of(q, s) : -1;
    float win[H > 0 ? H : 1][V];
    int from, to;
    if (first) {
      from = begin;
      to = min(end, max(r1, begin + H));
      const bool cont = p.start != nullptr && entry >= 0 && resumes(q, s);
      const IO* st = static_cast<const IO*>(p.start) + entry * H * p.D + d;
#pragma unroll
      for (int k = 0; k < H; ++k) {
        if (cont) Vec<IO, V>::load(st + (long long)k * p.D, win[k]);
        else
#pragma unroll
          for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
      }
    } else {
      from = max(r0, begin + H);
      to = min(end, r1);
      if (from < to) {
#pragma unroll
        for (int k = 0; k < H; ++k) Vec<IO, V>::load(x + (from - H + k) * p.ldx, win[k]);
      }
    }
    auto step = [&](const float (&now)[V], int t) {
      float y[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a = bias[v];
#pragma unroll
        for (int k = 0; k < H; ++k) a = fmaf(w[k][v], win[k][v], a);
        a = fmaf(w[H][v], now[v], a);
        y[v] = a * sigmoid(a);
      }
      Vec<IO, V>::store(out + t * p.ldo, y);
#pragma unroll
      for (int k = 0; k + 1 < H; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) win[k][v] = win[k + 1][v];
      if (H > 0)
#pragma unroll
        for (int v = 0; v < V; ++v) win[H > 0 ? H - 1 : 0][v] = now[v];
    };
    int t = from;
    for (; t + 4 <= to; t += 4) {
      float now[4][V];
#pragma unroll
      for (int j = 0; j < 4; ++j) Vec<IO, V>::load(x + (t + j) * p.ldx, now[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) step(now[j], t + j);
    }
    for (; t < to; ++t) {
      float now[V];
      Vec<IO, V>::load(x + t * p.ldx, now);
      step(now, t);
    }
    if (H > 0 && first && entry >= 0 && p.end != nullptr) {
      IO* en = static_cast<IO*>(p.end) + entry * H * p.D + d;
      if (to < end) {   // at least K - 1 rows of its own lie before the end
#pragma unroll
        for (int k = 0; k < H; ++k) Vec<IO, V>::load(x + (end - H + k) * p.ldx, win[k]);
      }
#pragma unroll
      for (int k = 0; k < H; ++k) Vec<IO, V>::store(en + (long long)k * p.D, win[k]);
    }
    begin = end;
    ++s;
  }
  if (p.zero_rest && s == q.count) zero_rows<IO, V>(out, p.ldo, max(r0, begin), r1);
}

// One token of each sequence against its cached window, which moves on by it.
template <typename IO, typename WT, int V, int K>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvPacked p) {
  constexpr int H = K - 1;
  const int d = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  const long long b = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (d >= p.D || b >= p.q.count) return;
  const long long entry = entry_of(p.q, (int)b);
  float win[K][V], w[K][V], bias[V], y[V];
  IO* en = static_cast<IO*>(p.end) + entry * H * p.D + d;
#pragma unroll
  for (int k = 0; k < H; ++k) {
    if (entry >= 0) Vec<IO, V>::load(en + (long long)k * p.D, win[k]);
    else
#pragma unroll
      for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
  }
  Vec<IO, V>::load(static_cast<const IO*>(p.x) + b * p.ldx + d, win[H]);
  load_taps<WT, V, K>(p, d, w, bias);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float a = bias[v];
#pragma unroll
    for (int k = 0; k < K; ++k) a = fmaf(w[k][v], win[k][v], a);
    y[v] = a * sigmoid(a);
  }
  Vec<IO, V>::store(static_cast<IO*>(p.out) + b * p.ldo + d, y);
  if (entry >= 0) {
#pragma unroll
    for (int k = 0; k < H; ++k) Vec<IO, V>::store(en + (long long)k * p.D, win[k + 1]);
  }
}

// Gradients.  With g = grad * silu'(pre): grad_x[r] = sum_k w[k] g[r + K - 1 - k] over the rows of r's own sequence (a
// row before its beginning is one of its window), grad_w[k] = sum_t g[t] x[t - (K - 1) + k], grad_bias = sum_t g[t].  A
// run walks K - 1 rows past its end to finish its own rows; its sums for the parameters go to `partial`, which
// conv_packed_sums_kernel adds up in a fixed order.
template <typename IO, typename WT, int V, int K>
__global__ void __launch_bounds__(128) conv_packed_backward_kernel(const ConvPacked p) {
  constexpr int H = K - 1;
  const int d = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  const long long at = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (d >= p.D || at >= p.runs) return;
  const Sequences& q = p.q;
  const int r0 = (int)(at * p.run);
  const bool last = at == p.runs - 1;
  const int r1 = last ? q.rows : r0 + p.run;
  const IO* x = static_cast<const IO*>(p.x) + d;
  const IO* grad = static_cast<const IO*>(p.grad) + d;
  IO* gx = static_cast<IO*>(p.grad_x) + d;
  float w[K][V], bias[V], dw[K][V] = {}, db[V] = {};
  load_taps<WT, V, K>(p, d, w, bias);

  int s = first_sequence(q, r0);
  int begin = s < q.count ? offset_at(q, s) : (q.count ? offset_at(q, q.count) : 0);
  if (s == 0) zero_rows<IO, V>(gx, p.D, r0, min(begin, r1));
  while (s < q.count && (begin < r1 || last)) {
    const int end = end_of(q, s, begin);
    const bool first = begin >= r0;
    const IO* st = p.start ? static_cast<const IO*>(p.start) + (long long)s * H * p.D + d : nullptr;
    const IO* ge = p.grad_end ? static_cast<const IO*>(p.grad_end) + (long long)s * H * p.D + d : nullptr;
    IO* gs = p.grad_start ? static_cast<IO*>(p.grad_start) + (long long)s * H * p.D + d : nullptr;
    const int from = max(begin, r0), to = min(end, last ? end : r1 + H);
    float win[K][V], acc[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[k][v] = win[k][v] = 0.0f;
#pragma unroll
    for (int k = 0; k < H; ++k) {
      const int r = from - H + k;
      if (r >= begin) Vec<IO, V>::load(x + r * p.ldx, win[k]);
      else if (st) Vec<IO, V>::load(st + (long long)(r - begin + H) * p.D, win[k]);
    }
    // the gradient of row r (of the window where r < begin) is complete
    auto emit = [&](float (&g)[V], int r) {
      if (r >= r1 || r < (first ? begin - H : r0)) return;
      if (ge && r >= end - H) {
        float more[V];
        Vec<IO, V>::load(ge + (long long)(r - end + H) * p.D, more);
#pragma unroll
        for (int v = 0; v < V; ++v) g[v] += more[v];
      }
      if (r >= begin) Vec<IO, V>::store(gx + (long long)r * p.D, g);
      else if (gs) Vec<IO, V>::store(gs + (long long)(r - begin + H) * p.D, g);
    };
    for (int t = from; t < to; ++t) {
      float up[V];
      Vec<IO, V>::load(x + t * p.ldx, win[H]);
      Vec<IO, V>::load(grad + t * p.ldg, up);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a = bias[v];
#pragma unroll
        for (int k = 0; k < K; ++k) a = fmaf(w[k][v], win[k][v], a);
        const float sg = sigmoid(a);
        const float g = up[v] * sg * fmaf(a, 1.0f - sg, 1.0f);
        if (t < r1) {
#pragma unroll
          for (int k = 0; k < K; ++k) dw[k][v] = fmaf(g, win[k][v], dw[k][v]);
          db[v] += g;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) acc[k][v] = fmaf(w[k][v], g, acc[k][v]);
      }
      emit(acc[0], t - H);
#pragma unroll
      for (int k = 0; k < H; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          acc[k][v] = acc[k + 1][v];
          win[k][v] = win[k + 1][v];
        }
#pragma unroll
      for (int v = 0; v < V; ++v) acc[H][v] = 0.0f;
    }
    if (to == end) {
#pragma unroll
      for (int k = 0; k < H; ++k) emit(acc[k], end - H + k);
    }
    begin = end;
    ++s;
  }
  if (s == q.count) zero_rows<IO, V>(gx, p.D, max(r0, begin), r1);
  float* part = p.partial + at * (K + 1) * p.D + d;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) part[(long long)k * p.D + v] = dw[k][v];
    part[(long long)K * p.D + v] = db[v];
  }
}

// grad_w[d, k] and grad_bias[d] from the runs' sums, in a fixed order: 8 threads share the runs of a channel.
template <typename WT, int K>
__global__ void __launch_bounds__(256) conv_packed_sums_kernel(const float* partial, int runs, int D, WT* grad_w, WT* grad_bias) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, d = blockIdx.x * 32 + lane, k = blockIdx.y;
  float a = 0.0f;
  if (d < D)
    for (int r = row; r < runs; r += 8) a += partial[((long long)r * (K + 1) + k) * D + d];
  part[row][lane] = a;
  __syncthreads();
  if (row != 0 || d >= D) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) a += part[i][lane];
  if (k < K) grad_w[(long long)d * K + k] = from_float<WT>(a);
  else if (grad_bias) grad_bias[d] = from_float<WT>(a);
}

enum class ConvPass { kForward, kStep, kBackward };

struct ConvShape {
  int vec;          // channels of a thread
  dim3 block;
  unsigned column_blocks;
};

static ConvShape conv_shape(int D, size_t element, bool aligned) {
  ConvShape c;
  const int wide = (int)(16 / element);
  c.vec = aligned && D % wide == 0 ? wide : 1;
  const int threads = (D + c.vec - 1) / c.vec;
  int x = 1;
  while (x < threads && x < 128) x *= 2;
  c.block = dim3(x, 128 / x);
  c.column_blocks = (threads + x - 1) / x;
  return c;
}

template <typename IO, typename WT, int V, int K>
static void launch_conv_k(const ConvPacked& p, ConvPass pass, const ConvShape& c, cudaStream_t stream) {
  const long long units = pass == ConvPass::kStep ? p.q.count : p.runs;
  const dim3 grid((unsigned)((units + c.block.y - 1) / c.block.y), c.column_blocks);
  if (pass == ConvPass::kForward) conv_packed_forward_kernel<IO, WT, V, K><<<grid, c.block, 0, stream>>>(p);
  else if (pass == ConvPass::kStep) conv_step_kernel<IO, WT, V, K><<<grid, c.block, 0, stream>>>(p);
  else conv_packed_backward_kernel<IO, WT, V, K><<<grid, c.block, 0, stream>>>(p);
}

template <typename IO, typename WT, int V>
static void launch_conv_v(const ConvPacked& p, int taps, ConvPass pass, const ConvShape& c, cudaStream_t stream) {
  switch (taps) {
    case 1: return launch_conv_k<IO, WT, V, 1>(p, pass, c, stream);
    case 2: return launch_conv_k<IO, WT, V, 2>(p, pass, c, stream);
    case 3: return launch_conv_k<IO, WT, V, 3>(p, pass, c, stream);
    default: return launch_conv_k<IO, WT, V, 4>(p, pass, c, stream);
  }
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static int launch_conv(const ConvPacked& p, int taps, int io, int wt, ConvPass pass, cudaStream_t stream) {
  const size_t element = io == OSSM_B200_DTYPE_BF16 ? 2 : 4;
  const bool aligned = aligned16(p.x) && aligned16(p.out) && aligned16(p.start) && aligned16(p.end) && aligned16(p.grad) &&
                       aligned16(p.grad_x) && aligned16(p.grad_end) && aligned16(p.grad_start) &&
                       p.ldx * element % 16 == 0 && p.ldo * element % 16 == 0 && p.ldg * element % 16 == 0;
  const ConvShape c = conv_shape(p.D, element, aligned);
  if (io == OSSM_B200_DTYPE_F32) {
    if (c.vec == 1) launch_conv_v<float, float, 1>(p, taps, pass, c, stream);
    else launch_conv_v<float, float, 4>(p, taps, pass, c, stream);
  } else if (wt == OSSM_B200_DTYPE_F32) {
    if (c.vec == 1) launch_conv_v<__nv_bfloat16, float, 1>(p, taps, pass, c, stream);
    else launch_conv_v<__nv_bfloat16, float, 8>(p, taps, pass, c, stream);
  } else {
    if (c.vec == 1) launch_conv_v<__nv_bfloat16, __nv_bfloat16, 1>(p, taps, pass, c, stream);
    else launch_conv_v<__nv_bfloat16, __nv_bfloat16, 8>(p, taps, pass, c, stream);
  }
  return check_cuda(cudaGetLastError(), "packed conv launch");
}

template <typename WT>
static void launch_sums(const ConvPacked& p, int taps, void* grad_w, void* grad_bias, cudaStream_t stream) {
  const dim3 grid((p.D + 31) / 32, taps + 1);
  WT* gw = static_cast<WT*>(grad_w);
  WT* gb = static_cast<WT*>(grad_bias);
  switch (taps) {
    case 1: conv_packed_sums_kernel<WT, 1><<<grid, 256, 0, stream>>>(p.partial, p.runs, p.D, gw, gb); break;
    case 2: conv_packed_sums_kernel<WT, 2><<<grid, 256, 0, stream>>>(p.partial, p.runs, p.D, gw, gb); break;
    case 3: conv_packed_sums_kernel<WT, 3><<<grid, 256, 0, stream>>>(p.partial, p.runs, p.D, gw, gb); break;
    default: conv_packed_sums_kernel<WT, 4><<<grid, 256, 0, stream>>>(p.partial, p.runs, p.D, gw, gb); break;
  }
}

// Rows of a run.  Long runs re-read few rows at their seams and leave few partial sums; short ones fill the GPU.
static int run_rows(int64_t rows, int64_t D, size_t element) {
  const int64_t threads = D * (int64_t)element / 16 + 1;
  const int64_t want = rows * threads / ((int64_t)sm_count() * 1024) + 1;
  return (int)(want < 8 ? 8 : (want > 256 ? 256 : want));
}

static int check_conv(const char* fn, int64_t rows, int64_t D, int64_t count, int64_t entries, int taps, int io, int wt) {
  if (rows < 0 || D < 0 || count < 0 || entries < 0) { set_last_error("%s: negative extent", fn); return kErrInvalidArgument; }
  if (taps < 1 || taps > 4) { set_last_error("%s: kernel size must be 1..4", fn); return kErrUnsupported; }
  if (rows > 0x7ffffff0ll || count > 0x7ffffff0ll || D > (1 << 22)) { set_last_error("%s: too many rows, sequences or channels", fn); return kErrUnsupported; }
  if ((io != OSSM_B200_DTYPE_F32 && io != OSSM_B200_DTYPE_BF16) || (wt != io && wt != OSSM_B200_DTYPE_F32)) {
    set_last_error("%s: element types must be float32, or bfloat16 with bfloat16 or float32 weights", fn);
    return kErrInvalidArgument;
  }
  return kOk;
}

}  // namespace packed
}  // namespace ossm_b200

extern "C" {

using namespace ossm_b200;

int ossm_b200_conv1d_silu_packed_forward(const void* x, int64_t ldx, const void* weight, const void* bias,
                                         const int* offsets, const int* slots, const void* resume, int resume_all,
                                         const void* start, void* end, int64_t entries, void* out, int64_t ldo,
                                         int zero_rest, int64_t rows, int64_t count, int64_t D, int taps, int io_dtype,
                                         int weight_dtype, ossm_b200_stream_t stream) {
  if (int rc = packed::check_conv("conv1d_silu_packed_forward", rows, D, count, entries, taps, io_dtype, weight_dtype)) return rc;
  if (D == 0 || (rows == 0 && count == 0)) return kOk;
  if (!weight || !offsets || (rows > 0 && (!x || !out))) { set_last_error("conv1d_silu_packed_forward: null pointer"); return kErrInvalidArgument; }
  if (ldx < D || ldo < D) { set_last_error("conv1d_silu_packed_forward: row pitch smaller than the channel count"); return kErrInvalidArgument; }
  packed::ConvPacked p{};
  p.q = {offsets, slots, static_cast<const unsigned char*>(resume), resume_all, (int)count, (int)rows, entries};
  p.x = x; p.w = weight; p.bias = bias; p.start = start; p.end = end; p.out = out; p.zero_rest = zero_rest;
  p.ldx = ldx; p.ldo = ldo; p.D = (int)D;
  p.run = packed::run_rows(rows, D, io_dtype == OSSM_B200_DTYPE_BF16 ? 2 : 4);
  p.runs = rows ? (int)((rows + p.run - 1) / p.run) : 1;
  return packed::launch_conv(p, taps, io_dtype, weight_dtype, packed::ConvPass::kForward, stream);
}

int ossm_b200_conv1d_silu_step(const void* x, int64_t ldx, const void* weight, const void* bias, const int* slots,
                               void* cache, int64_t entries, void* out, int64_t ldo, int64_t count, int64_t D, int taps,
                               int io_dtype, int weight_dtype, ossm_b200_stream_t stream) {
  if (int rc = packed::check_conv("conv1d_silu_step", 0, D, count, entries, taps, io_dtype, weight_dtype)) return rc;
  if (D == 0 || count == 0) return kOk;
  if (!x || !weight || !out || (!cache && taps > 1 && entries > 0)) { set_last_error("conv1d_silu_step: null pointer"); return kErrInvalidArgument; }
  if (ldx < D || ldo < D) { set_last_error("conv1d_silu_step: row pitch smaller than the channel count"); return kErrInvalidArgument; }
  packed::ConvPacked p{};
  p.q.slots = slots; p.q.count = (int)count; p.q.entries = entries;
  p.x = x; p.w = weight; p.bias = bias; p.end = cache; p.out = out;
  p.ldx = ldx; p.ldo = ldo; p.D = (int)D;
  return packed::launch_conv(p, taps, io_dtype, weight_dtype, packed::ConvPass::kStep, stream);
}

size_t ossm_b200_conv1d_silu_packed_backward_workspace_bytes(int64_t rows, int64_t D, int taps, int io_dtype) {
  if (rows <= 0 || D <= 0 || taps < 1) return 0;
  const int64_t run = packed::run_rows(rows, D, io_dtype == OSSM_B200_DTYPE_BF16 ? 2 : 4);
  return (size_t)((rows + run - 1) / run * (taps + 1) * D) * sizeof(float);
}

int ossm_b200_conv1d_silu_packed_backward(const void* grad, int64_t ldg, const void* x, int64_t ldx, const void* weight,
                                          const void* bias, const int* offsets, const void* start, const void* grad_end,
                                          void* grad_x, void* grad_weight, void* grad_bias, void* grad_start,
                                          void* workspace, size_t workspace_bytes, int64_t rows, int64_t count,
                                          int64_t D, int taps, int io_dtype, int weight_dtype,
                                          ossm_b200_stream_t stream) {
  if (int rc = packed::check_conv("conv1d_silu_packed_backward", rows, D, count, count, taps, io_dtype, weight_dtype)) return rc;
  if (D == 0) return kOk;
  if (rows == 0) { set_last_error("conv1d_silu_packed_backward: no rows"); return kErrInvalidArgument; }
  if (!grad || !x || !weight || !offsets || !grad_x || !grad_weight) { set_last_error("conv1d_silu_packed_backward: null pointer"); return kErrInvalidArgument; }
  if (ldx < D || ldg < D) { set_last_error("conv1d_silu_packed_backward: row pitch smaller than the channel count"); return kErrInvalidArgument; }
  if (!workspace || workspace_bytes < ossm_b200_conv1d_silu_packed_backward_workspace_bytes(rows, D, taps, io_dtype)) {
    set_last_error("conv1d_silu_packed_backward: workspace too small");
    return kErrWorkspace;
  }
  packed::ConvPacked p{};
  p.q = {offsets, nullptr, nullptr, 1, (int)count, (int)rows, count};
  p.x = x; p.w = weight; p.bias = bias; p.start = start; p.grad = grad; p.grad_end = grad_end;
  p.grad_x = grad_x; p.grad_start = grad_start; p.partial = static_cast<float*>(workspace);
  p.ldx = ldx; p.ldg = ldg; p.D = (int)D;
  p.run = packed::run_rows(rows, D, io_dtype == OSSM_B200_DTYPE_BF16 ? 2 : 4);
  p.runs = (int)((rows + p.run - 1) / p.run);
  if (int rc = packed::launch_conv(p, taps, io_dtype, weight_dtype, packed::ConvPass::kBackward, stream)) return rc;
  if (weight_dtype == OSSM_B200_DTYPE_F32) packed::launch_sums<float>(p, taps, grad_weight, grad_bias, stream);
  else packed::launch_sums<__nv_bfloat16>(p, taps, grad_weight, grad_bias, stream);
  return check_cuda(cudaGetLastError(), "conv_packed_sums_kernel launch");
}

}  // extern "C"
