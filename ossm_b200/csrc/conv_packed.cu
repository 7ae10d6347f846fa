// Causal depthwise conv1d + bias + SiLU over a packed batch and over single tokens, with its gradients (sm_100a).
//
//   pre[t, d] = bias[d] + sum_k w[d, k] x[t - (K - 1) + k, d]        out = pre * sigmoid(pre)
//
// A tap that reaches before the first row of its sequence reads the sequence's window: the K - 1 inputs that came
// before it (zeros for a fresh sequence).  The window left behind a sequence is its last K - 1 inputs, its own window
// included.  HBM-bound: x is read and out written once (backward: x and grad read, grad_x written); everything else is
// small.  65536 rows x 4096 channels, 3 taps, bf16: forward 0.202 ms = 0.82 of the measured HBM rate, backward 0.367 ms =
// 0.68 at 51 % of the issue slots: 200 registers leave eight warps an SM, too few loads under way to reach either limit.
// The windows turn by their index instead of moving through registers, and two channels share an instruction.  Single
// tokens, 512 sequences x 4096 channels, 4 taps, bf16: 10.5 us where the bytes take 5 (every sequence's threads load the
// taps and the bias again); one sequence 2.5 us.
//
// Work is cut into runs of consecutive rows.  A thread takes V adjacent channels (16 bytes of them where bases, pitches
// and D allow) through one run and keeps the window in registers.  The run that holds the FIRST row of a sequence
// computes the sequence's first K - 1 rows even where they reach into the next run, and writes the window left behind
// it: so the cache entry of a sequence is read and written by one thread only, and a call may update it in place.
#include "packed.cuh"

#include <type_traits>
#include <utility>

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
  float* partial;                // [CTAs along the runs, K + 1, D]
  long long ldx, ldo, ldg;
  int D, run, runs;
  int vec_w;                     // the weights lie on 16 bytes
};

// The taps of V channels are V K adjacent elements: K vector loads where the weights lie on 16 bytes.
template <typename WT, int V, int K>
__device__ __forceinline__ void load_taps(const ConvPacked& p, int d, float (&w)[K][V], float (&bias)[V]) {
  const WT* wp = static_cast<const WT*>(p.w) + (long long)d * K;
  constexpr int kWide = V % (16 / (int)sizeof(WT)) == 0 ? 16 / (int)sizeof(WT) : V;
  if (V > 1 && p.vec_w) {
#pragma unroll
    for (int i = 0; i < V * K; i += kWide) {
      float v[kWide];
      Vec<WT, kWide>::load(wp + i, v);
#pragma unroll
      for (int j = 0; j < kWide; ++j)
        if (i + j < V * K) w[(i + j) % K][(i + j) / K] = v[j];
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][v] = to_float(wp[v * K + k]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = p.bias ? to_float(static_cast<const WT*>(p.bias)[d + v]) : 0.0f;
}

// c += a b over a thread's channels, two an instruction.
template <int V>
__device__ __forceinline__ void fma_v(const float (&a)[V], const float (&b)[V], float (&c)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      const float2 r = __ffma2_rn(make_float2(a[v], a[v + 1]), make_float2(b[v], b[v + 1]), make_float2(c[v], c[v + 1]));
      c[v] = r.x; c[v + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = fmaf(a[v], b[v], c[v]);
  }
}

template <typename IO, int V>
__device__ __forceinline__ void zero_rows(IO* out, long long ld, int from, int to) {
  const float zero[V] = {};
  for (int t = from; t < to; ++t) Vec<IO, V>::store(out + t * ld, zero);
}

template <int K, int V>
__device__ __forceinline__ void shift(float (&win)[K][V]) {
#pragma unroll
  for (int k = 0; k + 1 < K; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) win[k][v] = win[k + 1][v];
}
// f(0), f(1), ... with the index known when it is compiled
template <int kCount, typename F, int... kIndex>
__device__ __forceinline__ void turns_of(F&& f, std::integer_sequence<int, kIndex...>) {
  (f(std::integral_constant<int, kIndex>()), ...);
}
template <int kCount, typename F>
__device__ __forceinline__ void turns(F&& f) {
  turns_of<kCount>(f, std::make_integer_sequence<int, kCount>());
}

template <typename IO, typename WT, int V, int K>
__global__ void __launch_bounds__(128, 4) conv_packed_forward_kernel(const ConvPacked p) {
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
    float win[K][V];                             // the K - 1 inputs before a row, oldest first, and the row's own
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
    // row t, its input in win[(o + K - 1) % K]: the window turns with o instead of being moved
    auto step = [&](auto turn, int t) {
      constexpr int o = decltype(turn)::value;
      float y[V];
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = bias[v];
#pragma unroll
      for (int k = 0; k < K; ++k) fma_v<V>(w[k], win[(o + k) % K], y);
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] *= sigmoid(y[v]);
      Vec<IO, V>::store(out + t * p.ldo, y);
    };
    // kAhead rows at a time, a multiple of K, as many more on their way
    constexpr int kAhead = K == 3 ? 3 : 4;
    typename Vec<IO, V>::Raw next[kAhead];
    auto fetch = [&](int t) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (t + j < to) next[j] = Vec<IO, V>::fetch(x + (t + j) * p.ldx);
    };
    fetch(from);
    int t = from;
    for (; t + kAhead <= to; t += kAhead) {
      typename Vec<IO, V>::Raw now[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) now[j] = next[j];
      fetch(t + kAhead);
      turns<kAhead>([&](auto j) {
        constexpr int r = decltype(j)::value, o = r % K;
        Vec<IO, V>::unpack(now[r], win[(o + H) % K]);
        step(std::integral_constant<int, o>(), t + r);
      });
    }
#pragma unroll
    for (int j = 0; j + 1 < kAhead; ++j)
      if (t + j < to) {
        Vec<IO, V>::unpack(next[j], win[H]);
        step(std::integral_constant<int, 0>(), t + j);
        shift<K, V>(win);
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
__device__ __forceinline__ void conv_backward_run(const ConvPacked& p, int d, long long at, float (&dw)[K][V], float (&db)[V]) {
  constexpr int H = K - 1;
  const Sequences& q = p.q;
  const int r0 = (int)(at * p.run);
  const bool last = at == p.runs - 1;
  const int r1 = last ? q.rows : r0 + p.run;
  const IO* x = static_cast<const IO*>(p.x) + d;
  const IO* grad = static_cast<const IO*>(p.grad) + d;
  IO* gx = static_cast<IO*>(p.grad_x) + d;
  float w[K][V], bias[V];
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
    // row t: its input in win[(o + H) % K], the gradients of the K rows that it reads in acc[o % K] ...: both turn with o
    auto step = [&](auto turn, const float (&up)[V], int t) {
      constexpr int o = decltype(turn)::value;
      float a[V], g[V];
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = bias[v];
#pragma unroll
      for (int k = 0; k < K; ++k) fma_v<V>(w[k], win[(o + k) % K], a);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float sg = sigmoid(a[v]);
        g[v] = up[v] * sg * fmaf(a[v], 1.0f - sg, 1.0f);
      }
      if (t < r1) {
#pragma unroll
        for (int k = 0; k < K; ++k) fma_v<V>(g, win[(o + k) % K], dw[k]);
#pragma unroll
        for (int v = 0; v < V; ++v) db[v] += g[v];
      }
#pragma unroll
      for (int k = 0; k < K; ++k) fma_v<V>(w[k], g, acc[(o + k) % K]);
      emit(acc[o % K], t - H);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[o % K][v] = 0.0f;
    };
    // kAhead rows of both operands at a time, a multiple of K, as many more on their way
    constexpr int kAhead = K == 1 ? 2 : K;
    typename Vec<IO, V>::Raw next_x[kAhead], next_g[kAhead];
    auto fetch = [&](int t) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (t + j < to) {
          next_x[j] = Vec<IO, V>::fetch(x + (t + j) * p.ldx);
          next_g[j] = Vec<IO, V>::fetch(grad + (t + j) * p.ldg);
        }
    };
    fetch(from);
    int t = from;
    for (; t + kAhead <= to; t += kAhead) {
      typename Vec<IO, V>::Raw now_x[kAhead], now_g[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) { now_x[j] = next_x[j]; now_g[j] = next_g[j]; }
      fetch(t + kAhead);
      turns<kAhead>([&](auto j) {
        constexpr int r = decltype(j)::value, o = r % K;
        float up[V];
        Vec<IO, V>::unpack(now_x[r], win[(o + H) % K]);
        Vec<IO, V>::unpack(now_g[r], up);
        step(std::integral_constant<int, o>(), up, t + r);
      });
    }
#pragma unroll
    for (int j = 0; j + 1 < kAhead; ++j)
      if (t + j < to) {
        float up[V];
        Vec<IO, V>::unpack(next_x[j], win[H]);
        Vec<IO, V>::unpack(next_g[j], up);
        step(std::integral_constant<int, 0>(), up, t + j);
        shift<K, V>(win);
        float done[V];
#pragma unroll
        for (int v = 0; v < V; ++v) done[v] = acc[0][v];
        shift<K, V>(acc);
#pragma unroll
        for (int v = 0; v < V; ++v) acc[H][v] = done[v];
      }
    if (to == end) {
#pragma unroll
      for (int k = 0; k < H; ++k) emit(acc[k], end - H + k);
    }
    begin = end;
    ++s;
  }
  if (s == q.count) zero_rows<IO, V>(gx, p.D, max(r0, begin), r1);
}

template <typename IO, typename WT, int V, int K>
__global__ void __launch_bounds__(128, 2) conv_packed_backward_kernel(const ConvPacked p) {
  const int d = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  const long long at = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  float dw[K][V] = {}, db[V] = {};
  if (d < p.D && at < p.runs) conv_backward_run<IO, WT, V, K>(p, d, at, dw, db);
  // the runs of the CTA, in order
  __shared__ float sums[128][V];
  float* part = p.partial + (long long)blockIdx.x * (K + 1) * p.D + d;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    float a[V];
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = k < K ? dw[k < K ? k : 0][v] : db[v];
    if (blockDim.y > 1) {
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) sums[threadIdx.y * blockDim.x + threadIdx.x][v] = a[v];
      __syncthreads();
      if (threadIdx.y == 0)
        for (int y = 1; y < blockDim.y; ++y)
#pragma unroll
          for (int v = 0; v < V; ++v) a[v] += sums[y * blockDim.x + threadIdx.x][v];
    }
    if (threadIdx.y == 0 && d < p.D)
#pragma unroll
      for (int v = 0; v < V; ++v) part[(long long)k * p.D + v] = a[v];
  }
}

// grad_w[d, k] and grad_bias[d] from the runs' sums, in a fixed order: 32 threads share the runs of a channel, eight
// loads under way in each.
template <typename WT, int K>
__global__ void __launch_bounds__(1024) conv_packed_sums_kernel(const float* partial, int runs, int D, WT* grad_w, WT* grad_bias) {
  __shared__ float part[32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, d = blockIdx.x * 32 + lane, k = blockIdx.y;
  float a = 0.0f;
  if (d < D) {
#pragma unroll 8
    for (int r = row; r < runs; r += 32) a += partial[((long long)r * (K + 1) + k) * D + d];
  }
  part[row][lane] = a;
  __syncthreads();
  a = part[lane][row];                           // a warp has the 32 sums of channel `row`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  const int c = blockIdx.x * 32 + row;
  if (lane != 0 || c >= D) return;
  if (k < K) grad_w[(long long)c * K + k] = from_float<WT>(a);
  else if (grad_bias) grad_bias[c] = from_float<WT>(a);
}

enum class ConvPass { kForward, kStep, kBackward };

struct ConvShape {
  int vec;          // channels of a thread
  dim3 block;
  unsigned column_blocks;
};

static ConvShape conv_shape(int D, int wide, bool aligned) {
  ConvShape c;
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

static int launch_conv(ConvPacked p, int taps, int io, int wt, ConvPass pass, cudaStream_t stream, int* parts = nullptr) {
  const size_t element = io == OSSM_B200_DTYPE_BF16 ? 2 : 4;
  const bool aligned = aligned16(p.x) && aligned16(p.out) && aligned16(p.start) && aligned16(p.end) && aligned16(p.grad) &&
                       aligned16(p.grad_x) && aligned16(p.grad_end) && aligned16(p.grad_start) &&
                       p.ldx * element % 16 == 0 && p.ldo * element % 16 == 0 && p.ldg * element % 16 == 0;
  p.vec_w = aligned16(p.w);
  const ConvShape c = conv_shape(p.D, (int)(16 / element), aligned);
  if (parts) *parts = (int)((p.runs + c.block.y - 1) / c.block.y);
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
static void launch_sums(const ConvPacked& p, int parts, int taps, void* grad_w, void* grad_bias, cudaStream_t stream) {
  const dim3 grid((p.D + 31) / 32, taps + 1);
  WT* gw = static_cast<WT*>(grad_w);
  WT* gb = static_cast<WT*>(grad_bias);
  switch (taps) {
    case 1: conv_packed_sums_kernel<WT, 1><<<grid, 1024, 0, stream>>>(p.partial, parts, p.D, gw, gb); break;
    case 2: conv_packed_sums_kernel<WT, 2><<<grid, 1024, 0, stream>>>(p.partial, parts, p.D, gw, gb); break;
    case 3: conv_packed_sums_kernel<WT, 3><<<grid, 1024, 0, stream>>>(p.partial, parts, p.D, gw, gb); break;
    default: conv_packed_sums_kernel<WT, 4><<<grid, 1024, 0, stream>>>(p.partial, parts, p.D, gw, gb); break;
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
  if (taps > 1 && (start || end) && !slots && entries < count) { set_last_error("conv1d_silu_packed_forward: fewer entries than sequences, and no slots"); return kErrInvalidArgument; }
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
  if (taps > 1 && cache && !slots && entries < count) { set_last_error("conv1d_silu_step: fewer entries than sequences, and no slots"); return kErrInvalidArgument; }
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
  int parts = 0;
  if (int rc = packed::launch_conv(p, taps, io_dtype, weight_dtype, packed::ConvPass::kBackward, stream, &parts)) return rc;
  if (weight_dtype == OSSM_B200_DTYPE_F32) packed::launch_sums<float>(p, parts, taps, grad_weight, grad_bias, stream);
  else packed::launch_sums<__nv_bfloat16>(p, parts, taps, grad_weight, grad_bias, stream);
  return check_cuda(cudaGetLastError(), "conv_packed_sums_kernel launch");
}

}  // extern "C"
