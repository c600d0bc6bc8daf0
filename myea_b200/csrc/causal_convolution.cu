// Short causal convolution over time, one filter per channel, forward and backward:
//   a[t] = bias + sum_j w[j] x[t - W + 1 + j],   y = a sigmoid(a)  or  a
//   da = dy sigmoid(a) (1 + a (1 - sigmoid(a))),   dx[p] = sum_j w[j] da[p + W - 1 - j],   dw[j] = sum_t da[t] x[t - W + 1 + j]
// Bound by memory: a handful of multiply-adds per element.  A thread takes four channels (8 or 16 bytes) over a run of
// positions and keeps the last W inputs, and backward the W errors that are not complete yet, in registers, so each element is
// read from memory once; the W - 1 positions that neighbouring runs share come out of L2.  What holds it back is the number of warps
// that fit beside such registers: a thread's loads, arithmetic and stores take turns, and few others fill in.  4 x 2048 x 4096 bf16
// with 4 taps take 40 us forward (3.4 TB/s) and 73 us backward (2.8 TB/s), in fp32 58 and 128 (4.7 and 3.1 TB/s; backward
// 64 words of a thread go through local memory).
// Measured with shorter runs: two blocks per SM instead of three 52 us for 48, backward one instead of two 122 us for 81.  Loads
// eight positions ahead instead of four 38 us, but 4.4 us in place of 3.7 for single positions of 64 sequences.
#include <math.h>

#include "sequence.cuh"

namespace myea {
namespace {

struct ConvArgs {
  myea_convolution c;
  int batch, time, width;
  int vectors;     // groups of four channels
  int run, runs;   // positions of a run (at least 8, more than the taps before it reach back), runs of a sequence
  bool vec_x, vec_y, vec_dy, vec_dx, vec_state, vec_final, vec_d_final, vec_d_state, vec_w;
  float *partial;  // backward: [batch * blocks of runs][taps + 1][width]
};

// four channels as two pairs
struct Quad {
  float2 v[2];
};
__device__ __forceinline__ Quad quad(float4 x) { return {{lo(x), hi(x)}}; }
__device__ __forceinline__ float4 whole(const Quad &q) { return make_float4(q.v[0].x, q.v[0].y, q.v[1].x, q.v[1].y); }

template <int W>
__device__ __forceinline__ void load_filter(const ConvArgs &s, int ch, int n, Quad (&w)[W], Quad &bias) {
  const float *src = s.c.weight + static_cast<long long>(ch) * W;
  float flat[4 * W];
  if (s.vec_w && n == 4) {
#pragma unroll
    for (int i = 0; i < W; ++i) *reinterpret_cast<float4 *>(flat + 4 * i) = __ldg(reinterpret_cast<const float4 *>(src) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 4 * W; ++i) flat[i] = i < n * W ? src[i] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < W; ++j) w[j] = quad(make_float4(flat[j], flat[W + j], flat[2 * W + j], flat[3 * W + j]));
  bias = quad(parameters4(s.c.bias == nullptr ? nullptr : s.c.bias + ch, n));
}

// input of one position before the run, from x or, before the first one, from the state
template <typename T, int W>
__device__ __forceinline__ Raw4<T> input_before(const ConvArgs &s, long long b, int t, int ch, int n) {
  if (t >= 0) return load4(static_cast<const T *>(s.c.x.data) + b * s.c.x.stride_batch + t * s.c.x.stride_time + ch, n, s.vec_x);
  if (s.c.state == nullptr) return zero4<T>();
  return load4(static_cast<const T *>(s.c.state) + (b * (W - 1) + (W - 1 + t)) * s.width + ch, n, s.vec_state);
}

template <typename T, int W>
__global__ void __launch_bounds__(256, W <= 4 ? 3 : 1) convolution_forward_kernel(const ConvArgs s) {
  const long long id = blockIdx.x * 256ll + threadIdx.x;
  const int v = static_cast<int>(id % s.vectors);
  const long long row = id / s.vectors;
  const int r = static_cast<int>(row % s.runs);
  const long long b = row / s.runs;
  if (b >= s.batch) return;
  const int ch = v * 4, n = min(4, s.width - ch);
  const int length = sequence_length(s.c.lengths, b, s.time);
  const int t0 = r * s.run, t1 = min(t0 + s.run, s.time), live = min(t1, length);
  Quad w[W], bias;
  load_filter<W>(s, ch, n, w, bias);
  Quad win[W];   // the last W inputs, the newest at W - 1
#pragma unroll
  for (int k = 0; k < W - 1; ++k)
    win[k + 1] = quad(t0 < live || r == 0 ? widen(input_before<T, W>(s, b, t0 - (W - 1) + k, ch, n)) : make_float4(0.f, 0.f, 0.f, 0.f));
  const T *x = static_cast<const T *>(s.c.x.data) + b * s.c.x.stride_batch + ch;
  T *y_at = static_cast<T *>(s.c.y.data) + b * s.c.y.stride_batch + t0 * s.c.y.stride_time + ch;
  constexpr int U = 4;   // positions whose loads are under way while the ones before are computed
  Raw4<T> ahead[U];
  const auto load = [&](int t) {
    const T *at = x + t * s.c.x.stride_time;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ahead[u] = t + u < live ? load4(at, n, s.vec_x) : zero4<T>();
      at += s.c.x.stride_time;
    }
  };
  load(t0);
  for (int t = t0; t < t1; t += U) {
    Raw4<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = ahead[u];
    load(t + U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < W - 1; ++k) win[k] = win[k + 1];
      win[W - 1] = quad(widen(raw[u]));
      if (t + u < t1) {
        Quad y;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float2 a = bias.v[i], sig;
#pragma unroll
          for (int j = 0; j < W; ++j) a = fma2(w[j].v[i], win[j].v[i], a);
          y.v[i] = s.c.silu ? gate2(a, sig) : a;
          if (t + u >= live) y.v[i] = both(0.f);
        }
        store4(y_at, whole(y), n, s.vec_y);
        y_at += s.c.y.stride_time;
      }
    }
  }
  // The first run's thread is the only one that reads the state (a run is longer than W - 1), so it may write it in place:
  // entry k comes from entry length + k or from an input.
  if (r == 0 && s.c.final_state != nullptr) {
    T *f = static_cast<T *>(s.c.final_state) + b * (W - 1) * s.width + ch;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      const float4 e = widen(input_before<T, W>(s, b, length - (W - 1) + k, ch, n));
      store4(f + static_cast<long long>(k) * s.width, e, n, s.vec_final);
    }
  }
}

// 32 groups of four channels x 8 runs per block
template <typename T, int W>
__global__ void __launch_bounds__(256, W <= 4 ? 2 : 1) convolution_backward_kernel(const ConvArgs s, int tiles, int run_blocks) {
  __shared__ float4 join[8][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int tile = blockIdx.x % tiles;
  const long long rest = blockIdx.x / tiles;
  const int rb = static_cast<int>(rest % run_blocks), r = rb * 8 + strand;
  const long long b = rest / run_blocks;
  const int ch = (tile * 32 + lane) * 4, n = min(4, s.width - ch);
  Quad dw[W + 1];   // the last one: of the bias
#pragma unroll
  for (int j = 0; j <= W; ++j) dw[j].v[0] = dw[j].v[1] = both(0.f);
  if (r < s.runs && n > 0) {
    const int length = sequence_length(s.c.lengths, b, s.time);
    const int t0 = r * s.run, t1 = min(t0 + s.run, s.time);
    Quad w[W], bias, win[W], open[W];   // open[j]: error of position t - W + 1 + j, not complete before step t
    load_filter<W>(s, ch, n, w, bias);
#pragma unroll
    for (int k = 0; k < W - 1; ++k)
      win[k + 1] = quad(t0 < length || r == 0 ? widen(input_before<T, W>(s, b, t0 - (W - 1) + k, ch, n)) : make_float4(0.f, 0.f, 0.f, 0.f));
#pragma unroll
    for (int j = 0; j < W; ++j) open[j].v[0] = open[j].v[1] = both(0.f);
    const T *x = static_cast<const T *>(s.c.x.data) + b * s.c.x.stride_batch + ch;
    const T *dy = static_cast<const T *>(s.c.dy.data) + b * s.c.dy.stride_batch + ch;
    T *dx = static_cast<T *>(s.c.dx.data);
    const int end = t1 + W - 1;   // the errors of the run's last positions need the W - 1 steps behind it
    constexpr int U = 4;
    Raw4<T> ahead_x[U], ahead_dy[U];
    const int reach = min(length, end);
    const auto load = [&](int t) {
      const T *at_x = x + t * s.c.x.stride_time, *at_dy = dy + t * s.c.dy.stride_time;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ahead_x[u] = t + u < reach ? load4(at_x, n, s.vec_x) : zero4<T>();
        ahead_dy[u] = t + u < reach ? load4(at_dy, n, s.vec_dy) : zero4<T>();
        at_x += s.c.x.stride_time;
        at_dy += s.c.dy.stride_time;
      }
    };
    load(t0);
    for (int t = t0; t < end; t += U) {
      Raw4<T> raw_x[U], raw_dy[U];
#pragma unroll
      for (int u = 0; u < U; ++u) { raw_x[u] = ahead_x[u]; raw_dy[u] = ahead_dy[u]; }
      load(t + U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Quad e = quad(widen(raw_dy[u]));
#pragma unroll
        for (int k = 0; k < W - 1; ++k) { win[k] = win[k + 1]; open[k] = open[k + 1]; }
        win[W - 1] = quad(widen(raw_x[u]));
        open[W - 1].v[0] = open[W - 1].v[1] = both(0.f);
        const bool in = t + u < reach, own = in && t + u < t1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float2 da = e.v[i];
          if (s.c.silu) {   // sigmoid(a) (1 + a (1 - sigmoid(a)))
            float2 a = bias.v[i], sg;
#pragma unroll
            for (int j = 0; j < W; ++j) a = fma2(w[j].v[i], win[j].v[i], a);
            const float2 y = gate2(a, sg);
            da = mul2(da, add2(sg, fma2(y, make_float2(-sg.x, -sg.y), y)));
          }
          if (!in) da = both(0.f);
#pragma unroll
          for (int j = 0; j < W; ++j) open[j].v[i] = fma2(w[j].v[i], da, open[j].v[i]);
          if (own) {
#pragma unroll
            for (int j = 0; j < W; ++j) dw[j].v[i] = fma2(da, win[j].v[i], dw[j].v[i]);
            dw[W].v[i] = add2(dw[W].v[i], da);
          }
        }
        const int p = t + u - (W - 1);   // complete now
        if (t + u < end && (p >= t0 || r == 0)) {
          float4 d = whole(open[0]);
          const int k = p - length + W - 1;   // entry of the final state that this position is
          if (k >= 0 && k < W - 1 && s.c.d_final_state != nullptr) {
            const float4 f = widen(load4(static_cast<const T *>(s.c.d_final_state) + (b * (W - 1) + k) * s.width + ch, n, s.vec_d_final));
            d.x += f.x; d.y += f.y; d.z += f.z; d.w += f.w;
          }
          if (p >= 0) {
            if (dx != nullptr) store4(dx + b * s.c.dx.stride_batch + p * s.c.dx.stride_time + ch, d, n, s.vec_dx);
          } else if (s.c.d_state != nullptr) {
            store4(static_cast<T *>(s.c.d_state) + (b * (W - 1) + (W - 1 + p)) * s.width + ch, d, n, s.vec_d_state);
          }
        }
      }
    }
  }
  if (s.partial == nullptr) return;
  float *part = s.partial + (b * run_blocks + rb) * (W + 1) * static_cast<long long>(s.width);
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    join[strand][lane] = whole(dw[j]);
    __syncthreads();
    const int c = tile * 128 + threadIdx.x;   // 128 threads sum one channel each
    if (threadIdx.x < 128 && c < s.width) {
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += reinterpret_cast<const float *>(&join[k][threadIdx.x >> 2])[threadIdx.x & 3];
      part[j * static_cast<long long>(s.width) + c] = sum;
    }
    __syncthreads();
  }
}

struct StoreFilter {   // column j * width + c of the partial sums
  float *dw, *db;
  long long width;
  int taps, accumulate;
  __device__ void operator()(long long column, float sum) const {
    const long long j = column / width, c = column - j * width;
    float *to = j < taps ? (dw == nullptr ? nullptr : dw + c * taps + j) : (db == nullptr ? nullptr : db + c);
    if (to != nullptr) *to = accumulate ? *to + sum : sum;
  }
};

__global__ void __launch_bounds__(256) convolution_finish_kernel(const float *part, long long rows, long long columns, StoreFilter store) {
  sum_partials_block(part, rows, columns, blockIdx.x, store);
}

// A run's positions: the launch takes as long as its waves of blocks, each as long as a run, the positions that a run reads twice and
// what a thread does once (together some 8 positions).  4 x 2048 x 4096: 80 forward and 128 backward, one wave each.  (Above four taps one
// block per SM is reckoned with; forward, up to six taps and with 16-bit types seven, two fit.)
int run_length(const myea_convolution *c, bool backward) {
  const int64_t resident = kSms * (c->taps > 4 ? 1 : backward ? 2 : 3), batch = static_cast<int64_t>(c->batch), time = static_cast<int64_t>(c->time);
  const int64_t groups = (static_cast<int64_t>(c->width) + 3) / 4;
  int best = 8;
  double least = 1e300;
  for (int run = 8; run <= 128; run += 4) {
    const int64_t runs = (time + run - 1) / run;
    const double blocks = backward ? static_cast<double>((groups + 31) / 32) * ((runs + 7) / 8) * batch : static_cast<double>(groups) * runs * batch / 256;
    const double cost = ceil(blocks / resident) * (run + 8);
    if (cost < least) {
      least = cost;
      best = run;
    }
  }
  return best;
}

const char *check(const myea_convolution *c, bool backward) {
  if (c == nullptr) return "causal_convolution: no description";
  if (c->type > MYEA_TYPE_F16) return "causal_convolution: unknown type";
  if (c->taps < 1 || c->taps > 8) return "causal_convolution: 1 to 8 taps";
  if (c->batch > kSequenceMost || c->time > kSequenceMost || c->width > kSequenceMost) return "causal_convolution: a dimension above 2^30";
  if (c->batch == 0 || c->width == 0) return nullptr;
  if (c->weight == nullptr) return "causal_convolution: no weights";
  if (c->time > 0 && c->x.data == nullptr) return "causal_convolution: no input";
  if (!backward) {
    if (c->time > 0 && c->y.data == nullptr) return "causal_convolution: no output";
    if (c->time > 0 && c->x.data == c->y.data) return "causal_convolution: the output may not be the input's array";
  } else {
    if (c->time > 0 && c->dy.data == nullptr) return "causal_convolution: no error on the outputs";
    if (c->time > 0 && c->dx.data != nullptr && (c->dx.data == c->dy.data || c->dx.data == c->x.data))
      return "causal_convolution: the error on the inputs may not be another operand's array";
    if (c->d_state != nullptr && c->d_state == c->d_final_state) return "causal_convolution: d_state may not be d_final_state";
  }
  return nullptr;
}

ConvArgs arguments(const myea_convolution *c, bool backward) {
  ConvArgs s = {};
  s.c = *c;
  s.batch = static_cast<int>(c->batch); s.time = static_cast<int>(c->time); s.width = static_cast<int>(c->width);
  s.vectors = (s.width + 3) / 4;
  s.run = run_length(c, backward);
  s.runs = s.time > 0 ? (s.time + s.run - 1) / s.run : 1;
  const size_t bytes = 4 * type_bytes(c->type);
  const bool even = c->width % 4 == 0;
  s.vec_x = view_takes_vectors(c->x, c->type); s.vec_y = view_takes_vectors(c->y, c->type);
  s.vec_dy = view_takes_vectors(c->dy, c->type); s.vec_dx = view_takes_vectors(c->dx, c->type);
  s.vec_state = even && aligned(c->state, bytes); s.vec_final = even && aligned(c->final_state, bytes);
  s.vec_d_final = even && aligned(c->d_final_state, bytes); s.vec_d_state = even && aligned(c->d_state, bytes);
  s.vec_w = aligned(c->weight, 16);
  return s;
}

int run_blocks_of(const ConvArgs &s) { return (s.runs + 7) / 8; }

template <typename T, int W> void launch_forward(const ConvArgs &s, long long blocks, cudaStream_t stream) {
  convolution_forward_kernel<T, W><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(s);
}
template <typename T, int W> void launch_backward(const ConvArgs &s, long long blocks, int tiles, int run_blocks, cudaStream_t stream) {
  convolution_backward_kernel<T, W><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(s, tiles, run_blocks);
}

template <typename F> void with_taps(uint32_t taps, F f) {
  switch (taps) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 3: f(std::integral_constant<int, 3>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 5: f(std::integral_constant<int, 5>()); break;
    case 6: f(std::integral_constant<int, 6>()); break;
    case 7: f(std::integral_constant<int, 7>()); break;
    default: f(std::integral_constant<int, 8>()); break;
  }
}

}  // namespace
}  // namespace myea

extern "C" int myea_b200_causal_convolution(int device, const myea_convolution *c, void *stream, char *error_message, size_t error_capacity) {
  using namespace myea;
  if (const char *why = check(c, false)) return refuse(error_message, error_capacity, MYEA_E_INVALID, why);
  if (c->batch == 0 || c->width == 0) return MYEA_OK;
  const ConvArgs s = arguments(c, false);
  const long long blocks = (static_cast<long long>(s.vectors) * s.runs * s.batch + 255) / 256;
  if (s.vectors > (1ll << 62) / (static_cast<long long>(s.runs) * s.batch) || blocks > 0x7fffffffll)
    return refuse(error_message, error_capacity, MYEA_E_INVALID, "causal_convolution: more positions than one launch takes");
  DeviceScope scope(device);
  if (!scope.ok) return refuse(error_message, error_capacity, MYEA_E_CUDA, "causal_convolution: no such device");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  with_type(c->type, [&](auto t) { with_taps(c->taps, [&](auto w) { launch_forward<decltype(t), decltype(w)::value>(s, blocks, st); }); });
  return launched(error_message, error_capacity, "causal_convolution");
}

extern "C" size_t myea_b200_causal_convolution_backward_workspace(const myea_convolution *c) {
  using namespace myea;
  if (check(c, true) != nullptr || c->batch == 0 || c->width == 0 || (c->d_weight == nullptr && c->d_bias == nullptr)) return 0;
  const ConvArgs s = arguments(c, true);
  return round_up_256(c->batch * run_blocks_of(s) * (c->taps + 1) * c->width * sizeof(float));
}

extern "C" int myea_b200_causal_convolution_backward(int device, const myea_convolution *c, void *workspace, size_t workspace_bytes, void *stream,
                                                     char *error_message, size_t error_capacity) {
  using namespace myea;
  if (const char *why = check(c, true)) return refuse(error_message, error_capacity, MYEA_E_INVALID, why);
  if (c->width == 0) return MYEA_OK;
  const size_t need = myea_b200_causal_convolution_backward_workspace(c);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 256)))
    return refuse(error_message, error_capacity, MYEA_E_INVALID, "causal_convolution: the workspace is missing, too small or not 256-byte aligned");
  ConvArgs s = arguments(c, true);
  s.partial = need > 0 ? static_cast<float *>(workspace) : nullptr;
  const int tiles = (s.vectors + 31) / 32, run_blocks = run_blocks_of(s);
  const double blocks_wide = static_cast<double>(tiles) * run_blocks * s.batch;
  if (blocks_wide > 2147483647.0) return refuse(error_message, error_capacity, MYEA_E_INVALID, "causal_convolution: more positions than one launch takes");
  DeviceScope scope(device);
  if (!scope.ok) return refuse(error_message, error_capacity, MYEA_E_CUDA, "causal_convolution: no such device");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long blocks = static_cast<long long>(blocks_wide);
  if (blocks > 0)
    with_type(c->type, [&](auto t) { with_taps(c->taps, [&](auto w) { launch_backward<decltype(t), decltype(w)::value>(s, blocks, tiles, run_blocks, st); }); });
  if (c->d_weight != nullptr || c->d_bias != nullptr) {
    const long long columns = static_cast<long long>(c->taps + 1) * s.width;
    convolution_finish_kernel<<<static_cast<unsigned>((columns + 31) / 32), 256, 0, st>>>(
        s.partial, blocks > 0 ? static_cast<long long>(s.batch) * run_blocks : 0, columns,
        StoreFilter{c->d_weight, c->d_bias, s.width, static_cast<int>(c->taps), static_cast<int>(c->accumulate)});
  }
  return launched(error_message, error_capacity, "causal_convolution_backward");
}
