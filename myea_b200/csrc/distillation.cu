// Error of a row of logits against a teacher's best ones, with its gradient (the formulas stand at myea_distillation in
// myea_b200.h).  With x the row, m its maximum, c = 1 / temperature:
//   q_i = e^(c (x_i - m)) / s,  r_i = e^(x_i - m) / s1,   soft term = soft T^2 sum_k p_k (log p_k - c (x_k - m) + log s)
//   gradient = soft T (q_i - sum of the p of word i) + hard (r_i - [i = label])
//
// Bound by memory: the row is read once from memory for m, s and s1 (in one pass: a sum is scaled whenever its maximum rises)
// and a second time, out of L2, when the gradient is written.  A block, or a cluster of blocks where the rows alone leave SMs
// idle, takes a row; the cluster's parts of the sums are exchanged through shared memory and joined in rank order.  The
// teacher's few words are mended at the end: their gradients are formed again from the logits with the teacher's part, so every
// element is rounded once.
#include <cooperative_groups.h>

#include "sequence.cuh"

namespace myea {
namespace {

namespace cg = cooperative_groups;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTopMost = 1024;

template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); uint4 v; };
template <typename T> __device__ __forceinline__ void unpack(const Pack<T> &p, float (&x)[Pack<T>::N]) {
  const T *e = reinterpret_cast<const T *>(&p.v);
#pragma unroll
  for (int i = 0; i < Pack<T>::N; ++i) x[i] = to_float(e[i]);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Maximum and sums of exponentials of what has been seen
struct Running {
  float m = -INFINITY, s = 0.f, s1 = 0.f;   // s at the temperature, s1 at 1 (only where both are asked for)
  __device__ __forceinline__ void rise(float to, float c, bool two) {   // to >= m
    const float by = to == -INFINITY ? 0.f : m - to;
    s *= exp2_fast(by * c);
    if (two) s1 *= exp2_fast(by * kLog2e);
    m = to;
  }
  __device__ __forceinline__ void join(const Running &o, float c, bool two) {
    Running r = o;
    const float to = fmaxf(m, r.m);
    rise(to, c, two);
    r.rise(to, c, two);
    s += r.s;
    s1 += r.s1;
  }
};

template <typename T, bool TWO>
__global__ void __launch_bounds__(512) distillation_kernel(const myea_distillation d) {
  constexpr int E = Pack<T>::N;
  extern __shared__ float dynamic[];
  int *s_index = reinterpret_cast<int *>(dynamic);
  float *s_p = dynamic + d.top, *s_x = s_p + d.top;   // the teacher's probabilities, the logits of its words
  __shared__ Running s_warp[16], s_part;
  __shared__ float s_sum[17];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const long long V = static_cast<long long>(d.vocabulary);
  const int K = static_cast<int>(d.top);
  const T *x = static_cast<const T *>(d.logits) + row * d.logits_stride;
  T *out = d.d_logits == nullptr ? nullptr : static_cast<T *>(d.d_logits) + row * d.d_logits_stride;
  // the row from its first 16-byte boundary on in packs, the blocks' shares of them, the elements before and behind
  long long head = static_cast<long long>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T));
  head = head < V ? head : V;
  const long long packs = (V - head) / E, first = packs * part / parts, last = packs * (part + 1) / parts;
  const long long from = part == 0 ? 0 : head + first * E, to = part == parts - 1 ? V : head + last * E;   // this block's elements
  const Pack<T> *body = reinterpret_cast<const Pack<T> *>(x + head);
  const bool out_packs = out != nullptr && aligned_16(out + head);
  const float w = d.weight == nullptr ? 1.f : d.weight[row];
  if (w == 0.f) {   // (every block of the row's cluster)
    if (out != nullptr)
      for (long long i = from + tid; i < to; i += threads) out[i] = from_float<T>(0.f);
    if (part == 0 && tid == 0) d.losses[row] = 0.f;
    return;
  }
  const float c = kLog2e / d.temperature;

  // the teacher's words and their logits
  float t_max = -INFINITY;
  for (int k = tid; k < K; k += threads) {
    const int i = d.index[row * d.index_stride + k];
    const bool there = i >= 0 && i < V;
    const float t = there ? d.teacher[row * d.teacher_stride + k] : -INFINITY;
    s_index[k] = there ? i : -1;
    s_p[k] = t;
    s_x[k] = there ? to_float(x[i]) : 0.f;
    t_max = fmaxf(t_max, t);
  }
  const int label = d.labels == nullptr || d.hard == 0.f ? -1 : d.labels[row];
  const bool labelled = label >= 0 && label < V;
  const float x_label = labelled ? to_float(x[label]) : 0.f;
  t_max = block_max(t_max, s_sum);
  float t_sum = 0.f;
  for (int k = tid; k < K; k += threads) {
    const float e = s_index[k] >= 0 && s_p[k] != -INFINITY ? exp2_fast((s_p[k] - t_max) * c) : 0.f;   // (NaN stays NaN)
    s_p[k] = e;
    t_sum += e;
  }
  t_sum = block_sum(t_sum, s_sum);
  const bool taught = t_sum != 0.f;
  const float t_scale = taught ? 1.f / t_sum : 0.f;
  for (int k = tid; k < K; k += threads) s_p[k] *= t_scale;

  // one pass for the maximum and the sums
  Running run;
  const auto take = [&](const float *e, int n) {
    float m = run.m;
    for (int i = 0; i < n; ++i) m = fmaxf(m, e[i]);
    if (m > run.m) run.rise(m, c, TWO);
    const float base = run.m == -INFINITY ? 0.f : run.m;
    for (int i = 0; i < n; ++i) {
      run.s += exp2_fast((e[i] - base) * c);
      if (TWO) run.s1 += exp2_fast((e[i] - base) * kLog2e);
    }
  };
  if (part == 0)
    for (long long i = tid; i < head; i += threads) {
      const float e[1] = {to_float(x[i])};
      take(e, 1);
    }
  constexpr int U = 4;
  for (long long i = first + tid; i < last; i += U * threads) {
    Pack<T> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * threads < last) p[u] = body[i + u * threads];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * threads < last) {
        float e[E];
        unpack(p[u], e);
        take(e, E);
      }
  }
  if (part == parts - 1)
    for (long long i = head + packs * E + tid; i < V; i += threads) {
      const float e[1] = {to_float(x[i])};
      take(e, 1);
    }
  // lanes, warps, blocks of the cluster: every block ends with the same sums
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) {
    Running o;
    o.m = __shfl_xor_sync(0xffffffffu, run.m, m);
    o.s = __shfl_xor_sync(0xffffffffu, run.s, m);
    o.s1 = __shfl_xor_sync(0xffffffffu, run.s1, m);
    run.join(o, c, TWO);
  }
  if (lane == 0) s_warp[warp] = run;
  __syncthreads();
  run = s_warp[0];
  for (int k = 1; k < warps; ++k) run.join(s_warp[k], c, TWO);
  if (parts > 1) {
    if (tid == 0) s_part = run;
    cluster.sync();
    run = *cluster.map_shared_rank(&s_part, 0);
    for (int k = 1; k < parts; ++k) run.join(*cluster.map_shared_rank(&s_part, k), c, TWO);
    cluster.sync();   // nobody leaves, or writes over the logits, while others read
  }
  const float unit = TWO ? run.s1 : run.s;
  if (run.s == 0.f) {   // no open word
    if (out != nullptr)
      for (long long i = from + tid; i < to; i += threads) out[i] = from_float<T>(0.f);
    if (part == 0 && tid == 0) d.losses[row] = 0.f;
    return;
  }

  if (part == 0) {
    float kl = 0.f;
    const float log_s = logf(run.s), T_ = d.temperature;
    for (int k = tid; k < K; k += threads) {
      const float p = s_p[k];
      if (p != 0.f) kl += p * (logf(p) - (s_x[k] - run.m) / T_ + log_s);
    }
    kl = block_sum(kl, s_sum);
    if (tid == 0) {
      float loss = taught ? d.soft * T_ * T_ * kl : 0.f;
      if (labelled) loss += d.hard * (logf(unit) - (x_label - run.m));
      d.losses[row] = w * loss;
    }
  }
  if (out == nullptr) return;

  // without a second temperature both terms have the same exponentials
  const float soft = taught ? w * d.soft * d.temperature : 0.f, hard = labelled ? w * d.hard : 0.f;
  const float a = TWO ? soft / run.s : (soft + hard) / run.s, b = TWO ? hard / run.s1 : 0.f;
  const float base = run.m;
  const auto gradient = [&](float e) {
    float g = a * exp2_fast((e - base) * c);
    if (TWO) g += b * exp2_fast((e - base) * kLog2e);
    return g;
  };
  if (part == 0)
    for (long long i = tid; i < head; i += threads) out[i] = from_float<T>(gradient(to_float(x[i])));
  for (long long i = first + tid; i < last; i += U * threads) {
    Pack<T> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * threads < last) p[u] = body[i + u * threads];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * threads < last) {
        float e[E];
        unpack(p[u], e);
        Pack<T> g;
        T *ge = reinterpret_cast<T *>(&g.v);
#pragma unroll
        for (int k = 0; k < E; ++k) ge[k] = from_float<T>(gradient(e[k]));
        T *at = out + head + (i + u * threads) * E;
        if (out_packs) {
          *reinterpret_cast<uint4 *>(at) = g.v;
        } else {
#pragma unroll
          for (int k = 0; k < E; ++k) at[k] = ge[k];
        }
      }
  }
  if (part == parts - 1)
    for (long long i = head + packs * E + tid; i < V; i += threads) out[i] = from_float<T>(gradient(to_float(x[i])));
  __syncthreads();
  // the teacher's words of this block's share, each by its first entry, and the label if the teacher does not name it
  bool named = false;
  for (int k = tid; k < K; k += threads) {
    const int i = s_index[k];
    if (i < from || i >= to) continue;
    bool leads = true;
    float p = 0.f;
    for (int j = 0; j < K; ++j) {
      if (s_index[j] != i) continue;
      if (j < k) leads = false;
      p += s_p[j];
    }
    if (i == label) named = true;
    if (leads) out[i] = from_float<T>(gradient(s_x[k]) - soft * p - (i == label ? hard : 0.f));
  }
  named = __syncthreads_or(named);
  if (tid == 0 && labelled && !named && label >= from && label < to) out[label] = from_float<T>(gradient(x_label) - hard);
}

const char *check(const myea_distillation *d) {
  if (d == nullptr) return "distillation_error: no description";
  if (d->type > MYEA_TYPE_F16) return "distillation_error: unknown type";
  if (d->rows > kSequenceMost || d->vocabulary > kSequenceMost) return "distillation_error: a dimension above 2^30";
  if (d->top < 1 || d->top > kTopMost) return "distillation_error: 1 to 1024 teacher entries per row";
  if (!(d->temperature > 0.f) || d->temperature > 3e38f) return "distillation_error: the temperature has to be positive and finite";
  if (d->rows == 0) return nullptr;
  if (d->vocabulary == 0) return "distillation_error: an empty vocabulary";
  if (d->logits == nullptr || d->index == nullptr || d->teacher == nullptr || d->losses == nullptr) return "distillation_error: logits, index, teacher or losses is missing";
  return nullptr;
}

template <typename T> cudaError_t launch(const myea_distillation &d, cudaStream_t stream) {
  int threads = 512, parts = 1;
  while (threads > 128 && threads * (16 / sizeof(T)) * 2 > d.vocabulary) threads /= 2;
  // a row over several blocks where the rows leave SMs idle, as long as a block keeps 8 packs per thread
  while (parts < 8 && d.rows * parts * 2 <= 2ull * kSms && d.vocabulary / (parts * 2) >= threads * (16 / sizeof(T)) * 8) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(d.rows * parts));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = d.top * 12;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool two = d.hard != 0.f && d.temperature != 1.f && d.labels != nullptr;
  return two ? cudaLaunchKernelEx(&cfg, distillation_kernel<T, true>, d) : cudaLaunchKernelEx(&cfg, distillation_kernel<T, false>, d);
}

}  // namespace
}  // namespace myea

extern "C" int myea_b200_distillation_error(int device, const myea_distillation *d, void *stream, char *error_message, size_t error_capacity) {
  using namespace myea;
  if (const char *why = check(d)) return refuse(error_message, error_capacity, MYEA_E_INVALID, why);
  if (d->rows == 0) return MYEA_OK;
  DeviceScope scope(device);
  if (!scope.ok) return refuse(error_message, error_capacity, MYEA_E_CUDA, "distillation_error: no such device");
  with_type(d->type, [&](auto t) { (void)launch<decltype(t)>(*d, static_cast<cudaStream_t>(stream)); });
  return launched(error_message, error_capacity, "distillation_error");
}
