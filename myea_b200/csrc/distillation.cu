// Error of a row of logits against a teacher's best ones, with its gradient (the formulas stand at myea_distillation in
// myea_b200.h).  With x the row, m its maximum, c = 1 / temperature:
//   q_i = e^(c (x_i - m)) / s,  r_i = e^(x_i - m) / s1,   soft term = soft T^2 sum_k p_k (log p_k - c (x_k - m) + log s)
//   gradient = soft T (q_i - sum of the p of word i) + hard (r_i - [i = label])
//
// Bound by memory, and nearly as much by the exponentials (two per word, 16 a cycle and SM).  Rows of up to 4096 packs of 16 bytes
// stay in registers from the one time that they are read until their gradient is written.  Longer ones are read twice, the second
// time out of L2: 296 rows of 256 KB at a time fit there as long as the gradients, which nobody reads here, are stored past it
// (stored the ordinary way a third of the second reading came out of memory again).  2048 rows of 131072 bf16 logits: 252 us, 4.3 TB/s
// of 6.5 (115 us for the losses alone; the second reading asks for its packs right before it uses them); a block of 1024 threads per SM 272 us, registers of clusters of four 422 us, most of it waiting for one another.
// Many short rows are bound by a row's chain of steps, so as many blocks as can be lie side by side: 4096 rows of 1024 fp32 logits
// 18.3 us with 40 registers a thread, 19.3 with 54, 20.8 as clusters of one block, 28 with a warp per row.
// A cluster of blocks takes a row only where the rows leave SMs idle; the blocks' parts of the sums are exchanged through
// shared memory and joined in rank order.
// Exponents are formed from x - m, which is exact near the maximum, where it counts.  The first warp
// works on the teacher's few words meanwhile; they are mended at the end: their gradients are formed again from the logits with the
// teacher's part, so every element is rounded once.
#include <cooperative_groups.h>

#include "sequence.cuh"

namespace myea {
namespace {

namespace cg = cooperative_groups;
constexpr int kTopMost = 1024;

template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); uint4 v; };
// the k-th pair of a pack's words
__device__ __forceinline__ float2 pair(const Pack<float> &p, int k) {
  return k == 0 ? make_float2(__uint_as_float(p.v.x), __uint_as_float(p.v.y)) : make_float2(__uint_as_float(p.v.z), __uint_as_float(p.v.w));
}
__device__ __forceinline__ uint32_t word(const uint4 &v, int k) { return k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w; }
__device__ __forceinline__ float2 pair(const Pack<__nv_bfloat16> &p, int k) {
  const uint32_t w = word(p.v, k);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 pair(const Pack<__half> &p, int k) {
  const uint32_t w = word(p.v, k);
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ uint32_t packed(float2 x, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t packed(float2 x, __half) {
  const __half2 h = __floats2half2_rn(x.x, x.y);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// the largest of a pack's words, NaN passed over
template <typename T> __device__ __forceinline__ float largest(const Pack<T> &p) {
  float2 m = pair(p, 0);
#pragma unroll
  for (int k = 1; k < Pack<T>::N / 2; ++k) {
    const float2 x = pair(p, k);
    m = make_float2(fmaxf(m.x, x.x), fmaxf(m.y, x.y));
  }
  return fmaxf(m.x, m.y);
}

// Maximum and sums of exponentials of what has been seen
struct Running {
  float m = -INFINITY, s = 0.f, s1 = 0.f;   // s at the temperature, s1 at 1 (only where both are asked for)
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void rise(float to, float c, bool two) {   // to >= m
    if (to == m) return;
    const float by = m == -INFINITY ? 0.f : m - to;   // (nothing has been summed yet)
    s *= exp2_fast(by * c);
    if (two) s1 *= exp2_fast(by * kLog2e);
    m = to;
  }
  // the lanes of a warp, every lane ending with the same
  __device__ __forceinline__ void join_lanes(float c, bool two) {
    float to = m;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, k));
    rise(to, c, two);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, k);
      if (two) s1 += __shfl_xor_sync(0xffffffffu, s1, k);
    }
  }
};

// P: packs of a thread at a time
template <typename T, bool TWO, int P>
__global__ void __launch_bounds__(512, P == 2 ? 3 : 2) distillation_kernel(const myea_distillation d) {
  constexpr int E = Pack<T>::N;
  extern __shared__ float dynamic[];
  int *s_index = reinterpret_cast<int *>(dynamic);
  float *s_p = dynamic + d.top, *s_x = s_p + d.top;   // the teacher's probabilities, the logits of its words
  __shared__ Running s_warp[32], s_part;
  __shared__ bool s_taught;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const int V = static_cast<int>(d.vocabulary), K = static_cast<int>(d.top);
  const T *x = static_cast<const T *>(d.logits) + row * d.logits_stride;
  T *out = d.d_logits == nullptr ? nullptr : static_cast<T *>(d.d_logits) + row * d.d_logits_stride;
  // the row from its first 16-byte boundary on in packs, the blocks' shares of them, the elements before and behind
  const int head = min(V, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const int packs = (V - head) / E, first = static_cast<int>(static_cast<long long>(packs) * part / parts);
  const int last = static_cast<int>(static_cast<long long>(packs) * (part + 1) / parts);
  const int from = part == 0 ? 0 : head + first * E, to = part == parts - 1 ? V : head + last * E;   // this block's elements
  const Pack<T> *body = reinterpret_cast<const Pack<T> *>(x + head);
  const bool out_packs = out != nullptr && aligned_16(out + head);
  const float c = kLog2e / d.temperature;
  Pack<T> p[P];
  const int reach = P * threads;
  const auto load = [&](int at) {
#pragma unroll
    for (int u = 0; u < P; ++u)
      if (at + u * threads < last) p[u] = body[at + u * threads];
  };
  load(first + tid);   // (under way while the row's weight is)
  const float w = d.weight == nullptr ? 1.f : d.weight[row];
  const auto nothing = [&]() {
    if (out != nullptr)
      for (int i = from + tid; i < to; i += threads) out[i] = from_float<T>(0.f);
    if (part == 0 && tid == 0) d.losses[row] = 0.f;
  };
  if (w == 0.f) return nothing();   // (every block of the row's cluster)
  // an element outside the packs, one per thread at most (part 0: in front, the last part: behind)
  const int loose = part == 0 && tid < head ? tid : part == parts - 1 && head + packs * E + tid < V && tid < E ? head + packs * E + tid : -1;
  const int loose2 = parts == 1 && part == 0 && tid < head && head + packs * E + tid < V ? head + packs * E + tid : -1;
  const float x_loose = loose >= 0 ? to_float(x[loose]) : -INFINITY, x_loose2 = loose2 >= 0 ? to_float(x[loose2]) : -INFINITY;
  const int label = d.labels == nullptr || d.hard == 0.f ? -1 : d.labels[row];
  const bool labelled = label >= 0 && label < V;
  const float x_label = labelled ? to_float(x[label]) : 0.f;

  if (warp == 0) {   // the teacher's words, their logits and probabilities
    float t_max = -INFINITY;
#pragma unroll 4
    for (int k = lane; k < K; k += 32) {
      const int i = d.index[row * d.index_stride + k];
      const bool there = i >= 0 && i < V;
      const float t = there ? d.teacher[row * d.teacher_stride + k] : -INFINITY;
      s_index[k] = there ? i : -1;
      s_p[k] = t;
      s_x[k] = there ? to_float(x[i]) : 0.f;
      t_max = fmaxf(t_max, t);
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) t_max = fmaxf(t_max, __shfl_xor_sync(0xffffffffu, t_max, m));
    float t_sum = 0.f;
    for (int k = lane; k < K; k += 32) {
      const float e = s_index[k] >= 0 && s_p[k] != -INFINITY ? exp2_fast((s_p[k] - t_max) * c) : 0.f;   // (NaN stays NaN)
      s_p[k] = e;
      t_sum += e;
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) t_sum += __shfl_xor_sync(0xffffffffu, t_sum, m);
    const float t_scale = t_sum != 0.f ? 1.f / t_sum : 0.f;
    for (int k = lane; k < K; k += 32) s_p[k] *= t_scale;
    if (lane == 0) s_taught = t_sum != 0.f;
  }

  // maximum and sums
  Running run;
  for (int at = first + tid;;) {
    Pack<T> ahead[P];   // of a long row: the next packs are on their way while these are summed
    if constexpr (P == 4) {
#pragma unroll
      for (int u = 0; u < P; ++u)
        if (at + reach + u * threads < last) ahead[u] = body[at + reach + u * threads];
    }
    float m = fmaxf(run.m, fmaxf(x_loose, x_loose2));
#pragma unroll
    for (int u = 0; u < P; ++u)
      if (at + u * threads < last) m = fmaxf(m, largest(p[u]));
    run.rise(m, c, TWO);
    const float2 b = both(-run.base());
    float2 s = both(0.f), s1 = both(0.f);
#pragma unroll
    for (int u = 0; u < P; ++u)
      if (at + u * threads < last) {
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          const float2 e = add2(pair(p[u], k), b);
          s = add2(s, exp2_fast(mul2(e, both(c))));
          if (TWO) s1 = add2(s1, exp2_fast(mul2(e, both(kLog2e))));
        }
      }
    run.s += s.x + s.y;
    run.s1 += s1.x + s1.y;
    if (at - tid + reach >= last) break;
    at += reach;
    if constexpr (P == 4) {
#pragma unroll
      for (int u = 0; u < P; ++u) p[u] = ahead[u];
    } else {
      load(at);
    }
  }
  if (loose >= 0) {
    run.s += exp2_fast((x_loose - run.base()) * c);
    if (TWO) run.s1 += exp2_fast((x_loose - run.base()) * kLog2e);
  }
  if (loose2 >= 0) {
    run.s += exp2_fast((x_loose2 - run.base()) * c);
    if (TWO) run.s1 += exp2_fast((x_loose2 - run.base()) * kLog2e);
  }
  // lanes, warps, blocks of the cluster: every block ends with the same sums
  run.join_lanes(c, TWO);
  if (lane == 0) s_warp[warp] = run;
  __syncthreads();
  run = lane < warps ? s_warp[lane] : Running();
  run.join_lanes(c, TWO);
  if (parts > 1) {
    if (tid == 0) s_part = run;
    cluster.sync();
    run = lane < parts ? *cluster.map_shared_rank(&s_part, lane) : Running();
    run.join_lanes(c, TWO);
    cluster.sync();   // nobody leaves, or writes over the logits, while others read
  }
  if (run.s == 0.f) return nothing();   // no open word
  const bool taught = s_taught;
  const float top = run.m, unit = TWO ? run.s1 : run.s;

  if (part == 0 && warp == 0) {
    float kl = 0.f;
    const float log_s = logf(run.s);
    for (int k = lane; k < K; k += 32) {
      const float q = s_p[k];
      if (q != 0.f) kl += q * (logf(q) - (s_x[k] - top) / d.temperature + log_s);
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) kl += __shfl_xor_sync(0xffffffffu, kl, m);
    if (lane == 0) {
      float loss = taught ? d.soft * d.temperature * d.temperature * kl : 0.f;
      if (labelled) loss += d.hard * (logf(unit) - (x_label - top));
      d.losses[row] = w * loss;
    }
  }
  if (out == nullptr) return;

  // without a second temperature both terms have the same exponentials
  const float soft = taught ? w * d.soft * d.temperature : 0.f, hard = labelled ? w * d.hard : 0.f;
  const float a = TWO ? soft / run.s : (soft + hard) / run.s, b = TWO ? hard / run.s1 : 0.f;
  const auto gradient2 = [&](float2 e) {
    const float2 far = add2(e, both(-top));
    float2 g = mul2(both(a), exp2_fast(mul2(far, both(c))));
    if (TWO) g = fma2(both(b), exp2_fast(mul2(far, both(kLog2e))), g);
    return g;
  };
  const auto gradient = [&](float e) { return gradient2(both(e)).x; };
  const bool again = last - first > reach;
  for (int at = first + tid; at - tid < last; at += reach) {
    if (again) load(at);
#pragma unroll
    for (int u = 0; u < P; ++u)
      if (at + u * threads < last) {
        Pack<T> g;
        if constexpr (E == 4) {
          const float2 lo = gradient2(pair(p[u], 0)), hi = gradient2(pair(p[u], 1));
          g.v = make_uint4(__float_as_uint(lo.x), __float_as_uint(lo.y), __float_as_uint(hi.x), __float_as_uint(hi.y));
        } else {
          g.v = make_uint4(packed(gradient2(pair(p[u], 0)), T()), packed(gradient2(pair(p[u], 1)), T()), packed(gradient2(pair(p[u], 2)), T()),
                           packed(gradient2(pair(p[u], 3)), T()));
        }
        T *to_ = out + head + static_cast<long long>(at + u * threads) * E;
        if (out_packs) {
          __stcs(reinterpret_cast<uint4 *>(to_), g.v);   // (nobody reads it here: what is read again stays in L2)
        } else {
          const T *ge = reinterpret_cast<const T *>(&g.v);
#pragma unroll
          for (int k = 0; k < E; ++k) to_[k] = ge[k];
        }
      }
  }
  if (loose >= 0) out[loose] = from_float<T>(gradient(x_loose));
  if (loose2 >= 0) out[loose2] = from_float<T>(gradient(x_loose2));
  __syncthreads();
  // the teacher's words of this block's share, each by its first entry, and the label if the teacher does not name it
  bool named = false;
  for (int k = tid; k < K; k += threads) {
    const int i = s_index[k];
    if (i < from || i >= to) continue;
    bool leads = true;
    float q = 0.f;
    for (int j = 0; j < K; ++j) {
      if (s_index[j] != i) continue;
      if (j < k) leads = false;
      q += s_p[j];
    }
    if (i == label) named = true;
    if (leads) out[i] = from_float<T>(gradient(s_x[k]) - soft * q - (i == label ? hard : 0.f));
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

bool two_temperatures(const myea_distillation &d) { return d.hard != 0.f && d.temperature != 1.f && d.labels != nullptr; }

template <typename T, int P> cudaError_t launch(const myea_distillation &d, int threads, int parts, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(d.rows * parts));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = d.top * 12;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return two_temperatures(d) ? cudaLaunchKernelEx(&cfg, distillation_kernel<T, true, P>, d) : cudaLaunchKernelEx(&cfg, distillation_kernel<T, false, P>, d);
}

template <typename T> cudaError_t launch(const myea_distillation &d, cudaStream_t stream) {
  const uint64_t packs = (d.vocabulary * sizeof(T) + 15) / 16;
  int parts = 1;
  // Blocks that fill one SM and leave the next with half the work are halved where a block's exponentials outweigh the exchange between two:
  // with 8 words in a pack and two temperatures (us, whole / halved: 203 rows of 16801, 25601, 32001 fp16 words 12.4 / 12.5, 15.4 / 14.5, 17.5 /
  // 15.7; of as many packs in fp32 10.9 / 11.2, 12.2 / 12.6, 13.2 / 13.7, and in fp16 at one temperature 10.5 / 11.0, 12.1 / 12.5, 13.1 /
  // 13.4), and in rows that are in blocks already (111 rows of 64001 fp16 words 19.1 / 17.7, at one temperature 14.3 / 14.1, of as many packs in
  // fp32 14.6 / 14.3; 75 rows 17.9 / 15.1, 13.6 / 12.5, 13.8 / 12.7).
  const bool heavy = sizeof(T) == 2 && two_temperatures(d);
  while (parts < 8 && ((d.rows * parts * 2 <= 2ull * kSms && packs >= parts * 2 * 256) ||
                       (d.rows * parts * 2 <= 3ull * kSms && packs > parts * 2048 && packs <= parts * 4096 && (parts > 1 || heavy))))
    parts *= 2;
  const uint64_t share = (packs + parts - 1) / parts;
  // Many rows: few threads with eight packs each, so that more rows lie side by side and the join of a row's warps is short (2000 rows of
  // 16001 bf16 words 46 us against 65 with 512 threads, 4000 rows of 8000 45 against 69 with two packs each, of 4000 35 against 41).
  // Of some 256 to 512 packs only in plenty: 400 rows of 4000 took 9.8 us against 7.7; with 256 packs and fewer never (28 against 18).
  const bool many = d.rows * parts > 2ull * kSms;
  if (many && share > (d.rows >= 8ull * kSms ? 256 : 512) && share <= 2048) return launch<T, 8>(d, static_cast<int>((share + 255) / 256 * 32), parts, stream);
  if (share <= 1024) return launch<T, 2>(d, share <= 64 ? 32 : static_cast<int>((share + 63) / 64 * 32), parts, stream);
  if (share <= 4096) return launch<T, 8>(d, 512, parts, stream);
  // (rows of 256 threads only while those under way fit L2: 1024 rows of 40000 bf16 words 42 us against 50, but of 131072 140 against 128)
  return launch<T, 4>(d, many && share * 16 * 4 * kSms <= (96u << 20) ? 256 : 512, parts, stream);
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
