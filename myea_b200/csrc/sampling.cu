// Draws one token per row from what temperature, top-k, top-p and min-p leave of it (defined at myea_sampling in myea_b200.h).
//
// All three limits keep a prefix of the row ordered by falling logit and rising index, so what is kept is a threshold on the
// logit and, among those equal to it, on the index.  The threshold is found without sorting: radix selection on the logits'
// bits (mapped to integers of the same order), 11, 11 and 10 at a time, with a histogram of counts and weights per digit.
// Weights are 64-bit integers, w * 2^shift: their sums are exact whatever the order of the atomics, and the same draw is
// made every time.
#include "sequence.cuh"

namespace myea {
namespace {

using u64 = unsigned long long;
constexpr int kThreads = 1024;
constexpr int kBins = 2048;

// integers in the order of the floats; 0: a closed word
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0;
  if (x == 0.f) x = 0.f;   // both zeros are equal
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

struct Row {
  float m, inv;        // largest logit
  double per;          // 1 / temperature
  int shift;
  // the weight of a logit as an integer
  __device__ __forceinline__ u64 weight(float x) const {
    if (!(x > -INFINITY)) return 0;
    const double w = x == m ? 1.0 : m == INFINITY ? 0.0 : exp((static_cast<double>(x) - static_cast<double>(m)) * per);
    return static_cast<u64>(__double2ll_rn(ldexp(w, shift)));
  }
};

__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

struct Shared {
  unsigned int count[kBins];
  u64 mass[kBins];
  u64 warp[32];
  float warp_m[32];
  int warp_i[32];
  int digit;
  u64 before_count, before_mass, bin_count, bin_mass;
  int token;
  u64 chance;
};

// What is kept: keys above `key`, and those equal to it up to index `last`
struct Kept {
  uint32_t key = 1;
  long long last = 1ll << 62;
  __device__ __forceinline__ bool has(uint32_t k, long long i) const { return k > key || (k == key && i <= last); }
};

// The first index, in rising order, at which the running sum of f(index) exceeds `target`; -1: none does.  before, own: the sum in front of it and its own
template <typename F> __device__ long long first_beyond(Shared &s, long long from, long long to, u64 target, F f, u64 *own) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  while (true) {
    const long long n = to - from, share = (n + 31) / 32, lo = from + share * warp, hi = min(lo + share, to);
    u64 sum = 0;
    for (long long i = lo + lane; i < hi; i += 32) sum += f(i);
    sum = warp_sum(sum);
    __syncthreads();
    if (lane == 0) s.warp[warp] = sum;
    __syncthreads();
    int w = 0;
    u64 before = 0;
    for (; w < 32; ++w) {
      if (before + s.warp[w] > target) break;
      before += s.warp[w];
    }
    if (w == 32) return -1;
    if (share == 1) {
      if (own != nullptr) *own = s.warp[w];
      __syncthreads();
      return from + w;
    }
    target -= before;
    from += share * w;
    to = min(from + share, to);
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sampling_kernel(const myea_sampling a, int shift) {
  __shared__ Shared s;
  const long long row = blockIdx.x, V = static_cast<long long>(a.vocabulary);
  const T *x = static_cast<const T *>(a.logits) + row * a.logits_stride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float temperature = a.temperature == nullptr ? 1.f : a.temperature[row];
  const float top_p = a.top_p == nullptr ? 1.f : a.top_p[row], min_p = a.min_p == nullptr ? 0.f : a.min_p[row];
  const long long top_k = a.top_k == nullptr ? 0 : a.top_k[row];
  const bool greedy = !(temperature > 0.f);

  float m = -INFINITY;
  long long at = -1;
  for (long long i = tid; i < V; i += kThreads) {
    const float e = to_float(x[i]);
    if (e > m) { m = e; at = i; }
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) {
    const float o = __shfl_xor_sync(0xffffffffu, m, k);
    const long long oi = __shfl_xor_sync(0xffffffffu, at, k);
    if (o > m || (o == m && oi < at && oi >= 0)) { m = o; at = oi; }
  }
  if (lane == 0) { s.warp_m[warp] = m; s.warp_i[warp] = static_cast<int>(at); }
  __syncthreads();
  m = s.warp_m[0];
  at = s.warp_i[0];
  for (int k = 1; k < 32; ++k)
    if (s.warp_m[k] > m || (s.warp_m[k] == m && s.warp_i[k] < at && s.warp_i[k] >= 0)) { m = s.warp_m[k]; at = s.warp_i[k]; }
  if (at < 0 || greedy) {
    if (tid == 0) {
      a.tokens[row] = static_cast<int>(at);
      if (a.chances != nullptr) a.chances[row] = at < 0 ? 0.f : 1.f;
    }
    return;
  }
  Row r;
  r.m = m; r.per = 1.0 / static_cast<double>(temperature); r.shift = shift;

  Kept kept;
  // keeps the first n words (by count), or those before which less than `mass` lies
  const auto limit = [&](bool by_mass, u64 target) {
    uint32_t prefix = 0;
    u64 before_count = 0, before_mass = 0;
    int low = 21;
    for (int round = 0; round < 3; ++round) {
      const int bits = round < 2 ? 11 : 10;
      low = round == 0 ? 21 : round == 1 ? 10 : 0;
      __syncthreads();
      for (int k = tid; k < kBins; k += kThreads) { s.count[k] = 0; s.mass[k] = 0; }
      __syncthreads();
      for (long long i = tid; i < V; i += kThreads) {
        const float e = to_float(x[i]);
        const uint32_t key = key_of(e);
        if (key == 0 || !kept.has(key, i) || (round > 0 && (key >> (low + bits)) != prefix)) continue;
        const uint32_t digit = (key >> low) & ((1u << bits) - 1);
        atomicAdd(&s.count[digit], 1u);
        if (by_mass) atomicAdd(&s.mass[digit], r.weight(e));
      }
      __syncthreads();
      if (tid == 0) {
        int d = (1 << bits) - 1;
        for (; d >= 0; --d) {
          if (s.count[d] == 0) continue;
          if (by_mass ? before_mass + s.mass[d] >= target : before_count + s.count[d] >= target) break;
          before_count += s.count[d];
          before_mass += s.mass[d];
        }
        s.digit = d;
        if (d >= 0) {
          s.before_count = before_count; s.before_mass = before_mass;
          s.bin_count = s.count[d]; s.bin_mass = s.mass[d];
        }
      }
      __syncthreads();
      if (s.digit < 0) return;   // fewer words than the limit
      prefix = (prefix << bits) | static_cast<uint32_t>(s.digit);
      before_count = s.before_count;
      before_mass = s.before_mass;
    }
    // of the words equal to the threshold
    u64 ties;
    if (by_mass) {
      const u64 each = s.bin_count > 0 ? s.bin_mass / s.bin_count : 0;
      ties = each == 0 ? s.bin_count : (target > before_mass ? (target - before_mass + each - 1) / each : 0);
      if (before_count == 0 && ties == 0) ties = 1;
    } else {
      ties = target - before_count;
    }
    if (ties < s.bin_count) {
      const Kept was = kept;
      const uint32_t key = prefix;
      const long long last = first_beyond(s, 0, V, ties - 1, [&](long long i) -> u64 { const uint32_t k = key_of(to_float(x[i])); return k == key && was.has(k, i); }, nullptr);
      kept.last = last;
      kept.key = key;
    } else if (prefix > kept.key) {
      kept.key = prefix;
      kept.last = 1ll << 62;
    }
    __syncthreads();
  };
  const auto sum_kept = [&]() {
    u64 sum = 0;
    for (long long i = tid; i < V; i += kThreads) {
      const float e = to_float(x[i]);
      const uint32_t k = key_of(e);
      if (k != 0 && kept.has(k, i)) sum += r.weight(e);
    }
    sum = warp_sum(sum);
    __syncthreads();
    if (lane == 0) s.warp[warp] = sum;
    __syncthreads();
    sum = 0;
    for (int k = 0; k < 32; ++k) sum += s.warp[k];
    return sum;
  };
  if (top_k > 0 && top_k < V) limit(false, static_cast<u64>(top_k));
  u64 total = sum_kept();
  if (top_p < 1.f) {
    const double part = top_p > 0.f ? static_cast<double>(top_p) * static_cast<double>(total) : 0.0;
    limit(true, static_cast<u64>(ceil(part)));
  }
  // the least weight, as an integer of the same scale
  u64 least = 0;
  if (min_p > 0.f) least = min_p >= 1.f ? 1ull << shift : static_cast<u64>(ceil(ldexp(static_cast<double>(min_p), shift)));
  const auto weigh = [&](long long i) -> u64 {
    const float e = to_float(x[i]);
    const uint32_t k = key_of(e);
    if (k == 0 || !kept.has(k, i)) return 0;
    const u64 w = r.weight(e);
    return w >= least ? w : 0;
  };
  u64 sum = 0;
  for (long long i = tid; i < V; i += kThreads) sum += weigh(i);
  sum = warp_sum(sum);
  __syncthreads();
  if (lane == 0) s.warp[warp] = sum;
  __syncthreads();
  total = 0;
  for (int k = 0; k < 32; ++k) total += s.warp[k];
  const float uniform = a.uniform[row];
  u64 target = uniform > 0.f ? static_cast<u64>(static_cast<double>(uniform) * static_cast<double>(total)) : 0;
  if (target >= total) target = total - 1;
  u64 own = 0;
  const long long token = first_beyond(s, 0, V, target, weigh, &own);
  if (tid == 0) {
    a.tokens[row] = static_cast<int>(token);
    if (a.chances != nullptr) a.chances[row] = static_cast<float>(static_cast<double>(own) / static_cast<double>(total));
  }
}

const char *check(const myea_sampling *s) {
  if (s == nullptr) return "sample: no description";
  if (s->type > MYEA_TYPE_F16) return "sample: unknown type";
  if (s->rows > kSequenceMost || s->vocabulary > kSequenceMost) return "sample: a dimension above 2^30";
  if (s->rows == 0) return nullptr;
  if (s->vocabulary == 0) return "sample: an empty vocabulary";
  if (s->logits == nullptr || s->uniform == nullptr || s->tokens == nullptr) return "sample: logits, uniform or tokens is missing";
  return nullptr;
}

// bits behind the point of a weight: the sum over the vocabulary stays below 2^62
int shift_for(uint64_t vocabulary) {
  int bits = 0;
  while ((uint64_t(1) << bits) < vocabulary) ++bits;
  return 62 - bits < 51 ? 62 - bits : 51;
}

}  // namespace
}  // namespace myea

extern "C" int myea_b200_sample(int device, const myea_sampling *s, void *stream, char *error_message, size_t error_capacity) {
  using namespace myea;
  if (const char *why = check(s)) return refuse(error_message, error_capacity, MYEA_E_INVALID, why);
  if (s->rows == 0) return MYEA_OK;
  DeviceScope scope(device);
  if (!scope.ok) return refuse(error_message, error_capacity, MYEA_E_CUDA, "sample: no such device");
  with_type(s->type, [&](auto t) {
    sampling_kernel<decltype(t)><<<static_cast<unsigned>(s->rows), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(*s, shift_for(s->vocabulary));
  });
  return launched(error_message, error_capacity, "sample");
}
