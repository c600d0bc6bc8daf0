// Draws one token per row from what temperature, top-k, top-p and min-p leave of it (defined at myea_sampling in myea_b200.h).
//
// All three limits keep a prefix of the row ordered by falling logit and rising index, so what is kept is a threshold on the
// logit and, among those equal to it, on the index.  The threshold is found without sorting, by histograms of counts or
// weights: first 2048 bins in the distance from the maximum, which spread the words of any ordinary row, then bins in the logits' bits
// (mapped to integers of the same order) within the bin that holds the threshold, until one value is left.
//
// Weights are integers, w * 2^shift: their sums are exact whatever the order of the atomics, and the same draw is made every
// time.  A draw from 1e5 words goes through as many borders, so a weight good to 24 bits would move a token of every few
// hundred rows; these are good to 2^-44 or better.  2^t is a table of 2^(k / 256) times the polynomial 1 + r + ... of the rest
// |r| < 2^-9.5 (its first term left out is below 2^-54), in 64-bit floating point, which this chip does at half the 32-bit rate.
//
// A cluster of up to eight blocks takes a row, each keeps its slice in shared memory, so the row is read from memory once whatever
// is asked of it; rows beyond the clusters' memory are read again in every pass.  A warp works on a contiguous part of a slice, so
// that the draw, which goes by rising index, finds its word from the warps' sums and one warp's walk over its part.
#include <cooperative_groups.h>

#include "sequence.cuh"

namespace myea {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;
constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2048, kParts = 8;
constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); uint4 v; };

// integers in the order of the floats; 0: a closed word
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t b = __float_as_uint(x + 0.f);   // (both zeros are equal)
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// What is kept: keys above `key`, and those equal to it up to index `last`
struct Kept {
  uint32_t key = 1;
  int last = 0x7fffffff;
  __device__ __forceinline__ bool has(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

struct alignas(16) Shared {
  unsigned int count[kBins], low[kBins], high[kBins];   // of a histogram: words, and their weights' lower and upper 32 bits
  double table[256];                                    // 2^(k / 256)
  u64 warp[kWarps];
  float warp_m[kWarps];
  float m;
  unsigned int key_min, key_max;
  int best, found;
  u64 own;
  // the bin that holds a limit
  int bin;
  u64 before_count, before_mass, bin_count, bin_mass, total_mass;
  u64 scan_count[kWarps], scan_mass[kWarps];
};

template <typename T, bool RES> struct Draw {
  static constexpr int E = Pack<T>::N;
  cg::cluster_group cluster;
  Shared &s;
  const T *x;          // the row
  uint4 *slice;        // this block's vectors of it (RES)
  int V, lead;         // words; elements by which the first vector begins before the row
  int first, last;     // this block's vectors
  int from, to;        // this warp's
  int parts, part, lane, warp;
  float m, half_scale; // the maximum; (m - x) / temperature = (m / 2 - x / 2) * half_scale
  double md, per;      // 256 log2(e) / temperature
  int shift;
  float beyond;        // distances from here on weigh nothing
  u64 warps[4], upto_warps;   // of total(): up to four warps' sums, and the running sum up to them

  __device__ __forceinline__ Draw(Shared &s_) : cluster(cg::this_cluster()), s(s_) {}

  // vector v of the row, -infinity where there is no word
  __device__ __forceinline__ Pack<T> from_memory(int v) const {
    const long long at = static_cast<long long>(v) * E - lead;
    Pack<T> p;
    if (at >= 0 && at + E <= V) {
      p.v = *reinterpret_cast<const uint4 *>(x + at);
    } else {
      T *e = reinterpret_cast<T *>(&p.v);
#pragma unroll
      for (int k = 0; k < E; ++k) e[k] = at + k >= 0 && at + k < V ? x[at + k] : from_float<T>(-INFINITY);
    }
    return p;
  }
  __device__ __forceinline__ void words(int v, float (&e)[E]) const {
    Pack<T> p;
    if constexpr (RES) p.v = slice[v - first];
    else p = from_memory(v);
    const T *w = reinterpret_cast<const T *>(&p.v);
#pragma unroll
    for (int k = 0; k < E; ++k) e[k] = to_float(w[k]);
  }
  __device__ __forceinline__ float distance(float e) const { return (0.5f * m - 0.5f * e) * half_scale; }
  // the weight of a word as an integer
  __device__ __forceinline__ u64 weight(float e) const {
    if (e == m) return 1ull << shift;
    if (!(distance(e) < beyond) || m == INFINITY) return 0;
    constexpr double magic = 6755399441055744.0;   // 1.5 * 2^52: the sum's lower bits are the nearest integer
    constexpr double c1 = kLn2 / 256, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6, c4 = c1 * c1 * c1 * c1 / 24;
    const double d = static_cast<double>(e) - md;
    const double z = fma(d, per, magic);
    const int i = __double2loint(z);
    const double r = fma(d, per, magic - z);
    double q = fma(fma(fma(fma(r, c4, c3), r, c2), r, c1), r, 1.0);
    q *= s.table[i & 255];
    const u64 bits = static_cast<u64>(__double_as_longlong(q));
    const int right = 52 - (static_cast<int>(bits >> 52) - 1023) - (i >> 8) - shift;   // (q > 0; i <= 0)
    return right > 63 ? 0 : ((bits & ((1ull << 52) - 1)) | (1ull << 52)) >> right;
  }
  // f(word, its index) for this warp's words, lanes side by side
  template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll 2
    for (int v = from + lane; v < to; v += 32) {
      float e[E];
      words(v, e);
#pragma unroll
      for (int k = 0; k < E; ++k) f(e[k], v * E + k - lead);
    }
  }
  static __device__ __forceinline__ u64 warp_sum(u64 y) {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) y += __shfl_xor_sync(0xffffffffu, y, k);
    return y;
  }
  // Sums of f over the row's words by warps (put into s.warp): their total, in every block
  template <typename F> __device__ u64 total(F f) {
    u64 sum = 0;
    each([&](float e, int i) { sum += f(e, i); });
    sum = warp_sum(sum);
    if (lane == 0) s.warp[warp] = sum;
    cluster.sync();
    // up to four neighbouring warps' sums per lane, and the running sum up to them
    const int each_lane = (parts * kWarps + 31) / 32;
    upto_warps = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = lane * each_lane + j;
      warps[j] = j < each_lane && k < parts * kWarps ? cluster.map_shared_rank(&s, k / kWarps)->warp[k % kWarps] : 0;
      upto_warps += warps[j];
    }
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const u64 o = __shfl_up_sync(0xffffffffu, upto_warps, k);
      if (lane >= k) upto_warps += o;
    }
    return __shfl_sync(0xffffffffu, upto_warps, 31);
  }
  // The first index, in rising order, at which the running sum of f exceeds `target` (below the total, after total(f)), and f there:
  // known to every block behind the next cluster.sync(), in s.found and s.own
  template <typename F> __device__ void find(u64 target, F f) {
    const int each_lane = (parts * kWarps + 31) / 32;
    const int with = __ffs(__ballot_sync(0xffffffffu, upto_warps > target)) - 1;   // the lane that has the warp
    u64 before = upto_warps - (warps[0] + warps[1] + warps[2] + warps[3]);
    int at = 0;
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (at == j && before + warps[j] <= target) {
        before += warps[j];
        ++at;
      }
    before = __shfl_sync(0xffffffffu, before, with);
    at = with * each_lane + __shfl_sync(0xffffffffu, at, with);
    if (at != part * kWarps + warp) return;
    for (int v0 = from; v0 < to; v0 += 32) {
      const int v = v0 + lane;
      float e[E];
      u64 own[E], sum = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) own[k] = 0;
      if (v < to) {
        words(v, e);
#pragma unroll
        for (int k = 0; k < E; ++k) { own[k] = f(e[k], v * E + k - lead); sum += own[k]; }
      }
      u64 upto = sum;
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) {
        const u64 o = __shfl_up_sync(0xffffffffu, upto, k);
        if (lane >= k) upto += o;
      }
      const unsigned beyond_ = __ballot_sync(0xffffffffu, before + upto > target);
      if (beyond_ != 0) {
        if (lane == __ffs(beyond_) - 1) {
          u64 run = before + upto - sum;
          int k = 0;
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (k == j) {
              if (run + own[j] > target) break;
              run += own[j];
              ++k;
            }
          u64 mine = 0;
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (k == j) mine = own[j];
          for (int o = 0; o < parts; ++o) {
            Shared *to_ = cluster.map_shared_rank(&s, o);
            to_->found = v * E + k - lead;
            to_->own = mine;
          }
        }
        return;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  // Histogram of the words for which bin(word, index) >= 0, over the cluster, and the bin that holds the limit: the first, from bin 0
  // on, with `target` words (or `target` of weight) up to its end.  part_of_all < 1: the target is that part of the whole weight.
  // s.bin is -1 where there is less.  On entry before_count / before_mass: what lies in front of bin 0.
  template <typename F> __device__ void limit_bin(bool by_mass, double part_of_all, u64 target, u64 before_count, u64 before_mass, F bin) {
    for (int k = threadIdx.x; k < kBins; k += kThreads) s.count[k] = s.low[k] = s.high[k] = 0;
    if (threadIdx.x == 0) { s.bin = -1; s.total_mass = 0; }
    __syncthreads();
    each([&](float e, int i) {
      const int b = bin(e, i);
      if (b < 0) return;
      atomicAdd(&s.count[b], 1u);
      if (by_mass) {
        const u64 w = weight(e);
        const unsigned l = static_cast<unsigned>(w);
        const unsigned old = atomicAdd(&s.low[b], l);
        const unsigned up = static_cast<unsigned>(w >> 32) + (old + l < l ? 1u : 0u);
        if (up != 0) atomicAdd(&s.high[b], up);
      }
    });
    cluster.sync();
    constexpr int B = kBins / kThreads;
    u64 c[B], w[B], sum_c = 0, sum_w = 0;
#pragma unroll
    for (int k = 0; k < B; ++k) { c[k] = 0; w[k] = 0; }
    for (int o = 0; o < parts; ++o) {
      const Shared *h = cluster.map_shared_rank(&s, o);
      const uint4 n = *reinterpret_cast<const uint4 *>(&h->count[threadIdx.x * B]);
      c[0] += n.x; c[1] += n.y; c[2] += n.z; c[3] += n.w;
      if (by_mass) {
        const uint4 l = *reinterpret_cast<const uint4 *>(&h->low[threadIdx.x * B]), u = *reinterpret_cast<const uint4 *>(&h->high[threadIdx.x * B]);
        w[0] += l.x + (static_cast<u64>(u.x) << 32); w[1] += l.y + (static_cast<u64>(u.y) << 32);
        w[2] += l.z + (static_cast<u64>(u.z) << 32); w[3] += l.w + (static_cast<u64>(u.w) << 32);
      }
    }
#pragma unroll
    for (int k = 0; k < B; ++k) { sum_c += c[k]; sum_w += w[k]; }
    u64 upto_c = sum_c, upto_w = sum_w;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const u64 oc = __shfl_up_sync(0xffffffffu, upto_c, k), ow = __shfl_up_sync(0xffffffffu, upto_w, k);
      if (lane >= k) { upto_c += oc; upto_w += ow; }
    }
    if (lane == 31) { s.scan_count[warp] = upto_c; s.scan_mass[warp] = upto_w; }
    __syncthreads();
    u64 all_w = 0;
    for (int k = 0; k < kWarps; ++k) {
      if (k < warp) { before_count += s.scan_count[k]; before_mass += s.scan_mass[k]; }
      all_w += s.scan_mass[k];
    }
    if (part_of_all < 1.0) target = static_cast<u64>(ceil(part_of_all * static_cast<double>(all_w)));
    before_count += upto_c - sum_c;
    before_mass += upto_w - sum_w;
#pragma unroll
    for (int k = 0; k < B; ++k) {
      if (c[k] != 0) {
        // the first bin of words with enough up to its end
        const bool enough = by_mass ? before_mass + w[k] >= target : before_count + c[k] >= target;
        const bool was = by_mass ? before_count != 0 && before_mass >= target : before_count >= target;
        if (enough && !was) {
          s.bin = threadIdx.x * B + k;
          s.before_count = before_count;
          s.before_mass = before_mass;
          s.bin_count = c[k];
          s.bin_mass = w[k];
        }
      }
      before_count += c[k];
      before_mass += w[k];
    }
    if (threadIdx.x == 0) s.total_mass = target;
    cluster.sync();   // nobody clears its bins while others read them
  }

  // keeps the first `target` words, or those before which less than the part `part_of_all` of the weight of what was kept lies
  __device__ void limit(Kept &kept, bool by_mass, double part_of_all, u64 target) {
    // bins by distance: 64 to a unit, of the logits for counts and of the logarithm of the weights for weights
    const float scale = by_mass ? 64.f * half_scale : 128.f;
    const auto far = [&](float e) {
      const float t = (0.5f * m - 0.5f * e) * scale;
      return e == m ? 0 : t < static_cast<float>(kBins - 1) ? static_cast<int>(t) : kBins - 1;
    };
    const Kept was = kept;
    limit_bin(by_mass, by_mass ? part_of_all : 1.0, target, 0, 0, [&](float e, int i) { const uint32_t k = key_of(e); return k != 0 && was.has(k, i) ? far(e) : -1; });
    if (s.bin < 0) return;   // fewer words than that
    target = s.total_mass;
    const int bin = s.bin;
    // the logits in that bin
    if (threadIdx.x == 0) { s.key_min = 0xffffffffu; s.key_max = 0; }
    __syncthreads();
    uint32_t lowest = 0xffffffffu, highest = 0;
    each([&](float e, int i) {
      const uint32_t k = key_of(e);
      if (k != 0 && was.has(k, i) && far(e) == bin) { lowest = min(lowest, k); highest = max(highest, k); }
    });
    lowest = __reduce_min_sync(0xffffffffu, lowest);
    highest = __reduce_max_sync(0xffffffffu, highest);
    if (lane == 0) { atomicMin(&s.key_min, lowest); atomicMax(&s.key_max, highest); }
    cluster.sync();
    for (int o = 0; o < parts; ++o) {
      const Shared *h = cluster.map_shared_rank(&s, o);
      lowest = min(lowest, h->key_min);
      highest = max(highest, h->key_max);
    }
    while (lowest != highest) {
      int narrow = 0;
      while (((highest - lowest) >> narrow) >= kBins) ++narrow;
      const uint32_t lo = lowest, hi = highest;
      const u64 before_count = s.before_count, before_mass = s.before_mass;
      __syncthreads();
      limit_bin(by_mass, 1.0, target, before_count, before_mass,
                [&](float e, int i) { const uint32_t k = key_of(e); return k >= lo && k <= hi && was.has(k, i) ? static_cast<int>((hi - k) >> narrow) : -1; });
      highest = hi - (static_cast<uint32_t>(s.bin) << narrow);
      lowest = highest - ((1u << narrow) - 1);
      lowest = lowest < lo || lowest > highest ? lo : lowest;
      if (narrow == 0) lowest = highest;
    }
    const uint32_t key = highest;
    // of the words equal to the threshold
    u64 ties;
    if (by_mass) {
      const u64 one = s.bin_mass / s.bin_count;
      ties = one == 0 ? s.bin_count : target > s.before_mass ? (target - s.before_mass + one - 1) / one : 0;
      if (s.before_count == 0 && ties == 0) ties = 1;
    } else {
      ties = target - s.before_count;
    }
    if (ties < s.bin_count) {
      const auto tie = [&](float e, int i) -> u64 { const uint32_t k = key_of(e); return k == key && was.has(k, i) ? 1 : 0; };
      if (ties > 0) {
        total(tie);
        find(ties - 1, tie);
        cluster.sync();
        kept.last = s.found;
        kept.key = key;
      } else {
        kept.key = key;
        kept.last = -1;
      }
    } else if (key > kept.key) {
      kept.key = key;
      kept.last = 0x7fffffff;
    }
    __syncthreads();   // what has been read here is written by the next limit
  }
};

template <typename T, bool RES>
__global__ void __launch_bounds__(kThreads) sampling_kernel(const myea_sampling a, int shift) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  Shared &s = *reinterpret_cast<Shared *>(dynamic);
  Draw<T, RES> d(s);
  constexpr int E = Pack<T>::N;
  d.parts = static_cast<int>(d.cluster.num_blocks());
  d.part = static_cast<int>(d.cluster.block_rank());
  d.lane = threadIdx.x & 31;
  d.warp = threadIdx.x >> 5;
  const long long row = blockIdx.x / d.parts;
  d.x = static_cast<const T *>(a.logits) + row * a.logits_stride;
  d.V = static_cast<int>(a.vocabulary);
  d.lead = static_cast<int>(reinterpret_cast<uintptr_t>(d.x) % 16 / sizeof(T));
  const long long vectors = (d.lead + static_cast<long long>(d.V) + E - 1) / E;
  d.first = static_cast<int>(vectors * d.part / d.parts);
  d.last = static_cast<int>(vectors * (d.part + 1) / d.parts);
  d.slice = reinterpret_cast<uint4 *>(dynamic + sizeof(Shared));
  const int share = (d.last - d.first + kWarps - 1) / kWarps;
  d.from = min(d.first + d.warp * share, d.last);
  d.to = min(d.from + share, d.last);
  const float temperature = a.temperature == nullptr ? 1.f : a.temperature[row];
  const float top_p = a.top_p == nullptr ? 1.f : a.top_p[row], min_p = a.min_p == nullptr ? 0.f : a.min_p[row], uniform = a.uniform[row];
  const int top_k = a.top_k == nullptr ? 0 : a.top_k[row];

  float m = -INFINITY;
  constexpr int U = 4;
  for (int v = d.from + d.lane; v < d.to; v += 32 * U) {
    Pack<T> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + 32 * u < d.to) p[u] = d.from_memory(v + 32 * u);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + 32 * u < d.to) {
        if constexpr (RES) d.slice[v + 32 * u - d.first] = p[u].v;
        const T *e = reinterpret_cast<const T *>(&p[u].v);
#pragma unroll
        for (int k = 0; k < E; ++k) m = fmaxf(m, to_float(e[k]));   // (NaN is passed over)
      }
  }
  if (threadIdx.x < 256) s.table[threadIdx.x] = exp2(static_cast<double>(threadIdx.x) / 256.0);
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
  if (d.lane == 0) s.warp_m[d.warp] = m;
  if (threadIdx.x == 0) s.best = 0x7fffffff;
  __syncthreads();
  for (int k = 0; k < kWarps; ++k) m = fmaxf(m, s.warp_m[k]);
  if (threadIdx.x == 0) s.m = m;
  d.cluster.sync();
  for (int k = 0; k < d.parts; ++k) m = fmaxf(m, d.cluster.map_shared_rank(&s, k)->m);
  if (m == -INFINITY || !(temperature > 0.f)) {
    int best = 0x7fffffff;
    if (m != -INFINITY) d.each([&](float e, int i) { if (e == m) best = min(best, i); });
    best = __reduce_min_sync(0xffffffffu, best);
    if (d.lane == 0) atomicMin(&s.best, best);
    d.cluster.sync();
    if (d.part == 0 && threadIdx.x == 0) {
      for (int k = 0; k < d.parts; ++k) best = min(best, d.cluster.map_shared_rank(&s, k)->best);
      a.tokens[row] = m == -INFINITY ? -1 : best;
      if (a.chances != nullptr) a.chances[row] = m == -INFINITY ? 0.f : 1.f;
    }
    d.cluster.sync();
    return;
  }
  d.m = m;
  d.md = static_cast<double>(m);
  d.half_scale = 2.f / temperature;
  d.per = 256.0 * kLog2e / static_cast<double>(temperature);
  d.shift = shift;
  d.beyond = static_cast<float>((shift + 1) * kLn2) + 0.5f;

  Kept kept;
  if (top_k > 0 && top_k < d.V) d.limit(kept, false, 1.0, static_cast<u64>(top_k));
  if (top_p < 1.f) d.limit(kept, true, top_p > 0.f ? static_cast<double>(top_p) : 0.0, 0);
  // the least weight, as an integer of the same scale, and the distance behind which no weight reaches it
  u64 least = 1;
  float reach = d.beyond;
  if (min_p > 0.f) {
    least = min_p >= 1.f ? 1ull << shift : static_cast<u64>(ceil(ldexp(static_cast<double>(min_p), shift)));
    reach = fminf(reach, -logf(min_p) * 1.0001f + 1e-3f);
  }
  const auto weigh = [&](float e, int i) -> u64 {
    if (!(d.distance(e) < reach) && e != m) return 0;
    const uint32_t k = key_of(e);
    if (k == 0 || !kept.has(k, i)) return 0;
    const u64 w = d.weight(e);
    return w >= least ? w : 0;
  };
  const u64 total = d.total(weigh);
  u64 target = uniform > 0.f ? static_cast<u64>(static_cast<double>(uniform) * static_cast<double>(total)) : 0;
  if (target >= total) target = total - 1;
  d.find(target, weigh);
  d.cluster.sync();
  if (d.part == 0 && threadIdx.x == 0) {
    a.tokens[row] = s.found;
    if (a.chances != nullptr) a.chances[row] = static_cast<float>(static_cast<double>(s.own) / static_cast<double>(total));
  }
}

const char *check(const myea_sampling *s) {
  if (s == nullptr) return "sample: no description";
  if (s->type > MYEA_TYPE_F16) return "sample: unknown type";
  if (s->rows > kSequenceMost || s->vocabulary > kSequenceMost) return "sample: a dimension above 2^30";
  if (s->rows == 0) return nullptr;
  if (s->vocabulary == 0) return "sample: an empty vocabulary";
  if (s->logits == nullptr || s->uniform == nullptr || s->tokens == nullptr) return "sample: logits, uniform or tokens is missing";
  if (s->rows * kParts > 0x7fffffffull) return "sample: more rows than one launch takes";
  return nullptr;
}

// bits behind the point of a weight: the sum over the vocabulary stays below 2^62
int shift_for(uint64_t vocabulary) {
  int bits = 0;
  while ((uint64_t(1) << bits) < vocabulary) ++bits;
  return 62 - bits < 51 ? 62 - bits : 51;
}

template <typename T, bool RES> cudaError_t launch(const myea_sampling &a, int parts, size_t smem, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(sampling_kernel<T, RES>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sampling_kernel<T, RES>, a, shift_for(a.vocabulary));
}

template <typename T> cudaError_t launch(const myea_sampling &a, cudaStream_t stream) {
  // a slice of at most 64 KB leaves room for two blocks on an SM; more blocks per row while the rows leave SMs idle and a
  // slice has 4096 words
  const uint64_t bytes = a.vocabulary * sizeof(T) + 32;
  int parts = 1;
  while (parts < kParts && (bytes / parts > (64u << 10) || (a.rows * parts * 2 <= 2 * kSms && a.vocabulary / (parts * 2) >= 4096))) parts *= 2;
  const size_t slice = (bytes / parts + 64) / 16 * 16;
  if (sizeof(Shared) + slice > (200u << 10)) return launch<T, false>(a, parts, sizeof(Shared), stream);
  return launch<T, true>(a, parts, sizeof(Shared) + slice, stream);
}

}  // namespace
}  // namespace myea

extern "C" int myea_b200_sample(int device, const myea_sampling *s, void *stream, char *error_message, size_t error_capacity) {
  using namespace myea;
  if (const char *why = check(s)) return refuse(error_message, error_capacity, MYEA_E_INVALID, why);
  if (s->rows == 0) return MYEA_OK;
  DeviceScope scope(device);
  if (!scope.ok) return refuse(error_message, error_capacity, MYEA_E_CUDA, "sample: no such device");
  cudaError_t e = cudaSuccess;
  with_type(s->type, [&](auto t) { e = launch<decltype(t)>(*s, static_cast<cudaStream_t>(stream)); });
  if (e != cudaSuccess) (void)cudaGetLastError();
  if (e != cudaSuccess) return refuse(error_message, error_capacity, MYEA_E_CUDA, "sample: the launch was refused");
  return launched(error_message, error_capacity, "sample");
}
