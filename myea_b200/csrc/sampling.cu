// Draws one token per row from what temperature, top-k, top-p and min-p leave of it (defined at myea_sampling in myea_b200.h).
//
// All three limits keep a prefix of the row ordered by falling logit and rising index, so what is kept is a threshold on the
// logit and, among those equal to it, on the index.  The threshold is found without sorting, by histograms of counts or
// weights: first 1024 bins in the distance from the maximum, which spread the words of any ordinary row, then bins in the logits' bits
// (mapped to integers of the same order) within the bin that holds the threshold, until one value is left.
//
// Weights are integers, w * 2^shift: their sums are exact whatever the order of the atomics, and the same draw is made every
// time.  A draw from 1e5 words goes through as many borders, so a weight good to 24 bits would move a token of every few
// hundred rows; these are good to 2^-45 of the largest one or better.  2^t is a table of 2^(k / 256) times the polynomial 1 + r + ... of the rest
// |r| < 2^-9.5 (its first term left out is below 2^-54), in 64-bit floating point, which this chip does at half the 32-bit rate.
//
// Bound by instructions and, with rows for fewer than two waves of blocks, by a row's chain of passes: 256 rows of 131072 bf16 words take
// 30 us for the largest word alone (2.2 TB/s), 83 for a draw from all words, 118 from the 50 best, 275 from top-p 0.9.  A bound from a
// sample for top-p, too, left out most additions to bins, but its code cost more (335 us).
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
constexpr int kThreads = 256, kWarps = kThreads / 32, kBins = 1024, kParts = 8, kList = 1024, kLongRow = 32;
constexpr size_t kSharedMost = 200u << 10;   // bytes of a block
static_assert(kThreads == 256, "a thread makes one entry of the table");
constexpr double kLog2e64 = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

template <typename T> struct Pack { static constexpr int N = 16 / sizeof(T); uint4 v; };

// integers in the order of the floats
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);   // (both zeros are equal)
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key); }

// What is kept: words above `value`, and those equal to it up to index `last` (closed words, -infinity and NaN, never)
struct Kept {
  float value = -INFINITY;
  int last = -1;
  __device__ __forceinline__ bool has(float e, int i) const { return e > value || (e == value && i <= last); }
};

// the largest of a vector's words, NaN passed over
__device__ __forceinline__ float largest(const uint4 &v, float) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
template <typename H2, typename H> __device__ __forceinline__ float largest_half(const uint4 &v) {
  const H2 *h = reinterpret_cast<const H2 *>(&v);
  const H2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(to_float(m.x), to_float(m.y));
}
__device__ __forceinline__ float largest(const uint4 &v, __nv_bfloat16) { return largest_half<__nv_bfloat162, __nv_bfloat16>(v); }
__device__ __forceinline__ float largest(const uint4 &v, __half) { return largest_half<__half2, __half>(v); }

struct alignas(16) Shared {
  // A histogram: words, and their weights in parts of 16, 16 and more bits (RES: sums of up to 65536 words do not carry), or as the
  // 64 bits of the first two.  Afterwards: the words of the bin that holds the limit.
  unsigned int count[kBins], mass[3][kBins];
  double table[256];                                    // 2^(shift + k / 256)
  u64 warp[kWarps];
  float warp_m[kWarps];
  float m;
  unsigned int key_min, key_max;
  int best, found;
  u64 own;
  // the bin that holds a limit
  int bin;
  unsigned int listed;
  u64 before_count, before_mass, bin_count, bin_mass, total_mass, all_count, all_mass;
  u64 scan_count[kWarps], scan_mass[kWarps];
  float cut_value;
  int cut_last;
  // a list of the bin's words, in the memory of the histogram: key and index, so that larger ones come first
  __device__ __forceinline__ u64 *list() { return reinterpret_cast<u64 *>(mass[0]); }
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
  float lowest;        // words below it weigh nothing
  bool steep;          // the word below m, or one that is not finite, may be too far off for the arithmetic:
  double least_d;      // differences are limited to this
  float own;           // the largest word of this thread
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
  __device__ __forceinline__ Pack<T> words(int v) const {
    Pack<T> p;
    if constexpr (RES) p.v = slice[v - first];
    else p = from_memory(v);
    return p;
  }
  // four of a vector's words, from h on
  static __device__ __forceinline__ float4 words4(const Pack<T> &p, int h) {
    if constexpr (sizeof(T) == 4) {
      return make_float4(__uint_as_float(p.v.x), __uint_as_float(p.v.y), __uint_as_float(p.v.z), __uint_as_float(p.v.w));
    } else {
      Raw4<T> r;
      r.v = h == 0 ? make_uint2(p.v.x, p.v.y) : make_uint2(p.v.z, p.v.w);
      return widen(r);
    }
  }
  __device__ __forceinline__ float distance(float e) const { return (0.5f * m - 0.5f * e) * half_scale; }
  // The weight of a word as an integer.  Most of it is 64-bit floating point, since selects and shifts of 64-bit integers cost more: the
  // rounding to an integer is the addition of 2^52, and words so far off that they round to 0, closed ones among them, stand for one
  // that just does.
  __device__ __forceinline__ u64 weight(float e) const {
    constexpr double magic = 6755399441055744.0, whole = 4503599627370496.0;   // 1.5 * 2^52: the sum's lower bits are the nearest integer; 2^52
    constexpr double c1 = kLn2 / 256, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6, c4 = c1 * c1 * c1 * c1 / 24;
    double d = static_cast<double>(fmaxf(e, lowest)) - md;
    if (steep) d = e == m ? 0.0 : fmax(d, -least_d);
    const double z = fma(d, per, magic);
    const int i = __double2loint(z);
    const double r = fma(d, per, magic - z);
    double q = fma(fma(fma(fma(r, c4, c3), r, c2), r, c1), r, 1.0);
    q *= s.table[i & 255];
    q = __hiloint2double(__double2hiint(q) + static_cast<int>(static_cast<unsigned>(i) << 12 & 0xfff00000u), __double2loint(q)) + whole;   // (times 2^(i >> 8))
    return static_cast<u64>(__double_as_longlong(q)) & ((1ull << 52) - 1);
  }
  // f(word, its index) for this warp's words from `least` up, lanes side by side; vectors without one are passed over
  template <typename F> __device__ __forceinline__ void each(float least, F f) const {
#pragma unroll 1
    for (int v = from + lane; v < to; v += 32) {
      const Pack<T> p = words(v);
      if (!(largest(p.v, T()) >= least)) continue;
      const T *w = reinterpret_cast<const T *>(&p.v);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float e = to_float(w[k]);
        if (e >= least) f(e, v * E + k - lead);
      }
    }
  }
  static __device__ __forceinline__ u64 warp_sum(u64 y) {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) y += __shfl_xor_sync(0xffffffffu, y, k);
    return y;
  }
  // Sums of f, which is 0 below `least`, over the row's words by warps (put into s.warp): their total, in every block
  template <typename F> __device__ u64 total(float least, F f) {
    u64 sum = 0;
    for (int v = from + lane; v < to; v += 32) {
      const Pack<T> p = words(v);
      if (!(largest(p.v, T()) >= least)) continue;
      u64 y[E];
#pragma unroll
      for (int h = 0; h < E; h += 4) {   // four chains of arithmetic at a time
        const float4 e = words4(p, h);
        y[h] = f(e.x, v * E + h - lead); y[h + 1] = f(e.y, v * E + h + 1 - lead); y[h + 2] = f(e.z, v * E + h + 2 - lead); y[h + 3] = f(e.w, v * E + h + 3 - lead);
        sum += (y[h] + y[h + 1]) + (y[h + 2] + y[h + 3]);
      }
    }
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
  // The first index, in rising order, at which the running sum of f exceeds `target` (below the total, after total(least, f)), and f there:
  // known to every block behind the next cluster.sync(), in s.found and s.own
  template <typename F> __device__ void find(float least, u64 target, F f) {
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
    if (at / kWarps != part) return;
    // the block that has it: the warp's part among all its threads, neighbouring words to each
    const int share = (last - first + kWarps - 1) / kWarps, begin = min(first + at % kWarps * share, last), words_ = (min(begin + share, last) - begin) * E;
    const int mine = (words_ + kThreads - 1) / kThreads, w0 = static_cast<int>(threadIdx.x) * mine;
    const auto value = [&](int w) -> u64 {   // of word w of the part
      const int i = begin * E + w - lead;
      if (w >= words_ || i < 0 || i >= V) return 0;
      float e;
      if constexpr (RES) e = to_float(reinterpret_cast<const T *>(slice)[(begin - first) * E + w]);
      else e = to_float(x[i]);
      return e >= least ? f(e, i) : 0;
    };
    u64 sum = 0;
#pragma unroll 1
    for (int k = 0; k < mine; ++k) sum += value(w0 + k);
    u64 upto = sum;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const u64 o = __shfl_up_sync(0xffffffffu, upto, k);
      if (lane >= k) upto += o;
    }
    if (lane == 31) s.scan_count[warp] = upto;
    __syncthreads();
    for (int k = 0; k < warp; ++k) before += s.scan_count[k];
    u64 run = before + upto - sum;
    if (run <= target && run + sum > target) {
#pragma unroll 1
      for (int k = 0; k < mine; ++k) {
        const u64 own = value(w0 + k);
        if (run + own > target) {
          for (int o = 0; o < parts; ++o) {
            Shared *to_ = cluster.map_shared_rank(&s, o);
            to_->found = begin * E + w0 + k - lead;
            to_->own = own;
          }
          break;
        }
        run += own;
      }
    }
  }

  // Counts the words from `least` up by bin(word, index), those with bin < 0 left out; by_mass: and adds up their weights
  template <typename F> __device__ __forceinline__ void histogram(float least, bool by_mass, F bin) {
    if (!by_mass) {
      each(least, [&](float e, int i) {
        const int b = bin(e, i);
        if (b >= 0) atomicAdd(&s.count[b], 1u);
      });
      return;
    }
    for (int v = from + lane; v < to; v += 32) {
      const Pack<T> p = words(v);
      if (!(largest(p.v, T()) >= least)) continue;
#pragma unroll
      for (int h = 0; h < E; h += 4) {   // four chains of arithmetic at a time
        const float4 e4 = words4(p, h);
        const float e[4] = {e4.x, e4.y, e4.z, e4.w};
        u64 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = weight(e[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int b = e[k] >= least ? bin(e[k], v * E + h + k - lead) : -1;
          if (b < 0) continue;
          atomicAdd(&s.count[b], 1u);
          if constexpr (RES) {
            atomicAdd(&s.mass[0][b], static_cast<unsigned>(w[k] & 0xffff));
            atomicAdd(&s.mass[1][b], static_cast<unsigned>(w[k] >> 16) & 0xffffu);
            atomicAdd(&s.mass[2][b], static_cast<unsigned>(w[k] >> 32));
          } else {
            atomicAdd(reinterpret_cast<u64 *>(s.mass[0]) + b, w[k]);
          }
        }
      }
    }
  }
  // Makes a histogram by fill(), over the cluster, and finds the bin that holds the limit: the first, from bin 0 on, with `target`
  // words (or `target` of weight) up to its end.  part_of_all < 1: the target is that part of the whole weight.
  // s.bin is -1 where there is less.  before_count / before_mass: what lies in front of bin 0.
  template <typename F> __device__ void limit_bin(bool by_mass, double part_of_all, u64 target, u64 before_count, u64 before_mass, F fill) {
    for (int k = threadIdx.x; k < kBins; k += kThreads) s.count[k] = s.mass[0][k] = s.mass[1][k] = s.mass[2][k] = 0;
    if (threadIdx.x == 0) { s.bin = -1; s.total_mass = 0; s.listed = 0; }
    __syncthreads();
    fill();
    cluster.sync();
    // Every block adds up its share of the bins (all of them in every block took four times as long): one to four neighbouring bins per
    // thread.
    const int bins = kBins / parts, each_thread = bins > kThreads ? bins / kThreads : 1, mine = static_cast<int>(threadIdx.x) * each_thread;
    const int first_bin = part * bins + mine;
    const auto bin_sums = [&](int k, u64 &c, u64 &w) {   // of bin k, over the blocks
      c = w = 0;
#pragma unroll 4
      for (int o = 0; o < parts; ++o) {
        const Shared *h = cluster.map_shared_rank(&s, o);
        c += h->count[k];
        if (by_mass) {
          if constexpr (RES) w += h->mass[0][k] + (static_cast<u64>(h->mass[1][k]) << 16) + (static_cast<u64>(h->mass[2][k]) << 32);
          else w += reinterpret_cast<const u64 *>(h->mass[0])[k];
        }
      }
    };
    u64 sum_c = 0, sum_w = 0;
    if (mine < bins) {
#pragma unroll 1
      for (int k = 0; k < each_thread; ++k) {
        u64 c, w;
        bin_sums(first_bin + k, c, w);
        sum_c += c;
        sum_w += w;
      }
    }
    u64 upto_c = sum_c, upto_w = sum_w;
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) {
      const u64 oc = __shfl_up_sync(0xffffffffu, upto_c, k), ow = __shfl_up_sync(0xffffffffu, upto_w, k);
      if (lane >= k) { upto_c += oc; upto_w += ow; }
    }
    if (lane == 31) { s.scan_count[warp] = upto_c; s.scan_mass[warp] = upto_w; }
    cluster.sync();
    // the sums of all the warps of all the blocks: up to two per lane
    u64 all_c = 0, all_w = 0, in_front_c = 0, in_front_w = 0;
    for (int k = lane; k < parts * kWarps; k += 32) {
      const Shared *h = cluster.map_shared_rank(&s, k / kWarps);
      const u64 n = h->scan_count[k % kWarps], y = h->scan_mass[k % kWarps];
      all_c += n;
      all_w += y;
      if (k < part * kWarps + warp) { in_front_c += n; in_front_w += y; }
    }
    all_c = warp_sum(all_c);
    before_count += warp_sum(in_front_c) + upto_c - sum_c;
    if (by_mass) {
      all_w = warp_sum(all_w);
      before_mass += warp_sum(in_front_w) + upto_w - sum_w;
    }
    if (part_of_all < 1.0) target = static_cast<u64>(ceil(part_of_all * static_cast<double>(all_w)));
    // the first bin of words with enough up to its end
    const bool enough = by_mass ? before_mass + sum_w >= target : before_count + sum_c >= target;
    const bool was = by_mass ? before_count != 0 && before_mass >= target : before_count >= target;
    if (sum_c != 0 && enough && !was) {
      u64 c, w;
      for (int k = first_bin;; ++k) {
        bin_sums(k, c, w);
        if (c != 0 && (by_mass ? before_mass + w >= target : before_count + c >= target)) {
          for (int o = 0; o < parts; ++o) {
            Shared *to_ = cluster.map_shared_rank(&s, o);
            to_->bin = k;
            to_->before_count = before_count;
            to_->before_mass = before_mass;
            to_->bin_count = c;
            to_->bin_mass = w;
          }
          break;
        }
        before_count += c;
        before_mass += w;
      }
    }
    if (threadIdx.x == 0) { s.total_mass = target; s.all_count = all_c; s.all_mass = all_w; }
    cluster.sync();   // nobody clears its bins, or writes the next sums, while others read them
  }

  // keeps the first `target` words, or those before which less than the part `part_of_all` of the weight of what was kept lies
  __device__ void limit(Kept &kept, bool by_mass, double part_of_all, u64 target) {
    // bins by distance: 32 to a unit, of the logits for counts and of the logarithm of the weights for weights (behind the last
    // bin those weigh nothing: 2^-46)
    const float scale = by_mass ? 32.f * half_scale : 64.f;
    float fine = 1.f;   // the bins are so many times finer
    const auto far = [&](float e) {
      const float t = (0.5f * m - 0.5f * e) * scale * fine;
      return e == m ? 0 : t < static_cast<float>(kBins - 1) ? static_cast<int>(t) : kBins - 1;
    };
    const auto reach_of = [&](float bin) { return (bin + 2.f) * 1.0001f / scale * 2.f; };   // (the words up to that bin, of the first kind, are nearer)
    const Kept was = kept;
    const float lowest_open = fmaxf(was.value, -3.402823466e38f);
    float least = lowest_open;
    u64 before_count = 0, before_mass = 0;
    // Counts in a long row: most words are passed over by a bound that is found first.  So many threads have a word as far up as the
    // limit, so no word below the last of these counts.  (With 16 words per thread the second histogram costs what the bound saves, 19 us
    // for a row of 32000; with 128, 256 rows of 131072 take 118 us in place of 143.)
    if (!by_mass && V >= kLongRow * parts * kThreads && target <= static_cast<u64>(parts) * kThreads) {
      limit_bin(false, 1.0, target, 0, 0, [&]() {
        const int b = own > -INFINITY ? far(own) : kBins - 1;
        if (b < kBins - 1) atomicAdd(&s.count[b], 1u);
      });
      const int bin = s.bin;
      if (bin >= 0) {
        least = fmaxf(least, m - reach_of(bin));
        fine = static_cast<float>(kBins - 2) / ((static_cast<float>(bin) + 2.f) * 1.001f + 1.f);
      }
      __syncthreads();
    }
    // Counts beyond the last bin are taken only when the limit lies there: most words of a row may, and their additions to one bin
    // would wait for one another.
    bool by_distance = true;
    int bin = 0, narrow = 0;
    uint32_t lo = 0, hi = 0, lowest = 0xffffffffu, highest = 0;
#pragma unroll 1
    while (true) {
      limit_bin(by_mass, by_distance && by_mass ? part_of_all : 1.0, target, before_count, before_mass, [&]() {
        histogram(least, by_mass, [&](float e, int i) {
          if (!was.has(e, i)) return -1;
          if (by_distance) {
            const int b = far(e);
            return b < kBins - 1 ? b : -1;
          }
          const uint32_t k = key_of(e);
          return k >= lo && k <= hi ? static_cast<int>((hi - k) >> narrow) : -1;
        });
      });
      const int at = s.bin;
      before_count = at < 0 ? s.all_count : s.before_count;
      before_mass = at < 0 ? s.all_mass : s.before_mass;
      target = s.total_mass;
      __syncthreads();
      if (!by_distance) {
        if (at < 0) return;   // fewer words than the limit
        highest = hi - (static_cast<uint32_t>(at) << narrow);
        lowest = highest - ((1u << narrow) - 1);
        lowest = lowest < lo || lowest > highest ? lo : lowest;
        if (lowest == highest) break;
      } else {
        by_distance = false;
        bin = at;
        if (bin < 0) {   // all words of the bins: the limit lies beyond them, or there are fewer words
          if (by_mass) return;
          bin = kBins - 1;
        } else {
          least = fmaxf(least, m - reach_of(static_cast<float>(bin + 1) / fine));
        }
        if (bin < kBins - 1 && s.bin_count <= kList) {   // few words in the bin: the first block sorts them
          Shared *head = cluster.map_shared_rank(&s, 0);
          each(least, [&](float e, int i) {
            if (far(e) != bin || !was.has(e, i)) return;
            head->list()[atomicAdd(&head->listed, 1u)] = (static_cast<u64>(key_of(e)) << 32) | static_cast<unsigned>(~i);
          });
          cluster.sync();
          if (part == 0) {
            const int n = static_cast<int>(s.listed);
            u64 *list = s.list();
            int size = 1;
            while (size < n) size *= 2;
            for (int j = n + threadIdx.x; j < size; j += kThreads) list[j] = 0;
            __syncthreads();
            for (int run = 2; run <= size; run *= 2)   // (bitonic: comparisons of elements a power of two apart)
              for (int apart = run / 2; apart > 0; apart /= 2) {
                for (int j = threadIdx.x; j < size / 2; j += kThreads) {
                  const int i = 2 * j - (j & (apart - 1)), o = i + apart;
                  const u64 a = list[i], b = list[o];
                  if ((a < b) == ((i & run) == 0)) { list[i] = b; list[o] = a; }
                }
                __syncthreads();
              }
            int keep;   // so many of them
            if (by_mass) {
              constexpr int L = kList / kThreads;
              u64 w[L], sum = 0;
#pragma unroll
              for (int j = 0; j < L; ++j) {
                const int at = threadIdx.x * L + j;
                w[j] = at < n ? weight(value_of(static_cast<uint32_t>(list[at] >> 32))) : 0;
                sum += w[j];
              }
              u64 upto = sum;
#pragma unroll
              for (int k = 1; k < 32; k <<= 1) {
                const u64 o = __shfl_up_sync(0xffffffffu, upto, k);
                if (lane >= k) upto += o;
              }
              if (lane == 31) s.scan_mass[warp] = upto;
              __syncthreads();
              u64 before = before_mass + upto - sum;
              for (int k = 0; k < warp; ++k) before += s.scan_mass[k];
              int mine = 0;
#pragma unroll
              for (int j = 0; j < L; ++j) {
                const int at = threadIdx.x * L + j;
                if (at < n && (before < target || before_count + at == 0)) ++mine;
                before += w[j];
              }
              if (threadIdx.x == 0) s.best = 0;
              __syncthreads();
              mine = __reduce_add_sync(0xffffffffu, mine);
              if (lane == 0) atomicAdd(&s.best, mine);
              __syncthreads();
              keep = s.best;
            } else {
              keep = static_cast<int>(target - before_count);
            }
            if (threadIdx.x < parts) {
              const u64 last_kept = list[keep - 1];
              Shared *to_ = cluster.map_shared_rank(&s, threadIdx.x);
              to_->cut_value = value_of(static_cast<uint32_t>(last_kept >> 32));
              to_->cut_last = static_cast<int>(~static_cast<unsigned>(last_kept));
            }
          }
          cluster.sync();
          kept.value = s.cut_value;
          kept.last = s.cut_last;
          __syncthreads();
          return;
        }
        // the logits in that bin
        if (threadIdx.x == 0) { s.key_min = 0xffffffffu; s.key_max = 0; }
        __syncthreads();
        each(least, [&](float e, int i) {
          if (far(e) == bin && was.has(e, i)) {
            const uint32_t k = key_of(e);
            lowest = min(lowest, k);
            highest = max(highest, k);
          }
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
        if (lowest > highest) return;   // no word there
        if (lowest == highest && bin < kBins - 1) break;   // (the last bin has not been counted)
      }
      lo = lowest;
      hi = highest;
      least = value_of(lo);
      narrow = 0;
      while (((hi - lo) >> narrow) >= kBins) ++narrow;
    }
    const float value = value_of(highest);
    // of the words equal to the threshold
    u64 ties;
    if (by_mass) {
      const u64 one = s.bin_mass / s.bin_count;
      ties = one == 0 ? s.bin_count : target > before_mass ? (target - before_mass + one - 1) / one : 0;
      if (before_count == 0 && ties == 0) ties = 1;
    } else {
      ties = target - before_count;
    }
    if (ties < s.bin_count) {
      kept.last = -1;
      if (ties > 0) {
        const auto tie = [&](float e, int i) -> u64 { return e == value && was.has(e, i) ? 1 : 0; };
        total(value, tie);
        find(value, ties - 1, tie);
        cluster.sync();
        kept.last = s.found;
      }
      kept.value = value;
    } else if (value > kept.value) {
      kept.value = value;
      kept.last = 0x7fffffff;
    }
    __syncthreads();   // what has been read here is written by the next limit
  }
};

template <typename T, bool RES>
__global__ void __launch_bounds__(kThreads, 4) sampling_kernel(const myea_sampling a, int shift) {
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
  const float top_p = a.top_p == nullptr ? 1.f : a.top_p[row], uniform = a.uniform[row];
  float min_p = a.min_p == nullptr ? 0.f : a.min_p[row];
  if (min_p > 1.f) min_p = 1.f;   // (the largest word's weight: it always stays)
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
        m = fmaxf(m, largest(p[u].v, T()));
      }
  }
  d.own = m;
  s.table[threadIdx.x] = ldexp(exp2(static_cast<double>(threadIdx.x) / 256.0), shift);
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
    if (m != -INFINITY) d.each(m, [&](float, int i) { best = min(best, i); });
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
  d.per = fmax(256.0 * kLog2e64 / static_cast<double>(temperature), 1e-300);
  d.shift = shift;
  d.beyond = static_cast<float>((shift + 1) * kLn2) + 0.5f;
  d.least_d = 256.0 * (shift + 2) / d.per;
  d.lowest = __double2float_rd(__dadd_rd(d.md, -d.least_d));   // (below m whatever is rounded off)
  d.steep = !(d.md - static_cast<double>(d.lowest) <= 2.0 * d.least_d);   // (too coarse a float for the distance, or an infinity)
  if (d.steep) d.lowest = -INFINITY;

  Kept kept;
#pragma unroll 1
  for (int by_mass = 0; by_mass < 2; ++by_mass)
    if (by_mass ? top_p < 1.f : top_k > 0 && top_k < d.V)
      d.limit(kept, by_mass, top_p > 0.f ? static_cast<double>(top_p) : 0.0, by_mass ? 0 : static_cast<u64>(top_k));
  // the least weight, as an integer of the same scale, and the distance behind which no weight reaches it
  u64 least = 1;
  float reach = d.beyond;
  if (min_p > 0.f) {
    least = static_cast<u64>(ceil(ldexp(static_cast<double>(min_p), shift)));
    reach = fminf(reach, -logf(min_p) * 1.0001f + 1e-3f);
  }
  const float nearest = fmaxf(m - reach * 1.001f * temperature, fmaxf(kept.value, -3.402823466e38f));
  u64 total = 0;
  const auto draw = [&](auto weigh) {
    total = d.total(nearest, weigh);
    u64 target = uniform > 0.f ? static_cast<u64>(static_cast<double>(uniform) * static_cast<double>(total)) : 0;
    if (target >= total) target = total - 1;
    d.find(nearest, target, weigh);
  };
  if (kept.value == -INFINITY && least == 1) {   // nothing is left out
    draw([&](float e, int) -> u64 { return d.weight(e); });
  } else if (least == 1) {
    draw([&](float e, int i) -> u64 {
      const u64 w = d.weight(e);
      return kept.has(e, i) ? w : 0;
    });
  } else {
    draw([&](float e, int i) -> u64 {
      const u64 w = d.weight(e);
      return kept.has(e, i) && w >= least ? w : 0;
    });
  }
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
  // the most that any call takes, not this call's: the limit belongs to the function, whoever launches it
  cudaError_t e = cudaFuncSetAttribute(sampling_kernel<T, RES>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSharedMost));
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
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sampling_kernel<T, RES>, a, shift_for(a.vocabulary));
}

template <typename T> cudaError_t launch(const myea_sampling &a, cudaStream_t stream) {
  // A slice of some 32 KB leaves room for four blocks on an SM (256 rows of 131072 bf16 words: two of 64 KB took a tenth longer).  More
  // blocks per row while the rows leave SMs idle and a slice has 4096 words.
  const uint64_t bytes = a.vocabulary * sizeof(T) + 32;
  int parts = 1;
  while (parts < kParts && (bytes / parts > (36u << 10) || (a.rows * parts * 2 <= 2 * kSms && a.vocabulary / (parts * 2) >= 4096))) parts *= 2;
  const size_t slice = (bytes / parts + 64) / 16 * 16;
  if (sizeof(Shared) + slice > kSharedMost || slice / sizeof(T) > 65536) return launch<T, false>(a, parts, sizeof(Shared), stream);
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
