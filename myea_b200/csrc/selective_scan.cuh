// Selective state space scan, forward (selective_scan.cu) and backward (selective_scan_backward.cu); the formulas stand at myea_scan
// in myea_b200.h.
//
// The work is one exponential and some four multiply-adds for each (position, channel, state); the arrays in memory hold one
// element per (position, channel).  With 16 states the special-function unit (16 results a cycle and SM) is busy three times as
// long as the memory, and what is done once per element (step length, gate) takes as many issue slots as the states.
//
// Layout: a thread keeps four states of CPT channels in registers, LPC = states / 4 (rounded up to a power of two) neighbouring
// lanes share the channels, a block has NT threads and CH channels of one group and walks over the positions in tiles of 16.  A tile's
// inputs come through registers (loaded one tile ahead, four channels at a time) into shared memory as fp32, after the softplus,
// so that per step a lane reads two words of each channel and four of B and of C.  A word read from shared memory costs a
// cycle of the SM whatever the access's width: two channels per thread share the eight words of B and C (measured with one
// channel: 12 cycles a step of 8 channels and 16 states, more than the exponentials' 8).  Sums over a channel's states leave as up to
// four parts in shared memory and are added where they are read.  Positions behind a sequence's end count as steps of length 0:
// they leave the state as it is.
//
// Few channels and a long time: the time is cut into chunks.  Because A does not depend on time, a chunk's decay is exp(A *
// sum of its steps); a first kernel computes every chunk's state from a zero start, a small one chains them, and the main
// kernel runs all chunks side by side from their true starts.  This costs the exponentials twice.
#pragma once

#include "sequence.cuh"

namespace myea {
namespace scan {

constexpr int TT = 16;   // positions of a tile, and between checkpoints
constexpr float kLog2eRest = 1.925963033500e-8f, kLn2 = 0.6931471805599453f;

struct ScanArgs {
  myea_scan s;
  int batch, time, width, states, groups, per_group;
  int tiles;           // of channels in a group
  int chunk, chunks;   // positions of a chunk (a multiple of TT), chunks
  bool vec_u, vec_delta, vec_z, vec_y, vec_dy, vec_du, vec_ddelta, vec_dz, vec_B, vec_C, vec_dB, vec_dC, vec_A, vec_state, vec_final, vec_d_final, vec_d_state;
  float *carry;        // [batch][chunks][width][NP]: states (errors on the states) of chunks from a zero start, then where they start
  float *steps;        // [batch][chunks][width]: sum of a chunk's step lengths
  float *part_bc;      // [tiles][batch][time][groups][LPC][dB, dC][4]
  float *part_a;       // [batch * chunks][width][NP]
  float *part_d;       // [batch * chunks][dD, d_delta_bias][width]
};

// where the workspace's parts begin, in bytes
struct Layout {
  size_t carry = 0, steps = 0, part_bc = 0, part_a = 0, part_d = 0, bytes = 0;
};

const char *check(const myea_scan *s, bool backward);
ScanArgs arguments(const myea_scan *s);
Layout layout_of(const ScanArgs &a, bool backward);
void place(ScanArgs &a, const Layout &w, void *workspace);
bool too_many_blocks(const ScanArgs &a);   // more than a grid holds, in any launch
int lanes_of(uint64_t states);

template <typename F> void with_lanes(int lanes, F f) {
  switch (lanes) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 8: f(std::integral_constant<int, 8>()); break;
    case 16: f(std::integral_constant<int, 16>()); break;
    default: f(std::integral_constant<int, 32>()); break;
  }
}

#ifdef __CUDACC__
template <int LPC_, int CPT_> struct Shape {
  static constexpr int LPC = LPC_, CPT = CPT_;
  static constexpr int NT = 128;   // threads that walk over the steps; as many do the work per element
  static constexpr int CH = NT * CPT / LPC;                          // channels of a block
  static constexpr int NP = 4 * LPC;                                 // states, padded
  static constexpr int V = TT * CH / 4;                              // groups of four channels in a tile
  static constexpr int VI = V > NT ? V / NT : 1;                     // of them per thread
  static constexpr int BV = TT * LPC;                                // groups of four values in a tile of B or C
  static constexpr int BI = BV > NT ? BV / NT : 1;
  static constexpr int ROWS = (V < NT ? V : NT) / (CH / 4);          // rows that the loading threads cover at once
  // Words of a tile in shared memory.  Values per channel lie twice, as the two halves of the packed arithmetic read them; sums over the
  // states lie in P parts per channel, [position][channel of a thread][thread][part].
  static constexpr int PAIRS = TT * CH * 2;
  static constexpr int P = LPC < 4 ? LPC : 4;
  static constexpr int SUMS = TT * CH * P;
  static constexpr int BC = TT * NP;
};


__device__ __forceinline__ float min_nan(float a, float b) {   // (NaN stays)
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^(s A).  The unit's results lie 2.0e-8 below 2^x on the average of x in -0.35 .. 0 (measured against 64 bits), the same way at every
// step, which a state of long memory adds up: 2^-25 in the exponent takes that off.  (A step of length 0 still keeps the state.)
__device__ __forceinline__ float2 decay2(float2 s, float2 A) { return exp2_fast(fma2(s, A, both(2.98023224e-8f))); }
// A rate as a finite number (NaN stays), so that a step of length 0 has the product 0 and keeps the state whatever its rate
__device__ __forceinline__ float finite_rate(float a) { return max_nan(a, -3.402823466e38f); }
// the rates of four states, for decay2
__device__ __forceinline__ void rates2(float4 a, float2 (&A)[2]) {
  A[0] = make_float2(finite_rate(a.x * kLog2e), finite_rate(a.y * kLog2e));
  A[1] = make_float2(finite_rate(a.z * kLog2e), finite_rate(a.w * kLog2e));
}

// log(1 + e^x) of two values, and its slope.  With e = e^-|x| <= 1 and q = e / (2 + e) <= 1/3:  log(1 + e) = 2 atanh(q) = 2 (q + q^3 / 3 +
// ...), whose first term left out, q^15 / 15, is below 2^-26 of the sum.  The product |x| log2(e) is carried to 48 bits.
template <bool SLOPE> __device__ __forceinline__ float2 softplus2(float2 x, float2 &slope) {
  const float2 a = make_float2(min_nan(fabsf(x.x), 100.f), min_nan(fabsf(x.y), 100.f));
  const float2 h = mul2(a, both(-kLog2e));
  float2 rest = fma2(a, both(-kLog2e), make_float2(-h.x, -h.y));
  rest = fma2(a, both(-kLog2eRest), rest);
  float2 e = exp2_fast(h);
  e = fma2(e, mul2(rest, both(kLn2)), e);
  const float2 q = mul2(e, inverse2(add2(e, both(2.f)))), q2 = mul2(q, q);
  float2 p = fma2(q2, both(2.f / 13.f), both(2.f / 11.f));
  p = fma2(p, q2, both(2.f / 9.f));
  p = fma2(p, q2, both(2.f / 7.f));
  p = fma2(p, q2, both(2.f / 5.f));
  p = fma2(p, q2, both(2.f / 3.f));
  p = fma2(p, q2, both(2.f));
  if (SLOPE) {
    const float2 r = inverse2(add2(e, both(1.f))), er = mul2(e, r);
    slope = make_float2(x.x > 0.f ? r.x : er.x, x.y > 0.f ? r.y : er.y);
  }
  return fma2(p, q, make_float2(max_nan(x.x, 0.f), max_nan(x.y, 0.f)));
}
// the step lengths of four channels (0 where there is no step)
__device__ __forceinline__ float4 step_lengths(float4 raw, float4 bias, bool soft, bool there) {
  float2 s0 = add2(lo(raw), lo(bias)), s1 = add2(hi(raw), hi(bias)), slope;
  if (soft) {
    s0 = softplus2<false>(s0, slope);
    s1 = softplus2<false>(s1, slope);
  }
  return there ? make_float4(s0.x, s0.y, s1.x, s1.y) : make_float4(0.f, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ float4 gated(float4 y, float4 z) {
  float2 sig;
  const float2 a = mul2(lo(y), gate2(lo(z), sig)), b = mul2(hi(y), gate2(hi(z), sig));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 times(float4 a, float4 b) {
  const float2 x = mul2(lo(a), lo(b)), y = mul2(hi(a), hi(b));
  return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ float4 &at4(float *p) { return *reinterpret_cast<float4 *>(p); }
__device__ __forceinline__ const float4 &at4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
// four channels' values, each twice
__device__ __forceinline__ void put_pairs(float *p, float4 v) {
  at4(p) = make_float4(v.x, v.x, v.y, v.y);
  at4(p + 4) = make_float4(v.z, v.z, v.w, v.w);
}

// all warps of a block whose halves run different code: each warp arrives from where it is
__device__ __forceinline__ void meet() { asm volatile("barrier.sync 0;" ::: "memory"); }

// Which channels and positions a block works on, and a thread in it
template <typename S> struct Place {
  int group, first, channels;   // channels: of the block's CH that exist
  int chunk;
  long long b;
  int t0, t1, live;             // positions of the chunk; those from `live` on lie behind the sequence's end
  int c, l, n;                  // this thread's first channel in the block, its lane among the channel's, its first state
  int c4, row;                  // the four channels that it loads and stores, and the first row
  int me;                      // the thread among NT
  bool loads;
  __device__ __forceinline__ Place(const ScanArgs &a, int chunks, int first_chunk) {
    long long id = blockIdx.x;
    const int per = a.tiles * a.groups, tile = static_cast<int>(id % per);
    id /= per;
    chunk = first_chunk + static_cast<int>(id % chunks);
    b = id / chunks;
    group = tile / a.tiles;
    const int in_group = (tile - group * a.tiles) * S::CH;
    first = group * a.per_group + in_group;
    channels = min(S::CH, a.per_group - in_group);
    t0 = chunk * a.chunk;
    t1 = min(t0 + a.chunk, a.time);
    live = min(t1, sequence_length(a.s.lengths, b, a.time));
    me = static_cast<int>(threadIdx.x) % S::NT;   // (a block may have NT threads twice, for two kinds of work)
    c = me / S::LPC * S::CPT;
    l = me % S::LPC;
    n = l * 4;
    c4 = me % (S::CH / 4) * 4;
    row = me / (S::CH / 4);
    loads = S::V >= S::NT || me < S::V;
  }
  __device__ __forceinline__ int have(const ScanArgs &a, int q) const { return c + q < channels ? min(4, a.states - n) : 0; }   // states of channel q that exist
  // four states of this thread's channel q in an array [rows][width][NP]
  __device__ __forceinline__ float4 &states_at(float *array, long long row_, const ScanArgs &a, int q) const {
    return *reinterpret_cast<float4 *>(array + (row_ * a.width + first + c + q) * S::NP + n);
  }
  __device__ __forceinline__ float4 four(const float *p) const { return parameters4(p == nullptr ? nullptr : p + first + c4, channels - c4); }
};

// A thread's place in a [time][channels] array that is read or written tile by tile
template <typename T, typename S> struct ChannelRows {
  T *at;             // the first of its rows, from position 0 of the sequence on
  long long stride;  // of a position
  int n;             // channels that exist, of four; 4 only if they can be accessed at once, 5: one by one
  __device__ __forceinline__ ChannelRows(const myea_view &v, bool vec, const Place<S> &p) {
    at = static_cast<T *>(v.data) + p.b * v.stride_batch + p.row * v.stride_time + p.first + p.c4;
    stride = v.stride_time;
    n = min(4, p.channels - p.c4);
    if (n == 4 && !vec) n = 5;
    if (!p.loads) n = 0;
  }
  __device__ __forceinline__ Raw4<T> load(long long position) const {
    const T *from = at + position * stride;
    if (n == 4) return *reinterpret_cast<const Raw4<T> *>(from);
    return load4(from, n, false);
  }
  __device__ __forceinline__ void store(long long position, float4 x) const {
    T *to = at + position * stride;
    if (n == 4) *reinterpret_cast<Raw4<T> *>(to) = narrow(x, T());
    else store4(to, x, n, false);
  }
};
template <typename T, typename S> struct ChannelTile {
  Raw4<T> raw[S::VI];
  // positions t .. of the block's channels; those from p.live on read as 0
  __device__ __forceinline__ void load(const ChannelRows<T, S> &rows, const Place<S> &p, int t) {
#pragma unroll
    for (int i = 0; i < S::VI; ++i) raw[i] = t + p.row + i * S::ROWS < p.live ? rows.load(t + i * S::ROWS) : zero4<T>();
  }
};
// and one of B or C
template <typename T, typename S> struct StateTile {
  Raw4<T> raw[S::BI];
  __device__ __forceinline__ void load(const myea_view &v, bool vec, const Place<S> &p, int states, int t) {
#pragma unroll
    for (int i = 0; i < S::BI; ++i) {
      const int id = p.me + S::NT * i, at = t + id / S::LPC, n = (id % S::LPC) * 4;
      raw[i] = id < S::BV && at < p.live
                   ? load4(static_cast<const T *>(v.data) + p.b * v.stride_batch + at * v.stride_time + p.group * static_cast<long long>(states) + n, min(4, states - n), vec)
                   : zero4<T>();
    }
  }
  __device__ __forceinline__ void put(float *tile, const Place<S> &p) const {   // [TT][NP]
#pragma unroll
    for (int i = 0; i < S::BI; ++i) {
      const int id = p.me + S::NT * i;
      if (id < S::BV) at4(tile + id * 4) = widen(raw[i]);
    }
  }
};

// the values of a thread's CPT channels at one position of a tile of pairs
template <int CPT> __device__ __forceinline__ void get_pairs(const float *p, float2 (&x)[CPT]) {
  if constexpr (CPT == 2) {
    const float4 v = at4(p);
    x[0] = lo(v);
    x[1] = hi(v);
  } else {
    x[0] = *reinterpret_cast<const float2 *>(p);
  }
}
// What two (channels, steps) of a walk need: inputs, B, C and the decays of the states
template <typename S> struct Steps {
  static constexpr int G = 2 / S::CPT;
  float s[G][S::CPT];
  float2 x[G][S::CPT], decay[G][S::CPT][2];
  float4 b[G], c[G];
  __device__ __forceinline__ void fetch(const float *delta, const float *in, const float *B, const float *C, int k, const float2 (&A)[S::CPT][2], bool with_C) {
#pragma unroll
    for (int j = 0; j < G; ++j) {
      float2 pair[S::CPT];
      get_pairs<S::CPT>(delta + (k + j) * 2 * S::CH, pair);
#pragma unroll
      for (int q = 0; q < S::CPT; ++q) {
        s[j][q] = pair[q].x;
        decay[j][q][0] = decay2(pair[q], A[q][0]);
        decay[j][q][1] = decay2(pair[q], A[q][1]);
      }
      get_pairs<S::CPT>(in + (k + j) * 2 * S::CH, x[j]);
      b[j] = at4(B + (k + j) * S::NP);
      if (with_C) c[j] = at4(C + (k + j) * S::NP);
    }
  }
};
// a thread's part of a sum over the states, y[q] of its channel q; lanes beyond the P-th are added up first
template <typename S> __device__ __forceinline__ void put_part(float *tile, int position, const Place<S> &p, const float (&y)[S::CPT]) {
#pragma unroll
  for (int q = 0; q < S::CPT; ++q) {
    float x = y[q];
#pragma unroll
    for (int m = 4; m < S::LPC; m *= 2) x += __shfl_xor_sync(0xffffffffu, x, m);
    if (S::LPC <= 4 || p.l < 4) tile[((position * S::CPT + q) * (S::NT / S::LPC) + p.me / S::LPC) * S::P + p.l] = x;
  }
}
// the sums of four neighbouring channels
template <typename S> __device__ __forceinline__ float4 get_sums(const float *tile, int position, int c4) {
  constexpr int CPT = S::CPT, TH = S::NT / S::LPC;
  const float *base = tile + (position * CPT * TH + c4 / CPT) * S::P;
  float y[4];
#pragma unroll
  for (int o = 0; o < 4; ++o) {
    const float *from = base + (o % CPT * TH + o / CPT) * S::P;
    if constexpr (S::P == 4) {
      const float4 v = at4(from);
      y[o] = (v.x + v.y) + (v.z + v.w);
    } else if constexpr (S::P == 2) {
      const float2 v = *reinterpret_cast<const float2 *>(from);
      y[o] = v.x + v.y;
    } else {
      y[o] = from[0];
    }
  }
  return make_float4(y[0], y[1], y[2], y[3]);
}

// four states of an fp32 array [..][states] (vec: 16-byte rows) from or to registers
__device__ __forceinline__ float4 load_states(const float *p, int n, bool vec) {
  if (vec && n >= 4) return *reinterpret_cast<const float4 *>(p);
  return parameters4(p, n);
}
__device__ __forceinline__ void store_states(float *p, float2 h0, float2 h1, int n, bool vec) {
  if (vec && n >= 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(h0.x, h0.y, h1.x, h1.y);
  } else {
    if (n > 0) p[0] = h0.x;
    if (n > 1) p[1] = h0.y;
    if (n > 2) p[2] = h1.x;
    if (n > 3) p[3] = h1.y;
  }
}

// Chains the chunks: slot k of `carry` becomes the state before chunk k (backward: the error on the state behind chunk k)
template <int LPC, bool BACKWARD>
__global__ void __launch_bounds__(256) scan_chain_kernel(const ScanArgs a) {
  constexpr int NP = 4 * LPC;
  const long long id = blockIdx.x * 256ll + threadIdx.x;
  const int n = static_cast<int>(id % LPC) * 4;
  const long long row = id / LPC, b = row / a.width, d = row - b * a.width;
  if (b >= a.batch) return;
  const int have = min(4, a.states - n);
  float4 a4 = parameters4(a.s.A + d * a.states + n, have);
  a4 = make_float4(finite_rate(a4.x), finite_rate(a4.y), finite_rate(a4.z), finite_rate(a4.w));
  const float *start = BACKWARD ? a.s.d_final_state : a.s.state;
  float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
  if (start != nullptr) h = load_states(start + row * a.states + n, have, BACKWARD ? a.vec_d_final : a.vec_state);
#pragma unroll 4
  for (int i = 0; i < a.chunks; ++i) {
    const int k = BACKWARD ? a.chunks - 1 - i : i;
    float4 *slot = reinterpret_cast<float4 *>(a.carry + ((b * a.chunks + k) * a.width + d) * NP + n);
    const float4 own = i + 1 < a.chunks ? *slot : h;
    const float s = i + 1 < a.chunks ? a.steps[(b * a.chunks + k) * a.width + d] * kLog2e : 0.f;
    *slot = h;
    h = make_float4(fmaf(exp2_fast(s * a4.x), h.x, own.x), fmaf(exp2_fast(s * a4.y), h.y, own.y), fmaf(exp2_fast(s * a4.z), h.z, own.z),
                    fmaf(exp2_fast(s * a4.w), h.w, own.w));
  }
}
#endif

}  // namespace scan
}  // namespace myea
