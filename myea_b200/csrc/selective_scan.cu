// Selective state space scan, forward and backward (the formulas stand at myea_scan in myea_b200.h).
//
// The work is one exponential and some four multiply-adds for each (position, channel, state); the arrays in memory hold one
// element per (position, channel).  With 16 states the special-function unit (16 exponentials a cycle and SM) takes about
// three times as long as the memory, so that unit bounds the forward pass and the issue slots bound the backward pass.
//
// Layout: a thread keeps four states of one channel in registers, LPC = states / 4 (rounded up to a power of two) neighbouring
// lanes share a channel, a block of 256 threads has 256 / LPC channels of one group and walks over the positions in tiles of
// 16.  A tile's inputs come through registers (loaded one tile ahead, four channels at a time) into shared memory as fp32,
// after the softplus, so that per step a lane reads two words of its channel and four of B and C each.  Sums over a channel's
// states are made for four steps at a time by exchanging halves between the lanes.  Positions behind a sequence's end count as
// steps of length 0: they leave the state as it is.
//
// Few channels and a long time: the time is cut into chunks.  Because A does not depend on time, a chunk's decay is exp(A *
// sum of its steps); a first kernel computes every chunk's state from a zero start, a small one chains them, and the main
// kernel runs all chunks side by side from their true starts.  This costs the exponentials twice.
//
// Backward: with g_t = dy_t C_t + a_{t+1} g_{t+1} (a: the decay of a step)
//   dC_t = sum over channels of dy h_t        dB_t = sum over channels of g s u        du = s sum(g B) + D dy
//   ds = sum(A g a h_{t-1}) + u sum(g B)      dA = sum over t of s g a h_{t-1}
// in tiles from the last to the first: the states of a tile are computed again from the checkpoint before it and stay in
// registers (64 of them), then the tile is walked backwards.  g a h_{t-1} is formed from the kept state rather than as
// g (h_t - s u B): the difference would lose the small values of fast states.  Sums over channels go through lanes, warps and,
// between blocks, partial arrays that a last kernel adds up in a fixed order.
#include "sequence.cuh"

namespace myea {
namespace {

constexpr int TT = 16;   // positions of a tile, and between checkpoints
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct ScanArgs {
  myea_scan s;
  int batch, time, width, states, groups, per_group;
  int tiles;           // of channels in a group
  int chunk, chunks;   // positions of a chunk (a multiple of TT), chunks
  bool vec_u, vec_delta, vec_z, vec_y, vec_dy, vec_du, vec_ddelta, vec_dz, vec_B, vec_C, vec_state, vec_final, vec_d_final, vec_d_state;
  float *carry;        // [batch][chunks][width][NP]: states (errors on the states) of chunks from a zero start, then where they start
  float *steps;        // [batch][chunks][width]: sum of a chunk's step lengths
  float *part_bc;      // [tiles][batch][time][groups][LPC][dB, dC][4]
  float *part_a;       // [batch * chunks][width][NP]
  float *part_d;       // [batch * chunks][dD, d_delta_bias][width]
};

template <int LPC> struct Shape {
  static constexpr int CH = 256 / LPC;       // channels of a block
  static constexpr int CW = 32 / LPC;        // of a warp
  static constexpr int RS = CH + CW;         // pitch of a tile's rows: lanes that write neighbouring steps of CW channels hit different banks
  static constexpr int NP = 4 * LPC;         // states, padded
  static constexpr int V = TT * CH / 4;      // groups of four channels in a tile
  static constexpr int VI = V > 256 ? V / 256 : 1;           // of them per thread
  static constexpr int BV = TT * LPC;        // groups of four values in a tile of B or C
  static constexpr int BI = BV > 256 ? BV / 256 : 1;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 lo(float4 v) { return make_float2(v.x, v.y); }
__device__ __forceinline__ float2 hi(float4 v) { return make_float2(v.z, v.w); }
__device__ __forceinline__ float2 exp2_fast(float2 x) { return make_float2(exp2_fast(x.x), exp2_fast(x.y)); }

__device__ __forceinline__ float step_length(float raw, bool softplus) {
  return softplus ? (raw > 20.f ? raw : log1pf(expf(raw))) : raw;
}

// Which channels and positions a block works on
template <int LPC> struct Place {
  int group, first, channels;   // channels: of the block's CH that exist
  int chunk;
  long long b;
  int t0, t1, length;
  __device__ __forceinline__ Place(const ScanArgs &a, int chunks, int first_chunk) {
    long long id = blockIdx.x;
    const int per = a.tiles * a.groups, tile = static_cast<int>(id % per);
    id /= per;
    chunk = first_chunk + static_cast<int>(id % chunks);
    b = id / chunks;
    group = tile / a.tiles;
    const int in_group = (tile - group * a.tiles) * Shape<LPC>::CH;
    first = group * a.per_group + in_group;
    channels = min(Shape<LPC>::CH, a.per_group - in_group);
    t0 = chunk * a.chunk;
    t1 = min(t0 + a.chunk, a.time);
    length = sequence_length(a.s.lengths, b, a.time);
  }
};

// One tile of a [time][channels] array on its way into shared memory
template <typename T, int LPC> struct ChannelTile {
  using S = Shape<LPC>;
  Raw4<T> raw[S::VI];
  // loads positions t .. of the block's channels; positions from `end` on read as 0
  __device__ __forceinline__ void load(const myea_view &v, bool vec, const Place<LPC> &p, int t, int end) {
    const int c = (threadIdx.x % (S::CH / 4)) * 4;
    const T *base = static_cast<const T *>(v.data) + p.b * v.stride_batch + p.first + c;
#pragma unroll
    for (int i = 0; i < S::VI; ++i) {
      const int at = t + static_cast<int>(threadIdx.x + 256 * i) / (S::CH / 4);
      raw[i] = (S::V >= 256 || threadIdx.x < S::V) && at < end ? load4(base + at * v.stride_time, min(4, p.channels - c), vec) : zero4<T>();
    }
  }
  __device__ __forceinline__ void store(const myea_view &v, bool vec, const Place<LPC> &p, int t, int end, int i, float4 x) const {
    const int c = (threadIdx.x % (S::CH / 4)) * 4;
    const int at = t + static_cast<int>(threadIdx.x + 256 * i) / (S::CH / 4);
    if (at < end) store4(static_cast<T *>(v.data) + p.b * v.stride_batch + at * v.stride_time + p.first + c, x, min(4, p.channels - c), vec);
  }
};
// and one of B or C
template <typename T, int LPC> struct StateTile {
  using S = Shape<LPC>;
  Raw4<T> raw[S::BI];
  __device__ __forceinline__ void load(const myea_view &v, bool vec, const Place<LPC> &p, int states, int t, int end) {
#pragma unroll
    for (int i = 0; i < S::BI; ++i) {
      const int id = threadIdx.x + 256 * i, at = t + id / LPC, n = (id % LPC) * 4;
      raw[i] = id < S::BV && at < end
                   ? load4(static_cast<const T *>(v.data) + p.b * v.stride_batch + at * v.stride_time + p.group * static_cast<long long>(states) + n, min(4, states - n), vec)
                   : zero4<T>();
    }
  }
  __device__ __forceinline__ void put(float *tile) const {   // [TT][NP]
#pragma unroll
    for (int i = 0; i < S::BI; ++i) {
      const int id = threadIdx.x + 256 * i;
      if (id < S::BV) *reinterpret_cast<float4 *>(tile + id * 4) = widen(raw[i]);
    }
  }
};

// tile[t + j][c] = p[j] summed over the LPC lanes of channel c, for four steps: halves change sides until a lane has one step
template <int LPC> __device__ __forceinline__ void put_sums(float *tile, int t, int c, float (&p)[4], int l) {
  constexpr int RS = Shape<LPC>::RS;
  if constexpr (LPC == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) tile[(t + j) * RS + c] = p[j];
  } else {
    const bool up = l & 1;
    float a = up ? p[2] : p[0], b = up ? p[3] : p[1];
    a += __shfl_xor_sync(0xffffffffu, up ? p[0] : p[2], 1);
    b += __shfl_xor_sync(0xffffffffu, up ? p[1] : p[3], 1);
    if constexpr (LPC == 2) {
      tile[(t + 2 * l) * RS + c] = a;
      tile[(t + 2 * l + 1) * RS + c] = b;
    } else {
      const bool up2 = l & 2;
      float s = up2 ? b : a;
      s += __shfl_xor_sync(0xffffffffu, up2 ? a : b, 2);
#pragma unroll
      for (int m = 4; m < LPC; m *= 2) s += __shfl_xor_sync(0xffffffffu, s, m);
      if (l < 4) tile[(t + 2 * (l & 1) + (l >> 1)) * RS + c] = s;
    }
  }
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

// STATES: only the states at the chunks' ends from a zero start, and the sums of their step lengths
template <typename T, int LPC, bool STATES>
__global__ void __launch_bounds__(256) scan_forward_kernel(const ScanArgs a) {
  using S = Shape<LPC>;
  __shared__ __align__(16) float s_delta[TT * S::RS];
  __shared__ __align__(16) float s_in[TT * S::RS];   // step length * input, then the sums over the states
  __shared__ __align__(16) float s_B[TT * S::NP], s_C[STATES ? 4 : TT * S::NP];
  const Place<LPC> p(a, STATES ? a.chunks - 1 : a.chunks, 0);
  const int c = threadIdx.x / LPC, l = threadIdx.x % LPC, n = l * 4;
  const int have = c < p.channels ? min(4, a.states - n) : 0;   // states that exist
  const long long d = p.first + c;                              // this lane's channel in the scan,
  const int c4 = (threadIdx.x % (S::CH / 4)) * 4;               // and the four it loads and stores
  const bool loads = S::V >= 256 || threadIdx.x < S::V;
  const float4 bias = parameters4(a.s.delta_bias == nullptr ? nullptr : a.s.delta_bias + p.first + c4, p.channels - c4);
  const float4 skip = STATES ? make_float4(0.f, 0.f, 0.f, 0.f) : parameters4(a.s.D == nullptr ? nullptr : a.s.D + p.first + c4, p.channels - c4);
  const float4 a4 = parameters4(a.s.A + d * a.states + n, have);
  const float2 A0 = make_float2(a4.x * kLog2e, a4.y * kLog2e), A1 = make_float2(a4.z * kLog2e, a4.w * kLog2e);
  float2 h0 = both(0.f), h1 = both(0.f);
  if (!STATES) {
    float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.chunks > 1) {
      if (have > 0) h = *reinterpret_cast<const float4 *>(a.carry + ((p.b * a.chunks + p.chunk) * a.width + d) * S::NP + n);
    } else if (a.s.state != nullptr) {
      h = load_states(a.s.state + (p.b * a.width + d) * a.states + n, have, a.vec_state);
    }
    h0 = lo(h); h1 = hi(h);
  }
  float sum = 0.f;
  const int live = min(p.t1, p.length);
  ChannelTile<T, LPC> u, delta, z, u_next, z_next;
  StateTile<T, LPC> B, C;
  u.load(a.s.u, a.vec_u, p, p.t0, live);
  delta.load(a.s.delta, a.vec_delta, p, p.t0, live);
  B.load(a.s.B, a.vec_B, p, a.states, p.t0, live);
  if (!STATES) {
    C.load(a.s.C, a.vec_C, p, a.states, p.t0, live);
    if (a.s.z.data != nullptr) z.load(a.s.z, a.vec_z, p, p.t0, live);
  }
  for (int t = p.t0; t < p.t1; t += TT) {
    if (loads) {
#pragma unroll
      for (int i = 0; i < S::VI; ++i) {
        const int row = static_cast<int>(threadIdx.x + 256 * i) / (S::CH / 4);
        const float4 raw = widen(delta.raw[i]), x = widen(u.raw[i]);
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (t + row < live)
          s = make_float4(step_length(raw.x + bias.x, a.s.softplus), step_length(raw.y + bias.y, a.s.softplus), step_length(raw.z + bias.z, a.s.softplus),
                          step_length(raw.w + bias.w, a.s.softplus));
        float *to_delta = s_delta + row * S::RS + c4, *to_in = s_in + row * S::RS + c4;
        to_delta[0] = s.x; to_delta[1] = s.y; to_delta[2] = s.z; to_delta[3] = s.w;
        to_in[0] = s.x * x.x; to_in[1] = s.y * x.y; to_in[2] = s.z * x.z; to_in[3] = s.w * x.w;
      }
    }
    B.put(s_B);
    if (!STATES) C.put(s_C);
    __syncthreads();
    if (t + TT < p.t1) {   // the next tile is on its way while this one is computed
      u_next.load(a.s.u, a.vec_u, p, t + TT, live);
      delta.load(a.s.delta, a.vec_delta, p, t + TT, live);
      B.load(a.s.B, a.vec_B, p, a.states, t + TT, live);
      if (!STATES) {
        C.load(a.s.C, a.vec_C, p, a.states, t + TT, live);
        if (a.s.z.data != nullptr) z_next.load(a.s.z, a.vec_z, p, t + TT, live);
      }
    }
    if (!STATES && a.s.checkpoints != nullptr && c < p.channels)
      *reinterpret_cast<float4 *>(a.s.checkpoints + ((p.b * ((a.time + TT - 1) / TT) + t / TT) * a.width + d) * S::NP + n) = make_float4(h0.x, h0.y, h1.x, h1.y);
    const int count = min(TT, p.t1 - t);
#pragma unroll 2
    for (int k = 0; k < count; k += 4) {   // (steps behind the last one have length 0)
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float s = s_delta[(k + j) * S::RS + c], in = s_in[(k + j) * S::RS + c];
        const float4 b4 = *reinterpret_cast<const float4 *>(s_B + (k + j) * S::NP + n);
        const float2 d0 = exp2_fast(mul2(both(s), A0)), d1 = exp2_fast(mul2(both(s), A1));
        h0 = fma2(d0, h0, mul2(both(in), lo(b4)));
        h1 = fma2(d1, h1, mul2(both(in), hi(b4)));
        if (STATES) {
          sum += s;
        } else {
          const float4 c4v = *reinterpret_cast<const float4 *>(s_C + (k + j) * S::NP + n);
          const float2 q = fma2(h1, hi(c4v), mul2(h0, lo(c4v)));
          y[j] = q.x + q.y;
        }
      }
      if (!STATES) {
        __syncwarp();   // (the lanes of this warp alone read these columns)
        put_sums<LPC>(s_in, k, c, y, l);
      }
    }
    __syncthreads();
    if (!STATES && loads) {
#pragma unroll
      for (int i = 0; i < S::VI; ++i) {
        const int row = static_cast<int>(threadIdx.x + 256 * i) / (S::CH / 4);
        const float4 x = widen(u.raw[i]);
        const float *from = s_in + row * S::RS + c4;
        float4 y = make_float4(fmaf(skip.x, x.x, from[0]), fmaf(skip.y, x.y, from[1]), fmaf(skip.z, x.z, from[2]), fmaf(skip.w, x.w, from[3]));
        if (a.s.z.data != nullptr) {
          const float4 g = widen(z.raw[i]);
          y.x *= g.x * sigmoid(g.x); y.y *= g.y * sigmoid(g.y); y.z *= g.z * sigmoid(g.z); y.w *= g.w * sigmoid(g.w);
        }
        if (t + row >= live) y = make_float4(0.f, 0.f, 0.f, 0.f);
        u.store(a.s.y, a.vec_y, p, t, p.t1, i, y);
      }
      u = u_next;
      z = z_next;
    } else if (STATES) {
      u = u_next;
    }
  }
  if (STATES) {
    if (c < p.channels) {
      *reinterpret_cast<float4 *>(a.carry + ((p.b * a.chunks + p.chunk) * a.width + d) * S::NP + n) = make_float4(h0.x, h0.y, h1.x, h1.y);
      if (l == 0) a.steps[(p.b * a.chunks + p.chunk) * a.width + d] = sum;
    }
  } else if (a.s.final_state != nullptr && p.chunk == a.chunks - 1 && have > 0) {
    store_states(a.s.final_state + (p.b * a.width + d) * a.states + n, h0, h1, have, a.vec_final);
  }
}

// Chains the chunks: slot k of `carry` becomes the state before chunk k (backward: the error on the state behind chunk k)
template <int LPC, bool BACKWARD>
__global__ void __launch_bounds__(256) scan_chain_kernel(const ScanArgs a) {
  constexpr int NP = Shape<LPC>::NP;
  const long long id = blockIdx.x * 256ll + threadIdx.x;
  const int n = static_cast<int>(id % LPC) * 4;
  const long long row = id / LPC, b = row / a.width, d = row - b * a.width;
  if (b >= a.batch) return;
  const int have = min(4, a.states - n);
  const float4 a4 = parameters4(a.s.A + d * a.states + n, have);
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

// error on y before the gate
__device__ __forceinline__ float4 before_gate(float4 dy, float4 z) {
  return make_float4(dy.x * z.x * sigmoid(z.x), dy.y * z.y * sigmoid(z.y), dy.z * z.z * sigmoid(z.z), dy.w * z.w * sigmoid(z.w));
}

// Errors on the state before each chunk when nothing comes from behind it, and the sums of the chunks' step lengths
template <typename T, int LPC>
__global__ void __launch_bounds__(256) scan_backward_states_kernel(const ScanArgs a) {
  using S = Shape<LPC>;
  __shared__ __align__(16) float s_delta[TT * S::RS];
  __shared__ __align__(16) float s_dy[TT * S::RS];
  __shared__ __align__(16) float s_C[TT * S::NP];
  const Place<LPC> p(a, a.chunks - 1, 1);
  const int c = threadIdx.x / LPC, l = threadIdx.x % LPC, n = l * 4;
  const int have = c < p.channels ? min(4, a.states - n) : 0;
  const long long d = p.first + c;
  const int c4 = (threadIdx.x % (S::CH / 4)) * 4;
  const bool loads = S::V >= 256 || threadIdx.x < S::V;
  const float4 bias = parameters4(a.s.delta_bias == nullptr ? nullptr : a.s.delta_bias + p.first + c4, p.channels - c4);
  const float4 a4 = parameters4(a.s.A + d * a.states + n, have);
  const float2 A0 = make_float2(a4.x * kLog2e, a4.y * kLog2e), A1 = make_float2(a4.z * kLog2e, a4.w * kLog2e);
  float2 g0 = both(0.f), g1 = both(0.f);
  float sum = 0.f;
  const int live = min(p.t1, p.length);
  ChannelTile<T, LPC> delta, z, dy;
  StateTile<T, LPC> C;
  int t = p.t0 + (p.t1 - p.t0 - 1) / TT * TT;
  delta.load(a.s.delta, a.vec_delta, p, t, live);
  dy.load(a.s.dy, a.vec_dy, p, t, live);
  C.load(a.s.C, a.vec_C, p, a.states, t, live);
  if (a.s.z.data != nullptr) z.load(a.s.z, a.vec_z, p, t, live);
  for (; t >= p.t0; t -= TT) {
    if (loads) {
#pragma unroll
      for (int i = 0; i < S::VI; ++i) {
        const int row = static_cast<int>(threadIdx.x + 256 * i) / (S::CH / 4);
        const float4 raw = widen(delta.raw[i]);
        float4 e = widen(dy.raw[i]), s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (a.s.z.data != nullptr) e = before_gate(e, widen(z.raw[i]));
        if (t + row < live)
          s = make_float4(step_length(raw.x + bias.x, a.s.softplus), step_length(raw.y + bias.y, a.s.softplus), step_length(raw.z + bias.z, a.s.softplus),
                          step_length(raw.w + bias.w, a.s.softplus));
        float *to_delta = s_delta + row * S::RS + c4, *to_dy = s_dy + row * S::RS + c4;
        to_delta[0] = s.x; to_delta[1] = s.y; to_delta[2] = s.z; to_delta[3] = s.w;
        to_dy[0] = e.x; to_dy[1] = e.y; to_dy[2] = e.z; to_dy[3] = e.w;
      }
    }
    C.put(s_C);
    __syncthreads();
    if (t - TT >= p.t0) {
      delta.load(a.s.delta, a.vec_delta, p, t - TT, live);
      dy.load(a.s.dy, a.vec_dy, p, t - TT, live);
      C.load(a.s.C, a.vec_C, p, a.states, t - TT, live);
      if (a.s.z.data != nullptr) z.load(a.s.z, a.vec_z, p, t - TT, live);
    }
#pragma unroll 4
    for (int k = TT - 1; k >= 0; --k) {
      const float s = s_delta[k * S::RS + c], e = s_dy[k * S::RS + c];
      const float4 c4v = *reinterpret_cast<const float4 *>(s_C + k * S::NP + n);
      g0 = mul2(exp2_fast(mul2(both(s), A0)), fma2(both(e), lo(c4v), g0));
      g1 = mul2(exp2_fast(mul2(both(s), A1)), fma2(both(e), hi(c4v), g1));
      sum += s;
    }
    __syncthreads();
  }
  if (c < p.channels) {
    *reinterpret_cast<float4 *>(a.carry + ((p.b * a.chunks + p.chunk) * a.width + d) * S::NP + n) = make_float4(g0.x, g0.y, g1.x, g1.y);
    if (l == 0) a.steps[(p.b * a.chunks + p.chunk) * a.width + d] = sum;
  }
}

// v[0..7] summed over the channels of a warp (lanes that differ in multiples of LPC): halves change sides for up to three
// rounds, so that a lane ends with 8 >> rounds of them, from `first` on
template <int LPC> __device__ __forceinline__ int sum_over_channels(float (&v)[8], int lane) {
  int first = 0;
  if constexpr (LPC < 32) {
    const bool up = lane & LPC;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float keep = up ? v[i + 4] : v[i], send = up ? v[i] : v[i + 4];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, LPC);
    }
    first += up ? 4 : 0;
  }
  if constexpr (LPC < 16) {
    const bool up = lane & (2 * LPC);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float keep = up ? v[i + 2] : v[i], send = up ? v[i] : v[i + 2];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, 2 * LPC);
    }
    first += up ? 2 : 0;
  }
  if constexpr (LPC < 8) {
    const bool up = lane & (4 * LPC);
    const float keep = up ? v[1] : v[0], send = up ? v[0] : v[1];
    v[0] = keep + __shfl_xor_sync(0xffffffffu, send, 4 * LPC);
    first += up ? 1 : 0;
  }
#pragma unroll
  for (int m = 8 * LPC; m < 32; m *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], m);
  return first;
}

template <int LPC> constexpr size_t backward_smem() {
  using S = Shape<LPC>;
  return (4 * TT * S::RS + 2 * TT * S::NP + 8 * TT * 8 * LPC) * sizeof(float);
}

template <typename T, int LPC>
__global__ void __launch_bounds__(256) scan_backward_kernel(const ScanArgs a) {
  using S = Shape<LPC>;
  extern __shared__ __align__(16) float shared[];
  float *s_B = shared, *s_C = s_B + TT * S::NP;
  float *s_part = s_C + TT * S::NP;                    // [warp][TT][LPC][dB, dC][4]
  float *s_delta = s_part + 8 * TT * 8 * LPC;
  float *s_in = s_delta + TT * S::RS, *s_dy = s_in + TT * S::RS;   // later: sum(g B), sum(A g a h)
  float *s_y = s_dy + TT * S::RS;
  const Place<LPC> p(a, a.chunks, 0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = threadIdx.x / LPC, l = threadIdx.x % LPC, n = l * 4;
  const int have = c < p.channels ? min(4, a.states - n) : 0;
  const long long d = p.first + c;
  const int c4 = (threadIdx.x % (S::CH / 4)) * 4;
  const bool loads = S::V >= 256 || threadIdx.x < S::V;
  const bool gate = a.s.z.data != nullptr;
  const float4 bias = parameters4(a.s.delta_bias == nullptr ? nullptr : a.s.delta_bias + p.first + c4, p.channels - c4);
  const float4 skip = parameters4(a.s.D == nullptr ? nullptr : a.s.D + p.first + c4, p.channels - c4);
  const float4 a4 = parameters4(a.s.A + d * a.states + n, have);
  const float2 A0 = make_float2(a4.x * kLog2e, a4.y * kLog2e), A1 = make_float2(a4.z * kLog2e, a4.w * kLog2e);
  float2 g0 = both(0.f), g1 = both(0.f), dA0 = both(0.f), dA1 = both(0.f);   // g: the error that comes from the later step
  {
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.chunks > 1) {
      if (have > 0) g = *reinterpret_cast<const float4 *>(a.carry + ((p.b * a.chunks + p.chunk) * a.width + d) * S::NP + n);
    } else if (a.s.d_final_state != nullptr) {
      g = load_states(a.s.d_final_state + (p.b * a.width + d) * a.states + n, have, a.vec_d_final);
    }
    g0 = lo(g); g1 = hi(g);
  }
  float4 sum_D = make_float4(0.f, 0.f, 0.f, 0.f), sum_bias = sum_D;
  const int live = min(p.t1, p.length);
  ChannelTile<T, LPC> u, delta, z, dy;
  StateTile<T, LPC> B, C;
  const float *kept = a.s.checkpoints + (p.b * ((a.time + TT - 1) / TT) * a.width + d) * S::NP + n;
  for (int t = p.t1 > p.t0 ? p.t0 + (p.t1 - p.t0 - 1) / TT * TT : p.t0 - TT; t >= p.t0; t -= TT) {
    u.load(a.s.u, a.vec_u, p, t, live);
    delta.load(a.s.delta, a.vec_delta, p, t, live);
    dy.load(a.s.dy, a.vec_dy, p, t, live);
    B.load(a.s.B, a.vec_B, p, a.states, t, live);
    C.load(a.s.C, a.vec_C, p, a.states, t, live);
    if (gate) z.load(a.s.z, a.vec_z, p, t, live);
    float4 start = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < p.channels) start = *reinterpret_cast<const float4 *>(kept + static_cast<long long>(t / TT) * a.width * S::NP);
    if (loads) {
#pragma unroll
      for (int i = 0; i < S::VI; ++i) {
        const int row = static_cast<int>(threadIdx.x + 256 * i) / (S::CH / 4);
        const float4 raw = widen(delta.raw[i]), x = widen(u.raw[i]);
        float4 e = widen(dy.raw[i]), s = make_float4(0.f, 0.f, 0.f, 0.f);
        if (gate) e = before_gate(e, widen(z.raw[i]));
        if (t + row < live)
          s = make_float4(step_length(raw.x + bias.x, a.s.softplus), step_length(raw.y + bias.y, a.s.softplus), step_length(raw.z + bias.z, a.s.softplus),
                          step_length(raw.w + bias.w, a.s.softplus));
        const int at = row * S::RS + c4;
        s_delta[at] = s.x; s_delta[at + 1] = s.y; s_delta[at + 2] = s.z; s_delta[at + 3] = s.w;
        s_in[at] = s.x * x.x; s_in[at + 1] = s.y * x.y; s_in[at + 2] = s.z * x.z; s_in[at + 3] = s.w * x.w;
        s_dy[at] = e.x; s_dy[at + 1] = e.y; s_dy[at + 2] = e.z; s_dy[at + 3] = e.w;
      }
    }
    B.put(s_B);
    C.put(s_C);
    __syncthreads();
    // the tile's states, and y for the gate's derivative
    float2 H0[TT], H1[TT];
    {
      float2 h0 = lo(start), h1 = hi(start);
#pragma unroll
      for (int k = 0; k < TT; k += 4) {
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float s = s_delta[(k + j) * S::RS + c], in = s_in[(k + j) * S::RS + c];
          const float4 b4 = *reinterpret_cast<const float4 *>(s_B + (k + j) * S::NP + n);
          h0 = fma2(exp2_fast(mul2(both(s), A0)), h0, mul2(both(in), lo(b4)));
          h1 = fma2(exp2_fast(mul2(both(s), A1)), h1, mul2(both(in), hi(b4)));
          H0[k + j] = h0;
          H1[k + j] = h1;
          if (gate) {
            const float4 c4v = *reinterpret_cast<const float4 *>(s_C + (k + j) * S::NP + n);
            const float2 q = fma2(h1, hi(c4v), mul2(h0, lo(c4v)));
            y[j] = q.x + q.y;
          }
        }
        if (gate) put_sums<LPC>(s_y, k, c, y, l);
      }
    }
#pragma unroll
    for (int k = TT - 4; k >= 0; k -= 4) {
      float sum_gB[4], sum_Aq[4];
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        const int i = k + j;
        const float s = s_delta[i * S::RS + c], in = s_in[i * S::RS + c], e = s_dy[i * S::RS + c];
        const float4 b4 = *reinterpret_cast<const float4 *>(s_B + i * S::NP + n), c4v = *reinterpret_cast<const float4 *>(s_C + i * S::NP + n);
        g0 = fma2(both(e), lo(c4v), g0);
        g1 = fma2(both(e), hi(c4v), g1);
        const float2 dB0 = mul2(g0, both(in)), dB1 = mul2(g1, both(in)), dC0 = mul2(both(e), H0[i]), dC1 = mul2(both(e), H1[i]);
        const float2 gB = fma2(g1, hi(b4), mul2(g0, lo(b4)));
        sum_gB[j] = gB.x + gB.y;
        g0 = mul2(g0, exp2_fast(mul2(both(s), A0)));
        g1 = mul2(g1, exp2_fast(mul2(both(s), A1)));
        const float2 q0 = mul2(g0, i > 0 ? H0[i > 0 ? i - 1 : 0] : lo(start)), q1 = mul2(g1, i > 0 ? H1[i > 0 ? i - 1 : 0] : hi(start));
        dA0 = fma2(q0, both(s), dA0);
        dA1 = fma2(q1, both(s), dA1);
        const float2 Aq = fma2(q1, A1, mul2(q0, A0));
        sum_Aq[j] = Aq.x + Aq.y;
        float v[8] = {dB0.x, dB0.y, dB1.x, dB1.y, dC0.x, dC0.y, dC1.x, dC1.y};
        const int first = sum_over_channels<LPC>(v, lane);
        constexpr int left = LPC >= 32 ? 8 : LPC == 16 ? 4 : LPC == 8 ? 2 : 1;
        if (lane < 8 * LPC) {
#pragma unroll
          for (int o = 0; o < left; ++o) s_part[((warp * TT + i) * LPC + l) * 8 + first + o] = v[o];
        }
      }
      __syncwarp();
      put_sums<LPC>(s_in, k, c, sum_gB, l);
      put_sums<LPC>(s_dy, k, c, sum_Aq, l);
    }
    __syncthreads();
    if (loads) {
#pragma unroll
      for (int i = 0; i < S::VI; ++i) {
        const int row = static_cast<int>(threadIdx.x + 256 * i) / (S::CH / 4), at = row * S::RS + c4;
        const float4 raw = widen(delta.raw[i]), x4 = widen(u.raw[i]), z4 = gate ? widen(z.raw[i]) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 e4 = widen(dy.raw[i]);
        const float r[4] = {raw.x + bias.x, raw.y + bias.y, raw.z + bias.z, raw.w + bias.w}, x[4] = {x4.x, x4.y, x4.z, x4.w};
        const float g[4] = {z4.x, z4.y, z4.z, z4.w}, e[4] = {e4.x, e4.y, e4.z, e4.w}, D[4] = {skip.x, skip.y, skip.z, skip.w};
        float du[4], ds[4], dz[4], dD[4];
        const bool on = t + row < live;
#pragma unroll
        for (int o = 0; o < 4; ++o) {
          const float s = s_delta[at + o], gB = s_in[at + o], Aq = s_dy[at + o];
          float ey = e[o];
          dz[o] = 0.f;
          if (gate) {
            const float sg = sigmoid(g[o]);
            dz[o] = on ? e[o] * fmaf(D[o], x[o], s_y[at + o]) * sg * (1.f + g[o] * (1.f - sg)) : 0.f;
            ey *= g[o] * sg;
          }
          du[o] = on ? fmaf(gB, s, D[o] * ey) : 0.f;
          ds[o] = on ? fmaf(gB, x[o], Aq * kLn2) * (a.s.softplus ? sigmoid(r[o]) : 1.f) : 0.f;
          dD[o] = on ? ey * x[o] : 0.f;
        }
        sum_D.x += dD[0]; sum_D.y += dD[1]; sum_D.z += dD[2]; sum_D.w += dD[3];
        sum_bias.x += ds[0]; sum_bias.y += ds[1]; sum_bias.z += ds[2]; sum_bias.w += ds[3];
        u.store(a.s.du, a.vec_du, p, t, p.t1, i, make_float4(du[0], du[1], du[2], du[3]));
        u.store(a.s.ddelta, a.vec_ddelta, p, t, p.t1, i, make_float4(ds[0], ds[1], ds[2], ds[3]));
        if (gate) u.store(a.s.dz, a.vec_dz, p, t, p.t1, i, make_float4(dz[0], dz[1], dz[2], dz[3]));
      }
    }
    // the block's share of dB and dC: warps in their order
    float *to = a.part_bc + ((((p.first - p.group * a.per_group) / S::CH * static_cast<long long>(a.batch) + p.b) * a.time + t) * a.groups + p.group) * (8 * LPC);
    for (int o = threadIdx.x; o < TT * 8 * LPC; o += 256) {
      const int row = o / (8 * LPC);
      if (t + row >= p.t1) break;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) sum += s_part[w * TT * 8 * LPC + o];
      to[static_cast<long long>(row) * a.groups * (8 * LPC) + (o - row * 8 * LPC)] = sum;
    }
    __syncthreads();
  }
  if (c < p.channels)
    *reinterpret_cast<float4 *>(a.part_a + ((p.b * a.chunks + p.chunk) * a.width + d) * S::NP + n) = make_float4(dA0.x, dA0.y, dA1.x, dA1.y);
  if (a.s.d_state != nullptr && p.chunk == 0 && have > 0) store_states(a.s.d_state + (p.b * a.width + d) * a.states + n, g0, g1, have, a.vec_d_state);
  // sums over the block's positions of what the loading threads have: rows of CH channels, added in their order
  constexpr int rows = (S::V < 256 ? S::V : 256) / (S::CH / 4);
  float *join = s_delta;   // [2][rows][CH] fits the tiles of the step lengths and inputs
  __syncthreads();
  if (loads) {
    const int at = static_cast<int>(threadIdx.x) / (S::CH / 4) * S::CH + c4;
    *reinterpret_cast<float4 *>(join + at) = sum_D;
    *reinterpret_cast<float4 *>(join + rows * S::CH + at) = sum_bias;
  }
  __syncthreads();
  for (int o = threadIdx.x; o < 2 * S::CH; o += 256) {
    const int k = o / S::CH, ch = o - k * S::CH;
    float sum = 0.f;
    for (int r = 0; r < rows; ++r) sum += join[(k * rows + r) * S::CH + ch];
    if (ch < p.channels) a.part_d[((p.b * a.chunks + p.chunk) * 2 + k) * a.width + p.first + ch] = sum;
  }
}

// Adds up the partial sums: blocks 0 .. of dB and dC, then dA, then dD and d_delta_bias
template <typename T, int LPC>
__global__ void __launch_bounds__(256) scan_finish_kernel(const ScanArgs a, long long blocks_bc, long long blocks_a) {
  constexpr int NP = Shape<LPC>::NP;
  const long long block = blockIdx.x, rows = static_cast<long long>(a.batch) * a.chunks;
  if (block < blocks_bc) {
    sum_partials_block(a.part_bc, a.tiles, static_cast<long long>(a.batch) * a.time * a.groups * 8 * LPC, block, [&](long long column, float sum) {
      const int e = static_cast<int>(column % (8 * LPC)), n = e / 8 * 4 + e % 4;
      long long at = column / (8 * LPC);
      const int g = static_cast<int>(at % a.groups);
      at /= a.groups;
      const int t = static_cast<int>(at % a.time);
      const myea_view &v = (e & 4) ? a.s.dC : a.s.dB;
      if (n < a.states) static_cast<T *>(v.data)[at / a.time * v.stride_batch + t * v.stride_time + g * static_cast<long long>(a.states) + n] = from_float<T>(sum);
    });
  } else if (block < blocks_bc + blocks_a) {
    sum_partials_block(a.part_a, rows, static_cast<long long>(a.width) * NP, block - blocks_bc, [&](long long column, float sum) {
      const int n = static_cast<int>(column % NP);
      float *to = a.s.d_A + column / NP * a.states + n;
      if (n < a.states) *to = a.s.accumulate ? *to + sum : sum;
    });
  } else {
    sum_partials_block(a.part_d, rows, 2ll * a.width, block - blocks_bc - blocks_a, [&](long long column, float sum) {
      float *to = column < a.width ? (a.s.d_D == nullptr ? nullptr : a.s.d_D + column) : (a.s.d_delta_bias == nullptr ? nullptr : a.s.d_delta_bias + column - a.width);
      if (to != nullptr) *to = a.s.accumulate ? *to + sum : sum;
    });
  }
}

int lanes_of(uint64_t states) {
  int lpc = 1;
  while (lpc * 4 < static_cast<int>(states)) lpc *= 2;
  return lpc;
}

const char *check(const myea_scan *s, bool backward) {
  if (s == nullptr) return "selective_scan: no description";
  if (s->type > MYEA_TYPE_F16) return "selective_scan: unknown type";
  if (s->states < 1 || s->states > 128) return "selective_scan: 1 to 128 states";
  if (s->batch > kSequenceMost || s->time > kSequenceMost || s->width > kSequenceMost) return "selective_scan: a dimension above 2^30";
  if (s->groups < 1 || (s->width % s->groups) != 0) return "selective_scan: the groups have to divide the width";
  if (s->batch == 0 || s->width == 0) return nullptr;
  if (s->A == nullptr) return "selective_scan: no decay rates (A)";
  if (s->time > 0 && (s->u.data == nullptr || s->delta.data == nullptr || s->B.data == nullptr || s->C.data == nullptr)) return "selective_scan: u, delta, B or C is missing";
  if (s->checkpoints != nullptr && !aligned(s->checkpoints, 16)) return "selective_scan: checkpoints that are not 16-byte aligned";
  if (!backward) {
    if (s->time > 0 && s->y.data == nullptr) return "selective_scan: no output";
    if (s->time > 0 && (s->y.data == s->u.data || s->y.data == s->delta.data || s->y.data == s->B.data || s->y.data == s->C.data || s->y.data == s->z.data))
      return "selective_scan: the output may not be an input's array";
    return nullptr;
  }
  if (s->time > 0 && (s->dy.data == nullptr || s->du.data == nullptr || s->ddelta.data == nullptr || s->dB.data == nullptr || s->dC.data == nullptr))
    return "selective_scan: dy, du, ddelta, dB or dC is missing";
  if (s->time > 0 && (s->z.data != nullptr) != (s->dz.data != nullptr)) return "selective_scan: dz goes with z";
  if (s->time > 0 && s->checkpoints == nullptr) return "selective_scan: the backward pass needs the forward pass's checkpoints";
  if (s->d_A == nullptr) return "selective_scan: no array for the derivatives of A";
  if (s->d_state != nullptr && s->d_state == s->d_final_state) return "selective_scan: d_state may not be d_final_state";
  return nullptr;
}

// Time is cut where the channels alone leave SMs without a block
ScanArgs arguments(const myea_scan *s) {
  ScanArgs a = {};
  a.s = *s;
  a.batch = static_cast<int>(s->batch); a.time = static_cast<int>(s->time); a.width = static_cast<int>(s->width);
  a.states = static_cast<int>(s->states); a.groups = static_cast<int>(s->groups); a.per_group = a.width / a.groups;
  const int ch = 256 / lanes_of(s->states);
  a.tiles = (a.per_group + ch - 1) / ch;
  const double blocks = static_cast<double>(a.tiles) * a.groups * a.batch;
  a.chunks = 1;
  a.chunk = (a.time + TT - 1) / TT * TT;
  if (blocks < kSms && a.time >= 8 * TT) {
    const int want = static_cast<int>(4 * kSms / blocks), most = a.time / (4 * TT);
    const int chunks = want < most ? want : most;
    a.chunk = ((a.time + chunks - 1) / chunks + TT - 1) / TT * TT;
    a.chunks = (a.time + a.chunk - 1) / a.chunk;
  }
  const uint32_t t = s->type;
  const bool even = s->states % 4 == 0;
  a.vec_u = view_takes_vectors(s->u, t); a.vec_delta = view_takes_vectors(s->delta, t); a.vec_z = view_takes_vectors(s->z, t);
  a.vec_y = view_takes_vectors(s->y, t); a.vec_dy = view_takes_vectors(s->dy, t); a.vec_du = view_takes_vectors(s->du, t);
  a.vec_ddelta = view_takes_vectors(s->ddelta, t); a.vec_dz = view_takes_vectors(s->dz, t);
  a.vec_B = even && view_takes_vectors(s->B, t); a.vec_C = even && view_takes_vectors(s->C, t);
  if (a.per_group % 4 != 0 && a.groups > 1)   // a group's first channel is on no boundary of four
    a.vec_u = a.vec_delta = a.vec_z = a.vec_y = a.vec_dy = a.vec_du = a.vec_ddelta = a.vec_dz = false;
  a.vec_state = even && aligned(s->state, 16); a.vec_final = even && aligned(s->final_state, 16);
  a.vec_d_final = even && aligned(s->d_final_state, 16); a.vec_d_state = even && aligned(s->d_state, 16);
  return a;
}

// where the workspace's parts begin, in bytes
struct Layout {
  size_t carry = 0, steps = 0, part_bc = 0, part_a = 0, part_d = 0, bytes = 0;
};
Layout layout_of(const ScanArgs &a, bool backward) {
  const size_t np = 4 * lanes_of(a.states), rows = static_cast<size_t>(a.batch) * a.chunks;
  Layout w;
  const auto take = [&](size_t floats) {
    const size_t at = w.bytes;
    w.bytes += round_up_256(floats * sizeof(float));
    return at;
  };
  if (a.chunks > 1) {
    w.carry = take(rows * a.width * np);
    w.steps = take(rows * a.width);
  }
  if (backward) {
    w.part_bc = take(static_cast<size_t>(a.tiles) * a.batch * a.time * a.groups * 2 * np);
    w.part_a = take(rows * a.width * np);
    w.part_d = take(rows * 2 * a.width);
  }
  return w;
}
void place(ScanArgs &a, const Layout &w, void *workspace) {
  char *base = static_cast<char *>(workspace);
  a.carry = reinterpret_cast<float *>(base + w.carry);
  a.steps = reinterpret_cast<float *>(base + w.steps);
  a.part_bc = reinterpret_cast<float *>(base + w.part_bc);
  a.part_a = reinterpret_cast<float *>(base + w.part_a);
  a.part_d = reinterpret_cast<float *>(base + w.part_d);
}

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

template <typename T, int LPC> void launch_forward(const ScanArgs &a, cudaStream_t stream) {
  const long long blocks = static_cast<long long>(a.tiles) * a.groups * a.batch;
  if (a.chunks > 1) {
    scan_forward_kernel<T, LPC, true><<<static_cast<unsigned>(blocks * (a.chunks - 1)), 256, 0, stream>>>(a);
    scan_chain_kernel<LPC, false><<<static_cast<unsigned>((static_cast<long long>(a.batch) * a.width * LPC + 255) / 256), 256, 0, stream>>>(a);
  }
  scan_forward_kernel<T, LPC, false><<<static_cast<unsigned>(blocks * a.chunks), 256, 0, stream>>>(a);
}

template <typename T, int LPC> cudaError_t launch_backward(const ScanArgs &a, cudaStream_t stream) {
  const long long blocks = static_cast<long long>(a.tiles) * a.groups * a.batch;
  constexpr size_t smem = backward_smem<LPC>();
  const cudaError_t e = cudaFuncSetAttribute(scan_backward_kernel<T, LPC>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  if (a.chunks > 1) {
    scan_backward_states_kernel<T, LPC><<<static_cast<unsigned>(blocks * (a.chunks - 1)), 256, 0, stream>>>(a);
    scan_chain_kernel<LPC, true><<<static_cast<unsigned>((static_cast<long long>(a.batch) * a.width * LPC + 255) / 256), 256, 0, stream>>>(a);
  }
  if (blocks > 0) scan_backward_kernel<T, LPC><<<static_cast<unsigned>(blocks * a.chunks), 256, smem, stream>>>(a);
  const long long blocks_bc = (static_cast<long long>(a.batch) * a.time * a.groups * 8 * LPC + 31) / 32;
  const long long blocks_a = (static_cast<long long>(a.width) * 4 * LPC + 31) / 32, blocks_d = (2ll * a.width + 31) / 32;
  scan_finish_kernel<T, LPC><<<static_cast<unsigned>(blocks_bc + blocks_a + blocks_d), 256, 0, stream>>>(a, blocks_bc, blocks_a);
  return cudaSuccess;
}

// every launch's blocks fit a grid
bool too_many_blocks(const ScanArgs &a) {
  const double lanes = lanes_of(a.states), batch = a.batch;
  const double main = static_cast<double>(a.tiles) * a.groups * batch * a.chunks, chain = batch * a.width * lanes / 256.0;
  const double finish = batch * a.time * a.groups * lanes / 4.0 + a.width * lanes / 8.0 + a.width / 16.0 + 3.0;
  return main > 2147483647.0 || chain > 2147483646.0 || finish > 2147483647.0;
}

}  // namespace
}  // namespace myea

extern "C" size_t myea_b200_selective_scan_checkpoint_bytes(const myea_scan *s) {
  using namespace myea;
  if (s == nullptr || s->states < 1 || s->states > 128 || s->batch > kSequenceMost || s->time > kSequenceMost || s->width > kSequenceMost) return 0;
  return static_cast<size_t>(s->batch) * ((s->time + TT - 1) / TT) * s->width * 4 * lanes_of(s->states) * sizeof(float);
}

extern "C" size_t myea_b200_selective_scan_workspace(const myea_scan *s) {
  using namespace myea;
  if (check(s, false) != nullptr || s->batch == 0 || s->width == 0) return 0;
  return layout_of(arguments(s), false).bytes;
}

extern "C" int myea_b200_selective_scan(int device, const myea_scan *s, void *workspace, size_t workspace_bytes, void *stream, char *error_message,
                                        size_t error_capacity) {
  using namespace myea;
  if (const char *why = check(s, false)) return refuse(error_message, error_capacity, MYEA_E_INVALID, why);
  if (s->batch == 0 || s->width == 0) return MYEA_OK;
  ScanArgs a = arguments(s);
  if (too_many_blocks(a)) return refuse(error_message, error_capacity, MYEA_E_INVALID, "selective_scan: more positions than one launch takes");
  const Layout w = layout_of(a, false);
  if (w.bytes > 0 && (workspace == nullptr || workspace_bytes < w.bytes || !aligned(workspace, 256)))
    return refuse(error_message, error_capacity, MYEA_E_INVALID, "selective_scan: the workspace is missing, too small or not 256-byte aligned");
  place(a, w, workspace);
  DeviceScope scope(device);
  if (!scope.ok) return refuse(error_message, error_capacity, MYEA_E_CUDA, "selective_scan: no such device");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  with_type(s->type, [&](auto t) { with_lanes(lanes_of(s->states), [&](auto n) { launch_forward<decltype(t), decltype(n)::value>(a, st); }); });
  return launched(error_message, error_capacity, "selective_scan");
}

extern "C" size_t myea_b200_selective_scan_backward_workspace(const myea_scan *s) {
  using namespace myea;
  if (check(s, true) != nullptr || s->width == 0) return 0;
  return layout_of(arguments(s), true).bytes;
}

extern "C" int myea_b200_selective_scan_backward(int device, const myea_scan *s, void *workspace, size_t workspace_bytes, void *stream, char *error_message,
                                                 size_t error_capacity) {
  using namespace myea;
  if (const char *why = check(s, true)) return refuse(error_message, error_capacity, MYEA_E_INVALID, why);
  if (s->width == 0) return MYEA_OK;
  ScanArgs a = arguments(s);
  if (too_many_blocks(a)) return refuse(error_message, error_capacity, MYEA_E_INVALID, "selective_scan: more positions than one launch takes");
  const Layout w = layout_of(a, true);
  if (w.bytes > 0 && (workspace == nullptr || workspace_bytes < w.bytes || !aligned(workspace, 256)))
    return refuse(error_message, error_capacity, MYEA_E_INVALID, "selective_scan: the workspace is missing, too small or not 256-byte aligned");
  place(a, w, workspace);
  DeviceScope scope(device);
  if (!scope.ok) return refuse(error_message, error_capacity, MYEA_E_CUDA, "selective_scan: no such device");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  with_type(s->type, [&](auto t) { with_lanes(lanes_of(s->states), [&](auto n) { e = launch_backward<decltype(t), decltype(n)::value>(a, st); }); });
  if (e != cudaSuccess) return refuse(error_message, error_capacity, MYEA_E_CUDA, "selective_scan: the shared memory was refused");
  return launched(error_message, error_capacity, "selective_scan_backward");
}
