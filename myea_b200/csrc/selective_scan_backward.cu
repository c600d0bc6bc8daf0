// Selective state space scan: the backward kernels and their entry points (layout: selective_scan.cuh).
//
// With g_t = dy_t C_t + a_{t+1} g_{t+1} (a: the decay of a step, s: its length)
//   dC_t = sum over channels of dy h_t        dB_t = sum over channels of g s u        du = s sum(g B) + D dy
//   ds = sum(A g a h_{t-1}) + u sum(g B)      dA = sum over t of s g a h_{t-1}
// in tiles from the last to the first.  The states of a quarter of a tile (4 positions) are kept in registers while it is walked backwards:
// a tile is walked once from the checkpoint before it, leaving the states at its quarters' edges in shared memory, then every
// quarter is computed again and walked backwards.  Keeping half a tile takes a quarter of an exponential per state less and twice
// the registers; with half the warps on an SM that was no faster (both 476 us for 8 x 1024 x 2048 x 16
// in bf16) and slower where there are few channels.
// g a h_{t-1} is formed from the kept state rather than as g (h_t - s u B): the difference would lose the small values of fast
// states.  Sums over channels go through a thread's channels, lanes, warps and, between blocks, partial arrays that a last kernel
// adds up in a fixed order.
#include "selective_scan.cuh"

namespace myea {
namespace scan {
namespace {

// Pitch of a tile's rows: lanes that write neighbouring steps hit different banks
template <typename S> constexpr int kPitch = (S::CH + 32 * S::CPT / S::LPC + 3) / 4 * 4;

// CPT neighbouring words of a tile's row
template <int CPT> __device__ __forceinline__ void get_words(const float *p, float (&x)[CPT]) {
  if constexpr (CPT == 2) {
    const float2 v = *reinterpret_cast<const float2 *>(p);
    x[0] = v.x;
    x[1] = v.y;
  } else {
    x[0] = p[0];
  }
}
template <int CPT> __device__ __forceinline__ void put_words(float *p, const float (&x)[CPT]) {
  if constexpr (CPT == 2) *reinterpret_cast<float2 *>(p) = make_float2(x[0], x[1]);
  else p[0] = x[0];
}

// tile[t + j][c + q] = y[q][j] summed over the LPC lanes of the channels, for four steps: halves change sides until a lane has one step
template <typename S> __device__ __forceinline__ void put_sums(float *tile, int t, int c, int l, const float (&y)[S::CPT][4]) {
  constexpr int LPC = S::LPC, CPT = S::CPT;
  if constexpr (LPC == 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x[CPT];
#pragma unroll
      for (int q = 0; q < CPT; ++q) x[q] = y[q][j];
      put_words<CPT>(tile + (t + j) * kPitch<S> + c, x);
    }
  } else {
    const bool up = l & 1, up2 = l & 2;
    float x0[CPT], x1[CPT];
#pragma unroll
    for (int q = 0; q < CPT; ++q) {
      x0[q] = (up ? y[q][2] : y[q][0]) + __shfl_xor_sync(0xffffffffu, up ? y[q][0] : y[q][2], 1);
      x1[q] = (up ? y[q][3] : y[q][1]) + __shfl_xor_sync(0xffffffffu, up ? y[q][1] : y[q][3], 1);
    }
    if constexpr (LPC == 2) {
      put_words<CPT>(tile + (t + 2 * l) * kPitch<S> + c, x0);
      put_words<CPT>(tile + (t + 2 * l + 1) * kPitch<S> + c, x1);
    } else {
#pragma unroll
      for (int q = 0; q < CPT; ++q) {
        x0[q] = (up2 ? x1[q] : x0[q]) + __shfl_xor_sync(0xffffffffu, up2 ? x0[q] : x1[q], 2);
#pragma unroll
        for (int m = 4; m < LPC; m *= 2) x0[q] += __shfl_xor_sync(0xffffffffu, x0[q], m);
      }
      if (l < 4) put_words<CPT>(tile + (t + 2 * (l & 1) + (l >> 1)) * kPitch<S> + c, x0);
    }
  }
}

// Errors on the state before each chunk when nothing comes from behind it, and the sums of the chunks' step lengths
template <typename T, typename S>
__global__ void __launch_bounds__(S::NT) scan_backward_states_kernel(const ScanArgs a) {
  constexpr int CPT = S::CPT;
  __shared__ __align__(16) float s_delta[TT * kPitch<S>];
  __shared__ __align__(16) float s_dy[TT * kPitch<S>];
  __shared__ __align__(16) float s_C[TT * S::NP];
  const Place<S> p(a, a.chunks - 1, 1);
  const bool gate = a.s.z.data != nullptr, soft = a.s.softplus;
  const float4 bias = p.four(a.s.delta_bias);
  float2 A[CPT][2], g[CPT][2];
  float sum[CPT];
#pragma unroll
  for (int q = 0; q < CPT; ++q) {
    rates2(parameters4(a.s.A + static_cast<long long>(p.first + p.c + q) * a.states + p.n, p.have(a, q)), A[q]);
    g[q][0] = g[q][1] = both(0.f);
    sum[q] = 0.f;
  }
  const ChannelRows<T, S> delta_rows(a.s.delta, a.vec_delta, p), dy_rows(a.s.dy, a.vec_dy, p), z_rows(a.s.z, a.vec_z, p);
  ChannelTile<T, S> delta, z, dy;
  StateTile<T, S> C;
  int t = p.t0 + (p.t1 - p.t0 - 1) / TT * TT;
  delta.load(delta_rows, p, t);
  dy.load(dy_rows, p, t);
  C.load(a.s.C, a.vec_C, p, a.states, t);
  if (gate) z.load(z_rows, p, t);
  for (; t >= p.t0; t -= TT) {
    if (p.loads) {
#pragma unroll
      for (int i = 0; i < S::VI; ++i) {
        const int row = p.row + i * S::ROWS;
        float4 e = widen(dy.raw[i]);
        if (gate) e = gated(e, widen(z.raw[i]));
        at4(s_delta + row * kPitch<S> + p.c4) = step_lengths(widen(delta.raw[i]), bias, soft, t + row < p.live);
        at4(s_dy + row * kPitch<S> + p.c4) = e;
      }
    }
    C.put(s_C, p);
    __syncthreads();
    if (t - TT >= p.t0) {
      delta.load(delta_rows, p, t - TT);
      dy.load(dy_rows, p, t - TT);
      C.load(a.s.C, a.vec_C, p, a.states, t - TT);
      if (gate) z.load(z_rows, p, t - TT);
    }
#pragma unroll 4
    for (int k = TT - 1; k >= 0; --k) {
      float s[CPT], e[CPT];
      get_words<CPT>(s_delta + k * kPitch<S> + p.c, s);
      get_words<CPT>(s_dy + k * kPitch<S> + p.c, e);
      const float4 c4 = at4(s_C + k * S::NP + p.n);
#pragma unroll
      for (int q = 0; q < CPT; ++q) {
        g[q][0] = mul2(decay2(both(s[q]), A[q][0]), fma2(both(e[q]), lo(c4), g[q][0]));
        g[q][1] = mul2(decay2(both(s[q]), A[q][1]), fma2(both(e[q]), hi(c4), g[q][1]));
        sum[q] += s[q];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < CPT; ++q)
    if (p.c + q < p.channels) {
      p.states_at(a.carry, p.b * a.chunks + p.chunk, a, q) = make_float4(g[q][0].x, g[q][0].y, g[q][1].x, g[q][1].y);
      if (p.l == 0) a.steps[(p.b * a.chunks + p.chunk) * a.width + p.first + p.c + q] = sum[q];
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

// Words of the backward kernel's shared memory, twice where tiles alternate: step lengths, steps * inputs and errors of a tile; sums over
// the states; B and C; dB and dC of each warp; the states at a tile's quarters
template <typename S> struct BackwardShared {
  static constexpr int TILE = TT * S::CH, SUMS = TT * kPitch<S>, PART = S::NT / 32 * TT * 8 * S::LPC, EDGES = 3 * S::CPT * 4 * S::NT;
  static constexpr size_t bytes = (2 * (3 * TILE + 3 * SUMS + 2 * S::BC + PART) + EDGES) * sizeof(float);
};

// One half of the block's warps walk over a tile while the other half prepare the tile before it and finish the one behind it, as in
// the forward pass.
template <typename T, typename S>
__global__ void __launch_bounds__(2 * S::NT, S::LPC <= 2 ? 1 : 2) scan_backward_kernel(const ScanArgs a) {
  using M = BackwardShared<S>;
  constexpr int CPT = S::CPT, LPC = S::LPC, Q = TT / 4, WARPS = S::NT / 32;
  extern __shared__ __align__(16) float shared[];
  float *s_delta = shared, *s_in = s_delta + 2 * M::TILE, *s_dy = s_in + 2 * M::TILE;
  float *s_y = s_dy + 2 * M::TILE, *s_gB = s_y + 2 * M::SUMS, *s_Aq = s_gB + 2 * M::SUMS;
  float *s_B = s_Aq + 2 * M::SUMS, *s_C = s_B + 2 * S::BC;
  float *s_part = s_C + 2 * S::BC;                     // [warp][TT][LPC][dB, dC][4]
  float *s_edge = s_part + 2 * M::PART;                // [quarter][channel of a thread][thread][4]
  const bool walks = threadIdx.x < S::NT;
  const Place<S> p(a, a.chunks, 0);
  const bool gate = a.s.z.data != nullptr;
  const int tiles = (p.t1 - p.t0 + TT - 1) / TT;
  const int t_last = p.t0 + (tiles - 1) * TT;          // tile i begins at t_last - i * TT
  if (walks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float2 A[CPT][2], g[CPT][2], dA[CPT][2];   // g: the error that comes from the later step
#pragma unroll
    for (int q = 0; q < CPT; ++q) {
      const int have = p.have(a, q);
      const long long d = p.first + p.c + q;
      rates2(parameters4(a.s.A + d * a.states + p.n, have), A[q]);
      float4 end = make_float4(0.f, 0.f, 0.f, 0.f);
      if (have > 0) {
        if (a.chunks > 1) end = p.states_at(a.carry, p.b * a.chunks + p.chunk, a, q);
        else if (a.s.d_final_state != nullptr) end = load_states(a.s.d_final_state + (p.b * a.width + d) * a.states + p.n, have, a.vec_d_final);
      }
      g[q][0] = lo(end);
      g[q][1] = hi(end);
      dA[q][0] = dA[q][1] = both(0.f);
    }
    const long long kept = p.b * ((a.time + TT - 1) / TT);
    float4 start[CPT];   // the state before the tile, on its way one tile ahead
    const auto load = [&](int t) {
#pragma unroll
      for (int q = 0; q < CPT; ++q)
        start[q] = p.c + q < p.channels ? p.states_at(a.s.checkpoints, kept + t / TT, a, q) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    if (tiles > 0) load(t_last);
    for (int i = 0; i < tiles + 2; ++i) {
      if (i >= 1 && i <= tiles) {
        const int buffer = (i - 1) & 1;
        const float *delta = s_delta + buffer * M::TILE + p.c, *in = s_in + buffer * M::TILE + p.c, *dy = s_dy + buffer * M::TILE + p.c;
        const float *B = s_B + buffer * S::BC + p.n, *C = s_C + buffer * S::BC + p.n;
        float *to_y = s_y + buffer * M::SUMS, *to_gB = s_gB + buffer * M::SUMS, *to_Aq = s_Aq + buffer * M::SUMS, *part = s_part + buffer * M::PART;
        float2 H[Q][CPT][2], before[CPT][2];   // states behind each step of a quarter, and the one before it
        // walks over the quarter from step `from` on; keep: the states stay in H, otherwise the last one becomes `before`
        const auto forward = [&](int from, auto keep, bool sums) {
          float2 h[CPT][2];
          float y[CPT][4];
#pragma unroll
          for (int q = 0; q < CPT; ++q) { h[q][0] = before[q][0]; h[q][1] = before[q][1]; }
#pragma unroll
          for (int j = 0; j < Q; ++j) {
            const int k = from + j;
            float s[CPT], x[CPT];
            get_words<CPT>(delta + k * S::CH, s);
            get_words<CPT>(in + k * S::CH, x);
            const float4 b4 = at4(B + k * S::NP);
#pragma unroll
            for (int q = 0; q < CPT; ++q) {
              h[q][0] = fma2(decay2(both(s[q]), A[q][0]), h[q][0], mul2(both(x[q]), lo(b4)));
              h[q][1] = fma2(decay2(both(s[q]), A[q][1]), h[q][1], mul2(both(x[q]), hi(b4)));
              if constexpr (decltype(keep)::value) { H[j][q][0] = h[q][0]; H[j][q][1] = h[q][1]; }
            }
            if (sums) {
              const float4 c4 = at4(C + k * S::NP);
#pragma unroll
              for (int q = 0; q < CPT; ++q) {
                const float2 r = fma2(h[q][1], hi(c4), mul2(h[q][0], lo(c4)));
                y[q][j] = r.x + r.y;
              }
            }
          }
          if (sums) put_sums<S>(to_y, from, p.c, p.l, y);
          if constexpr (!decltype(keep)::value) {
#pragma unroll
            for (int q = 0; q < CPT; ++q) { before[q][0] = h[q][0]; before[q][1] = h[q][1]; }
          }
        };
        const auto edge = [&](int quarter, int q) -> float4 & { return at4(s_edge + ((quarter * CPT + q) * S::NT + p.me) * 4); };   // (this thread's own)
#pragma unroll
        for (int q = 0; q < CPT; ++q) { before[q][0] = lo(start[q]); before[q][1] = hi(start[q]); }
        // to the last quarter, leaving the states at the quarters' edges
#pragma unroll 1
        for (int k = 0; k < 3; ++k) {
#pragma unroll
          for (int q = 0; q < CPT; ++q) edge(k, q) = make_float4(before[q][0].x, before[q][0].y, before[q][1].x, before[q][1].y);
          forward(k * Q, std::false_type(), gate);
        }
        if (i < tiles) load(t_last - i * TT);
#pragma unroll 1
        for (int quarter = 3; quarter >= 0; --quarter) {
          const int from = quarter * Q;
          if (quarter < 3) {
#pragma unroll
            for (int q = 0; q < CPT; ++q) {
              const float4 h = edge(quarter, q);
              before[q][0] = lo(h);
              before[q][1] = hi(h);
            }
          }
          forward(from, std::true_type(), gate && quarter == 3);
          float sum_gB[CPT][4], sum_Aq[CPT][4];
#pragma unroll
          for (int j = Q - 1; j >= 0; --j) {
            const int k = from + j;
            float s[CPT], x[CPT], e[CPT];
            get_words<CPT>(delta + k * S::CH, s);
            get_words<CPT>(in + k * S::CH, x);
            get_words<CPT>(dy + k * S::CH, e);
            const float4 b4 = at4(B + k * S::NP), c4 = at4(C + k * S::NP);
            float2 dB[2], dC[2];
#pragma unroll
            for (int q = 0; q < CPT; ++q) {
              g[q][0] = fma2(both(e[q]), lo(c4), g[q][0]);
              g[q][1] = fma2(both(e[q]), hi(c4), g[q][1]);
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                dB[w] = q == 0 ? mul2(g[q][w], both(x[q])) : fma2(g[q][w], both(x[q]), dB[w]);
                dC[w] = q == 0 ? mul2(H[j][q][w], both(e[q])) : fma2(H[j][q][w], both(e[q]), dC[w]);
              }
              const float2 gB = fma2(g[q][1], hi(b4), mul2(g[q][0], lo(b4)));
              sum_gB[q][j] = gB.x + gB.y;
              float2 r[2];
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                g[q][w] = mul2(g[q][w], decay2(both(s[q]), A[q][w]));
                r[w] = mul2(g[q][w], j > 0 ? H[j > 0 ? j - 1 : 0][q][w] : before[q][w]);
                dA[q][w] = fma2(r[w], both(s[q]), dA[q][w]);
              }
              const float2 Aq = fma2(r[1], A[q][1], mul2(r[0], A[q][0]));
              sum_Aq[q][j] = Aq.x + Aq.y;
            }
            float v[8] = {dB[0].x, dB[0].y, dB[1].x, dB[1].y, dC[0].x, dC[0].y, dC[1].x, dC[1].y};
            const int first = sum_over_channels<LPC>(v, lane);
            constexpr int left = LPC >= 32 ? 8 : LPC == 16 ? 4 : LPC == 8 ? 2 : 1;
            if (lane < 8 * LPC) {
#pragma unroll
              for (int o = 0; o < left; ++o) part[((warp * TT + k) * LPC + p.l) * 8 + first + o] = v[o];
            }
          }
          put_sums<S>(to_gB, from, p.c, p.l, sum_gB);
          put_sums<S>(to_Aq, from, p.c, p.l, sum_Aq);
        }
      }
      meet();
    }
#pragma unroll
    for (int q = 0; q < CPT; ++q) {
      const int have = p.have(a, q);
      if (p.c + q < p.channels)
        p.states_at(a.part_a, p.b * a.chunks + p.chunk, a, q) = make_float4(dA[q][0].x, dA[q][0].y, dA[q][1].x, dA[q][1].y);
      if (a.s.d_state != nullptr && p.chunk == 0 && have > 0)
        store_states(a.s.d_state + (p.b * a.width + p.first + p.c + q) * a.states + p.n, g[q][0], g[q][1], have, a.vec_d_state);
    }
    meet();
    meet();
  } else {
    const bool soft = a.s.softplus;
    const float4 bias = p.four(a.s.delta_bias), skip = p.four(a.s.D);
    const ChannelRows<T, S> u_rows(a.s.u, a.vec_u, p), delta_rows(a.s.delta, a.vec_delta, p), dy_rows(a.s.dy, a.vec_dy, p), z_rows(a.s.z, a.vec_z, p);
    const ChannelRows<T, S> du_rows(a.s.du, a.vec_du, p), ddelta_rows(a.s.ddelta, a.vec_ddelta, p), dz_rows(a.s.dz, a.vec_dz, p);
    ChannelTile<T, S> u, delta, z, dy, u_end, delta_end, z_end, dy_end;   // of the tile to prepare, and (read again) of the one to finish
    StateTile<T, S> B, C;
    float4 sum_D = make_float4(0.f, 0.f, 0.f, 0.f), sum_bias = sum_D;
    const auto load = [&](int t) {
      u.load(u_rows, p, t);
      delta.load(delta_rows, p, t);
      dy.load(dy_rows, p, t);
      B.load(a.s.B, a.vec_B, p, a.states, t);
      C.load(a.s.C, a.vec_C, p, a.states, t);
      if (gate) z.load(z_rows, p, t);
    };
    if (tiles > 0) load(t_last);
    for (int i = 0; i < tiles + 2; ++i) {
      const int buffer = i & 1, t_end = t_last - (i - 2) * TT;
      if (i >= 2) {
        if (p.loads) {
#pragma unroll
          for (int k = 0; k < S::VI; ++k) {
            const int row = p.row + k * S::ROWS, at = row * kPitch<S> + p.c4;
            const float4 x4 = widen(u_end.raw[k]), z4 = gate ? widen(z_end.raw[k]) : make_float4(0.f, 0.f, 0.f, 0.f), e4 = widen(dy_end.raw[k]);
            const float4 raw = widen(delta_end.raw[k]), s4 = at4(s_delta + buffer * M::TILE + row * S::CH + p.c4);
            const float4 gB4 = at4(s_gB + buffer * M::SUMS + at), Aq4 = at4(s_Aq + buffer * M::SUMS + at);
            const float4 y4 = gate ? at4(s_y + buffer * M::SUMS + at) : make_float4(0.f, 0.f, 0.f, 0.f);
            const bool on = t_end + row < p.live;
            const auto finish = [&](float2 x, float2 zz, float2 e, float2 r, float2 b, float2 s, float2 gB, float2 Aq, float2 y, float2 D, float2 &du_, float2 &ds_,
                                    float2 &dz_, float2 &dD_) {
              float2 ey = e;
              dz_ = both(0.f);
              if (gate) {   // z sigmoid(z), and its slope sigmoid(z) (1 + z (1 - sigmoid(z)))
                float2 sig;
                const float2 open = gate2(zz, sig), slope = add2(sig, fma2(open, make_float2(-sig.x, -sig.y), open));
                dz_ = mul2(mul2(e, fma2(D, x, y)), slope);
                ey = mul2(e, open);
              }
              du_ = fma2(gB, s, mul2(D, ey));
              ds_ = fma2(gB, x, mul2(Aq, both(kLn2)));
              if (soft) {   // times sigmoid(step before the softplus)
                const float2 v = add2(r, b);
                ds_ = mul2(ds_, inverse2(add2(exp2_fast(mul2(v, both(-kLog2e))), both(1.f))));
              }
              dD_ = mul2(ey, x);
              if (!on) du_ = ds_ = dz_ = dD_ = both(0.f);
            };
            float2 r0[4], r1[4];
            finish(lo(x4), lo(z4), lo(e4), lo(raw), lo(bias), lo(s4), lo(gB4), lo(Aq4), lo(y4), lo(skip), r0[0], r0[1], r0[2], r0[3]);
            finish(hi(x4), hi(z4), hi(e4), hi(raw), hi(bias), hi(s4), hi(gB4), hi(Aq4), hi(y4), hi(skip), r1[0], r1[1], r1[2], r1[3]);
            sum_D.x += r0[3].x; sum_D.y += r0[3].y; sum_D.z += r1[3].x; sum_D.w += r1[3].y;
            sum_bias.x += r0[1].x; sum_bias.y += r0[1].y; sum_bias.z += r1[1].x; sum_bias.w += r1[1].y;
            if (t_end + row < p.t1) {
              const int to = t_end + row - p.row;
              du_rows.store(to, make_float4(r0[0].x, r0[0].y, r1[0].x, r1[0].y));
              ddelta_rows.store(to, make_float4(r0[1].x, r0[1].y, r1[1].x, r1[1].y));
              if (gate) dz_rows.store(to, make_float4(r0[2].x, r0[2].y, r1[2].x, r1[2].y));
            }
          }
        }
        // the block's share of dB and dC: warps in their order
        const float *part = s_part + buffer * M::PART;
        float *to = a.part_bc + ((((p.first - p.group * a.per_group) / S::CH * static_cast<long long>(a.batch) + p.b) * a.time + t_end) * a.groups + p.group) * (8 * LPC);
        for (int o = p.me * 4; o < TT * 8 * LPC; o += S::NT * 4) {
          const int row = o / (8 * LPC);
          if (t_end + row >= p.t1) break;
          float4 sum = at4(part + o);
#pragma unroll
          for (int w = 1; w < WARPS; ++w) {
            const float4 x = at4(part + w * TT * 8 * LPC + o);
            sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
          }
          at4(to + static_cast<long long>(row) * a.groups * (8 * LPC) + (o - row * 8 * LPC)) = sum;
        }
      }
      if (i < tiles) {
        if (p.loads) {
#pragma unroll
          for (int k = 0; k < S::VI; ++k) {
            const int row = p.row + k * S::ROWS, at = buffer * M::TILE + row * S::CH + p.c4;
            const float4 s = step_lengths(widen(delta.raw[k]), bias, soft, t_last - i * TT + row < p.live);
            float4 e = widen(dy.raw[k]);
            if (gate) e = gated(e, widen(z.raw[k]));
            at4(s_delta + at) = s;
            at4(s_in + at) = times(s, widen(u.raw[k]));
            at4(s_dy + at) = e;
          }
        }
        B.put(s_B + buffer * S::BC, p);
        C.put(s_C + buffer * S::BC, p);
      }
      if (i + 1 < tiles) load(t_last - (i + 1) * TT);   // on its way until the next round,
      if (i >= 1 && i <= tiles) {                       // and the one to finish then
        const int t = t_last - (i - 1) * TT;
        u_end.load(u_rows, p, t);
        delta_end.load(delta_rows, p, t);
        dy_end.load(dy_rows, p, t);
        if (gate) z_end.load(z_rows, p, t);
      }
      meet();
    }
    // sums over the block's positions of what these threads have: rows of CH channels, added in their order
    meet();
    float *join = s_y;   // [2][ROWS][CH] fits the sums' tiles
    if (p.loads) {
      at4(join + p.row * S::CH + p.c4) = sum_D;
      at4(join + (S::ROWS + p.row) * S::CH + p.c4) = sum_bias;
    }
    meet();
    for (int o = p.me; o < 2 * S::CH; o += S::NT) {
      const int k = o / S::CH, ch = o - k * S::CH;
      float sum = 0.f;
      for (int r = 0; r < S::ROWS; ++r) sum += join[(k * S::ROWS + r) * S::CH + ch];
      if (ch < p.channels) a.part_d[((p.b * a.chunks + p.chunk) * 2 + k) * a.width + p.first + ch] = sum;
    }
  }
}

// Adds up the partial sums: blocks 0 .. of dB and dC, then dA, then dD and d_delta_bias
template <typename T, int LPC>
__global__ void __launch_bounds__(256) scan_finish_kernel(const ScanArgs a, long long blocks_bc, long long blocks_a) {
  constexpr int NP = 4 * LPC;
  const long long block = blockIdx.x, rows = static_cast<long long>(a.batch) * a.chunks;
  if (block < blocks_bc) {
    // four neighbouring values per thread, the tiles in their order: enough columns for every thread to have its own
    const long long columns = static_cast<long long>(a.batch) * a.time * a.groups * 8 * LPC, first = (block * 256 + threadIdx.x) * 4;
    if (first >= columns) return;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int r = 0; r < a.tiles; ++r) {
      const float4 x = *reinterpret_cast<const float4 *>(a.part_bc + r * columns + first);
      sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
    }
    const int e = static_cast<int>(first % (8 * LPC)), n = e / 8 * 4;   // (dB and dC of four states lie side by side)
    long long at = first / (8 * LPC);
    const int g = static_cast<int>(at % a.groups);
    at /= a.groups;
    const int t = static_cast<int>(at % a.time);
    const myea_view &v = (e & 4) ? a.s.dC : a.s.dB;
    store4(static_cast<T *>(v.data) + at / a.time * v.stride_batch + t * v.stride_time + g * static_cast<long long>(a.states) + n, sum, min(4, a.states - n),
           (e & 4) ? a.vec_dC : a.vec_dB);
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

template <typename T, typename S> cudaError_t launch_backward(const ScanArgs &a, cudaStream_t stream) {
  const long long blocks = static_cast<long long>(a.tiles) * a.groups * a.batch;
  constexpr int LPC = S::LPC;
  constexpr size_t smem = BackwardShared<S>::bytes;
  const cudaError_t e = cudaFuncSetAttribute(scan_backward_kernel<T, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  if (a.chunks > 1) {
    scan_backward_states_kernel<T, S><<<static_cast<unsigned>(blocks * (a.chunks - 1)), S::NT, 0, stream>>>(a);
    scan_chain_kernel<LPC, true><<<static_cast<unsigned>((static_cast<long long>(a.batch) * a.width * LPC + 255) / 256), 256, 0, stream>>>(a);
  }
  if (blocks > 0) scan_backward_kernel<T, S><<<static_cast<unsigned>(blocks * a.chunks), 2 * S::NT, smem, stream>>>(a);
  const long long blocks_bc = (static_cast<long long>(a.batch) * a.time * a.groups * 2 * LPC + 255) / 256;
  const long long blocks_a = (static_cast<long long>(a.width) * 4 * LPC + 31) / 32, blocks_d = (2ll * a.width + 31) / 32;
  scan_finish_kernel<T, LPC><<<static_cast<unsigned>(blocks_bc + blocks_a + blocks_d), 256, 0, stream>>>(a, blocks_bc, blocks_a);
  return cudaSuccess;
}

}  // namespace
}  // namespace scan
}  // namespace myea

extern "C" size_t myea_b200_selective_scan_backward_workspace(const myea_scan *s) {
  using namespace myea;
  using namespace myea::scan;
  if (check(s, true) != nullptr || s->width == 0) return 0;
  return layout_of(arguments(s), true).bytes;
}

extern "C" int myea_b200_selective_scan_backward(int device, const myea_scan *s, void *workspace, size_t workspace_bytes, void *stream, char *error_message,
                                                 size_t error_capacity) {
  using namespace myea;
  using namespace myea::scan;
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
  with_type(s->type, [&](auto t) {
    with_lanes(lanes_of(s->states), [&](auto n) {
      constexpr int lanes = decltype(n)::value;
      e = launch_backward<decltype(t), Shape<lanes, (lanes > 2 ? 2 : 1)>>(a, st);
    });
  });
  if (e != cudaSuccess) return refuse(error_message, error_capacity, MYEA_E_CUDA, "selective_scan: the shared memory was refused");
  return launched(error_message, error_capacity, "selective_scan_backward");
}
