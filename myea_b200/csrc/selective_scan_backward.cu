// Selective state space scan: the backward kernels and their entry points (layout: selective_scan.cuh).
//
// With g_t = dy_t C_t + a_{t+1} g_{t+1} (a: the decay of a step, s: its length)
//   dC_t = sum over channels of dy h_t        dB_t = sum over channels of g s u        du = s sum(g B) + D dy
//   ds = sum(A g a h_{t-1}) + u sum(g B)      dA = sum over t of s g a h_{t-1}
// in tiles from the last to the first.  The states of half a tile (8 positions) are kept in registers while it is walked
// backwards: a tile is computed again from the checkpoint before it, its second half walked, then its first half computed
// once more.  That is half an exponential per state more than keeping the whole tile, for half the registers.
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
    const float4 a4 = parameters4(a.s.A + static_cast<long long>(p.first + p.c + q) * a.states + p.n, p.have(a, q));
    A[q][0] = make_float2(a4.x * kLog2e, a4.y * kLog2e);
    A[q][1] = make_float2(a4.z * kLog2e, a4.w * kLog2e);
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
        g[q][0] = mul2(exp2_fast(mul2(both(s[q]), A[q][0])), fma2(both(e[q]), lo(c4), g[q][0]));
        g[q][1] = mul2(exp2_fast(mul2(both(s[q]), A[q][1])), fma2(both(e[q]), hi(c4), g[q][1]));
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

template <typename S> constexpr size_t backward_smem() {
  return (4 * TT * kPitch<S> + 2 * TT * S::NP + S::NT / 32 * TT * 8 * S::LPC) * sizeof(float);
}

template <typename T, typename S>
__global__ void __launch_bounds__(S::NT, 2) scan_backward_kernel(const ScanArgs a) {
  constexpr int CPT = S::CPT, LPC = S::LPC, HALF = TT / 2, WARPS = S::NT / 32;
  extern __shared__ __align__(16) float shared[];
  float *s_B = shared, *s_C = s_B + TT * S::NP;
  float *s_part = s_C + TT * S::NP;                    // [warp][TT][LPC][dB, dC][4]
  float *s_delta = s_part + WARPS * TT * 8 * LPC;
  float *s_in = s_delta + TT * kPitch<S>, *s_dy = s_in + TT * kPitch<S>;   // later: sum(g B), sum(A g a h)
  float *s_y = s_dy + TT * kPitch<S>;
  const Place<S> p(a, a.chunks, 0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool gate = a.s.z.data != nullptr, soft = a.s.softplus;
  const float4 bias = p.four(a.s.delta_bias), skip = p.four(a.s.D);
  float2 A[CPT][2], g[CPT][2], dA[CPT][2];   // g: the error that comes from the later step
#pragma unroll
  for (int q = 0; q < CPT; ++q) {
    const int have = p.have(a, q);
    const long long d = p.first + p.c + q;
    const float4 a4 = parameters4(a.s.A + d * a.states + p.n, have);
    A[q][0] = make_float2(a4.x * kLog2e, a4.y * kLog2e);
    A[q][1] = make_float2(a4.z * kLog2e, a4.w * kLog2e);
    float4 end = make_float4(0.f, 0.f, 0.f, 0.f);
    if (have > 0) {
      if (a.chunks > 1) end = p.states_at(a.carry, p.b * a.chunks + p.chunk, a, q);
      else if (a.s.d_final_state != nullptr) end = load_states(a.s.d_final_state + (p.b * a.width + d) * a.states + p.n, have, a.vec_d_final);
    }
    g[q][0] = lo(end);
    g[q][1] = hi(end);
    dA[q][0] = dA[q][1] = both(0.f);
  }
  float4 sum_D = make_float4(0.f, 0.f, 0.f, 0.f), sum_bias = sum_D;
  const ChannelRows<T, S> u_rows(a.s.u, a.vec_u, p), delta_rows(a.s.delta, a.vec_delta, p), dy_rows(a.s.dy, a.vec_dy, p), z_rows(a.s.z, a.vec_z, p);
  const ChannelRows<T, S> du_rows(a.s.du, a.vec_du, p), ddelta_rows(a.s.ddelta, a.vec_ddelta, p), dz_rows(a.s.dz, a.vec_dz, p);
  ChannelTile<T, S> u, delta, z, dy, u_next, z_next, dy_next;
  StateTile<T, S> B, C;
  const long long kept = p.b * ((a.time + TT - 1) / TT);
  int t = p.t1 > p.t0 ? p.t0 + (p.t1 - p.t0 - 1) / TT * TT : p.t0 - TT;
  if (t >= p.t0) {
    u.load(u_rows, p, t);
    delta.load(delta_rows, p, t);
    dy.load(dy_rows, p, t);
    B.load(a.s.B, a.vec_B, p, a.states, t);
    C.load(a.s.C, a.vec_C, p, a.states, t);
    if (gate) z.load(z_rows, p, t);
  }
  for (; t >= p.t0; t -= TT) {
    float2 start[CPT][2];
#pragma unroll
    for (int q = 0; q < CPT; ++q) {
      float4 h = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p.c + q < p.channels) h = p.states_at(a.s.checkpoints, kept + t / TT, a, q);
      start[q][0] = lo(h);
      start[q][1] = hi(h);
    }
    float4 slope[S::VI];
    if (p.loads) {
#pragma unroll
      for (int i = 0; i < S::VI; ++i) {
        const int row = p.row + i * S::ROWS, at = row * kPitch<S> + p.c4;
        const float4 raw = widen(delta.raw[i]), x = widen(u.raw[i]);
        float4 e = widen(dy.raw[i]);
        if (gate) e = gated(e, widen(z.raw[i]));
        float2 s0 = add2(lo(raw), lo(bias)), s1 = add2(hi(raw), hi(bias)), k0 = both(1.f), k1 = both(1.f);
        if (soft) {
          s0 = softplus2<true>(s0, k0);
          s1 = softplus2<true>(s1, k1);
        }
        slope[i] = make_float4(k0.x, k0.y, k1.x, k1.y);
        const float4 s = t + row < p.live ? make_float4(s0.x, s0.y, s1.x, s1.y) : make_float4(0.f, 0.f, 0.f, 0.f);
        at4(s_delta + at) = s;
        at4(s_in + at) = times(s, x);
        at4(s_dy + at) = e;
      }
    }
    B.put(s_B, p);
    C.put(s_C, p);
    __syncthreads();
    if (t - TT >= p.t0) {   // the next tile is on its way
      u_next.load(u_rows, p, t - TT);
      delta.load(delta_rows, p, t - TT);
      dy_next.load(dy_rows, p, t - TT);
      B.load(a.s.B, a.vec_B, p, a.states, t - TT);
      C.load(a.s.C, a.vec_C, p, a.states, t - TT);
      if (gate) z_next.load(z_rows, p, t - TT);
    }
    float2 H[HALF][CPT][2], before[CPT][2];   // states behind each step of a half, and the one before it
    // computes the states of the half from step `from` on, starting at `before`; Y: and y for the gate's derivative
    const auto forward = [&](int from, bool keep, bool sums) {
      float2 h[CPT][2];
#pragma unroll
      for (int q = 0; q < CPT; ++q) { h[q][0] = before[q][0]; h[q][1] = before[q][1]; }
#pragma unroll
      for (int k = 0; k < HALF; k += 4) {
        float y[CPT][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = from + k + j;
          float s[CPT], in[CPT];
          get_words<CPT>(s_delta + i * kPitch<S> + p.c, s);
          get_words<CPT>(s_in + i * kPitch<S> + p.c, in);
          const float4 b4 = at4(s_B + i * S::NP + p.n);
          float4 c4 = make_float4(0.f, 0.f, 0.f, 0.f);
          if (sums) c4 = at4(s_C + i * S::NP + p.n);
#pragma unroll
          for (int q = 0; q < CPT; ++q) {
            h[q][0] = fma2(exp2_fast(mul2(both(s[q]), A[q][0])), h[q][0], mul2(both(in[q]), lo(b4)));
            h[q][1] = fma2(exp2_fast(mul2(both(s[q]), A[q][1])), h[q][1], mul2(both(in[q]), hi(b4)));
            if (keep) { H[k + j][q][0] = h[q][0]; H[k + j][q][1] = h[q][1]; }
            if (sums) {
              const float2 r = fma2(h[q][1], hi(c4), mul2(h[q][0], lo(c4)));
              y[q][j] = r.x + r.y;
            }
          }
        }
        if (sums) put_sums<S>(s_y, from + k, p.c, p.l, y);
      }
      if (!keep) {
#pragma unroll
        for (int q = 0; q < CPT; ++q) { before[q][0] = h[q][0]; before[q][1] = h[q][1]; }
      }
    };
    const auto backward = [&](int from) {
#pragma unroll
      for (int k = HALF - 4; k >= 0; k -= 4) {
        float sum_gB[CPT][4], sum_Aq[CPT][4];
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          const int o = k + j, i = from + o;
          float s[CPT], in[CPT], e[CPT];
          get_words<CPT>(s_delta + i * kPitch<S> + p.c, s);
          get_words<CPT>(s_in + i * kPitch<S> + p.c, in);
          get_words<CPT>(s_dy + i * kPitch<S> + p.c, e);
          const float4 b4 = at4(s_B + i * S::NP + p.n), c4 = at4(s_C + i * S::NP + p.n);
          float2 dB[2], dC[2];
#pragma unroll
          for (int q = 0; q < CPT; ++q) {
            g[q][0] = fma2(both(e[q]), lo(c4), g[q][0]);
            g[q][1] = fma2(both(e[q]), hi(c4), g[q][1]);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              dB[w] = q == 0 ? mul2(g[q][w], both(in[q])) : fma2(g[q][w], both(in[q]), dB[w]);
              dC[w] = q == 0 ? mul2(H[o][q][w], both(e[q])) : fma2(H[o][q][w], both(e[q]), dC[w]);
            }
            const float2 gB = fma2(g[q][1], hi(b4), mul2(g[q][0], lo(b4)));
            sum_gB[q][j] = gB.x + gB.y;
            float2 r[2];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              g[q][w] = mul2(g[q][w], exp2_fast(mul2(both(s[q]), A[q][w])));
              r[w] = mul2(g[q][w], o > 0 ? H[o > 0 ? o - 1 : 0][q][w] : before[q][w]);
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
            for (int x = 0; x < left; ++x) s_part[((warp * TT + i) * LPC + p.l) * 8 + first + x] = v[x];
          }
        }
        __syncwarp();   // (the lanes of this warp alone read these columns)
        put_sums<S>(s_in, from + k, p.c, p.l, sum_gB);
        put_sums<S>(s_dy, from + k, p.c, p.l, sum_Aq);
      }
    };
#pragma unroll
    for (int q = 0; q < CPT; ++q) { before[q][0] = start[q][0]; before[q][1] = start[q][1]; }
    if (gate) {
      forward(0, false, true);
      forward(HALF, true, true);
    } else {
      forward(0, false, false);
      forward(HALF, true, false);
    }
    backward(HALF);
#pragma unroll
    for (int q = 0; q < CPT; ++q) { before[q][0] = start[q][0]; before[q][1] = start[q][1]; }
    forward(0, true, false);
    backward(0);
    __syncthreads();
    if (p.loads) {
#pragma unroll
      for (int i = 0; i < S::VI; ++i) {
        const int row = p.row + i * S::ROWS, at = row * kPitch<S> + p.c4;
        const float4 x4 = widen(u.raw[i]), z4 = gate ? widen(z.raw[i]) : make_float4(0.f, 0.f, 0.f, 0.f), e4 = widen(dy.raw[i]);
        const float4 s4 = at4(s_delta + at), gB4 = at4(s_in + at), Aq4 = at4(s_dy + at), y4 = gate ? at4(s_y + at) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float x[4] = {x4.x, x4.y, x4.z, x4.w}, gz[4] = {z4.x, z4.y, z4.z, z4.w}, e[4] = {e4.x, e4.y, e4.z, e4.w}, D[4] = {skip.x, skip.y, skip.z, skip.w};
        const float s[4] = {s4.x, s4.y, s4.z, s4.w}, gB[4] = {gB4.x, gB4.y, gB4.z, gB4.w}, Aq[4] = {Aq4.x, Aq4.y, Aq4.z, Aq4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
        const float k[4] = {slope[i].x, slope[i].y, slope[i].z, slope[i].w};
        float du[4], ds[4], dz[4], dD[4];
#pragma unroll
        for (int o = 0; o < 4; ++o) {
          float ey = e[o];
          dz[o] = 0.f;
          if (gate) {
            const float sg = sigmoid(gz[o]);
            dz[o] = e[o] * fmaf(D[o], x[o], y[o]) * sg * (1.f + gz[o] * (1.f - sg));
            ey *= gz[o] * sg;
          }
          du[o] = fmaf(gB[o], s[o], D[o] * ey);
          ds[o] = fmaf(gB[o], x[o], Aq[o] * kLn2) * k[o];
          dD[o] = ey * x[o];
          if (t + row >= p.live) du[o] = ds[o] = dz[o] = dD[o] = 0.f;
        }
        sum_D.x += dD[0]; sum_D.y += dD[1]; sum_D.z += dD[2]; sum_D.w += dD[3];
        sum_bias.x += ds[0]; sum_bias.y += ds[1]; sum_bias.z += ds[2]; sum_bias.w += ds[3];
        if (t + row < p.t1) {
          const int to = t + row - p.row;
          du_rows.store(to, make_float4(du[0], du[1], du[2], du[3]));
          ddelta_rows.store(to, make_float4(ds[0], ds[1], ds[2], ds[3]));
          if (gate) dz_rows.store(to, make_float4(dz[0], dz[1], dz[2], dz[3]));
        }
      }
    }
    u = u_next;
    z = z_next;
    dy = dy_next;
    // the block's share of dB and dC: warps in their order
    float *to = a.part_bc + ((((p.first - p.group * a.per_group) / S::CH * static_cast<long long>(a.batch) + p.b) * a.time + t) * a.groups + p.group) * (8 * LPC);
    for (int o = threadIdx.x; o < TT * 8 * LPC; o += S::NT) {
      const int row = o / (8 * LPC);
      if (t + row >= p.t1) break;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) sum += s_part[w * TT * 8 * LPC + o];
      to[static_cast<long long>(row) * a.groups * (8 * LPC) + (o - row * 8 * LPC)] = sum;
    }
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < CPT; ++q) {
    const int have = p.have(a, q);
    if (p.c + q < p.channels)
      p.states_at(a.part_a, p.b * a.chunks + p.chunk, a, q) = make_float4(dA[q][0].x, dA[q][0].y, dA[q][1].x, dA[q][1].y);
    if (a.s.d_state != nullptr && p.chunk == 0 && have > 0)
      store_states(a.s.d_state + (p.b * a.width + p.first + p.c + q) * a.states + p.n, g[q][0], g[q][1], have, a.vec_d_state);
  }
  // sums over the block's positions of what the loading threads have: rows of CH channels, added in their order
  float *join = s_delta;   // [2][ROWS][CH] fits the tiles of the step lengths and inputs
  __syncthreads();
  if (p.loads) {
    at4(join + p.row * S::CH + p.c4) = sum_D;
    at4(join + (S::ROWS + p.row) * S::CH + p.c4) = sum_bias;
  }
  __syncthreads();
  for (int o = threadIdx.x; o < 2 * S::CH; o += S::NT) {
    const int k = o / S::CH, ch = o - k * S::CH;
    float sum = 0.f;
    for (int r = 0; r < S::ROWS; ++r) sum += join[(k * S::ROWS + r) * S::CH + ch];
    if (ch < p.channels) a.part_d[((p.b * a.chunks + p.chunk) * 2 + k) * a.width + p.first + ch] = sum;
  }
}

// Adds up the partial sums: blocks 0 .. of dB and dC, then dA, then dD and d_delta_bias
template <typename T, int LPC>
__global__ void __launch_bounds__(256) scan_finish_kernel(const ScanArgs a, long long blocks_bc, long long blocks_a) {
  constexpr int NP = 4 * LPC;
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

template <typename T, typename S> cudaError_t launch_backward(const ScanArgs &a, cudaStream_t stream) {
  const long long blocks = static_cast<long long>(a.tiles) * a.groups * a.batch;
  constexpr int LPC = S::LPC;
  constexpr size_t smem = backward_smem<S>();
  const cudaError_t e = cudaFuncSetAttribute(scan_backward_kernel<T, S>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  if (a.chunks > 1) {
    scan_backward_states_kernel<T, S><<<static_cast<unsigned>(blocks * (a.chunks - 1)), S::NT, 0, stream>>>(a);
    scan_chain_kernel<LPC, true><<<static_cast<unsigned>((static_cast<long long>(a.batch) * a.width * LPC + 255) / 256), 256, 0, stream>>>(a);
  }
  if (blocks > 0) scan_backward_kernel<T, S><<<static_cast<unsigned>(blocks * a.chunks), S::NT, smem, stream>>>(a);
  const long long blocks_bc = (static_cast<long long>(a.batch) * a.time * a.groups * 8 * LPC + 31) / 32;
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
