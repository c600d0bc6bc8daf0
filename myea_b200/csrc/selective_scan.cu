// Selective state space scan: the forward kernels, the checks and the entry points (layout and reasons: selective_scan.cuh).
#include "selective_scan.cuh"

namespace myea {
namespace scan {
namespace {

// STATES: only the states at the chunks' ends from a zero start, and the sums of their step lengths.
// One half of the block's warps walk over the steps of a tile while the other half make the tile after it (step lengths, products)
// and finish the one before it (skip, gate, stores): the two kinds of work have different dependencies, and a chip that is
// not full of channels has twice the warps to hide them behind.  What bounds it are the warps that walk: with 16 states and 16-bit types two blocks
// fit on an SM, 8 such warps, and keep its unit for powers 61 % busy (4096 x 4096 channels in one sequence: 123 us, and 97 for STATES); fp32
// inputs on their way take 166 registers a thread, one block per SM and 176 us.
template <typename T, typename S, bool STATES>
__global__ void __launch_bounds__(2 * S::NT) scan_forward_kernel(const ScanArgs a) {
  constexpr int CPT = S::CPT, PAIRS = S::PAIRS, BC = S::BC;
  extern __shared__ __align__(16) float shared[];   // [2] of each: step lengths, steps * inputs, B, C, sums over the states
  float *s_delta = shared, *s_in = s_delta + 2 * PAIRS, *s_B = s_in + 2 * PAIRS, *s_C = s_B + 2 * BC, *s_y = s_C + 2 * BC;
  const bool walks = threadIdx.x < S::NT;
  const Place<S> p(a, STATES ? a.chunks - 1 : a.chunks, 0);
  const bool gate = !STATES && a.s.z.data != nullptr;
  const int tiles = (p.t1 - p.t0 + TT - 1) / TT;
  if (walks) {
    float2 A[CPT][2], h[CPT][2];
    float sum[CPT];
#pragma unroll
    for (int q = 0; q < CPT; ++q) {
      const int have = p.have(a, q);
      const long long d = p.first + p.c + q;
      rates2(parameters4(a.s.A + d * a.states + p.n, have), A[q]);
      float4 start = make_float4(0.f, 0.f, 0.f, 0.f);
      if (!STATES && have > 0) {
        if (a.chunks > 1) start = p.states_at(a.carry, p.b * a.chunks + p.chunk, a, q);
        else if (a.s.state != nullptr) start = load_states(a.s.state + (p.b * a.width + d) * a.states + p.n, have, a.vec_state);
      }
      h[q][0] = lo(start);
      h[q][1] = hi(start);
      sum[q] = 0.f;
    }
    for (int i = 0; i < tiles + 2; ++i) {
      if (i >= 1 && i <= tiles) {
        const int t = p.t0 + (i - 1) * TT, buffer = (i - 1) & 1;
        if (!STATES && a.s.checkpoints != nullptr) {
#pragma unroll
          for (int q = 0; q < CPT; ++q)
            if (p.c + q < p.channels)
              p.states_at(a.s.checkpoints, p.b * ((a.time + TT - 1) / TT) + t / TT, a, q) = make_float4(h[q][0].x, h[q][0].y, h[q][1].x, h[q][1].y);
        }
        const float *delta = s_delta + buffer * PAIRS + 2 * p.c, *in = s_in + buffer * PAIRS + 2 * p.c;
        const float *B = s_B + buffer * BC + p.n, *C = s_C + buffer * BC + p.n;
        float *to = s_y + buffer * S::SUMS;
        // (steps behind the last one have length 0)  What the next steps need is asked for, and their exponentials are begun, before
        // the steps at hand are finished: in order of issue, a lone warp would wait for each of them.
        Steps<S> now, next;
        now.fetch(delta, in, B, C, 0, A, !STATES);
#pragma unroll
        for (int k = 0; k < TT; k += Steps<S>::G) {
          if (k + Steps<S>::G < TT) next.fetch(delta, in, B, C, k + Steps<S>::G, A, !STATES);
#pragma unroll
          for (int j = 0; j < Steps<S>::G; ++j) {
            float y[CPT];
#pragma unroll
            for (int q = 0; q < CPT; ++q) {
              h[q][0] = fma2(now.decay[j][q][0], h[q][0], mul2(now.x[j][q], lo(now.b[j])));
              h[q][1] = fma2(now.decay[j][q][1], h[q][1], mul2(now.x[j][q], hi(now.b[j])));
              if (STATES) {
                sum[q] += now.s[j][q];
              } else {
                const float2 r = fma2(h[q][1], hi(now.c[j]), mul2(h[q][0], lo(now.c[j])));
                y[q] = r.x + r.y;
              }
            }
            if (!STATES) put_part<S>(to, k + j, p, y);
          }
          now = next;
        }
      }
      meet();
    }
#pragma unroll
    for (int q = 0; q < CPT; ++q) {
      const int have = p.have(a, q);
      const long long d = p.first + p.c + q;
      if (STATES) {
        if (p.c + q < p.channels) {
          p.states_at(a.carry, p.b * a.chunks + p.chunk, a, q) = make_float4(h[q][0].x, h[q][0].y, h[q][1].x, h[q][1].y);
          if (p.l == 0) a.steps[(p.b * a.chunks + p.chunk) * a.width + d] = sum[q];
        }
      } else if (a.s.final_state != nullptr && p.chunk == a.chunks - 1 && have > 0) {
        store_states(a.s.final_state + (p.b * a.width + d) * a.states + p.n, h[q][0], h[q][1], have, a.vec_final);
      }
    }
  } else {
    const bool soft = a.s.softplus;
    const float4 bias = p.four(a.s.delta_bias);
    const float4 skip = p.four(STATES ? nullptr : a.s.D);
    ChannelTile<T, S> delta, u, z, u1, z1, u2, z2;   // inputs of the tile to make, of the one being walked over and of the one to finish
    const ChannelRows<T, S> u_rows(a.s.u, a.vec_u, p), delta_rows(a.s.delta, a.vec_delta, p), z_rows(a.s.z, a.vec_z, p), y_rows(a.s.y, a.vec_y, p);
    StateTile<T, S> B, C;
    const auto load = [&](int t) {
      u.load(u_rows, p, t);
      delta.load(delta_rows, p, t);
      B.load(a.s.B, a.vec_B, p, a.states, t);
      if (!STATES) C.load(a.s.C, a.vec_C, p, a.states, t);
      if (gate) z.load(z_rows, p, t);
    };
    load(p.t0);
    for (int i = 0; i < tiles + 2; ++i) {
      const int t = p.t0 + i * TT;
      if (i < tiles) {
        float *to_delta = s_delta + (i & 1) * PAIRS + 2 * p.c4, *to_in = s_in + (i & 1) * PAIRS + 2 * p.c4;
        if (p.loads) {
#pragma unroll
          for (int k = 0; k < S::VI; ++k) {
            const int row = p.row + k * S::ROWS;
            const float4 s = step_lengths(widen(delta.raw[k]), bias, soft, t + row < p.live);
            put_pairs(to_delta + row * 2 * S::CH, s);
            put_pairs(to_in + row * 2 * S::CH, times(s, widen(u.raw[k])));
          }
        }
        B.put(s_B + (i & 1) * BC, p);
        if (!STATES) C.put(s_C + (i & 1) * BC, p);
      }
      const ChannelTile<T, S> u_end = u2, z_end = z2;
      if (!STATES) { u2 = u1; z2 = z1; u1 = u; z1 = z; }
      if (i + 1 < tiles) load(t + TT);   // on its way until the next round
      if (!STATES && i >= 2 && p.loads) {
        const float *from = s_y + (i & 1) * S::SUMS;
#pragma unroll
        for (int k = 0; k < S::VI; ++k) {
          const int row = p.row + k * S::ROWS;
          const float4 x = widen(u_end.raw[k]), sums = get_sums<S>(from, row, p.c4);
          const float2 y0 = fma2(lo(skip), lo(x), lo(sums)), y1 = fma2(hi(skip), hi(x), hi(sums));
          float4 y = make_float4(y0.x, y0.y, y1.x, y1.y);
          if (gate) y = gated(y, widen(z_end.raw[k]));
          const int at = t - 2 * TT + row;
          if (at >= p.live) y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (at < p.t1) y_rows.store(at - p.row, y);
        }
      }
      meet();
    }
  }
}

// A few positions: bound by the states' 8 bytes per value where many sequences are answered at once.  A thread takes four states of one
// channel in NB sequences, all of them under way at once; the step lengths, B and C come through shared memory, made once per channel
// and sequence.  The sums are made in the order of the kernel above: tokens one by one give the bits of the whole sequence.
template <typename T, int LPC, int NB>
__global__ void __launch_bounds__(256, 3) scan_steps_kernel(const ScanArgs a, int tiles) {
  constexpr int CH = 256 / LPC, NP = 4 * LPC, PAIRS = CH / 2 * NB, ITEMS = (PAIRS + 255) / 256;   // channels of a block; pairs of them in all sequences
  __shared__ __align__(16) float2 s_step[NB * CH];   // step length, and times the input
  __shared__ __align__(16) float s_y[NB * CH];
  __shared__ __align__(16) float s_B[NB * NP], s_C[NB * NP];
  const int tid = threadIdx.x, l = tid % LPC, n = l * 4, c = tid / LPC;
  const int group = blockIdx.x / tiles, in_group = (blockIdx.x - group * tiles) * CH;
  const int first = group * a.per_group + in_group, channels = min(CH, a.per_group - in_group);
  const int have = c < channels ? min(4, a.states - n) : 0;
  const bool gate = a.s.z.data != nullptr;
  float2 A[2];
  rates2(load_states(a.s.A + static_cast<long long>(first + c) * a.states + n, have, a.vec_A), A);
  for (int b0 = blockIdx.y * NB; b0 < a.batch; b0 += gridDim.y * NB) {
    float2 h[NB][2];
    const long long held = static_cast<long long>(a.width) * a.states, own = static_cast<long long>(first + c) * a.states + n;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const float4 start = a.s.state != nullptr && b0 + k < a.batch ? load_states(a.s.state + (b0 + k) * held + own, have, a.vec_state) : make_float4(0.f, 0.f, 0.f, 0.f);
      h[k][0] = lo(start);
      h[k][1] = hi(start);
    }
    if (a.s.checkpoints != nullptr && c < channels && a.time > 0) {
#pragma unroll
      for (int k = 0; k < NB; ++k)
        if (b0 + k < a.batch)
          *reinterpret_cast<float4 *>(a.s.checkpoints + (static_cast<long long>(b0 + k) * a.width + first + c) * NP + n) = make_float4(h[k][0].x, h[k][0].y, h[k][1].x, h[k][1].y);
    }
    for (int t = 0; t < a.time; ++t) {
      float2 x[ITEMS], z[ITEMS];
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int item = tid + 256 * i, k = item / (CH / 2), c2 = item % (CH / 2) * 2;
        const long long b = b0 + k;
        if (item >= PAIRS) break;
        const int count = b < a.batch && t < sequence_length(a.s.lengths, b, a.time) ? min(2, channels - c2) : 0;
        const auto two = [&](const myea_view &v) {
          const T *at = static_cast<const T *>(v.data) + b * v.stride_batch + t * v.stride_time + first + c2;
          return make_float2(count > 0 ? to_float(at[0]) : 0.f, count > 1 ? to_float(at[1]) : 0.f);
        };
        x[i] = two(a.s.u);
        float2 s = two(a.s.delta), slope;
        z[i] = gate ? two(a.s.z) : both(0.f);
        if (a.s.delta_bias != nullptr) s = add2(s, make_float2(count > 0 ? a.s.delta_bias[first + c2] : 0.f, count > 1 ? a.s.delta_bias[first + c2 + 1] : 0.f));
        if (a.s.softplus) s = softplus2<false>(s, slope);
        if (count == 0) s = both(0.f);
        const float2 in = mul2(s, x[i]);
        *reinterpret_cast<float4 *>(s_step + k * CH + c2) = make_float4(s.x, in.x, s.y, in.y);
      }
      for (int item = tid; item < 2 * NB * LPC; item += 256) {   // B, then C
        const bool is_B = item < NB * LPC;
        const int j = is_B ? item : item - NB * LPC, k = j / LPC, m = j % LPC * 4;
        const long long b = b0 + k;
        const myea_view &v = is_B ? a.s.B : a.s.C;
        const int count = b < a.batch && t < sequence_length(a.s.lengths, b, a.time) ? min(4, a.states - m) : 0;
        const T *at = static_cast<const T *>(v.data) + b * v.stride_batch + t * v.stride_time + group * static_cast<long long>(a.states) + m;
        at4((is_B ? s_B : s_C) + j * 4) = widen(load4(at, count, is_B ? a.vec_B : a.vec_C));
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const float2 step = s_step[k * CH + c];
        const float4 b4 = at4(s_B + k * NP + n), c4 = at4(s_C + k * NP + n);
        h[k][0] = fma2(decay2(both(step.x), A[0]), h[k][0], mul2(both(step.y), lo(b4)));
        h[k][1] = fma2(decay2(both(step.x), A[1]), h[k][1], mul2(both(step.y), hi(b4)));
        const float2 r = fma2(h[k][1], hi(c4), mul2(h[k][0], lo(c4)));
        float y = r.x + r.y;
#pragma unroll
        for (int m = 4; m < LPC; m *= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
#pragma unroll
        for (int m = 1; m < (LPC < 4 ? LPC : 4); m *= 2) y += __shfl_xor_sync(0xffffffffu, y, m);
        if (l == 0) s_y[k * CH + c] = y;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int item = tid + 256 * i, k = item / (CH / 2), c2 = item % (CH / 2) * 2;
        const long long b = b0 + k;
        if (item >= PAIRS || b >= a.batch || c2 >= channels) continue;
        const float2 skip = a.s.D == nullptr ? both(0.f) : make_float2(a.s.D[first + c2], c2 + 1 < channels ? a.s.D[first + c2 + 1] : 0.f);
        float2 out = fma2(skip, x[i], *reinterpret_cast<const float2 *>(s_y + k * CH + c2)), sig;
        if (gate) out = mul2(out, gate2(z[i], sig));
        if (t >= sequence_length(a.s.lengths, b, a.time)) out = both(0.f);
        T *to = static_cast<T *>(a.s.y.data) + b * a.s.y.stride_batch + t * a.s.y.stride_time + first + c2;
        to[0] = from_float<T>(out.x);
        if (c2 + 1 < channels) to[1] = from_float<T>(out.y);
      }
    }
    if (a.s.final_state != nullptr) {
#pragma unroll
      for (int k = 0; k < NB; ++k)
        if (b0 + k < a.batch) store_states(a.s.final_state + (b0 + k) * held + own, h[k][0], h[k][1], have, a.vec_final);
    }
    __syncthreads();
  }
}

template <typename T, int LPC, int NB> void launch_steps(const ScanArgs &a, cudaStream_t stream) {
  const int channels = 256 / LPC, tiles = (a.per_group + channels - 1) / channels, down = (a.batch + NB - 1) / NB;
  scan_steps_kernel<T, LPC, NB><<<dim3(static_cast<unsigned>(tiles * a.groups), static_cast<unsigned>(down < 65535 ? down : 65535)), 256, 0, stream>>>(a, tiles);
}

template <typename S> constexpr size_t forward_smem() { return (4 * S::PAIRS + 4 * S::BC + 2 * S::SUMS) * sizeof(float); }

template <typename T, typename S> cudaError_t launch_forward(const ScanArgs &a, cudaStream_t stream) {
  const long long blocks = static_cast<long long>(a.tiles) * a.groups * a.batch;
  // Measured at 4096 channels of 16 states in bf16: 256 sequences of 1 / 2 / 4 positions 40 / 57 / 88 us against 215 to 220 staged, whatever
  // number up to 16 it is (a whole tile is walked, and a block with one tile has nothing to do beside it); 16 sequences 5.2 / - / 11.5 against 16;
  // with a sequence per block, which a single one needs, 3.0 us against 4.0, but two positions 4.8.
  const bool many = blocks >= 4 * kSms;
  if (a.time <= (many ? 4 : 1)) {
    if (many) launch_steps<T, S::LPC, 8>(a, stream);
    else launch_steps<T, S::LPC, 1>(a, stream);
    return cudaSuccess;
  }
  constexpr int smem = static_cast<int>(forward_smem<S>());
  cudaError_t e = cudaFuncSetAttribute(scan_forward_kernel<T, S, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(scan_forward_kernel<T, S, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (a.chunks > 1) {
    scan_forward_kernel<T, S, true><<<static_cast<unsigned>(blocks * (a.chunks - 1)), 2 * S::NT, smem, stream>>>(a);
    scan_chain_kernel<S::LPC, false><<<static_cast<unsigned>((static_cast<long long>(a.batch) * a.width * S::LPC + 255) / 256), 256, 0, stream>>>(a);
  }
  scan_forward_kernel<T, S, false><<<static_cast<unsigned>(blocks * a.chunks), 2 * S::NT, smem, stream>>>(a);
  return cudaSuccess;
}

}  // namespace

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
  if (s->width == 0) return nullptr;
  if (backward && s->d_A == nullptr) return "selective_scan: no array for the derivatives of A";   // (written as 0 for no sequences)
  if (s->batch == 0) return nullptr;
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
  if (s->d_state != nullptr && s->d_state == s->d_final_state) return "selective_scan: d_state may not be d_final_state";
  return nullptr;
}

ScanArgs arguments(const myea_scan *s) {
  ScanArgs a = {};
  a.s = *s;
  a.batch = static_cast<int>(s->batch); a.time = static_cast<int>(s->time); a.width = static_cast<int>(s->width);
  a.states = static_cast<int>(s->states); a.groups = static_cast<int>(s->groups); a.per_group = a.width / a.groups;
  const int lanes = lanes_of(s->states);
  const int ch = 128 * (lanes > 2 ? 2 : 1) / lanes;
  a.tiles = (a.per_group + ch - 1) / ch;
  // Time is cut where the channels' blocks leave many SMs without one.  A cut walk costs 3.5 us for each block of 64 channels,
  // 16 states and 4096 positions (64 blocks: 222 us), a whole one 360 us for any number of blocks up to the SMs'.
  const double blocks = static_cast<double>(a.tiles) * a.groups * a.batch;
  a.chunks = 1;
  a.chunk = (a.time + TT - 1) / TT * TT;
  if (blocks > 0 && blocks < kSms * 2 / 3 && a.time >= 8 * TT) {
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
  a.vec_dB = even && view_takes_vectors(s->dB, t); a.vec_dC = even && view_takes_vectors(s->dC, t);
  a.vec_A = even && aligned(s->A, 16);
  a.vec_state = even && aligned(s->state, 16); a.vec_final = even && aligned(s->final_state, 16);
  a.vec_d_final = even && aligned(s->d_final_state, 16); a.vec_d_state = even && aligned(s->d_state, 16);
  return a;
}

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

// every launch's blocks fit a grid
bool too_many_blocks(const ScanArgs &a) {
  const double lanes = lanes_of(a.states), batch = a.batch;
  const double main = static_cast<double>(a.tiles) * a.groups * batch * a.chunks, chain = batch * a.width * lanes / 256.0;
  const double finish = batch * a.time * a.groups * lanes / 4.0 + a.width * lanes / 8.0 + a.width / 16.0 + 3.0;
  return static_cast<double>(a.width) * lanes > 2147483647.0 || main > 2147483647.0 || chain > 2147483646.0 || finish > 2147483647.0;
}

}  // namespace scan
}  // namespace myea

extern "C" size_t myea_b200_selective_scan_checkpoint_bytes(const myea_scan *s) {
  using namespace myea;
  using namespace myea::scan;
  if (s == nullptr || s->states < 1 || s->states > 128 || s->batch > kSequenceMost || s->time > kSequenceMost || s->width > kSequenceMost) return 0;
  return static_cast<size_t>(s->batch) * ((s->time + TT - 1) / TT) * s->width * 4 * lanes_of(s->states) * sizeof(float);
}

extern "C" size_t myea_b200_selective_scan_workspace(const myea_scan *s) {
  using namespace myea;
  using namespace myea::scan;
  if (check(s, false) != nullptr || s->batch == 0 || s->width == 0) return 0;
  return layout_of(arguments(s), false).bytes;
}

extern "C" int myea_b200_selective_scan(int device, const myea_scan *s, void *workspace, size_t workspace_bytes, void *stream, char *error_message,
                                        size_t error_capacity) {
  using namespace myea;
  using namespace myea::scan;
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
  cudaError_t e = cudaSuccess;
  with_type(s->type, [&](auto t) {
    with_lanes(lanes_of(s->states), [&](auto n) {
      constexpr int lanes = decltype(n)::value;
      e = launch_forward<decltype(t), Shape<lanes, (lanes > 2 ? 2 : 1)>>(a, st);
    });
  });
  if (e != cudaSuccess) return refuse(error_message, error_capacity, MYEA_E_CUDA, "selective_scan: the shared memory was refused");
  return launched(error_message, error_capacity, "selective_scan");
}
