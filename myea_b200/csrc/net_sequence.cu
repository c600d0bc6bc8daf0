// Where a network calls the operators for sequence models: selective scan layers, the output error against a teacher's best logits, and the
// draw of tokens from the output layer.
//
// A selective scan layer of D units with N states each reads a fully connected layer of 3 D + 2 N units, which projects its inputs to
// [x (D) | gate (D) | step (D) | B (N) | C (N)]; u = silu(causal convolution of x over the time steps), and the layer's output is the gated
// scan of u.  Its parameters lie in one run of the weights:
//   [convolution (D x taps) | its bias (D) | rates a (D x N), A = -e^a | skip (D) | step bias (D)]
// A stays negative whatever the optimizer does to a.  The arrays of a layer are [time step][row][units], which the operators read
// and write in place through their strides.  Rows that a short batch leaves unused are computed along, as in the other recurrent
// layers: their error is zero.
#include <stdio.h>

#include <algorithm>

#include "net.cuh"

namespace myea {

struct ScanLayer {
  long long D = 0, N = 0, taps = 0, count = 0;
  float *u = nullptr, *du = nullptr;      // [T * B, D] behind the convolution, and the error on it
  float *rates = nullptr;                 // [D, N] A
  float *checkpoints = nullptr;
  float *grads = nullptr;                 // [count] derivatives of the last backward pass, with respect to A in the place of a
  void *work = nullptr;
  size_t work_bytes = 0;
  long long at_bias() const { return D * taps; }
  long long at_rates() const { return at_bias() + D; }
  long long at_skip() const { return at_rates() + D * N; }
  long long at_step() const { return at_skip() + D; }
};

namespace {

int refused(myea_b200_net *net, int code, const char *msg) {
  net->ctx.error = msg;
  return code;
}

template <typename T> int device_array(myea_b200_net *net, T **p, size_t count) {
  void *q = nullptr;
  const size_t bytes = std::max<size_t>(count, 1) * sizeof(T);
  if (cudaMalloc(&q, bytes) != cudaSuccess) return refused(net, MYEA_E_CUDA, "cudaMalloc failed");
  net->allocations.push_back(q);
  if (cudaMemsetAsync(q, 0, bytes, net->ctx.stream) != cudaSuccess) return MYEA_E_CUDA;
  *p = static_cast<T *>(q);
  return MYEA_OK;
}

__global__ void __launch_bounds__(256) scan_rates_kernel(const float *a, float *A, long long n) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i < n) A[i] = -expf(a[i]);
}
// derivatives of the layer's run += the kept ones; dA / da = A
__global__ void __launch_bounds__(256) scan_derivatives_kernel(const float *kept, const float *A, long long first_rate, long long rates, long long n, float *to) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  const long long k = i - first_rate;
  to[i] += kept[i] * (k >= 0 && k < rates ? A[k] : 1.f);
}
// one block, in a fixed order
__global__ void __launch_bounds__(256) add_losses_kernel(const float *losses, long long rows, unsigned long long terms, double *acc, unsigned long long *count) {
  __shared__ double part[256];
  double sum = 0.0;
  for (long long r = threadIdx.x; r < rows; r += 256) sum += static_cast<double>(losses[r]);
  part[threadIdx.x] = sum;
  __syncthreads();
  for (int k = 128; k > 0; k >>= 1) {
    if (threadIdx.x < k) part[threadIdx.x] += part[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *acc += part[0];
    *count += terms;
  }
}

unsigned blocks_of(long long n) { return static_cast<unsigned>((n + 255) / 256); }

myea_view rows_of(const float *p, long long width, long long pitch) {   // [time][row][width] as [row][time][width]
  return {const_cast<float *>(p), width, pitch * width};
}

void describe(const myea_b200_net *net, const LayerPlan &L, myea_convolution *c, myea_scan *s) {
  const ScanLayer &S = *L.scan;
  const long long pitch = net->pitch();
  const LayerPlan &in = net->layers[L.input_layer];
  const float *x = in.values, *p = net->params + L.idx.first_connection_index;
  *c = myea_convolution();
  c->type = MYEA_TYPE_F32; c->taps = static_cast<uint32_t>(S.taps); c->silu = 1;
  c->batch = static_cast<uint64_t>(pitch); c->time = static_cast<uint64_t>(net->T); c->width = static_cast<uint64_t>(S.D);
  c->x = rows_of(x, L.n_in, pitch); c->y = rows_of(S.u, S.D, pitch);
  c->weight = p; c->bias = p + S.at_bias();
  *s = myea_scan();
  s->type = MYEA_TYPE_F32; s->softplus = 1;
  s->batch = c->batch; s->time = c->time; s->width = c->width; s->states = static_cast<uint64_t>(S.N); s->groups = 1;
  s->u = c->y;
  s->z = rows_of(x + S.D, L.n_in, pitch); s->delta = rows_of(x + 2 * S.D, L.n_in, pitch);
  s->B = rows_of(x + 3 * S.D, L.n_in, pitch); s->C = rows_of(x + 3 * S.D + S.N, L.n_in, pitch);
  s->y = rows_of(L.values, S.D, pitch);
  s->A = S.rates; s->D = p + S.at_skip(); s->delta_bias = p + S.at_step();
}

int failed(myea_b200_net *net, int rc, const char *message) {
  if (rc != MYEA_OK) net->ctx.error = message;
  return rc;
}

}  // namespace

// parameters of a selective scan layer, 0: its description is not valid (msg says why)
long long scan_layer_parameters(const myea_layer_desc &d, long long n_in, const char **msg) {
  const uint64_t D = d.unit_parameters[0], N = d.unit_parameters[1], taps = d.unit_parameters[2];
  *msg = nullptr;
  if (D < 1 || D > (1u << 24) || N < 1 || N > 128 || taps < 1 || taps > 8) *msg = "a selective scan layer has units, 1 to 128 states and 1 to 8 taps";
  else if (static_cast<long long>(3 * D + 2 * N) != n_in) *msg = "a selective scan layer reads a fully connected layer of 3 units + 2 states neurons";
  else if (d.type_dropout != MYEA_DROPOUT_NONE || d.type_normalization != MYEA_NORM_NONE) *msg = "selective scan layers take neither dropout nor normalization";
  return *msg != nullptr ? 0 : static_cast<long long>(D * (taps + 1) + D * N + 2 * D);
}

int scan_layer_create(myea_b200_net *net, LayerPlan &L) {
  const char *msg = nullptr;
  ScanLayer *S = new ScanLayer();
  L.scan = S;
  S->D = L.n_out;
  S->N = static_cast<long long>(L.desc.unit_parameters[1]);
  S->taps = static_cast<long long>(L.desc.unit_parameters[2]);
  S->count = scan_layer_parameters(L.desc, L.n_in, &msg);
  const long long rows = net->T * net->B;
  int rc = device_array(net, &S->u, rows * S->D);
  if (rc == MYEA_OK) rc = device_array(net, &S->du, rows * S->D);
  if (rc == MYEA_OK) rc = device_array(net, &S->rates, S->D * S->N);
  if (rc == MYEA_OK) rc = device_array(net, &S->grads, S->count);
  if (rc != MYEA_OK) return rc;
  // Working memory: shorter batches take no more.  With several time steps the arrays keep the rows of the longest batch, and a single
  // step is never cut, so that its sizes go by the rows.
  {
    myea_convolution c;
    myea_scan s;
    describe(net, L, &c, &s);
    // (addresses that stand for the backward pass's; only the sizes count here)
    c.d_weight = c.d_bias = s.d_A = S->grads;
    c.dy = c.y; c.dx = rows_of(S->du, S->D, net->B);
    s.checkpoints = S->du; s.dy = s.y; s.du = s.ddelta = s.dB = s.dC = s.dz = c.dx;
    S->work_bytes = std::max({myea_b200_selective_scan_workspace(&s), myea_b200_selective_scan_backward_workspace(&s),
                              myea_b200_causal_convolution_backward_workspace(&c)});
  }
  myea_scan s = {};
  s.batch = static_cast<uint64_t>(net->B); s.time = static_cast<uint64_t>(net->T); s.width = static_cast<uint64_t>(S->D); s.states = static_cast<uint64_t>(S->N);
  rc = device_array(net, &S->checkpoints, myea_b200_selective_scan_checkpoint_bytes(&s) / sizeof(float));
  char *work = nullptr;
  if (rc == MYEA_OK) rc = device_array(net, &work, S->work_bytes);
  S->work = work;
  return rc;
}

void scan_layer_destroy(LayerPlan &L) {
  delete L.scan;
  L.scan = nullptr;
}

int scan_layer_forward(myea_b200_net *net, LayerPlan &L) {
  const ScanLayer &S = *L.scan;
  Context &ctx = net->ctx;
  char message[256];
  myea_convolution c;
  myea_scan s;
  describe(net, L, &c, &s);
  s.checkpoints = net->training ? S.checkpoints : nullptr;
  ctx.begin(TC_RECURRENT);
  scan_rates_kernel<<<blocks_of(S.D * S.N), 256, 0, ctx.stream>>>(net->params + L.idx.first_connection_index + S.at_rates(), S.rates, S.D * S.N);
  int rc = myea_b200_causal_convolution(ctx.device, &c, ctx.stream, message, sizeof(message));
  if (rc == MYEA_OK) rc = myea_b200_selective_scan(ctx.device, &s, S.work, S.work_bytes, ctx.stream, message, sizeof(message));
  ctx.end(TC_RECURRENT, 3);
  return failed(net, rc, message);
}

// error on the layer's outputs (L.errors) -> error on the outputs of the layer that it reads, and the derivatives of its parameters
int scan_layer_backward(myea_b200_net *net, LayerPlan &L, float *d_input) {
  const ScanLayer &S = *L.scan;
  Context &ctx = net->ctx;
  const long long pitch = net->pitch();
  char message[256];
  myea_convolution c;
  myea_scan s;
  describe(net, L, &c, &s);
  s.checkpoints = S.checkpoints;
  s.dy = rows_of(L.errors, S.D, pitch); s.du = rows_of(S.du, S.D, pitch);
  s.dz = rows_of(d_input + S.D, L.n_in, pitch); s.ddelta = rows_of(d_input + 2 * S.D, L.n_in, pitch);
  s.dB = rows_of(d_input + 3 * S.D, L.n_in, pitch); s.dC = rows_of(d_input + 3 * S.D + S.N, L.n_in, pitch);
  s.d_A = S.grads + S.at_rates(); s.d_D = S.grads + S.at_skip(); s.d_delta_bias = S.grads + S.at_step();
  c.dy = s.du; c.dx = rows_of(d_input, L.n_in, pitch);
  c.d_weight = S.grads; c.d_bias = S.grads + S.at_bias();
  ctx.begin(TC_RECURRENT);
  int rc = myea_b200_selective_scan_backward(ctx.device, &s, S.work, S.work_bytes, ctx.stream, message, sizeof(message));
  if (rc == MYEA_OK) rc = myea_b200_causal_convolution_backward(ctx.device, &c, S.work, S.work_bytes, ctx.stream, message, sizeof(message));
  ctx.end(TC_RECURRENT, 4);
  return failed(net, rc, message);
}

int scan_layer_update_derivative_weight(myea_b200_net *net, LayerPlan &L) {
  const ScanLayer &S = *L.scan;
  net->ctx.begin(TC_RECURRENT);
  scan_derivatives_kernel<<<blocks_of(S.count), 256, 0, net->ctx.stream>>>(S.grads, S.rates, S.at_rates(), S.D * S.N, S.count,
                                                                            net->grads + L.idx.first_connection_index);
  net->ctx.end(TC_RECURRENT);
  return cudaGetLastError() == cudaSuccess ? MYEA_OK : MYEA_E_CUDA;
}

namespace {

int output_layer(myea_b200_net *net, uint64_t batch, LayerPlan **L) {
  if (static_cast<long long>(batch) != net->active_B) return refused(net, MYEA_E_INVALID, "batch must equal the batch of the last forward pass");
  if (net->pre_training_level != 0) return refused(net, MYEA_E_INVALID, "not while a pair of layers is pre-trained");
  *L = &net->layers.back();
  if ((*L)->desc.type_activation_function != MYEA_AF_SOFTMAX) return refused(net, MYEA_E_INVALID, "the output layer's activation function has to be softmax");
  return cudaSetDevice(net->ctx.device) == cudaSuccess ? MYEA_OK : MYEA_E_CUDA;
}

}  // namespace
}  // namespace myea

extern "C" int myea_b200_compute_error_distillation_device(myea_handle net, uint64_t batch, const int32_t *index, const float *teacher, uint64_t top,
                                                           const int32_t *labels, const float *weight, float temperature, float soft, float hard) {
  using namespace myea;
  if (net == nullptr) return MYEA_E_INVALID;
  LayerPlan *L = nullptr;
  int rc = output_layer(net, batch, &L);
  if (rc != MYEA_OK) return rc;
  if (index == nullptr || teacher == nullptr) return refused(net, MYEA_E_INVALID, "distillation: index or teacher is missing");
  if (net->desc.type_loss_function != MYEA_LOSS_CROSS_ENTROPY) return refused(net, MYEA_E_INVALID, "distillation: the network's loss function has to be the cross entropy");
  if (net->distillation_losses == nullptr) {
    rc = device_array(net, &net->distillation_losses, net->T * net->B);
    if (rc != MYEA_OK) return rc;
  }
  const long long pitch = net->pitch(), B = net->active_B, H = L->n_out;
  const long long t0 = net->T > 1 ? std::min<long long>(static_cast<long long>(net->desc.number_time_delays), net->T) : 0;
  // rows without an error: the steps before the delay, and those that a short batch leaves unused
  if (t0 > 0 || B < pitch) {
    rc = fill_zero(net->ctx, L->errors, net->T * pitch * H);
    if (rc != MYEA_OK) return rc;
  }
  char message[256];
  const long long runs = B == pitch ? (net->T > t0 ? 1 : 0) : net->T - t0, rows = B == pitch ? (net->T - t0) * pitch : B;
  for (long long k = 0; k < runs; ++k) {
    const long long from = B == pitch ? t0 * pitch : (t0 + k) * pitch, given = (t0 + k) * B;   // rows of the layer's arrays, and of the caller's
    myea_distillation d = {};
    d.type = MYEA_TYPE_F32;
    d.rows = static_cast<uint64_t>(rows); d.vocabulary = static_cast<uint64_t>(H); d.top = top;
    d.logits = L->summations + from * H; d.logits_stride = H;
    d.index = index + given * static_cast<long long>(top); d.index_stride = static_cast<int64_t>(top);
    d.teacher = teacher + given * static_cast<long long>(top); d.teacher_stride = static_cast<int64_t>(top);
    d.labels = labels == nullptr ? nullptr : labels + given;
    d.weight = weight == nullptr ? nullptr : weight + given;
    d.temperature = temperature; d.soft = soft; d.hard = hard;
    d.losses = net->distillation_losses;
    d.d_logits = L->errors + from * H; d.d_logits_stride = H;
    net->ctx.begin(TC_ELEMENTWISE);
    rc = myea_b200_distillation_error(net->ctx.device, &d, net->ctx.stream, message, sizeof(message));
    if (rc == MYEA_OK)
      add_losses_kernel<<<1, 256, 0, net->ctx.stream>>>(net->distillation_losses, rows, static_cast<unsigned long long>(rows * H), net->d_loss_acc, net->d_loss_count);
    net->ctx.end(TC_ELEMENTWISE, 2);
    if (rc != MYEA_OK) return failed(net, rc, message);
  }
  return cudaGetLastError() == cudaSuccess ? MYEA_OK : MYEA_E_CUDA;
}

extern "C" int myea_b200_sample_outputs_device(myea_handle net, uint64_t batch, const float *uniform, const float *temperature, const int32_t *top_k,
                                               const float *top_p, const float *min_p, int32_t *tokens, float *chances) {
  using namespace myea;
  if (net == nullptr) return MYEA_E_INVALID;
  LayerPlan *L = nullptr;
  int rc = output_layer(net, batch, &L);
  if (rc != MYEA_OK) return rc;
  if (uniform == nullptr || tokens == nullptr) return refused(net, MYEA_E_INVALID, "sample_outputs: uniform or tokens is missing");
  const long long pitch = net->pitch(), B = net->active_B, H = L->n_out;
  const long long runs = B == pitch ? 1 : net->T, rows = B == pitch ? net->T * pitch : B;
  char message[256];
  for (long long k = 0; k < runs; ++k) {
    const long long given = k * B;
    myea_sampling s = {};
    s.type = MYEA_TYPE_F32;
    s.rows = static_cast<uint64_t>(rows); s.vocabulary = static_cast<uint64_t>(H);
    s.logits = L->summations + k * pitch * H; s.logits_stride = H;
    s.uniform = uniform + given;
    s.temperature = temperature == nullptr ? nullptr : temperature + given;
    s.top_k = top_k == nullptr ? nullptr : top_k + given;
    s.top_p = top_p == nullptr ? nullptr : top_p + given;
    s.min_p = min_p == nullptr ? nullptr : min_p + given;
    s.tokens = tokens + given;
    s.chances = chances == nullptr ? nullptr : chances + given;
    net->ctx.begin(TC_ELEMENTWISE);
    rc = myea_b200_sample(net->ctx.device, &s, net->ctx.stream, message, sizeof(message));
    net->ctx.end(TC_ELEMENTWISE);
    if (rc != MYEA_OK) return failed(net, rc, message);
  }
  return MYEA_OK;
}
