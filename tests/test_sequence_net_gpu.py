"""Networks that use the operators for sequence models: a selective scan layer between fully connected ones, the error against a teacher's best
logits in the place of compute_error, the draw from the output layer, and a model that is trained with the three and then answers
token by token.

References are torch autograd in 64 bits on the same parameters; tolerances are those of the other parity tests: 1e-4 of a tensor's
largest value (the network's products carry 2e-6 of it, the scans 1e-5)."""
import numpy as np
import pytest
import torch

from myea_b200 import capi, sequence
from myea_b200.net import Net

pytestmark = pytest.mark.gpu
D, N, K = 12, 5, 4


def network(T, B, inputs=7, outputs=9, units=D, states=N, taps=K, af=capi.AF_TANH, softmax=False, below=None, time_delays=0):
    layers = [capi.fc(inputs), capi.fc(capi.selective_scan_inputs(units, states), af), capi.selective_scan(units, states, taps)]
    if below is not None:
        layers.insert(1, below)
    layers.append(capi.fc(outputs, capi.AF_SOFTMAX if softmax else capi.AF_LINEAR))
    return capi.net(layers, B, T=T, loss=capi.LOSS_CE if softmax else capi.LOSS_MSE, time_delays=time_delays)


def parameters(net, seed, scan_at, units=D, states=N, taps=K):
    rng = np.random.default_rng(seed)
    p = (rng.standard_normal(net.P) * 0.4).astype(np.float32)
    li = net.layer_index(scan_at)
    a = int(li.first_connection_index)
    assert int(li.last_connection_index) - a == units * (taps + 1) + units * states + 2 * units
    p[a + units * (taps + 2 + states):a + units * (taps + 3 + states)] -= 2.0   # short steps
    return p


def weights(net, p, l):
    li = net.layer_index(l)
    a, b = int(li.first_connection_index), int(li.first_bias_connection_index)
    return p[a:a + int(li.number_outputs) * int(li.number_inputs)].reshape(int(li.number_outputs), -1), p[b:b + int(li.number_outputs)]


def scan_parameters(net, p, l, units=D, states=N, taps=K):
    at = int(net.layer_index(l).first_connection_index)
    take = []
    for shape in ((units, taps), (units,), (units, states), (units,), (units,)):
        n = int(np.prod(shape))
        take.append(p[at:at + n].reshape(shape))
        at += n
    return take


def scan_layer(x, par):
    """[T, B, 3 D + 2 N] -> [T, B, D] by the formula"""
    conv, conv_bias, a, skip, step_bias = par
    d, n = a.shape
    T, B = x.shape[:2]
    xs, z, step, Bm, C = torch.split(x, [d, d, d, n, n], 2)
    padded = torch.cat([torch.zeros(conv.shape[1] - 1, B, d, dtype=x.dtype, device=x.device), xs], 0)
    u = torch.nn.functional.silu((padded.unfold(0, conv.shape[1], 1) * conv).sum(-1) + conv_bias)
    s = torch.nn.functional.softplus(step + step_bias, threshold=40.0)
    h, ys = torch.zeros(B, d, n, dtype=x.dtype, device=x.device), []
    for t in range(T):
        h = torch.exp(s[t][..., None] * -torch.exp(a)) * h + (s[t] * u[t])[..., None] * Bm[t][:, None]
        ys.append((h * C[t][:, None]).sum(-1) + skip * u[t])
    return torch.stack(ys) * torch.nn.functional.silu(z)


def read(net, layer, batch, what="outputs"):
    """[T, batch, units] outputs or errors of a batch that may be short"""
    out = np.empty((net.T, batch, int(net.layer_index(layer).number_outputs)), np.float32)
    net._ck(getattr(net.lib, "myea_b200_get_" + what)(net.h, layer, out.ctypes.data, out.size), what)
    return out


def near(got, want, what):
    got, want = np.asarray(got, np.float64), want.detach().cpu().numpy().astype(np.float64)
    scale = np.abs(want).max()
    assert np.abs(got - want).max() <= 1e-4 * max(scale, 1e-30), (what, np.abs(got - want).max(), scale)


@pytest.mark.parametrize("T,B,batch,af", [(6, 5, 5, capi.AF_TANH), (40, 3, 2, capi.AF_LINEAR), (1, 8, 3, capi.AF_TANH), (200, 2, 2, capi.AF_SIGMOID)])
def test_scan_layer_in_a_network(T, B, batch, af):
    desc = network(T, B, af=af)
    net = Net(desc, capi.opt(capi.OPT_GD, gd_lr=0.0))
    p = parameters(net, T + B, 2)
    net.set(capi.BUF_PARAMETERS, p)
    rng = np.random.default_rng(1)
    X, Y = rng.standard_normal((T, batch, 7)).astype(np.float32), rng.standard_normal((T, batch, 9)).astype(np.float32)
    for training in (False, True):
        net.forward(X, training, batch=batch)
    q = torch.tensor(p, dtype=torch.float64, requires_grad=True)
    w1, b1 = weights(net, q, 1)
    w3, b3 = weights(net, q, 3)
    act = {capi.AF_TANH: torch.tanh, capi.AF_LINEAR: lambda v: v, capi.AF_SIGMOID: torch.sigmoid}[af]
    y = scan_layer(act(torch.tensor(X).double() @ w1.T + b1), scan_parameters(net, q, 2)) @ w3.T + b3
    near(read(net, 3, batch), y, "outputs")
    (0.5 * ((y - torch.tensor(Y).double()) ** 2).sum()).backward()
    for _ in range(2):   # derivatives add up until they are used, and a backward pass may be repeated
        net.compute_error(Y)
        net.backward()
        net.update_derivative_weight()
    grads = net.get(capi.BUF_DERIVATIVES) / 2
    for l in (1, 2, 3):
        li = net.layer_index(l)
        a, b = int(li.first_connection_index), int(li.last_connection_index)
        near(grads[a:b], q.grad[a:b], "layer %d" % l)
    li = net.layer_index(2)
    at = int(li.first_connection_index)
    for name, n in (("convolution", D * K), ("its bias", D), ("rates", D * N), ("skip", D), ("step bias", D)):
        near(grads[at:at + n], q.grad[at:at + n], name)
        at += n
    net.close()


def test_scan_layers_stacked_with_other_recurrent_layers():
    """an LSTM layer below, a second scan above: runs, and its derivatives agree with differences of the loss"""
    T, B = 5, 3
    layers = [capi.fc(4), capi.lstm(6), capi.fc(capi.selective_scan_inputs(8, 4), capi.AF_TANH), capi.selective_scan(8, 4, 3),
              capi.fc(capi.selective_scan_inputs(8, 2), capi.AF_LINEAR), capi.selective_scan(8, 2, 2), capi.fc(8, capi.AF_LINEAR)]
    net = Net(capi.net(layers, B, T=T), capi.opt(capi.OPT_GD, gd_lr=0.0))
    rng = np.random.default_rng(5)
    p = (rng.standard_normal(net.P) * 0.3).astype(np.float32)
    X, Y = rng.standard_normal((T, B, 4)).astype(np.float32), rng.standard_normal((T, B, 8)).astype(np.float32)

    def loss(params):
        net.set(capi.BUF_PARAMETERS, params)
        net.forward(X)
        return 0.5 * float(((net.outputs(6).astype(np.float64) - Y) ** 2).sum())

    net.set(capi.BUF_PARAMETERS, p)
    net.forward(X)
    net.compute_error(Y)
    net.backward()
    net.update_derivative_weight()
    g = net.get(capi.BUF_DERIVATIVES).astype(np.float64)
    for l in range(1, 7):
        li = net.layer_index(l)
        a, b = int(li.first_connection_index), int(li.last_connection_index)
        way = np.zeros(net.P)
        way[a:b] = rng.standard_normal(b - a)
        way /= np.linalg.norm(way)
        h = 1e-2   # outputs good to 1e-6 of 1: a difference of losses of some 50 to 2e-3 of its slope; the third derivative adds h^2
        slope = (loss((p + h * way).astype(np.float32)) - loss((p - h * way).astype(np.float32))) / (2 * h)
        assert abs(slope - g @ way) <= 1e-2 * np.linalg.norm(g[a:b]) + 1e-2, (l, slope, g @ way)
    net.close()


@pytest.mark.parametrize("T,B,batch,delays", [(1, 9, 4, 0), (6, 5, 5, 2), (6, 5, 3, 0)])
def test_distillation_and_draw_through_the_output_layer(T, B, batch, delays):
    net = Net(network(T, B, outputs=21, softmax=True, time_delays=delays), capi.opt(capi.OPT_GD, gd_lr=0.0))
    net.set(capi.BUF_PARAMETERS, parameters(net, 3, 2))
    rng = np.random.default_rng(2)
    net.reset_loss()
    net.forward(rng.standard_normal((T, batch, 7)).astype(np.float32), True, batch=batch)
    gen = torch.Generator(device="cuda").manual_seed(4)
    index = torch.randint(21, (T, batch, 5), generator=gen, device="cuda", dtype=torch.int32)
    teacher = torch.randn(T, batch, 5, generator=gen, device="cuda")
    labels = torch.randint(21, (T, batch), generator=gen, device="cuda", dtype=torch.int32)
    weight = torch.rand(T, batch, generator=gen, device="cuda")
    torch.cuda.synchronize()
    net.compute_error_distillation(index, teacher, 2.0, 0.75, 0.25, labels, weight)
    # softmax outputs: logits up to a constant
    q = torch.tensor(np.log(read(net, 3, batch).astype(np.float64)), dtype=torch.float32, device="cuda")
    losses, d = sequence.distillation_error(q.reshape(-1, 21).contiguous(), index.reshape(-1, 5), teacher.reshape(-1, 5), 2.0, 0.75, 0.25, labels.reshape(-1),
                                            weight.reshape(-1))
    losses, d = losses.reshape(T, batch)[delays:], d.reshape(T, batch, 21)
    d[:delays] = 0.0
    near(read(net, 3, batch, "errors"), d, "errors")
    total, terms, _ = net.loss()
    assert terms == (T - delays) * batch * 21 and abs(total - losses.double().sum().item()) <= 1e-4 * abs(total)
    net.backward()
    net.update_derivative_weight()
    uniform = torch.rand(T, batch, generator=gen, device="cuda")
    tokens, chances = torch.empty(T, batch, dtype=torch.int32, device="cuda"), torch.empty(T, batch, device="cuda")
    top_k = torch.full((T, batch), 6, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    net.sample_outputs(uniform, tokens, top_k=top_k, chances=chances)
    net.synchronize()
    y = torch.softmax(q.double(), 2)
    kept = torch.topk(y, 6, dim=2)
    share = torch.gather(y, 2, tokens[..., None].long())[..., 0] / kept.values.sum(2)
    assert ((kept.indices == tokens[..., None]).any(2)).all() and torch.allclose(chances.double(), share, rtol=1e-4)
    net.close()


def test_a_model_trained_with_a_teacher_answers_token_by_token():
    """four steps against a teacher with Adam, then the trained network's answers: whole sequences through the network, and the same
    tokens one by one through the operators with their states; the draws agree"""
    T, B, V, units, states, taps = 24, 4, 33, 16, 8, 4
    desc = network(T, B, inputs=6, outputs=V, units=units, states=states, taps=taps, softmax=True, af=capi.AF_LINEAR)
    net = Net(desc, capi.opt(capi.OPT_ADAM, lr=1e-2))
    p0 = parameters(net, 8, 2, units, states, taps)
    net.set(capi.BUF_PARAMETERS, p0)
    gen = torch.Generator(device="cuda").manual_seed(9)
    rng = np.random.default_rng(9)
    index = torch.randint(V, (T, B, 8), generator=gen, device="cuda", dtype=torch.int32)
    teacher = torch.randn(T, B, 8, generator=gen, device="cuda") * 2
    X = rng.standard_normal((T, B, 6)).astype(np.float32)
    torch.cuda.synchronize()
    for _ in range(4):
        net.reset_loss()
        net.forward(X)
        net.compute_error_distillation(index, teacher, 1.5)
        assert np.isfinite(net.loss()[0])
        net.backward()
        net.update_derivative_weight()
        net.update_parameter()
    p = net.get(capi.BUF_PARAMETERS)
    assert np.isfinite(p).all() and (p != p0).any()
    net.forward(X, False)
    uniform = torch.rand(T, B, generator=gen, device="cuda")
    tokens = torch.empty(T, B, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    net.sample_outputs(uniform, tokens, top_p=torch.full((T, B), 0.9, device="cuda"))
    net.synchronize()
    dev = lambda a: torch.tensor(np.ascontiguousarray(a), device="cuda")  # noqa: E731
    w1, b1 = (dev(a) for a in weights(net, p, 1))
    w3, b3 = (dev(a) for a in weights(net, p, 3))
    conv, conv_bias, a, skip, step_bias = (dev(v) for v in scan_parameters(net, p, 2, units, states, taps))
    inputs, before, held = torch.tensor(X, device="cuda"), torch.zeros(B, taps - 1, units, device="cuda"), torch.zeros(B, units, states, device="cuda")
    x = inputs.double() @ w1.double().T + b1.double()
    whole = scan_layer(x, [v.double() for v in (conv, conv_bias, a, skip, step_bias)]) @ w3.double().T + b3.double()
    top_p = torch.full((B,), 0.9, device="cuda")
    agree = 0
    for t in range(T):
        row = (inputs[t].double() @ w1.double().T + b1.double()).float()[:, None]            # [B, 1, 3 D + 2 N]
        u, _ = sequence.causal_convolution(row[:, :, :units], conv, conv_bias, state=before, final_state=before)
        B_, C_ = (row[:, :, 3 * units + k * states:3 * units + (k + 1) * states].unflatten(2, (1, states)) for k in (0, 1))
        y, _ = sequence.selective_scan(u, row[:, :, 2 * units:3 * units], -torch.exp(a), B_, C_, D=skip, z=row[:, :, units:2 * units], delta_bias=step_bias,
                                       state=held, final_state=held)
        logits = (y[:, 0].double() @ w3.double().T + b3.double()).float()
        near(logits.cpu().numpy(), whole[t], "logits of step %d" % t)
        token, _ = sequence.sample(logits, uniform[t], top_p=top_p)
        agree += (token == tokens[t]).sum().item()
    # logits 1e-5 apart move a border of the draw by some 1e-5 of the row: 96 draws among 33 borders, a differing one in 30 runs
    assert agree >= T * B - 2
    net.close()


def test_refusals():
    ok = capi.fc(capi.selective_scan_inputs(D, N))
    for layers in ([capi.fc(46), capi.selective_scan(D, N), capi.fc(3)],                                  # reads the input layer
                   [capi.fc(5), capi.fc(45), capi.selective_scan(D, N), capi.fc(3)],                      # another width
                   [capi.fc(5), ok, capi.selective_scan(D, 0), capi.fc(3)], [capi.fc(5), ok, capi.selective_scan(D, 129), capi.fc(3)],
                   [capi.fc(5), ok, capi.selective_scan(D, N, 9), capi.fc(3)], [capi.fc(5), ok, capi.selective_scan(D, N)],
                   [capi.fc(5), ok, capi.selective_scan(D, N), capi.residual(1), capi.fc(D), capi.fc(3)]):
        with pytest.raises(RuntimeError):
            Net(capi.net(layers, 2, T=3))
    net = Net(network(2, 3), capi.opt())
    net.forward(np.zeros((2, 3, 7), np.float32))
    index, teacher = torch.zeros(2, 3, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, 1, device="cuda")
    with pytest.raises(RuntimeError, match="softmax"):
        net.compute_error_distillation(index, teacher)
    with pytest.raises(RuntimeError, match="softmax"):
        net.sample_outputs(teacher[..., 0].contiguous(), index[..., 0].contiguous())
    with pytest.raises(ValueError):
        net.compute_error_distillation(index.cpu(), teacher)
    with pytest.raises(RuntimeError):
        net.save("/tmp/selective_scan_layer.nn")
    net.close()
