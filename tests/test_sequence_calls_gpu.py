"""Calls that the documentation of the sequence operators allows and that their other tests do not make."""
import ctypes as C
import math
import threading

import numpy as np
import pytest
import torch

from myea_b200 import capi, sequence
from myea_b200.net import Net

from test_sequence_gpu import DEV, close, normal, run_scan, scan_inputs, scan_reference
from test_sequence_net_gpu import near, network, parameters, scan_layer, scan_parameters
from test_sequence_outputs_gpu import check_sampling, distillation_reference, teacher_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v", [1, 50, 4099, 131072])
def test_a_least_share_above_one_keeps_the_largest(v):
    """min_p counts as 1 at most: what weighs as much as the largest word stays, whatever else is asked for"""
    gen = torch.Generator(device=DEV).manual_seed(71)
    x = torch.randn(4, v, generator=gen, device=DEV)
    x[1] = x[1].round()                # several largest words
    x[2, ::2] = -math.inf
    x[3, v // 2] = math.inf
    u = torch.rand(4, generator=gen, device=DEV)
    top_k, top_p = torch.tensor([3, 0, 7, 1], dtype=torch.int32, device=DEV), torch.tensor([0.9, 0.3, 0.0, 1.0], device=DEV)
    for least in (1.0, 1.0005, 1.5, 100.0, 3e38, math.inf):
        min_p = torch.full((4,), least, device=DEV)
        for dtype in (torch.float32, torch.bfloat16):
            y = x.to(dtype)
            check_sampling(y, u, min_p=min_p)
            check_sampling(y, u, torch.full((4,), 0.7, device=DEV), top_k, top_p, min_p)
            check_sampling(y, u, torch.full((4,), 1e30, device=DEV), None, top_p, min_p)


def test_draws_from_several_host_threads():
    """threads whose launches take different amounts of shared memory, each a tight loop of calls (a refused one is counted, not lost)"""
    lib, rounds, sizes = capi.load(), 6000, (50, 32000, 1000, 60001)
    gen = torch.Generator(device=DEV).manual_seed(70)
    rows = [(torch.randn(1, v, generator=gen, device=DEV) * 2, torch.rand(1, generator=gen, device=DEV)) for v in sizes]
    want = [check_sampling(x, u) for x, u in rows]
    tokens = [torch.full_like(w, -7) for w in want]
    streams = [torch.cuda.Stream() for _ in sizes]
    torch.cuda.synchronize()
    begin, refused = threading.Barrier(len(sizes)), [None] * len(sizes)

    def draw(k):
        (x, u), message = rows[k], C.create_string_buffer(256)
        s = capi.Sampling(capi.TYPE_F32, 0, 1, sizes[k], logits=x.data_ptr(), logits_stride=sizes[k], uniform=u.data_ptr(), tokens=tokens[k].data_ptr())
        begin.wait(60)
        refused[k] = sum(lib.myea_b200_sample(0, C.byref(s), streams[k].cuda_stream, message, 256) != 0 for _ in range(rounds))

    threads = [threading.Thread(target=draw, args=(k,)) for k in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert refused == [0] * len(sizes)
    for a, b in zip(tokens, want):
        assert torch.equal(a, b)


def busy():
    """some 10 ms of work on the current stream"""
    a = torch.ones(4096, 4096, device=DEV, dtype=torch.bfloat16)
    for _ in range(100):
        a = a @ a * 0.0
    return a.sum().float()


def test_network_calls_keep_the_order_of_torchs_stream():
    """arguments that torch is still writing, that are written over or dropped behind the call, and results that torch reads next: no
    synchronization in between"""
    T, B, V = 3, 6, 21
    net = Net(network(T, B, outputs=V, softmax=True), capi.opt(capi.OPT_GD, gd_lr=0.0))
    net.set(capi.BUF_PARAMETERS, parameters(net, 3, 2))
    net.forward(np.random.default_rng(2).standard_normal((T, B, 7)).astype(np.float32))
    gen = torch.Generator(device=DEV).manual_seed(72)
    index = torch.randint(V, (T, B, 5), generator=gen, device=DEV, dtype=torch.int32)
    teacher, weight = torch.randn(T, B, 5, generator=gen, device=DEV), torch.rand(T, B, generator=gen, device=DEV)
    uniform, top_p = torch.rand(T, B, generator=gen, device=DEV), torch.rand(T, B, generator=gen, device=DEV) * 0.9 + 0.05
    busy()
    torch.cuda.synchronize()
    net.compute_error_distillation(index, teacher, weight=weight)
    errors = net.errors(3)
    tokens, chances = torch.full((T, B), -7, dtype=torch.int32, device=DEV), torch.zeros(T, B, device=DEV)
    net.sample_outputs(uniform, tokens, top_p=top_p, chances=chances)
    net.synchronize()
    torch.cuda.synchronize()
    assert (tokens >= 0).all() and np.abs(errors).max() > 0
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            late = [torch.zeros_like(v) for v in (index, teacher, weight)]
            torch.cuda.synchronize()
            late[2] += busy()
            for to, v in zip(late, (index, teacher, weight)):
                to += v
            net.compute_error_distillation(late[0], late[1], weight=late[2])
            for to in late:
                to.zero_()
            net.synchronize()
            assert np.array_equal(net.errors(3), errors)
            given, drawn, had = torch.zeros_like(uniform), torch.full_like(tokens, -7), torch.zeros_like(chances)
            torch.cuda.synchronize()
            given += busy()
            given += uniform
            net.sample_outputs(given, drawn, top_p=top_p * 1.0, chances=had)
            given.fill_(0.999)
            seen, share = drawn.clone(), had.clone()   # (torch reads behind the network's kernel)
            assert torch.equal(seen, tokens) and torch.equal(share, chances)
            torch.cuda.synchronize()
    net.close()


def test_tensors_that_want_a_gradient_are_refused():
    """autograd does not see these calls: rather an error than a result without history"""
    i = scan_inputs(73, torch.float32, 1, 4, 8, 4, 1)
    w = normal(torch.Generator(device=DEV).manual_seed(1), 8, 4)
    logits, index, teacher = normal(torch.Generator(device=DEV).manual_seed(2), 2, 9), torch.zeros(2, 1, dtype=torch.int32, device=DEV), torch.zeros(2, 1, device=DEV)
    scan = lambda j: sequence.selective_scan(j["u"], j["delta"], j["A"], j["B"], j["C"], D=j["D"], z=j["z"], delta_bias=j["bias"], state=j["state"])  # noqa: E731
    wants = lambda v: v.clone().requires_grad_()  # noqa: E731
    for name in ("u", "delta", "A", "B", "C", "D", "z", "bias", "state"):
        with pytest.raises(ValueError, match="gradient"):
            scan({**i, name: wants(i[name])})
    for call in (lambda: sequence.causal_convolution(wants(i["u"]), w), lambda: sequence.causal_convolution(i["u"], wants(w)),
                 lambda: sequence.causal_convolution(i["u"], w, out=wants(i["u"])), lambda: sequence.causal_convolution_backward(wants(i["dy"]), i["u"], w),
                 lambda: sequence.distillation_error(wants(logits), index, teacher), lambda: sequence.distillation_error(logits, index, wants(teacher)),
                 lambda: sequence.distillation_error(logits, index, teacher, weight=wants(teacher[:, 0]))):
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():   # and where nothing is recorded they are like any other
        for a, b in zip(scan({k: wants(v) for k, v in i.items()}), scan(i)):
            assert torch.equal(a, b)
        sequence.causal_convolution(i["u"], wants(w), out=torch.nn.Parameter(i["u"].clone()))
        assert torch.equal(sequence.distillation_error(wants(logits), index, teacher)[1], sequence.distillation_error(logits, index, teacher)[1])
    # a draw is whole numbers, which have no gradient anywhere
    u = torch.tensor([0.3, 0.6], device=DEV)
    assert torch.equal(sequence.sample(wants(logits), u)[0], sequence.sample(logits, u)[0])


@pytest.mark.parametrize("t,d,n", [(1, 20, 16), (21, 20, 16), (37, 9, 5), (600, 20, 16)])
def test_rates_of_minus_infinity_forget_and_leave_the_other_steps_alone(t, d, n):
    """a rate of minus infinity (or one that becomes it in the change of base) drops the state at every step; where there is no step, behind
    a sequence's end and in the rest of a tile, the state stays.  The reference has -1e30 in its place, whose decays are the same 0
    and 1; the tolerance is the one of the other scan tests, with the exponents of the finite rates."""
    i = scan_inputs(74, torch.float32, 3, t, d, n, 1)
    lengths = torch.tensor([t, t // 3, 0], dtype=torch.int32, device=DEV)
    behind = torch.arange(t, device=DEV)[None] >= lengths[:, None]
    for name in ("u", "delta", "B", "C", "z", "dy"):
        i[name][behind] = math.nan
    i["A"][::3, 1::2] = -math.inf
    i["A"][1::3, 0] = torch.finfo(torch.float32).min
    got = run_scan(i, True, lengths)
    clean = {k: torch.nan_to_num(v.double()) for k, v in i.items()}
    clean["A"] = i["A"].double().clamp(min=-1e30)
    want, big = scan_reference(clean, True, lengths, False), scan_reference(clean, True, lengths, True)
    exponents = scan_reference({**clean, "A": torch.where(clean["A"] < -1e20, -1.0, clean["A"])}, True, lengths, False)["exponents"]
    once = (t + 16) * 2.0 ** -22 + (exponents + 4) * 2.0 ** -21 + 80 * 2.0 ** -23 + n * 2.0 ** -24
    for name in want:
        if name != "exponents":
            sums = {"A": 3 * t, "D": 3 * t, "delta_bias": 3 * t, "B": d, "C": d}.get(name, 0)
            close(name, got[name], want[name], (once + sums * 2.0 ** -24) * big[name])


@pytest.mark.parametrize("dtype,r,v,tau,hard", [(torch.float32, 2, 50001, 4.0, 0.25), (torch.bfloat16, 2, 131072, 1.0, 0.0), (torch.float32, 300, 131072, 2.0, 0.5),
                                                (torch.bfloat16, 600, 60001, 1.0, 0.0), (torch.float16, 203, 32001, 1.5, 0.25), (torch.bfloat16, 1200, 8003, 1.5, 0.5),
                                                (torch.float32, 203, 16001, 1.5, 0.25), (torch.bfloat16, 203, 32001, 1.0, 0.0), (torch.float16, 111, 64001, 2.0, 0.5)])
def test_long_rows_of_the_distillation_lose_no_word(dtype, r, v, tau, hard):
    """Sums as exact as they are made: a thread adds up at most v / 256 + 128 words (a block has 256 threads or more, or eight packs of 8 words each), lanes,
    warps and blocks add 5 + 4 + 3 times: depth * 2^-24.  A thread's maximum rises at most once for each 2 packs of 4 words that it reads, every warp's
    and block's three times more; a rise multiplies by an exponential, which is off by E = 2^-22 + 2^-23 (R / T + 2) as the words' own are.  On random
    logits a thread's maximum rises about ln(v / 256) times, 8 at most here; 16 are allowed.  A sum, and with it a gradient, is good to (16 + 5) E +
    depth * 2^-24, below 2^-13 here: a share of the row that got lost shows."""
    gen = torch.Generator(device=DEV).manual_seed(v + r)
    x = (torch.randn(r, v, generator=gen, device=DEV) * 0.5).to(dtype)
    index, teacher = teacher_for(gen, r, v, 5)
    labels = torch.randint(v, (r,), generator=gen, device=DEV, dtype=torch.int32)
    losses, d = sequence.distillation_error(x, index, teacher, tau, 1.0 - hard, hard, labels)
    some = torch.arange(0, r, max(1, r // 6), device=DEV)
    want, grad, want_big, grad_big = distillation_reference(x[some], index[some], teacher[some], tau, 1.0 - hard, hard, labels[some], None)
    reach = (x.double().max() - x.double().min()).item()
    reach = max(reach, (teacher.max() - teacher.min()).item())
    e = 2.0 ** -22 + 2.0 ** -23 * (reach / min(tau, 1.0) + 2)
    share = 21 * e + (v / 256 + 140) * 2.0 ** -24
    assert share < 2.0 ** -13
    off = (losses[some].double().cpu() - want).abs() - (share * (want_big + 1.0) + 2.0 ** -24 * want.abs())
    assert off.max() <= 0, off.max()
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * (2.0 ** -10 if dtype == torch.float16 else 1)
    off = (d[some].double().cpu() - grad).abs() - (half * grad.abs() + (1 + half) * share * grad_big + tiny)
    assert off.max() <= 0, off.max()


def directions(net, X, Y, layers, out):
    """derivatives of every layer against differences of the loss: outputs good to 1e-6 of 1, a difference of losses of some 50 good to 2e-3 of its slope, and
    the third derivative adds h^2"""
    p = net.get(capi.BUF_PARAMETERS)
    rng = np.random.default_rng(5)

    def loss(params):
        net.set(capi.BUF_PARAMETERS, params)
        net.forward(X)
        return 0.5 * float(((net.outputs(out).astype(np.float64) - Y) ** 2).sum())

    net.forward(X)
    net.compute_error(Y)
    net.backward()
    net.update_derivative_weight()
    g = net.get(capi.BUF_DERIVATIVES).astype(np.float64)
    for l in layers:
        li = net.layer_index(l)
        a, b = int(li.first_connection_index), int(li.last_connection_index)
        way = np.zeros(net.P)
        way[a:b] = rng.standard_normal(b - a)
        way /= np.linalg.norm(way)
        h = 1e-2
        slope = (loss((p + h * way).astype(np.float32)) - loss((p - h * way).astype(np.float32))) / (2 * h)
        assert abs(slope - g @ way) <= 1e-2 * np.linalg.norm(g[a:b]) + 1e-2, (l, slope, g @ way)
    net.set(capi.BUF_PARAMETERS, p)


@pytest.mark.parametrize("T", [1, 6])
@pytest.mark.parametrize("kind", ["normalized", "recurrent below", "lstm above", "pooling above", "recurrent above", "pooling below"])
def test_scan_layer_among_layers_of_other_kinds(kind, T):
    B, d, n = 6, 8, 4
    wide = capi.selective_scan_inputs(d, n)
    below = {"normalized": [capi.fc(wide, capi.AF_TANH, norm=capi.NORM_BN)], "recurrent below": [capi.fc_ind_rnn(wide, capi.AF_TANH)],
             "pooling below": [capi.fc(wide, capi.AF_TANH), capi.pooling(capi.LAYER_AVERAGE_POOLING, 3, 1), capi.fc(wide, capi.AF_LINEAR)]}.get(kind, [capi.fc(wide, capi.AF_TANH)])
    above = {"lstm above": [capi.lstm(3)], "pooling above": [capi.pooling(capi.LAYER_AVERAGE_POOLING, 2, 2)],
             "recurrent above": [capi.fc_ind_rnn(7, capi.AF_TANH)]}.get(kind, [])
    layers = [capi.fc(4)] + below + [capi.selective_scan(d, n, 3)] + above + [capi.fc(3, capi.AF_LINEAR)]
    net = Net(capi.net(layers, B, T=T), capi.opt(capi.OPT_GD, gd_lr=0.0))
    rng = np.random.default_rng(6)
    p = (rng.standard_normal(net.P) * 0.3).astype(np.float32)
    if net.n_norm:
        p[net.W + net.n_bias:net.W + net.n_bias + net.n_norm] = 1.0
    net.set(capi.BUF_PARAMETERS, p)
    X, Y = rng.standard_normal((T, B, 4)).astype(np.float32), rng.standard_normal((T, B, 3)).astype(np.float32)
    directions(net, X, Y, [l for l in range(1, len(layers)) if layers[l].type_layer not in (capi.LAYER_AVERAGE_POOLING,)], len(layers) - 1)
    net.close()


def test_scan_layer_behind_dropout():
    """the scan reads the outputs that dropout leaves, and its error goes on to the layer below as for any other layer above it"""
    T, B, d, n, k = 5, 4, 12, 5, 4
    layers = [capi.fc(7), capi.fc(capi.selective_scan_inputs(d, n), capi.AF_TANH, dropout=capi.DROP_BERNOULLI, p=(0.7, 0.0, 0.0)), capi.selective_scan(d, n, k),
              capi.fc(9, capi.AF_LINEAR)]
    net = Net(capi.net(layers, B, T=T), capi.opt(capi.OPT_GD, gd_lr=0.0))
    p = parameters(net, 9, 2, d, n, k)
    net.set(capi.BUF_PARAMETERS, p)
    rng = np.random.default_rng(7)
    mask = (rng.random((T, capi.selective_scan_inputs(d, n))) < 0.7).astype(np.uint8)
    net.set_mask_bernoulli(1, mask)
    net.forward(rng.standard_normal((T, B, 7)).astype(np.float32))
    net.compute_error(rng.standard_normal((T, B, 9)).astype(np.float32))
    net.backward()
    net.update_derivative_weight()
    read = net.outputs(1)
    assert (read[np.broadcast_to(mask[:, None] == 0, read.shape)] == 0).all() and (read != 0).any()
    x, q = torch.tensor(read.astype(np.float64), requires_grad=True), torch.tensor(p.astype(np.float64), requires_grad=True)
    y = scan_layer(x, scan_parameters(net, q, 2, d, n, k))
    near(net.outputs(2), y, "outputs")
    (y * torch.tensor(net.errors(2).astype(np.float64))).sum().backward()
    near(net.errors(1), x.grad * (1 - x.detach() ** 2), "error below")   # (tanh's slope from its output)
    li = net.layer_index(2)
    a, b = int(li.first_connection_index), int(li.last_connection_index)
    near(net.get(capi.BUF_DERIVATIVES)[a:b], q.grad[a:b], "derivatives")
    net.close()


def test_network_calls_are_not_captured_from_another_stream():
    """the network's forward pass runs on its own stream, whatever torch captures: replays would draw from whatever lies there"""
    T, B, V = 2, 3, 9
    net = Net(network(T, B, outputs=V, softmax=True), capi.opt(capi.OPT_GD, gd_lr=0.0))
    net.set(capi.BUF_PARAMETERS, parameters(net, 4, 2))
    net.forward(np.random.default_rng(3).standard_normal((T, B, 7)).astype(np.float32))
    index, teacher = torch.zeros(T, B, 2, dtype=torch.int32, device=DEV), torch.zeros(T, B, 2, device=DEV)
    uniform, tokens = torch.full((T, B), 0.4, device=DEV), torch.full((T, B), -7, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        uniform.mul_(1.0)
        with pytest.raises(RuntimeError, match="captured"):
            net.sample_outputs(uniform, tokens)
        with pytest.raises(RuntimeError, match="captured"):
            net.compute_error_distillation(index, teacher)
    assert (tokens == -7).all()
    with torch.cuda.stream(torch.cuda.ExternalStream(net.lib.myea_b200_stream(net.h))):   # torch on the network's own stream: in order anyway
        net.sample_outputs(uniform, tokens)
        seen = tokens.clone()
    torch.cuda.synchronize()
    assert ((seen >= 0) & (seen < V)).all()
    net.compute_error_distillation(index, teacher)
    net.synchronize()
    net.close()
