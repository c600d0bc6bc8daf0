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
from test_sequence_net_gpu import network, parameters
from test_sequence_outputs_gpu import check_sampling

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
