"""The sequence operators at the sizes and orders of calls where another of their kernels answers: rows beyond the clusters' memory, long
rows in plenty, a few positions of many sequences, nothing at all, arrays whose offsets pass 32 bits, calls side by side.  What two ways
of asking for the same must give is compared bit by bit; the rest by the checks, and with the tolerances, of the operators' own tests."""
import math

import pytest
import torch

from myea_b200 import sequence

from test_sequence_gpu import DEV, normal, run_scan, scan_inputs
from test_sequence_outputs_gpu import check_distillation, check_sampling, teacher_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,v", [(torch.float32, 400003), (torch.bfloat16, 600001), (torch.float16, 530001)])
def test_sampling_beyond_the_clusters_memory(dtype, v):
    gen = torch.Generator(device=DEV).manual_seed(v)
    x = (torch.randn(2, v, generator=gen, device=DEV) * 3).to(dtype)
    u = torch.tensor([0.123, 0.876], device=DEV)
    top_k = torch.tensor([5000, 17], dtype=torch.int32, device=DEV)
    top_p, min_p = torch.tensor([0.35, 0.93], device=DEV), torch.tensor([0.02, 0.3], device=DEV)
    check_sampling(x, u)
    check_sampling(x, u, top_k=top_k)
    check_sampling(x, u, top_p=top_p)
    check_sampling(x, u, torch.tensor([0.7, 0.0], device=DEV), top_k, top_p, min_p)
    equal = torch.full_like(x, 0.5)   # every word on the threshold: the index decides
    check_sampling(equal, u, top_k=top_k, top_p=top_p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_of_many_long_rows(dtype):
    r, v, k = 150, 40003, 20
    gen = torch.Generator(device=DEV).manual_seed(21)
    x = (torch.randn(r, v, generator=gen, device=DEV) * 3).to(dtype)
    index, teacher = teacher_for(gen, r, v, k)
    index[:, 3] = index[:, 0]        # a word twice
    index[1, 5], index[2, 6] = -1, v
    labels = torch.randint(v, (r,), generator=gen, device=DEV, dtype=torch.int32)
    labels[:50] = index[:50, 0]
    weight = torch.rand(r, generator=gen, device=DEV)
    weight[7] = 0.0
    check_distillation(x, index, teacher, 2.0, 0.5, 0.5, labels, weight)
    check_distillation(x, index, teacher, 1.0, 0.75, 0.25, labels, weight, in_place=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,d,n,g", [(203, 66, 7, 3), (603, 64, 16, 1), (301, 130, 1, 1), (597, 8, 128, 1), (149, 300, 33, 2)])
def test_few_positions_of_many_sequences_follow_the_whole(dtype, b, d, n, g):
    t = 9
    i = scan_inputs(b, dtype, b, t, d, n, g)
    lengths = torch.randint(0, t + 1, (b,), device=DEV, dtype=torch.int32, generator=torch.Generator(device=DEV).manual_seed(b))
    behind = torch.arange(t, device=DEV)[None] >= lengths[:, None]
    for name in ("u", "delta", "B", "C", "z"):
        i[name][behind] = math.nan
    par = dict(D=i["D"], delta_bias=i["bias"])
    y, final = sequence.selective_scan(i["u"], i["delta"], i["A"], i["B"], i["C"], z=i["z"], lengths=lengths, state=i["state"], **par)
    state, at = i["state"].clone(), 0
    for piece in (4, 1, 3, 1):
        cut = lambda v: v[:, at:at + piece]  # noqa: E731
        s, _ = sequence.selective_scan(cut(i["u"]), cut(i["delta"]), i["A"], cut(i["B"]), cut(i["C"]), z=cut(i["z"]), lengths=lengths - at, state=state,
                                       final_state=state, **par)
        assert torch.equal(s, cut(y)), at
        at += piece
    assert torch.equal(state, final) and torch.isfinite(y.double()).all()


def test_nothing_to_do():
    for t in (0, 1, 300):
        i = scan_inputs(30, torch.float32, 0, t, 24, 16, 1)
        got = run_scan(i)
        assert got["y"].shape == (0, t, 24) and got["state"].shape == (0, 24, 16)
        for name in ("A", "D", "delta_bias"):
            assert not got[name].any(), name
        held = torch.full((24, 16), 3.0, device=DEV)
        run_scan(i, d_A=held, d_D=torch.zeros(24, device=DEV), d_delta_bias=torch.zeros(24, device=DEV), accumulate=True)
        assert (held == 3.0).all()
        w, bias = normal(torch.Generator(device=DEV).manual_seed(1), 24, 4), torch.zeros(24, device=DEV)
        y, final = sequence.causal_convolution(i["u"], w, bias)
        d = sequence.causal_convolution_backward(i["dy"], i["u"], w, bias)
        assert y.shape == (0, t, 24) and final.shape == (0, 3, 24) and not d["weight"].any() and not d["bias"].any()
    empty = torch.empty(0, 100, device=DEV)
    losses, grad = sequence.distillation_error(empty, torch.empty(0, 5, dtype=torch.int32, device=DEV), torch.empty(0, 5, device=DEV))
    tokens, chances = sequence.sample(empty, torch.empty(0, device=DEV))
    assert losses.shape == (0,) and grad.shape == (0, 100) and tokens.shape == chances.shape == (0,)


def test_derivatives_of_slices_of_wider_time_major_arrays():
    """every activation a slice off the 16-byte boundaries of an array with time in front"""
    i = scan_inputs(31, torch.bfloat16, 3, 150, 70, 16, 2)
    lengths = torch.tensor([150, 77, 1], dtype=torch.int32, device=DEV)
    want = run_scan(i, lengths=lengths)
    wide = dict(i)
    for name in ("u", "delta", "B", "C", "z", "dy"):
        v = i[name].flatten(2)
        store = torch.full((150, 3, v.shape[2] + 9), math.nan, device=DEV, dtype=v.dtype)
        store[:, :, 5:5 + v.shape[2]] = v.transpose(0, 1)
        view = store[:, :, 5:5 + v.shape[2]].transpose(0, 1)
        wide[name] = view if name not in ("B", "C") else view.unflatten(2, (2, 16))
    got = run_scan(wide, lengths=lengths)
    for name in want:
        assert torch.equal(got[name], want[name]), name
    w, bias = normal(torch.Generator(device=DEV).manual_seed(2), 70, 4), torch.zeros(70, device=DEV)
    plain = sequence.causal_convolution_backward(i["dy"], i["u"], w, bias, lengths=lengths)
    into = torch.full((150, 3, 79), 9.0, device=DEV, dtype=torch.bfloat16)
    sliced = sequence.causal_convolution_backward(wide["dy"], wide["u"], w, bias, lengths=lengths, dx=into[:, :, 5:75].transpose(0, 1))
    for name in ("x", "weight", "bias"):
        assert torch.equal(plain[name], sliced[name]), name
    assert (into[:, :, :5] == 9.0).all() and (into[:, :, 75:] == 9.0).all()


def test_offsets_beyond_32_bits():
    far = (1 << 31) + 8
    memory = torch.empty(far + (1 << 16), dtype=torch.bfloat16, device=DEV)

    def spread(v):   # a [2, ...] tensor with its halves 4 GB apart
        view = memory.as_strided((2,) + v.shape[1:], (far,) + v.stride()[1:], spread.at)
        spread.at += (v[0].numel() + 7) // 8 * 8
        return view.copy_(v)

    spread.at = 0
    i = scan_inputs(32, torch.bfloat16, 2, 40, 24, 16, 1)
    want = run_scan(i)
    got = run_scan({k: spread(v) if k in ("u", "delta", "B", "C", "z", "dy") else v for k, v in i.items()})
    for name in want:
        assert torch.equal(got[name], want[name]), name
    w = normal(torch.Generator(device=DEV).manual_seed(3), 24, 4)
    spread.at = 0
    x, dy = spread(i["u"]), spread(i["dy"])
    y, dx = spread(torch.zeros_like(i["u"])), spread(torch.zeros_like(i["u"]))
    sequence.causal_convolution(x, w, out=y)
    got, want = sequence.causal_convolution_backward(dy, x, w, dx=dx), sequence.causal_convolution_backward(i["dy"], i["u"], w)
    assert torch.equal(y, sequence.causal_convolution(i["u"], w)[0])
    assert torch.equal(got["x"], want["x"]) and torch.equal(got["weight"], want["weight"])
    gen = torch.Generator(device=DEV).manual_seed(33)
    logits = normal(gen, 2, 1003, scale=3.0, dtype=torch.bfloat16)
    index, teacher = teacher_for(gen, 2, 1003, 9)
    spread.at = 0
    apart = spread(logits)
    u = torch.tensor([0.2, 0.9], device=DEV)
    assert torch.equal(sequence.sample(apart, u)[0], sequence.sample(logits, u)[0])
    losses, grad = sequence.distillation_error(apart, index, teacher, d_logits=apart)
    for a, b in zip((losses, grad), sequence.distillation_error(logits, index, teacher)):
        assert torch.equal(a, b)


def test_calls_side_by_side():
    """two streams that work at the same time, each with its own arrays, give what each gives alone"""
    work = []
    for k in range(2):
        gen = torch.Generator(device=DEV).manual_seed(40 + k)
        i = scan_inputs(40 + k, torch.float32, 1, 512, 96, 16, 1)
        logits = normal(gen, 40, 20001, scale=3.0)
        work.append((i, normal(gen, 96, 4), logits, *teacher_for(gen, 40, 20001, 9), torch.rand(40, generator=gen, device=DEV), torch.full((40,), 0.9, device=DEV)))

    def run(i, w, logits, index, teacher, u, top_p):
        d = sequence.causal_convolution_backward(i["dy"], i["u"], w)
        return [v for v in run_scan(i).values() if v is not None] + [d["x"], d["weight"], *sequence.distillation_error(logits, index, teacher),
                                                                     *sequence.sample(logits, u, top_p=top_p)]

    alone = [run(*w) for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(5):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[k].append(run(*work[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for got in results[k]:
            for a, b in zip(got, alone[k]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["normal", "sorted", "steps", "closed", "peaked", "flat"])
def test_limits_of_long_rows(kind):
    """limits about the number of threads that a row has, and words of which every thread, few threads or one have the largest"""
    v, gen = 131072, torch.Generator(device=DEV).manual_seed(50)
    x = torch.randn(6, v, generator=gen, device=DEV) * 2
    if kind == "sorted":
        x = x.sort(1)[0]
    if kind == "steps":
        x = x.round()
    if kind == "closed":
        x[torch.rand(6, v, generator=gen, device=DEV) < 0.995] = -math.inf
    if kind == "peaked":
        x[:, v // 3] += 30.0
    if kind == "flat":
        x = torch.full_like(x, 1.5)
    u = torch.rand(6, generator=gen, device=DEV)
    top_k = torch.tensor([1, 1023, 2047, 2048, 2049, v - 1], dtype=torch.int32, device=DEV)
    top_p = torch.tensor([0.5, 0.9, 0.999, 0.01, 0.7, 0.95], device=DEV)
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        check_sampling(y, u, top_k=top_k)
        check_sampling(y, u, torch.full((6,), 0.6, device=DEV), top_k, top_p)


def test_a_captured_token_step_carries_its_states():
    """a step of answering in one graph, the states written in place and its logits scored against a teacher, replayed on new inputs"""
    b, d, n = 5, 200, 16
    gen = torch.Generator(device=DEV).manual_seed(60)
    w, bias, A = normal(gen, d, 4), normal(gen, d), -torch.exp(normal(gen, d, n))
    index, teacher = teacher_for(gen, b, d, 7)
    top_p = torch.full((b,), 0.8, device=DEV)
    inputs = [dict(x=normal(gen, b, 1, d), z=normal(gen, b, 1, d), delta=normal(gen, b, 1, d), B=normal(gen, b, 1, 1, n), C=normal(gen, b, 1, 1, n),
                   u=torch.rand(b, generator=gen, device=DEV)) for _ in range(4)]
    start = [normal(gen, b, 3, d), normal(gen, b, d, n)]

    def step(i, conv, h):
        x, _ = sequence.causal_convolution(i["x"], w, bias, state=conv, final_state=conv)
        y, _ = sequence.selective_scan(x, i["delta"], A, i["B"], i["C"], z=i["z"], state=h, final_state=h)
        tokens, chances = sequence.sample(y[:, 0], i["u"], top_p=top_p)
        losses, grad = sequence.distillation_error(y[:, 0], index, teacher, temperature=2.0)
        return [y, tokens, chances, losses, grad]

    conv, h = (s.clone() for s in start)
    want = [[v.clone() for v in step(i, conv, h)] + [conv.clone(), h.clone()] for i in inputs]
    held, states = {k: v.clone() for k, v in inputs[0].items()}, [s.clone() for s in start]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held, *states)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held, *states)
    for s, v in zip(states, start):
        s.copy_(v)
    for i, expected in zip(inputs, want):
        for k, v in i.items():
            held[k].copy_(v)
        graph.replay()
        for a, e in zip(out + states, expected):
            assert torch.equal(a, e)


@pytest.mark.parametrize("dtype,r,v", [(torch.bfloat16, 1200, 2500), (torch.float32, 300, 2305), (torch.float16, 300, 16003), (torch.bfloat16, 203, 32001),
                                       (torch.bfloat16, 320, 33003), (torch.float32, 1200, 700)])
def test_distillation_by_rows_and_lengths(dtype, r, v):
    """numbers of rows and lengths between which the threads of a row change"""
    gen = torch.Generator(device=DEV).manual_seed(v)
    x = (torch.randn(r, v, generator=gen, device=DEV) * 3).to(dtype)
    index, teacher = teacher_for(gen, r, v, 6)
    labels = torch.randint(v, (r,), generator=gen, device=DEV, dtype=torch.int32)
    check_distillation(x, index, teacher, 1.5, 0.5, 0.5, labels, torch.rand(r, generator=gen, device=DEV))
    check_distillation(x, index, teacher, in_place=True)
