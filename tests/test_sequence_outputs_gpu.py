"""The error against a teacher's best logits and the draw of tokens against their definitions in 64 bits.

Tolerances.  An exponential is good to 2 steps (2^-22) and its argument (x - m) c to 2 roundings, 2^-23 of its magnitude, at most R / T with R
the range of the row; a sum of n of them adds n * 2^-24 when its order is free.  With E = 2^-22 + 2^-23 (R / T + 2) + n * 2^-24 a
probability is good to 2 E of itself, a gradient weight * (soft T (q - p) + hard (r - 1)) to 2 E + 2^-22 of weight * (soft T (q + p) + hard (r + 1)),
and a loss to the same share of its terms' magnitudes.  Tokens are whole numbers and have to be equal: the kernel's sums are exact
to 1e-12, and no case here puts its random number that close to a border unless both sides compute it without rounding."""
import math

import numpy as np
import pytest
import torch

from myea_b200 import sequence

pytestmark = pytest.mark.gpu
DEV = "cuda"


def distillation_reference(x, index, teacher, tau, soft, hard, labels, weight):
    """(losses, gradient, magnitudes of both) in 64 bits, row by row"""
    x, teacher = x.double().cpu(), teacher.double().cpu()
    index, r, v = index.cpu().long(), *x.shape
    loss, grad = torch.zeros(r, dtype=torch.float64), torch.zeros(r, v, dtype=torch.float64)
    loss_big, grad_big = torch.zeros_like(loss), torch.zeros_like(grad)
    for i in range(r):
        w = 1.0 if weight is None else weight[i].item()
        if w == 0.0 or (x[i] == -math.inf).all():
            continue
        there = (index[i] >= 0) & (index[i] < v)
        there &= teacher[i] > -math.inf
        at = index[i][there]
        logq = torch.log_softmax(x[i] / tau, 0)
        if len(at):
            p = torch.softmax(teacher[i][there] / tau, 0)
            loss[i] += soft * tau * tau * (p * (p.log() - logq[at])).sum()
            loss_big[i] += abs(soft) * tau * tau * (p * (p.log().abs() + logq[at].abs())).sum()
            dense = torch.zeros(v, dtype=torch.float64).index_add_(0, at, p)
            grad[i] += soft * tau * (logq.exp() - dense)
            grad_big[i] += abs(soft) * tau * (logq.exp() + dense)
        label = -1 if labels is None else labels[i].item()
        if hard != 0.0 and 0 <= label < v:
            logr = torch.log_softmax(x[i], 0)
            one = torch.nn.functional.one_hot(torch.tensor(label), v).double()
            loss[i] -= hard * logr[label]
            loss_big[i] += abs(hard) * logr[label].abs()
            grad[i] += hard * (logr.exp() - one)
            grad_big[i] += abs(hard) * (logr.exp() + one)
        loss[i] *= w
        grad[i] *= w
        loss_big[i] *= abs(w)
        grad_big[i] *= abs(w)
    return loss, grad, loss_big, grad_big


def check_distillation(x, index, teacher, tau=1.0, soft=1.0, hard=0.0, labels=None, weight=None, in_place=False):
    want, grad, want_big, grad_big = distillation_reference(x, index, teacher, tau, soft, hard, labels, weight)
    open_ = x.double()[torch.isfinite(x.double())]
    reach = (open_.max() - open_.min()).item() if open_.numel() else 0.0
    tf = teacher[torch.isfinite(teacher)]
    reach = max(reach, (tf.max() - tf.min()).item() if tf.numel() else 0.0)
    e = 2.0 ** -22 + 2.0 ** -23 * (reach / min(tau, 1.0) + 2) + x.shape[1] * 2.0 ** -24
    share = 2 * e + 2.0 ** -22
    work = x.clone()
    losses, d = sequence.distillation_error(work, index, teacher, tau, soft, hard, labels, weight, d_logits=work if in_place else None)
    only, none = sequence.distillation_error(x, index, teacher, tau, soft, hard, labels, weight, derivatives=False)
    assert none is None and torch.equal(only, losses)
    off = (losses.double().cpu() - want).abs() - (share * (want_big + e) + 2.0 ** -24 * want.abs())
    assert off.max() <= 0, off.max()
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).tiny * (2.0 ** -10 if x.dtype == torch.float16 else 1)
    off = (d.double().cpu() - grad).abs() - (half * grad.abs() + (1 + half) * share * grad_big + tiny)
    assert torch.isfinite(d.double()).all() and off.max() <= 0, off.max()
    return losses, d


def teacher_for(gen, r, v, k):
    index = torch.stack([torch.randperm(v, generator=gen, device=DEV)[:k] for _ in range(r)]).to(torch.int32)
    return index, torch.randn(r, k, generator=gen, device=DEV) * 3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("r,v,k,tau,hard", [(3, 10, 4, 1.0, 0.0), (1, 1, 1, 2.0, 0.5), (5, 33, 33, 1.5, 0.25), (2, 1024, 16, 2.0, 0.5), (3, 4097, 50, 1.0, 0.5),
                                            (2, 50001, 64, 4.0, 0.25), (1, 131072, 7, 1.0, 0.0), (7, 75, 1, 0.5, 1.0), (2, 3001, 1024, 1.0, 0.1)])
def test_distillation(dtype, r, v, k, tau, hard):
    gen = torch.Generator(device=DEV).manual_seed(v + k)
    x = (torch.randn(r, v, generator=gen, device=DEV) * 3).to(dtype)
    index, teacher = teacher_for(gen, r, v, k)
    labels = torch.randint(v, (r,), generator=gen, device=DEV, dtype=torch.int32)
    weight = torch.rand(r, generator=gen, device=DEV)
    check_distillation(x, index, teacher, tau, 1.0 - hard, hard, labels, weight)
    check_distillation(x, index, teacher, tau, in_place=True)


def test_distillation_of_odd_rows():
    """entries that are not there, the same word twice, closed words, rows without weight, entries, label or open words"""
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(8, 41, generator=gen, device=DEV)
    index, teacher = teacher_for(gen, 8, 41, 6)
    labels = torch.tensor([3, -100, 41, 0, 7, 8, 9, 40], dtype=torch.int32, device=DEV)
    weight = torch.tensor([1.0, 0.0, 0.5, 2.0, 1.0, 1.0, 1.0, 1.0], device=DEV)
    x[1] = math.nan                       # weight 0: not read
    teacher[1] = math.nan
    index[2, 2:] = -1
    index[2, 4] = 1 << 30
    teacher[2, 2:] = math.nan             # nor are entries that are not there
    index[3] = -1                         # no entry at all
    index[4, :] = index[4, 0]             # one word, six times
    index[5, 3] = index[5, 1]
    index[5, 0] = 8                       # the label is one of the teacher's words
    x[6, 10:] = -math.inf
    index[6] = torch.arange(6, dtype=torch.int32, device=DEV)
    teacher[6, 2] = -math.inf
    x[7] = -math.inf
    losses, d = check_distillation(x, index, teacher, 2.0, 0.7, 0.3, labels, weight)
    assert losses[1] == 0 and (d[1] == 0).all() and losses[7] == 0 and (d[7] == 0).all() and (d[6, 10:] == 0).all()
    x[0] = torch.finfo(torch.float32).min   # lowest values instead of infinities: equal, so all open
    check_distillation(x[:1], index[:1], teacher[:1], 2.0, 0.7, 0.3, labels[:1], weight[:1])
    x[6, 10:] = torch.finfo(torch.float32).min
    _, d = sequence.distillation_error(x[6:7], index[6:7], teacher[6:7])
    assert (d[0, 10:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_reads_slices_and_leaves_their_neighbours(dtype):
    gen = torch.Generator(device=DEV).manual_seed(4)
    wide = (torch.randn(4, 517, generator=gen, device=DEV) * 2).to(dtype)
    index, teacher = teacher_for(gen, 4, 500, 9)
    x = wide[:, 3:503]
    out = torch.full((4, 519), 7.0, device=DEV, dtype=dtype)
    losses, d = sequence.distillation_error(x, index, teacher, d_logits=out[:, 5:505])
    want, dense = sequence.distillation_error(x.contiguous(), index, teacher)
    # (other boundaries, another order of the sums)
    assert torch.allclose(losses, want, rtol=1e-5, atol=0) and torch.allclose(d.float(), dense.float(), rtol=2.0 ** -7 if dtype == torch.bfloat16 else 1e-4, atol=1e-9)
    assert (out[:, :5] == 7).all() and (out[:, 505:] == 7).all()


def test_distillation_derivatives_against_differences():
    """central differences of fp32 losses of size 10, good to 1e-5, over 2 * 2^-5: good to 2e-4; the third derivative adds below 1e-3"""
    gen = torch.Generator(device=DEV).manual_seed(6)
    x = torch.randn(1, 12, generator=gen, device=DEV)
    index, teacher = teacher_for(gen, 1, 12, 5)
    label = torch.tensor([4], dtype=torch.int32, device=DEV)
    value = lambda y: sequence.distillation_error(y, index, teacher, 2.0, 0.6, 0.4, label, derivatives=False)[0].item()  # noqa: E731
    _, d = sequence.distillation_error(x, index, teacher, 2.0, 0.6, 0.4, label)
    for i in range(12):
        step = torch.zeros_like(x)
        step[0, i] = 2.0 ** -5
        assert abs((value(x + step) - value(x - step)) / 2.0 ** -4 - d[0, i].item()) < 2e-3


# ---- sampling --------------------------------------------------------------------------------------------------------------

def draw_reference(x, u, tau, top_k, top_p, min_p):
    """(token, chance) of one row of doubles, by the definition"""
    is_open = x > -math.inf
    if not is_open.any():
        return -1, 0.0
    order = np.array(sorted(np.flatnonzero(is_open), key=lambda i: (-x[i], i)))
    if not tau > 0.0:
        return int(order[0]), 1.0
    m = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == m, 1.0, np.exp((x[order] - m) / tau) if m < math.inf else 0.0)
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1.0:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((before < top_p * w.sum()).sum()))
        order, w = order[:n], w[:n]
    if min_p > 0.0:
        keep = w >= min(min_p, 1.0)
        order, w = order[keep], w[keep]
    back = np.argsort(order)
    order, w = order[back], w[back]
    sums = np.cumsum(w)
    j = int(np.argmax(sums > u * sums[-1]))
    return int(order[j]), w[j] / sums[-1]


def check_sampling(x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    tokens, chances = sequence.sample(x, u, temperature, top_k, top_p, min_p)
    again, _ = sequence.sample(x, u, temperature, top_k, top_p, min_p)
    assert torch.equal(tokens, again)
    rows = x.double().cpu().numpy()
    one = lambda a, r, none: none if a is None else a[r].item()  # noqa: E731
    for r in range(x.shape[0]):
        token, chance = draw_reference(rows[r], u[r].item(), one(temperature, r, 1.0), one(top_k, r, 0), one(top_p, r, 1.0), one(min_p, r, 0.0))
        assert tokens[r].item() == token, (r, tokens[r].item(), token)
        assert abs(chances[r].item() - chance) <= 2.0 ** -23 * chance, r
    return tokens


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("r,v", [(4, 1), (9, 10), (12, 333), (16, 1024), (6, 32001), (3, 131072)])
def test_sampling(dtype, r, v):
    gen = torch.Generator(device=DEV).manual_seed(v)
    for scale in (0.5, 3.0):
        x = (torch.randn(r, v, generator=gen, device=DEV) * scale).to(dtype)
        u = torch.rand(r, generator=gen, device=DEV)
        temperature = torch.rand(r, generator=gen, device=DEV) + 0.4
        top_k = torch.randint(0, min(v, 600) + 2, (r,), generator=gen, device=DEV, dtype=torch.int32)
        top_p = torch.rand(r, generator=gen, device=DEV) * 0.8 + 0.19
        min_p = torch.rand(r, generator=gen, device=DEV) * 0.3
        check_sampling(x, u)
        check_sampling(x, u, temperature, top_k)
        check_sampling(x, u, temperature, None, top_p)
        check_sampling(x, u, temperature, None, None, min_p)
        check_sampling(x, u, temperature, top_k, top_p, min_p)


def test_sampling_with_equal_logits():
    """few distinct values, so that every limit falls among equal ones: rising index decides"""
    gen = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randint(-2, 3, (40, 700), generator=gen, device=DEV).float()
    x[:8] = 0.0                     # all equal: sums without rounding
    x[8:10] = -0.0
    x[9, ::2] = 0.0                 # both zeros are one value
    u = torch.rand(40, generator=gen, device=DEV)
    top_k = torch.randint(1, 700, (40,), generator=gen, device=DEV, dtype=torch.int32)
    top_p = torch.rand(40, generator=gen, device=DEV) * 0.9 + 0.05
    check_sampling(x, u, None, top_k)
    check_sampling(x, u, None, None, top_p)
    check_sampling(x.bfloat16(), u, None, top_k, top_p)


def test_sampling_of_odd_rows():
    big = torch.finfo(torch.float32)
    x = torch.zeros(12, 50, device=DEV)
    x[0] = -math.inf                          # nothing left
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 17] = -5.0                           # one word left
    x[3] = big.min                            # the type's lowest value everywhere: equal words
    x[4] = big.min
    x[4, 30] = 1.0
    x[5, 20] = math.inf                       # shares the draw with nobody
    x[6, 5:8] = math.inf
    x[7, ::3] = math.nan
    x[8] = torch.arange(50, device=DEV) * 1000.0
    x[9] = big.max
    x[10, 1:] = big.min
    x[10, 0] = big.max                        # differences beyond the type's range
    u = torch.full((12,), 0.5, device=DEV)
    for value in (0.0, 0.25, 1.0 - 2.0 ** -24):
        u[:] = value
        tokens = check_sampling(x, u)
        assert tokens[0] == -1 and tokens[1] == -1 and tokens[2] == 17 and tokens[4] == 30 and tokens[5] == 20
        check_sampling(x, u, torch.full((12,), 1e-30, device=DEV))
        check_sampling(x, u, torch.full((12,), 1e30, device=DEV), torch.full((12,), 3, device=DEV, dtype=torch.int32))
        assert (check_sampling(x, u, torch.zeros(12, device=DEV))[3] == 0).all()          # greedy: the lowest index
        check_sampling(x, u, top_k=torch.full((12,), 1, device=DEV, dtype=torch.int32))
        check_sampling(x, u, top_k=torch.full((12,), 1000, device=DEV, dtype=torch.int32), top_p=torch.zeros(12, device=DEV))
        check_sampling(x, u, min_p=torch.ones(12, device=DEV))
        check_sampling(x, u, top_p=torch.full((12,), 1.5, device=DEV), min_p=torch.full((12,), -1.0, device=DEV))


def test_sampling_of_a_slice_on_another_stream_and_in_a_graph():
    gen = torch.Generator(device=DEV).manual_seed(13)
    wide = (torch.randn(6, 2005, generator=gen, device=DEV) * 2).bfloat16()
    x, u = wide[:, 3:2002], torch.rand(6, generator=gen, device=DEV)
    top_p = torch.full((6,), 0.9, device=DEV)
    want = check_sampling(x, u, top_p=top_p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = sequence.sample(x, u, top_p=top_p)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tokens, _ = sequence.sample(x, u, top_p=top_p)
    u.copy_(torch.rand(6, generator=gen, device=DEV))
    g.replay()
    assert torch.equal(tokens, check_sampling(x, u, top_p=top_p))


def test_sampling_follows_the_chances():
    """40000 draws with evenly spread random numbers: each token as often as its chance says, to one draw"""
    n = 40000
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, -math.inf, 0.5], device=DEV).expand(n, 6)
    u = (torch.arange(n, device=DEV, dtype=torch.float32) + 0.5) / n
    tokens, chances = sequence.sample(x, u)
    p = torch.softmax(x[0].double(), 0)
    for i in range(6):
        assert abs((tokens == i).sum().item() - n * p[i].item()) <= 2 + n * 2.0 ** -23
    assert torch.allclose(chances.double(), p[tokens.long()], rtol=2.0 ** -22)
