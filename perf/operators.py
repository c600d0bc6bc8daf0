"""What the operators for sequence models are measured on (myea_b200.sequence): the short causal convolution and the
selective state space scan in prompts, training and single tokens, the error against a teacher's top logits with its
gradient, and the draw of tokens from an output layer's logits.

`own` decides who computes: the library's kernels, or the same operators written out in elementary torch operations.
A case is a dict of plain values; "op" and "mode" say what one pass is:
  convolution  "train" forward and backward, "token" one position with its state carried on
  scan         "prompt" forward with the state behind it, "train" forward and backward, "token" one position
  distill      row losses and the gradient with respect to the logits
  sample       one token for every row, and the probability that it had
Parameters (convolution weights, A, D, biases) are held in 32 bits, activations and logits in the case's "type".
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    conv = dict(op="convolution", taps=4, ragged=False)
    scan = dict(op="scan", groups=1, gate=True, ragged=False, state=True)
    teach = dict(op="distill", masked=False)
    return [
        # training of a layer of ordinary width in the half-wide type: 4 sequences of 2048 positions
        dict(conv, name="convolution train", mode="train", type="bf16", batch=4, time=2048, width=4096),
        # 64 sequences answered token by token: one new position each, the last three inputs kept
        dict(conv, name="convolution tokens", mode="token", type="f32", batch=64, time=1, width=2048),
        # one long prompt alone: few channels, many positions, so the length has to give the parallel work
        dict(scan, name="scan long prompt", mode="prompt", type="bf16", batch=1, time=4096, width=4096, states=16, state=False),
        # a training step on 8 sequences
        dict(scan, name="scan train", mode="train", type="bf16", batch=8, time=1024, width=2048, states=16),
        # the width of the ragged regression network, sequences of different lengths, a number of states that divides by nothing
        dict(scan, name="scan ragged train", mode="train", type="f32", batch=7, time=203, width=333, states=7, groups=3, gate=False, ragged=True),
        # 256 sequences answered token by token: bound by their states
        dict(scan, name="scan tokens", mode="token", type="bf16", batch=256, time=1, width=4096, states=16),
        # a single sequence answered token by token: only latency counts
        dict(scan, name="scan one token", mode="token", type="f32", batch=1, time=1, width=1024, states=16),
        # a classifier of 1024 outputs taught by a larger one, labels mixed in: the batch of the wide network
        dict(teach, name="distill classes", type="f32", rows=4096, vocabulary=1024, top=16, temperature=2.0, hard=0.5),
        # 2048 positions of a large vocabulary, the teacher's 64 best logits stored for each
        dict(teach, name="distill large vocabulary", type="bf16", rows=2048, vocabulary=131072, top=64, temperature=1.0, hard=0.0),
        # a padded batch of few positions: rows without weight, lists that end early, a vocabulary off every boundary
        dict(teach, name="distill ragged", type="f16", rows=203, vocabulary=32001, top=50, temperature=1.5, hard=0.25, masked=True),
        # one row: a single sequence that waits for its next token
        dict(op="sample", name="sample one row", type="f32", rows=1, vocabulary=32000, settings="one", masked=False),
        # 256 sequences of a large vocabulary, each with settings of its own
        dict(op="sample", name="sample batch", type="bf16", rows=256, vocabulary=131072, settings="mixed", masked=False),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.4:
        v = v // 32 * 32
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["convolution", "scan", "scan", "scan", "distill", "distill", "sample", "sample"])
    c = dict(op=op, type=rng.choice(["f32", "bf16", "f16"]))
    if op == "convolution":
        c.update(mode=rng.choice(["train", "token"]), taps=rng.randint(2, 6), width=_log(rng, 8, 8192), ragged=rng.random() < 0.3)
        if c["mode"] == "token":
            c.update(batch=_log(rng, 1, 512), time=1, ragged=False)
        else:
            c.update(batch=_log(rng, 1, 32), time=_log(rng, 1, 4096))
    elif op == "scan":
        groups = rng.choice([1, 1, 1, 2, 3])
        c.update(mode=rng.choice(["prompt", "train", "token"]), groups=groups, width=_log(rng, 8, 4096) // groups * groups,
                 states=rng.choice([16, 16, 4, 7, 8, 24, 32, 64]), gate=rng.random() < 0.7, ragged=rng.random() < 0.3, state=rng.random() < 0.5)
        c["width"] = max(c["width"], groups)
        if c["mode"] == "token":
            c.update(batch=_log(rng, 1, 512), time=1, ragged=False, state=True)
        else:
            c.update(batch=_log(rng, 1, 16), time=_log(rng, 2, 4096))
    elif op == "distill":
        vocabulary = _log(rng, 10, 160000)
        c.update(rows=_log(rng, 1, 8192), vocabulary=vocabulary, top=min(vocabulary, _log(rng, 1, 256)),
                 temperature=rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]), hard=rng.choice([0.0, 0.25, 0.5]), masked=rng.random() < 0.4)
    else:
        c.update(rows=_log(rng, 1, 512), vocabulary=_log(rng, 10, 160000), settings=rng.choice(["one", "mixed", "plain"]), masked=rng.random() < 0.4)
    most = {}
    for x in listed():   # (a case costs no more than the largest one of its own operator)
        most[x["op"]] = max(most.get(x["op"], 0.0), _cost(x))
    while _cost(c) > most[op]:
        if "time" in c and c["time"] >= 2 * c["batch"]:
            c["time"] //= 2
        elif "batch" in c and c["batch"] > 1:
            c["batch"] = max(1, c["batch"] // 2)
        elif "rows" in c and c["rows"] > 1:
            c["rows"] = max(1, c["rows"] // 2)
        elif "width" in c:
            c["width"] = max(c.get("groups", 1), c["width"] // 2 // c.get("groups", 1) * c.get("groups", 1))
        else:
            c["vocabulary"] //= 2
    return c


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 8)


def work(case):
    c = case
    e = SIZE[c["type"]]
    if c["op"] == "convolution":
        n, w = float(c["batch"]) * c["time"] * c["width"], c["taps"]
        par, kept = c["width"] * (w + 1) * 4.0, float(c["batch"]) * (w - 1) * c["width"] * e
        if c["mode"] == "token":
            return {"bytes": 2 * n * e + par + 2 * kept, "flops": n * (2 * w + 6)}
        # forward x -> y; backward dy, x -> dx; parameters and their derivatives
        return {"bytes": 5 * n * e + 3 * par + 4 * kept, "flops": n * (8 * w + 22)}
    if c["op"] == "scan":
        b, t, d, s = float(c["batch"]), c["time"], c["width"], c["states"]
        n, bc, par, h = b * t * d * e, b * t * c["groups"] * s * e, d * (s + 2) * 4.0, b * d * s * 4.0
        g = 1 if c["gate"] else 0
        held = h * (2 if c["state"] else 1)
        # one step of one state: product and exponential for the decay, product of the input, two multiply-adds
        fwd = {"bytes": n * (3 + g) + 2 * bc + par + held, "flops": b * t * d * (s * 7 + 12 + 6 * g)}
        if c["mode"] != "train":
            return fwd
        # backward: the inputs and the error read, a derivative written for each; 22 operations for one step of one state
        return {"bytes": fwd["bytes"] + n * (3 + g) + n * (2 + g) + 4 * bc + 2 * par + held, "flops": fwd["flops"] + b * t * d * (s * 22 + 24)}
    r, v = float(c["rows"]), c["vocabulary"]
    if c["op"] == "distill":
        return {"bytes": r * v * 2 * e + r * c["top"] * 8 + r * 12, "flops": r * v * (8 if c["hard"] == 0.0 or c["temperature"] == 1.0 else 12)}
    return {"bytes": r * v * e + r * 28, "flops": r * v * 6}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _inputs(c, seed):
    """everything a program has in hand before the call, on the GPU, from the seed alone"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    tp = TYPES[c["type"]]

    def normal(*shape, scale=1.0, shift=0.0, dtype=None):
        x = torch.empty(shape, device="cuda").normal_(generator=gen).mul_(scale)
        return (x.add_(shift) if shift else x).to(dtype or tp)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.empty(shape, device="cuda").uniform_(lo, hi, generator=gen)

    if c["op"] in ("convolution", "scan"):
        b, t, d = c["batch"], c["time"], c["width"]
        lengths = None
        if c["ragged"]:
            lengths = torch.randint(0, t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
            lengths[0] = t
        train = c["mode"] == "train"
    if c["op"] == "convolution":
        k = c["taps"]
        return {"x": normal(b, t, d), "weight": uniform(d, k, lo=-k ** -0.5, hi=k ** -0.5), "bias": uniform(d, lo=-0.5, hi=0.5), "state": normal(b, k - 1, d),
                "lengths": lengths, "dy": normal(b, t, d, scale=0.1) if train else None, "d_final": normal(b, k - 1, d, scale=0.1) if train else None}
    if c["op"] == "scan":
        s, g = c["states"], c["groups"]
        # decays from slow to fast states, step lengths between 1e-3 and 1e-1 where the projection gives 0
        rate = torch.arange(1, s + 1, device="cuda", dtype=torch.float32).repeat(d, 1) * torch.exp(0.2 * normal(d, s, dtype=torch.float32))
        step = torch.exp(uniform(d, lo=math.log(1e-3), hi=math.log(1e-1)))
        return {"u": normal(b, t, d), "delta": normal(b, t, d, scale=0.5), "A": -rate, "B": normal(b, t, g, s), "C": normal(b, t, g, s),
                "D": 1.0 + 0.1 * normal(d, dtype=torch.float32), "z": normal(b, t, d) if c["gate"] else None,
                "delta_bias": step + torch.log(-torch.expm1(-step)), "state": normal(b, d, s, dtype=torch.float32) if c["state"] else None,
                "lengths": lengths, "dy": normal(b, t, d, scale=0.1) if train else None, "d_final": normal(b, d, s, scale=0.1, dtype=torch.float32) if train else None}
    r, v = c["rows"], c["vocabulary"]
    logits = normal(r, v, scale=2.5, dtype=torch.float32)
    favourites = torch.randint(v, (r, min(v, 8)), generator=gen, device="cuda")
    logits.scatter_add_(1, favourites, uniform(r, favourites.shape[1], lo=2.0, hi=8.0))
    if c["op"] == "distill":
        k = c["top"]
        near = logits + normal(r, v, scale=0.7, dtype=torch.float32)
        teacher, index = torch.topk(near, k, dim=1)
        del near
        index = index.to(torch.int32)
        weight = torch.ones(r, device="cuda")
        labels = torch.randint(v, (r,), generator=gen, device="cuda", dtype=torch.int32) if c["hard"] > 0.0 else None
        if c["masked"]:   # padded positions weigh nothing, some lists are shorter, some words are closed
            weight[uniform(r) < 0.3] = 0.0
            cut = torch.randint(1, k + 1, (r, 1), generator=gen, device="cuda")
            index = torch.where(torch.arange(k, device="cuda") < cut, index, torch.full_like(index, -1))
            closed = uniform(r, v) < 0.02
            closed.scatter_(1, index.clamp(min=0).long(), False)
            if labels is not None:
                closed.scatter_(1, labels[:, None].long(), False)
            logits.masked_fill_(closed, -math.inf)
            if labels is not None:
                labels[uniform(r) < 0.2] = -100
        weight /= max(1.0, float(r))
        return {"logits": logits.to(tp), "index": index, "teacher": teacher, "weight": weight, "labels": labels}
    if c["masked"]:
        logits.masked_fill_(uniform(r, v) < 0.5, -math.inf)
    got = {"logits": logits.to(tp), "uniform": uniform(r), "temperature": None, "top_k": None, "top_p": None, "min_p": None}
    if c["settings"] == "one":
        got.update(temperature=torch.full((r,), 0.8, device="cuda"), top_k=torch.full((r,), 50, device="cuda", dtype=torch.int32),
                   top_p=torch.full((r,), 0.9, device="cuda"))
    elif c["settings"] == "mixed":   # a sixth of the rows greedy, each limit on for some of them
        which = torch.randint(6, (r,), generator=gen, device="cuda")
        off = lambda on, x, none: torch.where(on, x, torch.full_like(x, none))  # noqa: E731
        got.update(temperature=off(which > 0, uniform(r, lo=0.5, hi=1.5), 0.0),
                   top_k=off((which == 1) | (which == 4), torch.randint(1, 1000, (r,), generator=gen, device="cuda", dtype=torch.int32), 0),
                   top_p=off((which == 2) | (which == 4), uniform(r, lo=0.5, hi=0.99), 1.0), min_p=off(which == 3, uniform(r, lo=0.01, hi=0.2), 0.0))
    return got


def prepare(case, seed):
    c = dict(case)
    s = {"case": c, "in": _inputs(c, seed)}
    i = s["in"]
    if own and c["op"] == "scan" and c["mode"] == "train":   # what the forward pass keeps for the backward pass
        from myea_b200 import sequence
        s["kept"] = sequence.scan_checkpoints(i["u"], i["A"])
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    c, i = state["case"], state["in"]
    if own:
        return _library(state, c, i)
    if c["op"] == "convolution":
        return _convolution(c, i)
    if c["op"] == "scan":
        return _scan(c, i)
    return _distill(c, i) if c["op"] == "distill" else _sample(c, i)


def _library(state, c, i):
    from myea_b200 import sequence
    if c["op"] == "convolution":
        par = dict(bias=i["bias"], silu=True, state=i["state"], lengths=i["lengths"])
        y, final = sequence.causal_convolution(i["x"], i["weight"], **par)
        if c["mode"] == "token":
            return {"y": y, "final": final}
        d = sequence.causal_convolution_backward(i["dy"], i["x"], i["weight"], d_final_state=i["d_final"], **par)
        return {"y": y, "final": final, "dx": d["x"], "dweight": d["weight"], "dbias": d["bias"], "dstate": d["state"]}
    if c["op"] == "scan":
        par = dict(D=i["D"], z=i["z"], delta_bias=i["delta_bias"], softplus=True, state=i["state"], lengths=i["lengths"])
        kept = state.get("kept")
        y, final = sequence.selective_scan(i["u"], i["delta"], i["A"], i["B"], i["C"], checkpoints=kept, **par)
        if c["mode"] != "train":
            return {"y": y, "final": final}
        d = sequence.selective_scan_backward(i["dy"], i["u"], i["delta"], i["A"], i["B"], i["C"], kept, d_final_state=i["d_final"], **par)
        got = {"y": y, "final": final, "du": d["u"], "ddelta": d["delta"], "dA": d["A"], "dB": d["B"], "dC": d["C"], "dD": d["D"], "dbias": d["delta_bias"]}
        if c["gate"]:
            got["dz"] = d["z"]
        if c["state"]:
            got["dstate"] = d["state"]
        return got
    if c["op"] == "distill":
        losses, d = sequence.distillation_error(i["logits"], i["index"], i["teacher"], temperature=c["temperature"], soft=1.0 - c["hard"], hard=c["hard"],
                                                labels=i["labels"], weight=i["weight"])
        return {"losses": losses, "dlogits": d}
    tokens, chance = sequence.sample(i["logits"], i["uniform"], temperature=i["temperature"], top_k=i["top_k"], top_p=i["top_p"], min_p=i["min_p"])
    return {"tokens": tokens, "chance": chance}


def _inside(i, b, t):
    """[b, t, 1]: positions of the sequences"""
    if i["lengths"] is None:
        return None
    return (torch.arange(t, device="cuda")[None, :] < i["lengths"][:, None])[:, :, None]


def _convolution(c, i):
    b, t, d, k, tp = c["batch"], c["time"], c["width"], c["taps"], TYPES[c["type"]]
    inside = _inside(i, b, t)
    w = i["weight"]
    x = torch.cat([i["state"], i["x"]], 1).float()
    acc = i["bias"].expand(b, t, d)
    for j in range(k):
        acc = acc + w[:, j] * x[:, j:j + t]
    sig = 1.0 / (1.0 + torch.exp(-acc))
    y = acc * sig
    if inside is not None:
        y = torch.where(inside, y, torch.zeros_like(y))
    ends = torch.full((b,), t, device="cuda") if i["lengths"] is None else i["lengths"].long()
    at = (ends[:, None] + torch.arange(k - 1, device="cuda"))[:, :, None].expand(b, k - 1, d)
    got = {"y": y.to(tp), "final": torch.gather(x, 1, at).to(tp)}
    if c["mode"] == "token":
        return got
    da = i["dy"].float() * sig * (1.0 + acc * (1.0 - sig))
    if inside is not None:
        da = torch.where(inside, da, torch.zeros_like(da))
    dx = torch.zeros_like(x)
    dw = torch.empty_like(w)
    for j in range(k):
        dx[:, j:j + t] += w[:, j] * da
        dw[:, j] = (da * x[:, j:j + t]).sum((0, 1), dtype=torch.float64).float()
    dx.scatter_add_(1, at, i["d_final"].float())
    got.update(dx=dx[:, k - 1:].to(tp), dweight=dw, dbias=da.sum((0, 1), dtype=torch.float64).float(), dstate=dx[:, :k - 1].to(tp))
    return got


def _scan(c, i):
    b, t, d, s, g, tp = c["batch"], c["time"], c["width"], c["states"], c["groups"], TYPES[c["type"]]
    inside = _inside(i, b, t)
    u, raw = i["u"].float(), i["delta"].float() + i["delta_bias"]
    wide = lambda x: x.float()[:, :, :, None, :].expand(b, t, g, d // g, s).reshape(b, t, d, s)  # noqa: E731
    delta = torch.where(raw > 20.0, raw, torch.log1p(torch.exp(raw.clamp(max=20.0))))
    if inside is not None:
        delta = torch.where(inside, delta, torch.zeros_like(delta))
    B, C = wide(i["B"]), wide(i["C"])
    decay = torch.exp(delta[..., None] * i["A"])
    add = (delta * u)[..., None] * B
    h0 = i["state"] if i["state"] is not None else torch.zeros(b, d, s, device="cuda")
    hs = torch.empty(b, t + 1, d, s, device="cuda")
    hs[:, 0] = h0
    for k in range(t):
        hs[:, k + 1] = decay[:, k] * hs[:, k] + add[:, k]
    y = (hs[:, 1:] * C).sum(-1) + i["D"] * u
    if c["gate"]:
        z = i["z"].float()
        sig = 1.0 / (1.0 + torch.exp(-z))
        out = y * z * sig
    else:
        out = y
    if inside is not None:
        out = torch.where(inside, out, torch.zeros_like(out))
    got = {"y": out.to(tp), "final": hs[:, t].clone()}
    if c["mode"] != "train":
        return got
    dout = i["dy"].float()
    if inside is not None:
        dout = torch.where(inside, dout, torch.zeros_like(dout))
    dy = dout
    if c["gate"]:
        got["dz"] = (dout * y * sig * (1.0 + z * (1.0 - sig))).to(tp)
        dy = dout * z * sig
    gs = dy[..., None] * C
    gs[:, t - 1] += i["d_final"]
    for k in range(t - 1, 0, -1):
        gs[:, k - 1] += decay[:, k] * gs[:, k]
    if c["state"]:
        got["dstate"] = decay[:, 0] * gs[:, 0]
    narrow = lambda x: x.reshape(b, t, g, d // g, s).sum(3)  # noqa: E731
    got["dC"] = narrow(dy[..., None] * hs[:, 1:]).to(tp)
    gB = (gs * B).sum(-1)
    got["dB"] = narrow(gs * (delta * u)[..., None]).to(tp)
    q = gs * decay * hs[:, :t]
    got["dA"] = (q * delta[..., None]).sum((0, 1), dtype=torch.float64).float()
    ddelta = ((q * i["A"]).sum(-1) + gB * u) / (1.0 + torch.exp(-raw))
    if inside is not None:
        ddelta = torch.where(inside, ddelta, torch.zeros_like(ddelta))
    got["ddelta"], got["du"] = ddelta.to(tp), (gB * delta + i["D"] * dy).to(tp)
    got["dD"], got["dbias"] = (dy * u).sum((0, 1), dtype=torch.float64).float(), ddelta.sum((0, 1), dtype=torch.float64).float()
    return got


def _distill(c, i):
    tau, hard, r, v = c["temperature"], c["hard"], c["rows"], c["vocabulary"]
    x, w = i["logits"].float(), i["weight"]
    on = w != 0.0
    there = (i["index"] >= 0) & (i["index"] < v)
    at = torch.where(there, i["index"], torch.zeros_like(i["index"])).long()
    t = torch.where(there, i["teacher"] / tau, torch.full_like(i["teacher"], -math.inf))
    t = t - t.amax(1, keepdim=True)
    p = torch.exp(t)
    p = p / p.sum(1, keepdim=True)
    top = x.amax(1, keepdim=True)
    e = torch.exp((x - top) / tau)
    total = e.sum(1, keepdim=True)
    logq = (torch.gather(x, 1, at) - top) / tau - torch.log(total)
    kl = torch.where(p > 0.0, p * (torch.log(p) - logq), torch.zeros_like(p)).sum(1)
    soft = (1.0 - hard) * tau * tau
    d = e * (soft / tau / total)
    d.scatter_add_(1, at, torch.where(there, p * (-soft / tau), torch.zeros_like(p)))
    losses = soft * kl
    if hard > 0.0:
        labelled = (i["labels"] >= 0) & (i["labels"] < v)
        name = torch.where(labelled, i["labels"], torch.zeros_like(i["labels"])).long()[:, None]
        e = torch.exp(x - top)
        total = e.sum(1, keepdim=True)
        ce = torch.log(total) - (torch.gather(x, 1, name) - top)
        losses = losses + torch.where(labelled, hard * ce[:, 0], torch.zeros_like(losses))
        share = torch.where(labelled, hard, 0.0)[:, None]
        d += e * (share / total)
        d.scatter_add_(1, name, -share.to(d.dtype))
    losses = torch.where(on, w * losses, torch.zeros_like(losses))
    return {"losses": losses, "dlogits": torch.where(on[:, None], d * w[:, None], torch.zeros_like(d)).to(TYPES[c["type"]])}


def _sample(c, i):
    r, v = c["rows"], c["vocabulary"]
    x = i["logits"].double()
    one = lambda name, none: (i[name] if i[name] is not None else torch.full((r,), none, device="cuda"))[:, None]  # noqa: E731
    tau, top_k, top_p, min_p = one("temperature", 1.0).double(), one("top_k", 0), one("top_p", 1.0).double(), one("min_p", 0.0).double()
    greedy = tau <= 0.0
    s, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((s - s[:, :1]) / torch.where(greedy, torch.ones_like(tau), tau))
    place = torch.arange(v, device="cuda")[None, :]
    keep = (place < torch.where(top_k > 0, top_k, torch.full_like(top_k, v))) & (w > 0.0)
    w = torch.where(keep, w, torch.zeros_like(w))
    before = torch.cumsum(w, 1) - w
    keep = keep & ((top_p >= 1.0) | (before < top_p * w.sum(1, keepdim=True)) | (place == 0)) & (w >= min_p) & (~greedy | (place == 0))
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, torch.zeros_like(w)))
    sums = torch.cumsum(w, 1)
    total = sums[:, -1:]
    token = (sums <= i["uniform"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=v - 1)
    return {"tokens": token[:, 0].to(torch.int32), "chance": (torch.gather(w, 1, token) / total)[:, 0].float()}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    c, i = dict(case), _inputs(dict(case), seed)
    with torch.enable_grad():
        return {"convolution": _exact_convolution, "scan": _exact_scan, "distill": _exact_distill, "sample": _exact_sample}[c["op"]](c, i)


def _exact_convolution(c, i):
    t, k = c["time"], c["taps"]
    train = c["mode"] == "train"
    leaves = {n: i[n].double().requires_grad_(train) for n in ("x", "weight", "bias", "state")}
    ends = i["lengths"].tolist() if i["lengths"] is not None else [t] * c["batch"]
    ys, finals = [], []
    for b, n in enumerate(ends):
        row = torch.cat([leaves["state"][b], leaves["x"][b, :n]], 0)                    # [k - 1 + n, d]
        a = leaves["bias"] + (row.unfold(0, k, 1) * leaves["weight"]).sum(-1) if n else row[:0]
        ys.append(torch.nn.functional.pad(torch.nn.functional.silu(a), (0, 0, 0, t - n)))
        finals.append(row[n:])
    y, final = torch.stack(ys), torch.stack(finals)
    got = {"y": y.detach(), "final": final.detach()}
    if train:
        ((y * i["dy"].double()).sum() + (final * i["d_final"].double()).sum()).backward()
        got.update(dx=leaves["x"].grad, dweight=leaves["weight"].grad, dbias=leaves["bias"].grad, dstate=leaves["state"].grad)
    return got


def _exact_scan(c, i):
    b, t, d, s, g = c["batch"], c["time"], c["width"], c["states"], c["groups"]
    train = c["mode"] == "train"
    leaf = lambda n: i[n].double().requires_grad_(train) if i[n] is not None else None  # noqa: E731
    L = {n: leaf(n) for n in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")}
    y, final = torch.zeros(b, t, d, dtype=torch.float64, device="cuda"), torch.zeros(b, d, s, dtype=torch.float64, device="cuda")
    live = 1.0 if i["lengths"] is None else (torch.arange(t, device="cuda")[None] < i["lengths"][:, None]).double()[:, :, None]
    slab = max(1, int(2e8 / (b * t * s * (3 * max(1, t.bit_length()) if train else 4))))
    for group in range(g):
        for lo in range(group * (d // g), (group + 1) * (d // g), slab):
            ch = slice(lo, min(lo + slab, (group + 1) * (d // g)))
            step = torch.nn.functional.softplus(L["delta"][:, :, ch] + L["delta_bias"][ch], threshold=40.0) * live
            # the scan by doubling: after k rounds every position holds the sum over the last 2^k positions
            decay = torch.exp(step[..., None] * L["A"][ch])
            h = (step * L["u"][:, :, ch])[..., None] * L["B"][:, :, group, None, :]
            if L["state"] is not None:
                h = torch.cat([(h[:, :1] + decay[:, :1] * L["state"][:, None, ch]), h[:, 1:]], 1)
            k = 1
            while k < t:
                h = torch.cat([h[:, :k], h[:, k:] + decay[:, k:] * h[:, :-k]], 1)
                decay = torch.cat([decay[:, :k], decay[:, k:] * decay[:, :-k]], 1)
                k *= 2
            out = (h * L["C"][:, :, group, None, :]).sum(-1) + L["D"][ch] * L["u"][:, :, ch]
            if L["z"] is not None:
                out = out * torch.nn.functional.silu(L["z"][:, :, ch])
            out = out * live
            y[:, :, ch], final[:, ch] = out.detach(), h[:, -1].detach()
            if train:
                ((out * i["dy"][:, :, ch].double()).sum() + (h[:, -1] * i["d_final"][:, ch].double()).sum()).backward()
            del h, decay, out, step
    got = {"y": y, "final": final}
    if train:
        got.update(du=L["u"].grad, ddelta=L["delta"].grad, dA=L["A"].grad, dB=L["B"].grad, dC=L["C"].grad, dD=L["D"].grad, dbias=L["delta_bias"].grad)
        if c["gate"]:
            got["dz"] = L["z"].grad
        if c["state"]:
            got["dstate"] = L["state"].grad
    return got


def _exact_distill(c, i):
    tau, hard, r, v = c["temperature"], c["hard"], c["rows"], c["vocabulary"]
    losses, grads = [], []
    rows = max(1, int(3e7) // v)
    for lo in range(0, r, rows):
        cut = slice(lo, min(lo + rows, r))
        x = i["logits"][cut].double().requires_grad_(True)
        w = i["weight"][cut].double()
        there = (i["index"][cut] >= 0) & (i["index"][cut] < v)
        at = i["index"][cut].long().clamp(min=0, max=v - 1)
        p = torch.softmax((i["teacher"][cut].double() / tau).masked_fill(~there, -math.inf), 1)
        logq = torch.log_softmax(x / tau, 1)
        each = (torch.xlogy(p, p) - torch.where(p > 0.0, p * torch.gather(logq, 1, at), 0.0)).sum(1) * (1.0 - hard) * tau * tau
        if hard > 0.0:
            label = i["labels"][cut].long()
            known = (label >= 0) & (label < v)
            logp = torch.log_softmax(x, 1)
            each = each - hard * torch.where(known, torch.gather(logp, 1, label.clamp(min=0, max=v - 1)[:, None])[:, 0], 0.0)
        each = each * w
        each.sum().backward()
        losses.append(each.detach())
        grads.append(x.grad.float() if c["type"] != "f32" else x.grad)   # (outputs of 16 bits: 32 hold the exact value well enough)
    return {"losses": torch.cat(losses), "dlogits": torch.cat(grads)}


def _exact_sample(c, i):
    row = lambda name, none: np.full(c["rows"], none) if i[name] is None else i[name].cpu().numpy().astype(np.float64)  # noqa: E731
    x, u = i["logits"].double().cpu().numpy(), i["uniform"].cpu().numpy().astype(np.float64)
    tau, top_k, top_p, min_p = row("temperature", 1.0), row("top_k", 0), row("top_p", 1.0), row("min_p", 0.0)
    tokens, chance = [], []
    for r in range(c["rows"]):
        order = np.lexsort((np.arange(c["vocabulary"]), -x[r]))
        if tau[r] <= 0.0:
            kept, w = order[:1], np.ones(1)
        else:
            if top_k[r] > 0:
                order = order[:int(top_k[r])]
            order = order[np.isfinite(x[r][order])]
            w = np.exp((x[r][order] - x[r][order[0]]) / tau[r])
            n = len(w)
            if top_p[r] < 1.0:
                n = max(1, int(np.searchsorted(np.concatenate([[0.0], np.cumsum(w)[:-1]]), top_p[r] * w.sum(), side="left")))
            n = min(n, int((w >= min_p[r]).sum()))
            kept, w = order[:n], w[:n]
        by_index = np.argsort(kept)
        kept, w = kept[by_index], w[by_index]
        sums = np.cumsum(w)
        j = min(len(w) - 1, int(np.searchsorted(sums, u[r] * sums[-1], side="right")))
        tokens.append(int(kept[j]))
        chance.append(w[j] / sums[-1])
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "chance": torch.tensor(chance, dtype=torch.float64)}
