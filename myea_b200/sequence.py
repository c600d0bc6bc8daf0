"""Operators for sequence models on tensors that lie on the GPU: thin calls into libmyea_b200.so (include/myea_b200.h, where the
formulas stand).  They stand beside the recurrent layers, the output error and the output layer of `net.Net` and need no network.

Tensors are torch tensors, used where they lie: an activation is [batch, time, width] with any strides over batch and time
and densely packed last dimensions (a time-major array is x.transpose(0, 1), a slice of a wider projection is read in place),
of float32, bfloat16 or float16, one type per call; parameters, states of a scan and losses are float32.  A call runs on the
current stream of the tensors' GPU, may be captured into a CUDA graph and does not wait.  ValueError: the arguments do not fit
together (nothing was launched); RuntimeError: the library refused the call or failed, with its message.
"""
import ctypes as C

import torch

from . import capi

_TYPES = {torch.float32: capi.TYPE_F32, torch.bfloat16: capi.TYPE_BF16, torch.float16: capi.TYPE_F16}


def _call(name, device, *args):
    message = C.create_string_buffer(256)
    rc = getattr(capi.load(), "myea_b200_" + name)(device.index, *args, torch.cuda.current_stream(device).cuda_stream, message, 256)
    if rc != 0:
        raise RuntimeError("%s failed (%d): %s" % (name, rc, message.value.decode()))


def _check(name, x, shape, dtype, device):
    if tuple(x.shape) != tuple(shape) or x.dtype != dtype or x.device != device:
        raise ValueError("%s: expected %s of %s on %s, got %s of %s on %s" % (name, tuple(shape), dtype, device, tuple(x.shape), x.dtype, x.device))


def _type(x):
    if x.device.type != "cuda":
        raise ValueError("tensors have to lie on a GPU, got one on %s" % x.device)
    if x.dtype not in _TYPES:
        raise ValueError("float32, bfloat16 or float16 expected, got %s" % x.dtype)
    return _TYPES[x.dtype]


def _dense(x, from_dim):
    """whether the dimensions from `from_dim` on lie densely"""
    step = 1
    for n, s in zip(reversed(x.shape[from_dim:]), reversed(x.stride()[from_dim:])):
        if n != 1 and s != step:
            return False
        step *= n
    return True


def _view(name, x, shape, dtype, device):
    """address and strides of a [batch, time, ...] tensor; nothing where there is none"""
    if x is None:
        return 0, 0, 0
    _check(name, x, shape, dtype, device)
    if not _dense(x, 2):
        raise ValueError("%s: the dimensions behind batch and time have to lie densely, strides are %s" % (name, x.stride()))
    return x.data_ptr(), x.stride(0), x.stride(1)


def _array(name, x, shape, dtype, device):
    """address of a densely packed tensor; None where there is none"""
    if x is None:
        return None
    _check(name, x, shape, dtype, device)
    if not x.is_contiguous():
        raise ValueError("%s has to be contiguous" % name)
    return x.data_ptr()


def _out(given, shape, dtype, device):
    return torch.empty(shape, dtype=dtype, device=device) if given is None else given


def _convolution(x, weight, bias, silu, state, lengths):
    if x.dim() != 3 or weight.dim() != 2:
        raise ValueError("x is [batch, time, width] and weight [width, taps]")
    (b, t, d), k, dev = x.shape, weight.shape[1], x.device
    s = capi.Convolution(_type(x), k, 1 if silu else 0, 0, b, t, d)
    s.x, s.x_batch, s.x_time = _view("x", x, (b, t, d), x.dtype, dev)
    s.weight = _array("weight", weight, (d, k), torch.float32, dev)
    s.bias = _array("bias", bias, (d,), torch.float32, dev)
    s.state = _array("state", state, (b, k - 1, d), x.dtype, dev)
    s.lengths = _array("lengths", lengths, (b,), torch.int32, dev)
    return s


def causal_convolution(x, weight, bias=None, silu=True, state=None, final_state=None, lengths=None, out=None):
    """(y, final_state): y[b, t, c] = act(bias[c] + sum over j of weight[c, j] * x[b, t - taps + 1 + j, c]), act = silu or nothing.
    weight [width, taps], 1 to 8 taps; state [batch, taps - 1, width]: the inputs before the first (None: zeros); final_state: where the
    last taps - 1 inputs go (None: a new tensor; `state` itself is allowed); lengths int32 [batch]: y is 0 behind a sequence's
    end.  A single token is time = 1 with both states."""
    s = _convolution(x, weight, bias, silu, state, lengths)
    (b, t, d), k = x.shape, weight.shape[1]
    y, final_state = _out(out, (b, t, d), x.dtype, x.device), _out(final_state, (b, k - 1, d), x.dtype, x.device)
    s.y, s.y_batch, s.y_time = _view("out", y, (b, t, d), x.dtype, x.device)
    s.final_state = _array("final_state", final_state, (b, k - 1, d), x.dtype, x.device)
    _call("causal_convolution", x.device, C.byref(s))
    return y, final_state


def causal_convolution_backward(dy, x, weight, bias=None, silu=True, state=None, lengths=None, d_final_state=None, dx=None, d_weight=None, d_bias=None,
                                accumulate=False):
    """{"x", "weight", "bias" (None without one), "state" (None without one)}: derivatives for the error `dy` on y and
    `d_final_state` on the final state.  d_weight / d_bias given: the derivatives go there, with `accumulate` onto what they hold."""
    s = _convolution(x, weight, bias, silu, state, lengths)
    (b, t, d), k, dev = x.shape, weight.shape[1], x.device
    dx, d_weight = _out(dx, (b, t, d), x.dtype, dev), _gradient("d_weight", d_weight, (d, k), dev, accumulate)
    d_bias = _gradient("d_bias", d_bias, (d,), dev, accumulate) if bias is not None else None
    d_state = torch.empty((b, k - 1, d), dtype=x.dtype, device=dev) if state is not None else None
    s.accumulate = 1 if accumulate else 0
    s.dy, s.dy_batch, s.dy_time = _view("dy", dy, (b, t, d), x.dtype, dev)
    s.dx, s.dx_batch, s.dx_time = _view("dx", dx, (b, t, d), x.dtype, dev)
    s.d_weight = _array("d_weight", d_weight, (d, k), torch.float32, dev)
    s.d_bias = _array("d_bias", d_bias, (d,), torch.float32, dev)
    s.d_final_state = _array("d_final_state", d_final_state, (b, k - 1, d), x.dtype, dev)
    s.d_state = _array("d_state", d_state, (b, k - 1, d), x.dtype, dev)
    work, size = _workspace("causal_convolution_backward_workspace", s, dev)
    _call("causal_convolution_backward", dev, C.byref(s), work.data_ptr() if size else None, size)
    return {"x": dx, "weight": d_weight, "bias": d_bias, "state": d_state}


def _gradient(name, given, shape, device, accumulate):
    if given is None and accumulate:
        raise ValueError("%s: accumulate needs an array to add to" % name)
    return _out(given, shape, torch.float32, device)


def _workspace(name, s, device):
    size = getattr(capi.load(), "myea_b200_" + name)(C.byref(s))
    return (torch.empty(size, dtype=torch.uint8, device=device) if size else None), size


def _scan(u, delta, A, B, Cm, D, z, delta_bias, softplus, state, lengths):
    if u.dim() != 3 or A.dim() != 2 or B.dim() != 4:
        raise ValueError("u is [batch, time, width], A [width, states], B and C [batch, time, groups, states]")
    (b, t, d), n, g, dev, tp = u.shape, A.shape[1], B.shape[2], u.device, u.dtype
    s = capi.Scan(_type(u), 1 if softplus else 0, 0, 0, b, t, d, n, g)
    s.u, s.u_batch, s.u_time = _view("u", u, (b, t, d), tp, dev)
    s.delta, s.delta_batch, s.delta_time = _view("delta", delta, (b, t, d), tp, dev)
    s.B, s.B_batch, s.B_time = _view("B", B, (b, t, g, n), tp, dev)
    s.C, s.C_batch, s.C_time = _view("C", Cm, (b, t, g, n), tp, dev)
    s.z, s.z_batch, s.z_time = _view("z", z, (b, t, d), tp, dev)
    s.A = _array("A", A, (d, n), torch.float32, dev)
    s.D = _array("D", D, (d,), torch.float32, dev)
    s.delta_bias = _array("delta_bias", delta_bias, (d,), torch.float32, dev)
    s.state = _array("state", state, (b, d, n), torch.float32, dev)
    s.lengths = _array("lengths", lengths, (b,), torch.int32, dev)
    return s


def _checkpoint_shape(b, t, d, n):
    lanes = 1
    while lanes * 4 < n:
        lanes *= 2
    return b, (t + 15) // 16, d, lanes * 4


def scan_checkpoints(u, A):
    """the array that a forward pass over `u` with decay rates `A` leaves its states in for the backward pass; a program may keep
    it for every step of the same sizes"""
    _type(u)
    return torch.empty(_checkpoint_shape(*u.shape, A.shape[1]), dtype=torch.float32, device=u.device)


def selective_scan(u, delta, A, B, C_, D=None, z=None, delta_bias=None, softplus=True, state=None, final_state=None, lengths=None, checkpoints=None,
                   out=None):
    """(y, final_state) of the selective state space scan over u, delta [batch, time, width] with A [width, states] (1 to 128 states),
    B, C [batch, time, groups, states], D and delta_bias [width], a gate z like u, a state [batch, width, states] to start from (None:
    zeros) and one to end in (None: a new tensor; `state` itself is allowed).  lengths int32 [batch]: y is 0 behind a sequence's
    end, and the state there stays.  checkpoints (scan_checkpoints): kept for selective_scan_backward.  A single token is
    time = 1 with both states."""
    s = _scan(u, delta, A, B, C_, D, z, delta_bias, softplus, state, lengths)
    (b, t, d), n, dev = u.shape, A.shape[1], u.device
    y, final_state = _out(out, (b, t, d), u.dtype, dev), _out(final_state, (b, d, n), torch.float32, dev)
    s.y, s.y_batch, s.y_time = _view("out", y, (b, t, d), u.dtype, dev)
    s.final_state = _array("final_state", final_state, (b, d, n), torch.float32, dev)
    s.checkpoints = _array("checkpoints", checkpoints, _checkpoint_shape(b, t, d, n), torch.float32, dev)
    work, size = _workspace("selective_scan_workspace", s, dev)
    _call("selective_scan", dev, C.byref(s), work.data_ptr() if size else None, size)
    return y, final_state


def selective_scan_backward(dy, u, delta, A, B, C_, checkpoints, D=None, z=None, delta_bias=None, softplus=True, state=None, lengths=None,
                            d_final_state=None, d_A=None, d_D=None, d_delta_bias=None, accumulate=False):
    """Derivatives for the error `dy` on y and `d_final_state` on the final state, by the names of the forward pass's arguments
    ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"; None where there was none).  d_A, d_D, d_delta_bias given: those go
    there, with `accumulate` onto what they hold."""
    s = _scan(u, delta, A, B, C_, D, z, delta_bias, softplus, state, lengths)
    (b, t, d), n, g, dev, tp = u.shape, A.shape[1], B.shape[2], u.device, u.dtype
    got = {"u": torch.empty((b, t, d), dtype=tp, device=dev), "delta": torch.empty((b, t, d), dtype=tp, device=dev),
           "B": torch.empty((b, t, g, n), dtype=tp, device=dev), "C": torch.empty((b, t, g, n), dtype=tp, device=dev),
           "z": torch.empty((b, t, d), dtype=tp, device=dev) if z is not None else None,
           "A": _gradient("d_A", d_A, (d, n), dev, accumulate), "D": _gradient("d_D", d_D, (d,), dev, accumulate) if D is not None else None,
           "delta_bias": _gradient("d_delta_bias", d_delta_bias, (d,), dev, accumulate) if delta_bias is not None else None,
           "state": torch.empty((b, d, n), dtype=torch.float32, device=dev) if state is not None else None}
    s.accumulate = 1 if accumulate else 0
    s.checkpoints = _array("checkpoints", checkpoints, _checkpoint_shape(b, t, d, n), torch.float32, dev)
    s.dy, s.dy_batch, s.dy_time = _view("dy", dy, (b, t, d), tp, dev)
    s.du, s.du_batch, s.du_time = _view("du", got["u"], (b, t, d), tp, dev)
    s.ddelta, s.ddelta_batch, s.ddelta_time = _view("ddelta", got["delta"], (b, t, d), tp, dev)
    s.dB, s.dB_batch, s.dB_time = _view("dB", got["B"], (b, t, g, n), tp, dev)
    s.dC, s.dC_batch, s.dC_time = _view("dC", got["C"], (b, t, g, n), tp, dev)
    s.dz, s.dz_batch, s.dz_time = _view("dz", got["z"], (b, t, d), tp, dev)
    s.d_A = _array("d_A", got["A"], (d, n), torch.float32, dev)
    s.d_D = _array("d_D", got["D"], (d,), torch.float32, dev)
    s.d_delta_bias = _array("d_delta_bias", got["delta_bias"], (d,), torch.float32, dev)
    s.d_final_state = _array("d_final_state", d_final_state, (b, d, n), torch.float32, dev)
    s.d_state = _array("d_state", got["state"], (b, d, n), torch.float32, dev)
    work, size = _workspace("selective_scan_backward_workspace", s, dev)
    _call("selective_scan_backward", dev, C.byref(s), work.data_ptr() if size else None, size)
    return got


def _rows(name, x, shape, dtype, device):
    """address and row pitch of a [rows, columns] tensor"""
    if x is None:
        return None, 0
    _check(name, x, shape, dtype, device)
    if not _dense(x, 1):
        raise ValueError("%s: the columns have to lie densely, strides are %s" % (name, x.stride()))
    return x.data_ptr(), x.stride(0)


def distillation_error(logits, index, teacher, temperature=1.0, soft=1.0, hard=0.0, labels=None, weight=None, derivatives=True, losses=None, d_logits=None):
    """(losses [rows], d_logits [rows, vocabulary] or None): the error of `logits` against a teacher's best logits, teacher[r, k] (float32) of
    word index[r, k] (int32, outside the vocabulary: no entry), with `soft` * temperature^2 * KL(teacher, logits) at that
    temperature plus `hard` * cross entropy to labels (int32 [rows], outside the vocabulary: none), times weight (float32 [rows]); and its
    derivatives, of the logits' type, unless derivatives = False.  d_logits may be `logits`."""
    if logits.dim() != 2 or index.dim() != 2:
        raise ValueError("logits is [rows, vocabulary], index and teacher are [rows, top]")
    (r, v), k, dev = logits.shape, index.shape[1], logits.device
    s = capi.Distillation(_type(logits), 0, r, v, k)
    losses = _out(losses, (r,), torch.float32, dev)
    d_logits = _out(d_logits, (r, v), logits.dtype, dev) if derivatives else None
    s.logits, s.logits_stride = _rows("logits", logits, (r, v), logits.dtype, dev)
    s.index, s.index_stride = _rows("index", index, (r, k), torch.int32, dev)
    s.teacher, s.teacher_stride = _rows("teacher", teacher, (r, k), torch.float32, dev)
    s.labels, s.weight = _array("labels", labels, (r,), torch.int32, dev), _array("weight", weight, (r,), torch.float32, dev)
    s.temperature, s.soft, s.hard = temperature, soft, hard
    s.losses = _array("losses", losses, (r,), torch.float32, dev)
    s.d_logits, s.d_logits_stride = _rows("d_logits", d_logits, (r, v), logits.dtype, dev)
    _call("distillation_error", dev, C.byref(s))
    return losses, d_logits


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, chances=None):
    """(tokens int32 [rows], chances [rows]): one token for every row of logits [rows, vocabulary], drawn with uniform (float32 [rows], in
    [0, 1)) from what temperature, top_k (int32), top_p and min_p leave of the row, each an array of one value per row or None; and
    the chance that it had.  temperature <= 0: the largest logit.  A row whose words are all closed (minus infinity): token -1."""
    if logits.dim() != 2:
        raise ValueError("logits is [rows, vocabulary]")
    (r, v), dev = logits.shape, logits.device
    s = capi.Sampling(_type(logits), 0, r, v)
    tokens, chances = _out(tokens, (r,), torch.int32, dev), _out(chances, (r,), torch.float32, dev)
    s.logits, s.logits_stride = _rows("logits", logits, (r, v), logits.dtype, dev)
    for name, x, dtype in (("uniform", uniform, torch.float32), ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32), ("tokens", tokens, torch.int32), ("chances", chances, torch.float32)):
        setattr(s, name, _array(name, x, (r,), dtype, dev))
    _call("sample", dev, C.byref(s))
    return tokens, chances
