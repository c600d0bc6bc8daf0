"""Operators for sequence models on tensors that lie on the GPU: thin calls into libmyea_b200.so (include/myea_b200.h, where the
formulas stand).  They stand beside the recurrent layers, the output error and the output layer of `net.Net` and need no network.

Tensors are torch tensors, used where they lie: an activation is [batch, time, width] with any strides over batch and time
and densely packed last dimensions (a time-major array is x.transpose(0, 1), a slice of a wider projection is read in place),
of float32, bfloat16 or float16, one type per call; parameters, states of a scan and losses are float32.  A call runs on the
current stream of the tensors' GPU, may be captured into a CUDA graph and does not wait.  Autograd does not follow it: derivatives come
from the *_backward functions and the errors, and tensors that want a gradient are refused where gradients are recorded.  ValueError: the arguments do not fit
together (nothing was launched); RuntimeError: the library refused the call or failed, with its message.
"""
import ctypes as C
import struct
import threading

import torch

from . import capi

_TYPES = {torch.float32: capi.TYPE_F32, torch.bfloat16: capi.TYPE_BF16, torch.float16: capi.TYPE_F16}
_F32, _I32 = torch.float32, torch.int32
# the descriptions of myea_b200.h, packed (a call for one token takes a few microseconds: so do forty attribute assignments)
_CONVOLUTION = struct.Struct("<4I3Q" + 4 * "Qqq" + "9Q")
_SCAN = struct.Struct("<4I5Q" + 6 * "Qqq" + "7Q" + 6 * "Qqq" + "5Q")
_DISTILLATION = struct.Struct("<2I3Q" + 3 * "Qq" + "2Q4f2Qq")
_SAMPLING = struct.Struct("<2I2QQq7Q")
_NO_VIEW = (0, 0, 0)
_local = threading.local()   # .message: where the library says why
# a stream's handle without the object around it (1.3 us of the 10 to 15 that a call takes on the host)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name, index, *args):
    try:
        message = _local.message
    except AttributeError:
        message = _local.message = C.create_string_buffer(256)
    rc = getattr(capi.load(), name)(index, *args, _stream(index), message, 256)
    if rc != 0:
        raise RuntimeError("%s failed (%d): %s" % (name, rc, message.value.decode()))


def _no_history(name):
    raise ValueError("%s wants a gradient, which autograd would lose here: detach it or call under torch.no_grad(), and use the operator's derivatives" % name)


def _mismatch(name, x, shape, dtype, index):
    raise ValueError("%s: expected %s of %s on cuda:%d, got %s of %s on %s" % (name, tuple(shape), dtype, index, tuple(x.shape), x.dtype, x.device))


def _type(x):
    if not x.is_cuda:
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


def _view(name, x, shape, dtype, index):
    """address and strides of a [batch, time, ...] tensor; nothing where there is none"""
    if x is None:
        return _NO_VIEW
    if x.shape != shape or x.dtype is not dtype or x.get_device() != index:
        _mismatch(name, x, shape, dtype, index)
    return _own_view(name, x)


def _own_view(name, x):
    """the same for the tensor that the others are compared with"""
    if x.requires_grad and torch.is_grad_enabled():
        _no_history(name)
    if not x.is_contiguous() and not _dense(x, 2):
        raise ValueError("%s: the dimensions behind batch and time have to lie densely, strides are %s" % (name, x.stride()))
    strides = x.stride()
    return x.data_ptr(), strides[0], strides[1]


def _output(name, given, like):
    """(tensor, its address and strides): the given one, or a new one like `like`"""
    if given is not None:
        return given, _view(name, given, like.shape, like.dtype, like.get_device())
    new = _empty_like(like)
    _, t, d = like.shape
    return new, (new.data_ptr(), t * d, d)


def _array(name, x, shape, dtype, index):
    """address of a densely packed tensor; 0 where there is none"""
    if x is None:
        return 0
    if x.shape != shape or x.dtype is not dtype or x.get_device() != index:
        _mismatch(name, x, shape, dtype, index)
    if x.requires_grad and torch.is_grad_enabled():
        _no_history(name)
    if not x.is_contiguous():
        raise ValueError("%s has to be contiguous" % name)
    return x.data_ptr()


def _gradient(name, given, shape, like, accumulate):
    if given is not None:
        return given
    if accumulate:
        raise ValueError("%s: accumulate needs an array to add to" % name)
    return like.new_empty(shape, dtype=_F32)


def _workspace(name, description, like):
    size = getattr(capi.load(), name)(description)
    if size == 0:
        return None, None, 0
    work = like.new_empty(size, dtype=torch.uint8)
    return work, work.data_ptr(), size


def _empty_like(x):
    """a densely packed tensor of x's shape and type"""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)   # (the first is quicker)


def causal_convolution(x, weight, bias=None, silu=True, state=None, final_state=None, lengths=None, out=None):
    """(y, final_state): y[b, t, c] = act(bias[c] + sum over j of weight[c, j] * x[b, t - taps + 1 + j, c]), act = silu or nothing.
    weight [width, taps], 1 to 8 taps; state [batch, taps - 1, width]: the inputs before the first (None: zeros); final_state: where the
    last taps - 1 inputs go (None: a new tensor; `state` itself is allowed); lengths int32 [batch]: y is 0 behind a sequence's
    end.  A single token is time = 1 with both states."""
    kind = _type(x)
    if x.dim() != 3 or weight.dim() != 2:
        raise ValueError("x is [batch, time, width] and weight [width, taps]")
    (b, t, d), k, tp, at = x.shape, weight.shape[1], x.dtype, x.get_device()
    before = (b, k - 1, d)
    out, to = _output("out", out, x)
    if final_state is None:
        final_state = x.new_empty(before)
    _call("myea_b200_causal_convolution", at, _CONVOLUTION.pack(
        kind, k, 1 if silu else 0, 0, b, t, d, *_own_view("x", x), *to, *_NO_VIEW, *_NO_VIEW,
        _array("weight", weight, (d, k), _F32, at), _array("bias", bias, (d,), _F32, at), _array("state", state, before, tp, at),
        _array("final_state", final_state, before, tp, at), _array("lengths", lengths, (b,), _I32, at), 0, 0, 0, 0))
    return out, final_state


def causal_convolution_backward(dy, x, weight, bias=None, silu=True, state=None, lengths=None, d_final_state=None, dx=None, d_weight=None, d_bias=None,
                                accumulate=False):
    """{"x", "weight", "bias" (None without one), "state" (None without one)}: derivatives for the error `dy` on y and
    `d_final_state` on the final state.  d_weight / d_bias given: the derivatives go there, with `accumulate` onto what they hold."""
    kind = _type(x)
    if x.dim() != 3 or weight.dim() != 2:
        raise ValueError("x is [batch, time, width] and weight [width, taps]")
    (b, t, d), k, tp, at = x.shape, weight.shape[1], x.dtype, x.get_device()
    whole, before = (b, t, d), (b, k - 1, d)
    dx, to = _output("dx", dx, x)
    d_weight = _gradient("d_weight", d_weight, (d, k), x, accumulate)
    d_bias = _gradient("d_bias", d_bias, (d,), x, accumulate) if bias is not None else None
    d_state = x.new_empty(before) if state is not None else None
    s = _CONVOLUTION.pack(
        kind, k, 1 if silu else 0, 1 if accumulate else 0, b, t, d, *_own_view("x", x), *_NO_VIEW, *_view("dy", dy, whole, tp, at),
        *to, _array("weight", weight, (d, k), _F32, at), _array("bias", bias, (d,), _F32, at), _array("state", state, before, tp, at),
        0, _array("lengths", lengths, (b,), _I32, at), _array("d_weight", d_weight, (d, k), _F32, at), _array("d_bias", d_bias, (d,), _F32, at),
        _array("d_final_state", d_final_state, before, tp, at), _array("d_state", d_state, before, tp, at))
    work, address, size = _workspace("myea_b200_causal_convolution_backward_workspace", s, x)
    _call("myea_b200_causal_convolution_backward", at, s, address, size)
    return {"x": dx, "weight": d_weight, "bias": d_bias, "state": d_state}


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


def _scan_inputs(u, delta, A, B, C_, D, z, delta_bias, state, lengths):
    """(type, sizes, device, views of the inputs, arrays of the parameters), checked"""
    kind = _type(u)
    if u.dim() != 3 or A.dim() != 2 or B.dim() != 4:
        raise ValueError("u is [batch, time, width], A [width, states], B and C [batch, time, groups, states]")
    (b, t, d), n, g, tp, at = u.shape, A.shape[1], B.shape[2], u.dtype, u.get_device()
    whole, narrow = (b, t, d), (b, t, g, n)
    views = _own_view("u", u) + _view("delta", delta, whole, tp, at) + _view("B", B, narrow, tp, at) + _view("C", C_, narrow, tp, at) + _view("z", z, whole, tp, at)
    arrays = (_array("A", A, (d, n), _F32, at), _array("D", D, (d,), _F32, at), _array("delta_bias", delta_bias, (d,), _F32, at),
              _array("state", state, (b, d, n), _F32, at))
    return kind, (b, t, d, n, g), at, views, arrays, _array("lengths", lengths, (b,), _I32, at)


def selective_scan(u, delta, A, B, C_, D=None, z=None, delta_bias=None, softplus=True, state=None, final_state=None, lengths=None, checkpoints=None,
                   out=None):
    """(y, final_state) of the selective state space scan over u, delta [batch, time, width] with A [width, states] (1 to 128 states),
    B, C [batch, time, groups, states], D and delta_bias [width], a gate z like u, a state [batch, width, states] to start from (None:
    zeros) and one to end in (None: a new tensor; `state` itself is allowed).  lengths int32 [batch]: y is 0 behind a sequence's
    end, and the state there stays.  checkpoints (scan_checkpoints): kept for selective_scan_backward.  A single token is
    time = 1 with both states."""
    kind, (b, t, d, n, g), at, views, arrays, lengths_at = _scan_inputs(u, delta, A, B, C_, D, z, delta_bias, state, lengths)
    out, to = _output("out", out, u)
    if final_state is None:
        final_state = u.new_empty((b, d, n), dtype=_F32) if state is None else torch.empty_like(state)
    kept = 0 if checkpoints is None else _array("checkpoints", checkpoints, _checkpoint_shape(b, t, d, n), _F32, at)
    s = _SCAN.pack(kind, 1 if softplus else 0, 0, 0, b, t, d, n, g, *views, *to, *arrays,
                   _array("final_state", final_state, (b, d, n), _F32, at), lengths_at, kept, *_NO_GRADIENTS)
    work, address, size = _workspace("myea_b200_selective_scan_workspace", s, u)
    _call("myea_b200_selective_scan", at, s, address, size)
    return out, final_state


_NO_GRADIENTS = (0,) * 23


def selective_scan_backward(dy, u, delta, A, B, C_, checkpoints, D=None, z=None, delta_bias=None, softplus=True, state=None, lengths=None,
                            d_final_state=None, d_A=None, d_D=None, d_delta_bias=None, accumulate=False):
    """Derivatives for the error `dy` on y and `d_final_state` on the final state, by the names of the forward pass's arguments
    ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"; None where there was none).  d_A, d_D, d_delta_bias given: those go
    there, with `accumulate` onto what they hold."""
    kind, (b, t, d, n, g), at, views, arrays, lengths_at = _scan_inputs(u, delta, A, B, C_, D, z, delta_bias, state, lengths)
    tp, whole, narrow, held = u.dtype, (b, t, d), (b, t, g, n), (b, d, n)
    got = {"u": _empty_like(u), "delta": _empty_like(u), "B": u.new_empty(narrow), "C": u.new_empty(narrow), "z": _empty_like(u) if z is not None else None,
           "A": _gradient("d_A", d_A, (d, n), u, accumulate), "D": _gradient("d_D", d_D, (d,), u, accumulate) if D is not None else None,
           "delta_bias": _gradient("d_delta_bias", d_delta_bias, (d,), u, accumulate) if delta_bias is not None else None,
           "state": u.new_empty(held, dtype=_F32) if state is not None else None}
    s = _SCAN.pack(kind, 1 if softplus else 0, 1 if accumulate else 0, 0, b, t, d, n, g, *views, *_NO_VIEW, *arrays, 0, lengths_at,
                   _array("checkpoints", checkpoints, _checkpoint_shape(b, t, d, n), _F32, at), *_view("dy", dy, whole, tp, at),
                   *_view("du", got["u"], whole, tp, at), *_view("ddelta", got["delta"], whole, tp, at), *_view("dB", got["B"], narrow, tp, at),
                   *_view("dC", got["C"], narrow, tp, at), *_view("dz", got["z"], whole, tp, at), _array("d_A", got["A"], (d, n), _F32, at),
                   _array("d_D", got["D"], (d,), _F32, at), _array("d_delta_bias", got["delta_bias"], (d,), _F32, at),
                   _array("d_final_state", d_final_state, held, _F32, at), _array("d_state", got["state"], held, _F32, at))
    work, address, size = _workspace("myea_b200_selective_scan_backward_workspace", s, u)
    _call("myea_b200_selective_scan_backward", at, s, address, size)
    return got


def _rows(name, x, shape, dtype, index):
    """address and row pitch of a [rows, columns] tensor"""
    if x is None:
        return 0, 0
    if x.shape != shape or x.dtype is not dtype or x.get_device() != index:
        _mismatch(name, x, shape, dtype, index)
    return _own_rows(name, x)


def _own_rows(name, x, history=False):
    """the same for the tensor that the others are compared with; history: autograd may follow it"""
    if not history and x.requires_grad and torch.is_grad_enabled():
        _no_history(name)
    if not x.is_contiguous() and not _dense(x, 1):
        raise ValueError("%s: the columns have to lie densely, strides are %s" % (name, x.stride()))
    return x.data_ptr(), x.stride(0)


def distillation_error(logits, index, teacher, temperature=1.0, soft=1.0, hard=0.0, labels=None, weight=None, derivatives=True, losses=None, d_logits=None):
    """(losses [rows], d_logits [rows, vocabulary] or None): the error of `logits` against a teacher's best logits, teacher[r, k] (float32) of
    word index[r, k] (int32, outside the vocabulary: no entry), with `soft` * temperature^2 * KL(teacher, logits) at that
    temperature plus `hard` * cross entropy to labels (int32 [rows], outside the vocabulary: none), times weight (float32 [rows]); and its
    derivatives, of the logits' type, unless derivatives = False.  d_logits may be `logits`."""
    kind = _type(logits)
    if logits.dim() != 2 or index.dim() != 2:
        raise ValueError("logits is [rows, vocabulary], index and teacher are [rows, top]")
    (r, v), k, tp, at = logits.shape, index.shape[1], logits.dtype, logits.get_device()
    if losses is None:
        losses = logits.new_empty((r,), dtype=_F32)
    if not derivatives:
        d_logits = None
    elif d_logits is None:
        d_logits = _empty_like(logits)
    _call("myea_b200_distillation_error", at, _DISTILLATION.pack(
        kind, 0, r, v, k, *_own_rows("logits", logits), *_rows("index", index, (r, k), _I32, at), *_rows("teacher", teacher, (r, k), _F32, at),
        _array("labels", labels, (r,), _I32, at), _array("weight", weight, (r,), _F32, at), temperature, soft, hard, 0.0,
        _array("losses", losses, (r,), _F32, at), *_rows("d_logits", d_logits, (r, v), tp, at)))
    return losses, d_logits


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, chances=None):
    """(tokens int32 [rows], chances [rows]): one token for every row of logits [rows, vocabulary], drawn with uniform (float32 [rows], in
    [0, 1)) from what temperature, top_k (int32), top_p and min_p leave of the row, each an array of one value per row or None; and
    the chance that it had.  temperature <= 0: the largest logit.  A row whose words are all closed (minus infinity): token -1.  A draw
    has no derivatives: the logits may want a gradient, the results have no history."""
    kind = _type(logits)
    if logits.dim() != 2:
        raise ValueError("logits is [rows, vocabulary]")
    (r, v), at = logits.shape, logits.get_device()
    one = (r,)
    if tokens is None:
        tokens = logits.new_empty(one, dtype=_I32)
    if chances is None:
        chances = torch.empty_like(uniform) if uniform is not None else logits.new_empty(one, dtype=_F32)
    _call("myea_b200_sample", at, _SAMPLING.pack(
        kind, 0, r, v, *_own_rows("logits", logits, True), _array("uniform", uniform, one, _F32, at), _array("temperature", temperature, one, _F32, at),
        _array("top_k", top_k, one, _I32, at), _array("top_p", top_p, one, _F32, at), _array("min_p", min_p, one, _F32, at),
        _array("tokens", tokens, one, _I32, at), _array("chances", chances, one, _F32, at)))
    return tokens, chances
