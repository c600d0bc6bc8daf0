"""The operators for sequence models without a GPU: descriptions that cannot be computed are refused with a reason before any device is
touched, and the Python side refuses arguments that do not fit together."""
import ctypes as C

import pytest
import torch

from myea_b200 import capi, sequence

MEMORY = C.create_string_buffer(1 << 16)
ADDRESS = (C.addressof(MEMORY) + 255) // 256 * 256   # never followed: every call here is refused first


def refused(name, s, *work):
    message = C.create_string_buffer(256)
    rc = getattr(capi.load(), "myea_b200_" + name)(0, C.byref(s) if s is not None else None, *work, None, message, 256)
    assert rc == -1, (name, rc, message.value)
    return message.value.decode()


def convolution(**kw):
    s = capi.Convolution(capi.TYPE_F32, 4, 1, 0, 2, 8, 16)
    for n in ("x", "y", "dy", "dx", "weight", "d_weight"):
        setattr(s, n, ADDRESS + 1024 * (1 + ["x", "y", "dy", "dx", "weight", "d_weight"].index(n)))
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def scan(**kw):
    names = ("u", "delta", "B", "C", "y", "dy", "du", "ddelta", "dB", "dC", "A", "d_A", "checkpoints")
    s = capi.Scan(capi.TYPE_F32, 1, 0, 0, 2, 8, 16, 16, 1)
    for k, n in enumerate(names):
        setattr(s, n, ADDRESS + 1024 * (k + 1))
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_struct_layouts_match_header():
    assert C.sizeof(capi.Convolution) == 4 * 4 + 3 * 8 + 4 * 24 + 9 * 8
    assert C.sizeof(capi.Scan) == 4 * 4 + 5 * 8 + 12 * 24 + 7 * 8 + 5 * 8
    for s, packed in ((capi.Convolution, sequence._CONVOLUTION), (capi.Scan, sequence._SCAN), (capi.Distillation, sequence._DISTILLATION),
                      (capi.Sampling, sequence._SAMPLING)):
        assert C.sizeof(s) == packed.size


@pytest.mark.parametrize("change,word", [(dict(type=3), "type"), (dict(taps=0), "taps"), (dict(taps=9), "taps"), (dict(time=1 << 31), "dimension"),
                                         (dict(weight=None), "weights"), (dict(x=None), "input"), (dict(y=None), "output"), (dict(y=ADDRESS + 1024), "output")])
def test_convolution_refusals(change, word):
    assert word in refused("causal_convolution", convolution(**change))


def test_convolution_backward_refusals():
    assert "workspace" in refused("causal_convolution_backward", convolution(), None, 0)
    assert "workspace" in refused("causal_convolution_backward", convolution(), ADDRESS, 16)
    assert "workspace" in refused("causal_convolution_backward", convolution(), ADDRESS + 4, 1 << 30)
    assert "error" in refused("causal_convolution_backward", convolution(dy=None), ADDRESS, 1 << 30)
    assert "operand" in refused("causal_convolution_backward", convolution(dx=ADDRESS + 1024), ADDRESS, 1 << 30)
    assert "d_state" in refused("causal_convolution_backward", convolution(d_state=ADDRESS, d_final_state=ADDRESS), ADDRESS, 1 << 30)
    assert refused("causal_convolution", None) and refused("causal_convolution_backward", None, None, 0)


@pytest.mark.parametrize("change,word", [(dict(type=7), "type"), (dict(states=0), "states"), (dict(states=129), "states"), (dict(groups=0), "groups"),
                                         (dict(groups=3), "groups"), (dict(width=1 << 31), "dimension"), (dict(A=None), "(A)"), (dict(delta=None), "delta"),
                                         (dict(y=None), "output"), (dict(y=ADDRESS + 1024), "output"), (dict(checkpoints=ADDRESS + 4), "aligned")])
def test_scan_refusals(change, word):
    assert word in refused("selective_scan", scan(**change), None, 0)


@pytest.mark.parametrize("change,word", [(dict(dy=None), "dy"), (dict(dB=None), "dB"), (dict(z=ADDRESS), "dz"), (dict(dz=ADDRESS), "dz"),
                                         (dict(checkpoints=None), "checkpoints"), (dict(d_A=None), "derivatives of A"),
                                         (dict(d_state=ADDRESS, d_final_state=ADDRESS), "d_state"), (dict(), "workspace")])
def test_scan_backward_refusals(change, word):
    assert word in refused("selective_scan_backward", scan(**change), None, 0)


def test_scan_refuses_a_missing_workspace_when_time_is_cut():
    s = scan(time=4096, batch=1)
    assert capi.load().myea_b200_selective_scan_workspace(C.byref(s)) > 0
    assert "workspace" in refused("selective_scan", s, None, 0)
    assert refused("selective_scan", None, None, 0) and refused("selective_scan_backward", None, None, 0)


def test_tensors_off_the_gpu_are_refused():
    x, w = torch.zeros(1, 4, 8), torch.zeros(8, 4)
    with pytest.raises(ValueError, match="GPU"):
        sequence.causal_convolution(x, w)
    with pytest.raises(ValueError, match="GPU"):
        sequence.selective_scan(x, x, torch.zeros(8, 16), torch.zeros(1, 4, 1, 16), torch.zeros(1, 4, 1, 16))


def distillation(**kw):
    s = capi.Distillation(capi.TYPE_F32, 0, 4, 100, 8, temperature=1.0, soft=1.0)
    for k, n in enumerate(("logits", "index", "teacher", "losses")):
        setattr(s, n, ADDRESS + 1024 * k)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def sampling(**kw):
    s = capi.Sampling(capi.TYPE_F32, 0, 4, 100)
    for k, n in enumerate(("logits", "uniform", "tokens")):
        setattr(s, n, ADDRESS + 1024 * k)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("change,word", [(dict(type=9), "type"), (dict(rows=1 << 31), "dimension"), (dict(vocabulary=1 << 31), "dimension"), (dict(top=0), "entries"),
                                         (dict(top=1025), "entries"), (dict(temperature=0.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
                                         (dict(temperature=float("inf")), "temperature"), (dict(vocabulary=0), "vocabulary"), (dict(logits=None), "logits"),
                                         (dict(index=None), "index"), (dict(teacher=None), "teacher"), (dict(losses=None), "losses")])
def test_distillation_refusals(change, word):
    assert word in refused("distillation_error", distillation(**change))


@pytest.mark.parametrize("change,word", [(dict(type=9), "type"), (dict(rows=1 << 31), "dimension"), (dict(vocabulary=1 << 31), "dimension"), (dict(vocabulary=0), "vocabulary"),
                                         (dict(logits=None), "logits"), (dict(uniform=None), "uniform"), (dict(tokens=None), "tokens")])
def test_sampling_refusals(change, word):
    assert word in refused("sample", sampling(**change))
    assert refused("sample", None) and refused("distillation_error", None)


def test_an_empty_batch_needs_little_memory_however_long_its_time():
    """no sequences of many positions: nothing is cut, and only the (empty) sums of the parameters are formed"""
    for time in (0, 127, 128, 4096):
        s = scan(batch=0, time=time)
        assert capi.load().myea_b200_selective_scan_workspace(C.byref(s)) == 0
        assert capi.load().myea_b200_selective_scan_backward_workspace(C.byref(s)) == 0
        assert capi.load().myea_b200_causal_convolution_backward_workspace(C.byref(convolution(batch=0, time=time))) == 0
