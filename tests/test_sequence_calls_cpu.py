"""Calls of the sequence operators that are refused before a GPU is touched, beside those of their other tests."""
import ctypes as C

import pytest
import torch

from myea_b200 import capi
from myea_b200.net import Net

from test_sequence_cpu import ADDRESS, convolution, refused, scan


class OnGpu:
    """what a network asks of a tensor, as if it lay on a GPU"""
    def __init__(self, index, shape=(2, 3), dtype=torch.float32, dense=True):
        self.index, self.shape, self.dtype, self.device, self.is_cuda, self.dense = index, torch.Size(shape), dtype, torch.device("cuda", index), True, dense

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return self.dense

    def data_ptr(self):
        return 4096


def test_a_network_takes_arrays_of_its_own_gpu():
    net = Net.__new__(Net)   # (without a handle: a GPU has to be there for one)
    net.h, net.device = None, 1
    assert net._device_array("weight", OnGpu(1), (2, 3), "float32") == 4096 and net._device_array("weight", None, (2, 3), "float32") is None
    for other in (OnGpu(0), OnGpu(1, (3, 2)), OnGpu(1, dtype=torch.int32), OnGpu(1, dense=False), torch.zeros(2, 3)):
        with pytest.raises(ValueError, match="cuda:1"):
            net._device_array("weight", other, (2, 3), "float32")


def test_a_scan_over_no_sequences_needs_its_derivative_arrays():
    """the derivatives of A are written (as 0) for an empty batch too"""
    assert "derivatives of A" in refused("selective_scan_backward", scan(batch=0, d_A=None), None, 0)
    assert "derivatives of A" in refused("selective_scan_backward", scan(batch=0, time=0, d_A=None, d_D=ADDRESS), None, 0)


@pytest.mark.parametrize("d,n,taps", [(1, 1, 1), (12, 5, 4), (64, 16, 4), (65, 128, 8)])
def test_single_steps_of_fewer_rows_take_no_more_working_memory(d, n, taps):
    """a network makes room for its whole batch and runs shorter ones"""
    lib, before = capi.load(), (0, 0, 0)
    for rows in list(range(1, 70)) + [148, 149, 296, 591, 592, 593, 1000, 4096, 65536]:
        s, c = scan(batch=rows, time=1, width=d, states=n), convolution(batch=rows, time=1, width=d, taps=taps)
        now = (lib.myea_b200_selective_scan_workspace(C.byref(s)), lib.myea_b200_selective_scan_backward_workspace(C.byref(s)),
               lib.myea_b200_causal_convolution_backward_workspace(C.byref(c)))
        assert now[1] > 0 and now[2] > 0 and all(a <= b for a, b in zip(before, now)), rows
        before = now
