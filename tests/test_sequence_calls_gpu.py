"""Calls that the documentation of the sequence operators allows and that their other tests do not make."""
import math

import pytest
import torch

from test_sequence_gpu import DEV
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
