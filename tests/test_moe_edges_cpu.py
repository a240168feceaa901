"""Sizes of the layer's operators that the C-ABI's 32 bits do not hold, without a GPU."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


def test_more_rows_than_32_bits_are_refused():
    """A count cut to 32 bits would leave rows without a result."""
    from vllm_expert_cache import moe
    with FakeTensorMode():
        x = torch.empty(2 ** 32 + 5, 8, dtype=torch.bfloat16, device="cuda")
        gate = torch.empty(4, 8, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(ValueError, match="rows of x"):
            moe.route(x, gate, 1)
        ids = torch.empty(2 ** 32 + 5, 1, dtype=torch.int32, device="cuda")
        weights = torch.empty(2 ** 32 + 5, 1, device="cuda")
        w = torch.empty(2, 16, 8, dtype=torch.bfloat16, device="cuda")
        with pytest.raises(ValueError, match="rows of x"):
            moe.experts(x, weights, ids, w, w.view(2, 8, 16)[:, :, :8])


@pytest.mark.parametrize("T", [2 ** 30, 2 ** 31 - 4, 2 ** 31 - 1])
def test_router_refuses_more_tokens_than_a_launch_takes(T):
    """Before CUDA is touched, and without a sum past the end of int."""
    import build_lib
    from vllm_expert_cache import _lib
    build_lib.build()
    at = 1 << 20                                    # never dereferenced
    assert _lib.lib().expert_cache_route(at, T, 8, 8, at, 4, 1, 0, 1, None, 1.0, at, at,
                                         None) == -1
