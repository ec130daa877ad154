"""Outputs of the serving calls are made where torch's modes see them."""
from __future__ import annotations

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu


class Made(TorchDispatchMode):
    """Addresses of the tensors that operators return."""

    def __init__(self):
        super().__init__()
        self.seen = set()

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if isinstance(out, torch.Tensor):
            self.seen.add(out.data_ptr())
        return out


def calls():
    from pallas_flash.kernels import paged
    k = torch.randn(4, 2, 16, 64, device="cuda").to(torch.bfloat16)
    q = torch.randn(2, 4, 1, 64, device="cuda").to(torch.bfloat16)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    n = torch.tensor([20, 30], dtype=torch.int32, device="cuda")
    bounds = paged.empty_bounds(k)
    shared = torch.tensor([16], dtype=torch.int32, device="cuda")
    return [lambda: paged.paged_decode(q, k, k, table, n, return_lse=True), lambda: paged.paged_decode(q[:, :2], k, k, table, n, return_lse=True),
            lambda: paged.paged_decode(q, k, k, table, n, return_lse=True, shared_lens=shared), lambda: paged.select_pages(q, bounds, table, n, 2, page_size=16)]


def test_dispatch_modes_see_outputs(built_lib):
    for call in calls():
        with Made() as mode:
            out = call()
        assert {t.data_ptr() for t in out} <= mode.seen


def test_deterministic_fill(built_lib):
    """New memory is filled where torch is told so (and the results do not depend on it)."""
    from pallas_flash import _lib
    want = [[t.clone() for t in call()] for call in calls()]
    dev = torch.device("cuda", torch.cuda.current_device())
    torch.use_deterministic_algorithms(True)
    try:
        assert _lib.empty((1000,), (1,), torch.float32, dev).isnan().all()
        got = [call() for call in calls()]
    finally:
        torch.use_deterministic_algorithms(False)
    assert all(a.shape == b.shape and a.dtype == b.dtype for x, y in zip(got, want) for a, b in zip(x, y))
    assert _lib.device_status() == (0, 0)
