"""Caches in pages at the edges of what their calls take: calls without rows."""
import gc

import numpy as np
import pytest
import torch

import q3h
from test_gpu_draft import dev_i

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_handles_left():
    """Handles that a refusal's traceback still holds go before the device does."""
    yield
    gc.collect()


def test_append_of_no_rows_at_positions(device):
    """A step in which no sequence has a row: tensors without elements, which have no address."""
    rope = q3h.Rope(device, 64, 100, 1e4, axes=[i % 3 for i in range(32)])
    for pages in (0, 4):
        cache = q3h.Cache(device, 2, 2, 64, 100, q3h.KV_Q4, pages=pages, page_positions=32)
        for n, rows in ((2, 0), (0, 3)):
            x = torch.zeros((n, rows, 2, 64), device="cuda")
            at = torch.zeros((3, n, rows), dtype=torch.int32, device="cuda")
            q = cache.append(x, x, dev_i(np.zeros(n)), q=x, rope=rope, positions=at)
            assert q.shape == x.shape
            cache.append(x, x, dev_i(np.zeros(n)), rope=rope)
