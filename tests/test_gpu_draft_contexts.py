"""Drafted trees and rows over int8 caches on contexts, where the attention's
groups are cut into shares that leave parts (contexts of more than a few hundred
positions), and what other calls on a context do to a pending tree."""
import gc

import numpy as np
import pytest

import q3h
from test_gpu_draft_forward import Setup, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_handles_left():
    yield
    gc.collect()


@pytest.mark.parametrize("fmt", [q3h.KV_F32, q3h.KV_F16])
def test_a_measured_attention_drops_the_tree(device, fmt):
    """q3h_context_time_attention writes position len, where the tree's first row
    waits: nothing of the tree can be kept after it."""
    s = Setup(device, fmt=fmt)
    c = s.context(60)
    x = rows_of(1, 4)
    c.forward(x[:2])
    c.forward_tree(x, [-1, 0, 1, 0])
    c.time_attention(iters=1)
    with pytest.raises(q3h.Q3HError) as e:
        c.keep([0, 1])
    assert e.value.code == q3h.E_STATE and c.length == 2
    c.forward_tree(x, [-1, 0, 1, 0])
    c.keep([0, 1])
    assert c.length == 4
    s.destroy(c)
