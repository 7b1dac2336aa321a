"""Scores of rows of logits (q3h_token_logprobs) whose values do not set their
largest apart."""
import gc

import pytest
import torch

import q3h

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_handles_left():
    yield
    gc.collect()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [20, 64])
def test_rows_of_logits_alike(device, dtype, k):
    """Rows whose logits are all alike, or the type's lowest value but for a few:
    the lowest tokens, and no more than 12 times the time of rows of all values
    (ranks are counted among the few hundred keys that are left, not among all of
    them, which takes 1000 times as long)."""
    rows, vocab = 40, 151936
    g = torch.Generator(device="cuda").manual_seed(k)
    few = torch.randint(0, vocab, (rows, 10), generator=g, device="cuda")
    values = torch.randn(rows, vocab, generator=g, device="cuda")
    masked = torch.full((rows, vocab), torch.finfo(dtype).min, device="cuda")
    masked.scatter_(1, few, values[:, :10])
    tokens = few[:, :1].to(torch.int32).contiguous()
    times = {}
    for name, x in (("values", values), ("alike", torch.zeros_like(values)), ("masked", masked)):
        x = x.to(dtype)
        got = q3h.token_logprobs(device, x, tokens, top_k=k)
        want = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(got["top_ids"].long(), want), name
        best = float("inf")
        for _ in range(5):
            e0, e1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            e0.record()
            for _ in range(4):
                q3h.token_logprobs(device, x, tokens, top_k=k)
            e1.record()
            e1.synchronize()
            best = min(best, e0.elapsed_time(e1) / 4)
        times[name] = best * 1e3
    print(times, flush=True)
    assert max(times["alike"], times["masked"]) < 12 * times["values"], times
