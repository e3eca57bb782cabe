"""Attention at the last positions that a length can name."""
import pytest

from kv_plain import TYPES, Device, attention, torch_type
from test_gpu_attention_accuracy import append, attend, read, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("count", [None, 2, 100])
@pytest.mark.parametrize("short", [0, 1, 17])
def test_lengths_up_to_the_largest(ctx, type, count, short):
    """2^31 - 1 tokens and a few less, on one page in every place of the table: the last tile's
    end lies beyond 31 bits, and what it holds behind the length is not seen."""
    import torch
    page, window, n = 65536, 50, count or 1
    length = 2 ** 31 - 1 - short
    gen = torch.Generator(device="cuda").manual_seed(short)
    cache = ctx.kv_cache(kv_heads=1, head_dim=32, page_tokens=page, pages=1)
    x, v = torch.randn(page, 1, 32, generator=gen, device="cuda"), torch.randn(page, 1, 32, generator=gen, device="cuda")
    v[length % page:] = 100.0
    append(ctx, cache, [[0]], [page], [page], x, v)
    keys, values = read(ctx, cache, [[0]], page)
    q = torch.randn(n, 4, 32, generator=gen, device="cuda").to(torch_type(type))
    out = attend(ctx, cache, [[0] * (2 ** 31 // page)], [length], None if count is None else [count], q, window)
    # the window's keys alone, as positions of a short sequence
    first = length - n - window + 1
    at = torch.arange(first, length, device="cuda") % page
    want = attention(q.double(), keys[at], values[at], window - 1, 0.125, window)
    assert bool(((out.double() - want[0]).abs() <= tolerance(want, len(at), type)).all())
    # the same rows, appended there, read back
    new, v_new = torch.randn(n, 1, 32, generator=gen, device="cuda"), torch.randn(n, 1, 32, generator=gen, device="cuda")
    table = [[0] * (2 ** 31 // page)]
    append(ctx, cache, table, [length], [n], new, v_new)
    end = length % page
    k2, v2 = read(ctx, cache, [[0]], page)
    dev, back = Device(table, [length], [n]), torch.zeros(n, 1, 32, device="cuda")
    torch.cuda.synchronize()
    cache.read_device(dev.batch, back.data_ptr(), 0)
    ctx.sync()
    assert bool((back.double() == k2[end - n:end]).all()) and bool((k2[:end - n] == keys[:end - n]).all())
    assert bool((v2[end:] == values[end:]).all())
    cache.close()


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("counts", [None, [1, 1, 0], [90, 40, 7]], ids=str)
def test_infinite_sinks(ctx, type, counts):
    """An infinite sink takes all weight, one of -inf none, a NaN gives NaNs: in that head alone, with keys and
    without."""
    import numpy as np
    import torch

    from kv_plain import random_table
    inf = float("inf")
    lengths = [300, 200, 5]
    gen = torch.Generator(device="cuda").manual_seed(8)
    table, _, pages = random_table(np.random.default_rng(8), lengths, 16)
    cache = ctx.kv_cache(kv_heads=2, head_dim=64, page_tokens=16, pages=pages)
    append(ctx, cache, table, lengths, lengths, torch.randn(505, 2, 64, generator=gen, device="cuda"),
           torch.randn(505, 2, 64, generator=gen, device="cuda"))
    n = 3 if counts is None else sum(counts)
    q = torch.randn(n, 4, 64, generator=gen, device="cuda").to(torch_type(type))
    plain = attend(ctx, cache, table, lengths, counts, q)
    out = attend(ctx, cache, table, lengths, counts, q, sinks=torch.tensor([inf, -inf, 3e38, float("nan")], device="cuda"))
    assert not bool(out[:, 0].any()) and not bool(out[:, 2].any()) and bool(torch.isnan(out[:, 3]).all())
    off = (out[:, 1].float() - plain[:, 1].float()).abs()  # the same sums, divided by them plus 0
    assert bool((off <= plain[:, 1].float().abs() * 2.0 ** -22).all()) or type != "f32" and bool((off == 0).all())
    cache.close()
