"""Attention's results to the last bit that its rows' type can hold, where the
roundings inside the kernels would show."""
import numpy as np
import pytest

from kv_plain import TYPES, Device, attention, attention_tolerance, random_table, spt, torch_type

pytestmark = pytest.mark.gpu


def tolerance(want, length, type):
    """What f32 rows are allowed (attention_tolerance), and one rounding of the result to the rows' type."""
    import torch
    tol = attention_tolerance(*want, length, "f32")
    if type == "f32":
        return tol
    eps = torch.finfo(torch_type(type)).eps / 2
    return tol + (want[0].abs() + tol) * eps + (2.0 ** -25 if type == "f16" else 0.0)


def append(ctx, cache, table, lengths, counts, k, v):
    import torch
    dev = Device(table, lengths, counts)
    torch.cuda.synchronize()
    cache.append_device(dev.batch, k.data_ptr(), v.data_ptr())
    ctx.sync()


def read(ctx, cache, table, length):
    """Keys and values of one sequence as the cache holds them, in 64 bits."""
    import torch
    dev = Device(table, [length], [length])
    k = torch.zeros(length, cache.kv_heads, cache.head_dim, device="cuda")
    v = torch.zeros_like(k)
    torch.cuda.synchronize()
    cache.read_device(dev.batch, k.data_ptr(), v.data_ptr())
    ctx.sync()
    return k.double(), v.double()


def attend(ctx, cache, table, lengths, counts, q, window=0, sinks=None, scale=0.125):
    import torch
    type = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[q.dtype]
    out = torch.full_like(q, 7)
    dev = Device(table, lengths, counts)
    torch.cuda.synchronize()
    cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), q.shape[1], type, scale=scale, window=window,
                           sinks_ptr=0 if sinks is None else sinks.data_ptr())
    ctx.sync()
    return out


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("length,counts", [(24, None), (24, [2]), (24, [24]), (500, None), (500, [2]), (500, [300])])
def test_values_that_nearly_cancel(ctx, type, dim, length, counts):
    """Neighbouring keys have opposite values and nearly equal weights: the results are far smaller
    than the values, and so is their rounding, but not that of a weight held in fewer bits."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(dim + length)
    table, _, pages = random_table(np.random.default_rng(dim), [length], 16)
    cache = ctx.kv_cache(kv_heads=2, head_dim=dim, page_tokens=16, pages=pages)
    k = torch.randn(length, 2, dim, generator=gen, device="cuda")
    v = torch.randn(length // 2, 2, dim, generator=gen, device="cuda").repeat_interleave(2, 0)
    v[1::2] *= -1
    append(ctx, cache, table, [length], [length], k, v)
    keys, values = read(ctx, cache, table, length)
    n = 1 if counts is None else counts[0]
    q = (0.02 * torch.randn(n, 16, dim, generator=gen, device="cuda")).to(torch_type(type))
    out = attend(ctx, cache, table, [length], counts, q)
    want = attention(q.double(), keys, values, length - n, 0.125)
    off, tol = (out.double() - want[0]).abs(), tolerance(want, length, type)
    assert bool((off <= tol).all()), float((off / tol).max())
    cache.close()
