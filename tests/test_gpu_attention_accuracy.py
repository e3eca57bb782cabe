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


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("counts", [None, [2, 2], [90, 40]], ids=str)
@pytest.mark.parametrize("junk", [1e3, 1e6, -6e5])
def test_large_values_in_masked_places(ctx, type, counts, junk):
    """Finite numbers of any size behind the length and before the window, beside small values in
    sight, change no bit: neither of single rows nor of chunks."""
    import torch
    lengths, whole = [300, 200], [320, 256]
    n = [1, 1] if counts is None else counts
    gen = torch.Generator(device="cuda").manual_seed(2)
    table, _, pages = random_table(np.random.default_rng(3), whole, 32)
    cache = ctx.kv_cache(kv_heads=2, head_dim=64, page_tokens=32, pages=pages)
    k = torch.randn(500, 2, 64, generator=gen, device="cuda")
    v = 1e-3 * torch.randn(500, 2, 64, generator=gen, device="cuda")
    append(ctx, cache, table, lengths, lengths, k, v)
    held = [read(ctx, cache, table[b:b + 1], lengths[b]) for b in range(2)]
    q = torch.randn(sum(n), 16, 64, generator=gen, device="cuda").to(torch_type(type))
    window = 37
    want, seen = attend(ctx, cache, table, lengths, counts, q), attend(ctx, cache, table, lengths, counts, q, window)
    at = 0
    for b, c in enumerate(n):
        for out, w in ((want, 0), (seen, window)):
            exact = attention(q[at:at + c].double(), *held[b], lengths[b] - c, 0.125, w)
            assert bool(((out[at:at + c].double() - exact[0]).abs() <= tolerance(exact, lengths[b], type)).all())
        at += c
    # behind the lengths
    tail = [w - m for w, m in zip(whole, lengths)]
    x = torch.full((sum(tail), 2, 64), junk, device="cuda")
    append(ctx, cache, table, whole, tail, x, x)
    assert bool((attend(ctx, cache, table, lengths, counts, q) == want).all())
    assert bool((attend(ctx, cache, table, lengths, counts, q, window) == seen).all())
    # and up to the first key that a row with the window sees
    head = [m - c + 1 - window for m, c in zip(lengths, n)]
    x = torch.full((sum(head), 2, 64), junk, device="cuda")
    append(ctx, cache, table, head, head, x, x)
    assert bool((attend(ctx, cache, table, lengths, counts, q, window) == seen).all())
    cache.close()


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("count", [2, 60])
def test_a_later_token_stays_out_of_earlier_rows(ctx, type, count):
    """The last token's key and value change, up to 2^20 times their neighbours': the rows before it keep every bit."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(4)
    length = 150
    table, _, pages = random_table(np.random.default_rng(4), [length], 16)
    cache = ctx.kv_cache(kv_heads=2, head_dim=64, page_tokens=16, pages=pages)
    k = torch.randn(length, 2, 64, generator=gen, device="cuda")
    v = torch.randn(length, 2, 64, generator=gen, device="cuda")
    append(ctx, cache, table, [length], [length], k, 1e-2 * v)
    q = torch.randn(count, 16, 64, generator=gen, device="cuda").to(torch_type(type))
    want = attend(ctx, cache, table, [length], [count], q)
    for size in (1.0, 100.0, 1e4):
        append(ctx, cache, table, [length], [1], -k[:1].contiguous(), size * v[:1])
        out = attend(ctx, cache, table, [length], [count], q)
        assert bool((out[:-1] == want[:-1]).all()) and not bool((out[-1] == want[-1]).all())
    cache.close()


@pytest.mark.parametrize("type", list(TYPES))
def test_single_tokens_with_and_without_offsets(ctx, type):
    """The same batch either way, to the last bit."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(6)
    lengths = [4000, 3, 900, 1, 77]
    table, _, pages = random_table(np.random.default_rng(6), lengths, 16)
    cache = ctx.kv_cache(kv_heads=2, head_dim=64, page_tokens=16, pages=pages)
    n = sum(lengths)
    append(ctx, cache, table, lengths, lengths, torch.randn(n, 2, 64, generator=gen, device="cuda"),
           torch.randn(n, 2, 64, generator=gen, device="cuda"))
    q = torch.randn(5, 16, 64, generator=gen, device="cuda").to(torch_type(type))
    a, b = attend(ctx, cache, table, lengths, None, q), attend(ctx, cache, table, lengths, [1] * 5, q)
    assert bool((a == b).all())
    cache.close()
