"""Attention over the 4-bit cache against 64-bit arithmetic on what the cache
holds, within the tolerance that the kernel's roundings add up to."""
import numpy as np
import pytest

from kv_plain import TYPES, Device, attention, attention_tolerance, random_table, spt, torch_type

pytestmark = pytest.mark.gpu


def filled(ctx, seed, lengths, heads, dim, page, k_scale=1.0, v_scale=1.0):
    """A cache of random tokens, its table, and what it holds [sequence] in 64 bits."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    table, spare, pages = random_table(rng, lengths, page)
    n = int(sum(lengths))
    k = torch.randn(max(n, 1), heads, dim, generator=gen, device="cuda") * k_scale
    v = torch.randn(max(n, 1), heads, dim, generator=gen, device="cuda") * v_scale
    cache = ctx.kv_cache(kv_heads=heads, head_dim=dim, page_tokens=page, pages=pages)
    dev = Device(table, lengths, lengths)
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    torch.cuda.synchronize()
    cache.append_device(dev.batch, k.data_ptr(), v.data_ptr())
    cache.read_device(dev.batch, ko.data_ptr(), vo.data_ptr())
    ctx.sync()
    at = np.concatenate([[0], np.cumsum(lengths)])
    held = [(ko[a:b].double(), vo[a:b].double()) for a, b in zip(at[:-1], at[1:])]
    return cache, table, held


def check(ctx, cache, table, held, lengths, counts, heads, type="f32", window=0, sinks=None, seed=9, tail=0,
          q_scale=1.0, scale=None, q=None):
    import torch
    dim = cache.head_dim
    scale = dim ** -0.5 if scale is None else scale
    n = int(sum(counts)) if counts is not None else len(lengths)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if q is None:
        q = (torch.randn(n + tail, heads, dim, generator=gen, device="cuda") * q_scale).to(torch_type(type))
    out = torch.full_like(q, 7)
    dev = Device(table, lengths, counts, tokens=n + tail)
    torch.cuda.synchronize()
    cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), heads, TYPES[type], scale=scale, window=window,
                           sinks_ptr=0 if sinks is None else sinks.data_ptr())
    ctx.sync()
    assert (out[n:] == 7).all()
    at = 0
    for b, (length, (keys, values)) in enumerate(zip(lengths, held)):
        c = 1 if counts is None else counts[b]
        rows = q[at:at + c].double()
        if c:
            want = attention(rows, keys[:length], values[:length], length - c, scale, window, sinks)
            tol = attention_tolerance(*want, length, type)
            off = (out[at:at + c].double() - want[0]).abs()
            assert bool((off <= tol).all()), (b, length, float((off / tol).max()))
        at += c
    return out


EDGES = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 513, 1025]


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("dim,kv,group,page", [(64, 8, 8, 64), (128, 2, 4, 16), (32, 1, 3, 48), (96, 2, 1, 32),
                                              (64, 1, 13, 16), (128, 1, 16, 128)])
def test_decode(ctx, type, dim, kv, group, page):
    """One new token a sequence, at the lengths around tiles, steps and pages."""
    import torch
    cache, table, held = filled(ctx, dim + kv, EDGES, kv, dim, page)
    sinks = torch.randn(kv * group, device="cuda")
    check(ctx, cache, table, held, EDGES, None, kv * group, type, sinks=sinks)
    check(ctx, cache, table, held, EDGES, None, kv * group, type, window=37)
    cache.close()


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("dim,kv,group,page,window", [(64, 4, 8, 64, 0), (64, 2, 5, 16, 33), (128, 2, 4, 32, 0),
                                                     (32, 1, 1, 16, 1), (96, 1, 6, 48, 100)])
def test_chunks(ctx, type, dim, kv, group, page, window):
    """Ragged chunks: whole prompts, tails of longer contexts, single tokens, sequences with none; rows behind the last."""
    import torch
    lengths = [70, 1, 300, 16, 0, 129, 33, 500]
    counts = [70, 1, 17, 0, 0, 128, 1, 65]
    cache, table, held = filled(ctx, dim + page, lengths, kv, dim, page)
    sinks = torch.randn(kv * group, device="cuda")
    check(ctx, cache, table, held, lengths, counts, kv * group, type, window=window, sinks=sinks, tail=3)
    cache.close()


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_long_context(ctx, type):
    """One long sequence, split over all SMs, beside short ones."""
    lengths = [40001, 5, 3000]
    cache, table, held = filled(ctx, 1, lengths, 2, 64, 128)
    a = check(ctx, cache, table, held, lengths, None, 16, type)
    b = check(ctx, cache, table, held, lengths, None, 16, type)
    assert bool((a == b).all())  # the order in which CTAs arrive changes nothing
    check(ctx, cache, table, held, lengths, [4, 1, 2], 16, type, window=5000)
    cache.close()


@pytest.mark.parametrize("k_scale,v_scale,q_scale", [(1e-3, 1e-4, 1e-3), (30.0, 1e3, 1.0), (1e-30, 3e4, 1e30),
                                                     (6.0, 1e-6, 6.0)])
def test_magnitudes(ctx, k_scale, v_scale, q_scale):
    """Small and large keys, values and queries, and sharp softmaxes."""
    lengths = [7, 260, 1100]
    cache, table, held = filled(ctx, 2, lengths, 2, 64, 16, k_scale, v_scale)
    check(ctx, cache, table, held, lengths, None, 16, q_scale=q_scale)
    check(ctx, cache, table, held, lengths, [7, 5, 1], 16, "bf16", q_scale=q_scale)
    cache.close()


def test_values_of_very_different_sizes(ctx):
    """Tokens whose values are 2^20 larger than their neighbours', early or late."""
    import torch
    length = 400
    gen = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randn(length, 1, 64, generator=gen, device="cuda")
    v = torch.randn(length, 1, 64, generator=gen, device="cuda")
    v[3] *= 2.0 ** 10
    v[390] *= 2.0 ** 13
    v[100:200] *= 2.0 ** -7
    table = np.arange(7, dtype=np.int32)[None, :]
    cache = ctx.kv_cache(kv_heads=1, head_dim=64, page_tokens=64, pages=7)
    dev = Device(table, [length], [length])
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    torch.cuda.synchronize()
    cache.append_device(dev.batch, k.data_ptr(), v.data_ptr())
    cache.read_device(dev.batch, ko.data_ptr(), vo.data_ptr())
    ctx.sync()
    check(ctx, cache, table, [(ko.double(), vo.double())], [length], [300], 8)
    cache.close()


def test_sinks(ctx):
    """A sink far above, far below and at -inf; rows without keys are 0 with and without one."""
    import torch
    lengths = [50, 3]
    cache, table, held = filled(ctx, 3, lengths, 1, 64, 16)
    sinks = torch.tensor([100.0, -100.0, float("-inf"), 0.0], device="cuda")
    check(ctx, cache, table, held, lengths, None, 4, sinks=sinks)
    # more new rows than the length has places: the first have no position
    q = torch.randn(8, 4, 64, device="cuda")
    for s in (0, sinks.data_ptr()):
        out = torch.full_like(q, 7)
        dev = Device(table, [50, 3], [0, 8])
        torch.cuda.synchronize()
        cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 4, scale=0.125, sinks_ptr=s)
        ctx.sync()
        assert not out[:5].any() and bool(torch.isfinite(out).all()) and bool(out[5:, 3].any(-1).all())
    cache.close()


def test_masked_places_hold_anything(ctx):
    """NaN keys and values behind the length, before the window, and on pages of no sequence change nothing."""
    import torch
    cache, table, held = filled(ctx, 4, [100, 64], 2, 64, 16)
    junk = torch.full((100, 2, 64), float("nan"), device="cuda")
    want = check(ctx, cache, table, held, [60, 40], None, 16)
    windowed = check(ctx, cache, table, held, [60, 40], None, 16, window=20)
    # overwrite positions 60 .. 99 and 40 .. 63 with NaN
    dev = Device(table, [100, 64], [40, 24])
    torch.cuda.synchronize()
    cache.append_device(dev.batch, junk.data_ptr(), junk.data_ptr())
    ctx.sync()
    assert bool((check(ctx, cache, table, held, [60, 40], None, 16) == want).all())
    # and positions 0 .. 39 / 0 .. 19, which the windows leave out
    dev = Device(table, [40, 20], [40, 20])
    torch.cuda.synchronize()
    cache.append_device(dev.batch, junk.data_ptr(), junk.data_ptr())
    ctx.sync()
    clean = [(k.clone(), v.clone()) for k, v in held]
    assert bool((check(ctx, cache, table, clean, [60, 40], None, 16, window=20) == windowed).all())
    # without the window the NaNs are in sight
    q = torch.randn(2, 16, 64, device="cuda")
    out = torch.zeros_like(q)
    dev = Device(table, [60, 40])
    torch.cuda.synchronize()
    cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 16, scale=0.125)
    ctx.sync()
    assert bool(torch.isnan(out).all())
    cache.close()


@pytest.mark.parametrize("type", list(TYPES))
def test_masked_places_of_chunks_hold_anything(ctx, type):
    """The same for chunks of rows: NaNs behind a row's position or before its window stay out
    of it, and one in sight of some rows reaches those alone, in the value blocks that hold it."""
    import torch
    lengths, counts = [300, 200], [90, 40]
    cache, table, held = filled(ctx, 15, lengths, 2, 64, 16)
    gen = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(130, 16, 64, generator=gen, device="cuda").to(torch_type(type))
    want = check(ctx, cache, table, held, lengths, counts, 16, type, window=50, q=q)
    # positions 0 .. 150 of sequence 0 (its rows see 161 ..) and 0 .. 99 of sequence 1 (111 ..)
    junk = torch.full((251, 2, 64), float("nan"), device="cuda")
    dev = Device(table, [151, 100], [151, 100])
    torch.cuda.synchronize()
    cache.append_device(dev.batch, junk.data_ptr(), junk.data_ptr())
    ctx.sync()
    out = torch.zeros_like(q)
    dev = Device(table, lengths, counts)
    torch.cuda.synchronize()

    def attend():
        cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 16, TYPES[type], scale=0.125, window=50)
        ctx.sync()

    attend()
    assert bool((out == want).all())
    # a value block with a NaN at position 250 of sequence 0: head 1, dims 32 .. 63
    k, v = (x.float()[250:251].contiguous() for x in held[0])
    v = v.clone()
    v[0, 1, 40] = float("nan")
    one = Device(table[:1], [251], [1])
    torch.cuda.synchronize()
    cache.append_device(one.batch, k.data_ptr(), v.data_ptr())
    ctx.sync()
    attend()
    hit = torch.zeros(130, 16, 64, dtype=torch.bool, device="cuda")
    first = 250 - 210  # row of position 250; windows of 50 see it from there to position 299
    hit[first:90, 8:, 32:] = True
    assert bool(torch.isnan(out[hit]).all()) and bool((out[~hit] == want[~hit]).all())
    # a key with one: every value of the rows that see it
    k[0, 0, 3] = float("nan")
    torch.cuda.synchronize()
    cache.append_device(one.batch, k.data_ptr(), k.data_ptr())
    ctx.sync()
    attend()
    assert bool(torch.isnan(out[first:90, :8]).all()) and bool((out[:first] == want[:first]).all())
    assert bool((out[90:] == want[90:]).all())
    cache.close()


def test_waits_that_run_out(ctx):
    """A tile that is never loaded: the waits for it give up, the call is reported as timed out, and
    the next is right again."""
    import torch
    lengths, counts = [3000, 500], [300, 64]
    cache, table, held = filled(ctx, 16, lengths, 2, 64, 16)
    q = torch.randn(364, 16, 64, device="cuda")
    out = torch.zeros_like(q)
    dev = Device(table, lengths, counts)
    torch.cuda.synchronize()
    old = ctx.get_option(spt.OPT_WAIT_LIMIT)
    ctx.set_option(spt.OPT_WAIT_LIMIT, 18)
    ctx.set_option(spt.OPT_FAULT_STAGE, 2)
    try:
        cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 16, scale=0.125)
        with pytest.raises(spt.SptError) as e:
            ctx.sync()
        assert e.value.status == spt.ERR_TIMEOUT
    finally:
        ctx.set_option(spt.OPT_WAIT_LIMIT, old)
        ctx.set_option(spt.OPT_FAULT_STAGE, -1)
    for _ in range(2):
        check(ctx, cache, table, held, lengths, counts, 16, q=q)
    cache.close()


def test_bad_query_rows_stay_alone(ctx):
    """A NaN or an infinity in one row of q gives NaNs there and touches no other row."""
    import torch
    lengths, counts = [90, 30], [20, 1]
    cache, table, held = filled(ctx, 6, lengths, 2, 64, 16)
    for type in TYPES:
        q = torch.randn(21, 16, 64, device="cuda").to(torch_type(type))
        good = check(ctx, cache, table, held, lengths, counts, 16, type, q=q)
        bad = q.clone()
        bad[4, 3, 10], bad[7, 9, 0], bad[20, 15, 63] = float("nan"), float("inf"), float("-inf")
        out = torch.zeros_like(q)
        dev = Device(table, lengths, counts)
        torch.cuda.synchronize()
        cache.attention_device(dev.batch, bad.data_ptr(), out.data_ptr(), 16, TYPES[type], scale=0.125)
        ctx.sync()
        hit = torch.zeros(21, 16, dtype=torch.bool, device="cuda")
        hit[4, 3] = hit[7, 9] = hit[20, 15] = True
        assert bool(torch.isnan(out[hit]).all()) and bool((out[~hit] == good[~hit]).all()), type
    cache.close()


def test_keys_on_bad_pages_are_left_out(ctx):
    """Device tables with pages outside the pool, or too short for the length: those keys do not count."""
    import torch
    cache, table, held = filled(ctx, 7, [64], 1, 64, 16)
    q = torch.randn(1, 8, 64, device="cuda")
    keys, values = held[0]
    for bad, keep in (([[table[0, 0], -1, table[0, 2], 1 << 30]], [0, 2]), ([table[0, :2]], [0, 1])):
        out = torch.zeros_like(q)
        dev = Device(bad, [64])
        torch.cuda.synchronize()
        cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 8, scale=0.125)
        ctx.sync()
        seen = torch.cat([torch.arange(16 * i, 16 * i + 16) for i in keep]).cuda()
        want = attention(q.double(), keys[seen], values[seen], 31, 0.125)
        tol = attention_tolerance(*want, 64, "f32")
        assert bool(((out.double() - want[0]).abs() <= tol).all())
    cache.close()


@pytest.mark.parametrize("type", list(TYPES))
def test_strides(ctx, type):
    """q as a slice of a fused projection at any alignment, out with gaps that stay as they were."""
    import torch
    lengths, counts, heads = [40, 7], [5, 2], 8
    cache, table, held = filled(ctx, 8, lengths, 1, 64, 16)
    width = heads * 64
    wide = torch.randn(7, width + 131, device="cuda").to(torch_type(type))
    out = torch.full((7, width + 5), 7.0, device="cuda").to(torch_type(type))
    q = wide[:, 3:3 + width].reshape(7, heads, 64).contiguous()
    want = check(ctx, cache, table, held, lengths, counts, heads, type, q=q)
    dev = Device(table, lengths, counts)
    torch.cuda.synchronize()
    cache.attention_device(dev.batch, wide.data_ptr() + 3 * wide.element_size(), out.data_ptr() + out.element_size(),
                           heads, TYPES[type], scale=0.125, q_stride=width + 131, out_stride=width + 5)
    ctx.sync()
    assert bool((out[:, 1:1 + width].reshape(7, heads, 64) == want).all())
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 1 + width:] == 7).all())
    cache.close()


def test_many_sequences(ctx):
    """More sequences than a CTA has threads, most of them short, some without rows."""
    rng = np.random.default_rng(12)
    lengths = [int(n) for n in rng.integers(1, 40, 700)]
    counts = [int(min(n, c)) for n, c in zip(lengths, rng.integers(0, 3, 700))]
    cache, table, held = filled(ctx, 12, lengths, 1, 32, 16)
    check(ctx, cache, table, held, lengths, counts, 4)
    check(ctx, cache, table, held, lengths, None, 4)
    cache.close()


def test_long_pool_offsets(ctx):
    """Pages whose bytes lie beyond 2^32 of the pool's start."""
    import torch
    pages = 7600  # x 1024 tokens x 8 heads x 72 bytes = 4.48 GB
    cache = ctx.kv_cache(kv_heads=8, head_dim=64, page_tokens=1024, pages=pages)
    assert cache.nbytes > 1 << 32
    table, n = [[pages - 1, 3]], 1100
    k, v = torch.randn(n, 8, 64, device="cuda"), torch.randn(n, 8, 64, device="cuda")
    dev = Device(table, [n], [n])
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    torch.cuda.synchronize()
    cache.append_device(dev.batch, k.data_ptr(), v.data_ptr())
    cache.read_device(dev.batch, ko.data_ptr(), vo.data_ptr())
    ctx.sync()
    assert bool(((ko - k).abs() <= k.abs().amax(-1, keepdim=True) / 7).all())
    check(ctx, cache, table, [(ko.double(), vo.double())], [n], [2], 64)
    cache.close()


def test_host_call_and_refusals(ctx):
    rng = np.random.default_rng(13)
    lengths = np.array([20, 3], np.int32)
    table, _, pages = random_table(rng, lengths, 16)
    cache = ctx.kv_cache(kv_heads=2, head_dim=64, page_tokens=16, pages=pages)
    every = spt.KvBatch(2, 23, table.shape[1], table, lengths, [0, 20, 23])
    k, v = (rng.standard_normal((23, 2, 64)).astype(np.float32) for _ in range(2))
    cache.append(every, k, v)
    ko, vo = cache.read(every)
    import torch
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    sinks = rng.standard_normal(4).astype(np.float32)
    batch = spt.KvBatch(2, 3, table.shape[1], table, lengths)
    out = np.full((3, 4, 64), 7, np.float32)
    cache.attention(batch, q, 4, scale=0.125, sinks=sinks, out=out)
    assert (out[2] == 7).all()
    for b, (a, e) in enumerate(((0, 20), (20, 23))):
        want = attention(torch.tensor(q[b:b + 1]).double(), torch.tensor(ko[a:e]).double(),
                         torch.tensor(vo[a:e]).double(), e - a - 1, 0.125, 0, torch.tensor(sinks))
        tol = attention_tolerance(*want, e - a, "f32")
        assert bool(((torch.tensor(out[b:b + 1]).double() - want[0]).abs() <= tol).all())

    def refused(status, call):
        with pytest.raises(spt.SptError) as e:
            call()
        assert e.value.status == status, e.value

    dim = spt.ERR_DIMENSIONS
    refused(dim, lambda: cache.attention(batch, q[:, :3], 3, scale=0.125))          # heads on key heads
    refused(dim, lambda: cache.attention(batch, q, 4, scale=0.0))
    refused(dim, lambda: cache.attention(batch, q, 4, scale=float("nan")))
    refused(dim, lambda: cache.attention(batch, q, 4, scale=0.125, window=-1))
    refused(dim, lambda: cache.attention(batch, q[:2], 4, scale=0.125))
    refused(dim, lambda: cache.attention(batch, q, 4, scale=0.125, layer=1))
    refused(spt.ERR_OVERLAP, lambda: cache.attention(batch, q, 4, scale=0.125, out=q))
    refused(dim, lambda: cache.attention(spt.KvBatch(2, 3, 2, table, [20, 40]), q, 4, scale=0.125))
    with pytest.raises(spt.CanceledError):
        cache.attention(batch, q, 4, scale=0.125, cancel=np.ones(1, np.int32))
    d = torch.zeros(4096, device="cuda")
    dev = Device(table, lengths)
    refused(spt.ERR_OVERLAP, lambda: cache.attention_device(dev.batch, d.data_ptr(), d.data_ptr() + 256, 4, scale=1.0))
    refused(dim, lambda: cache.attention_device(dev.batch, d.data_ptr() + 1, d.data_ptr() + 8192, 4, scale=1.0))
    cache.close()


def test_captured_and_replayed(ctx):
    """Append and attention in a graph, replayed on new rows and lengths in the same buffers."""
    import torch
    lengths = [300, 37]
    cache, table, held = filled(ctx, 14, lengths, 2, 64, 16)
    table = np.concatenate([table, np.full((2, 1), -1, np.int32)], 1)
    stream = torch.cuda.Stream()
    dev = Device(table, [301, 38])
    k, v = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    q, out = torch.zeros(2, 16, 64, device="cuda"), torch.zeros(2, 16, 64, device="cuda")
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            cache.append_device(dev.batch, k.data_ptr(), v.data_ptr())
            cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 16, scale=0.125)
        for step in range(3):
            gen = torch.Generator(device="cuda").manual_seed(step)
            for x in (k, v, q):
                x.copy_(torch.randn(x.shape, generator=gen, device="cuda"))
            dev.lengths.copy_(torch.tensor([301 + step, 38 + step]))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            every = Device(table, [301 + step, 38 + step], [301 + step, 38 + step])
            ko = torch.empty(339 + 2 * step, 2, 64, device="cuda")
            vo = torch.empty_like(ko)
            torch.cuda.synchronize()
            cache.read_device(every.batch, ko.data_ptr(), vo.data_ptr())
            ctx.sync()
            for b, (a, e) in enumerate(((0, 301 + step), (301 + step, 339 + 2 * step))):
                want = attention(q[b:b + 1].double(), ko[a:e].double(), vo[a:e].double(), e - a - 1, 0.125)
                tol = attention_tolerance(*want, e - a, "f32")
                assert bool(((out[b:b + 1].double() - want[0]).abs() <= tol).all()), (step, b)
    finally:
        ctx.set_stream(0)
    cache.close()
