"""Attention's bounded waits when they run out: the call is reported, nothing is
left behind, and no other call is touched."""
import contextlib

import pytest

from kv_plain import Device, spt
from test_gpu_attention import check, filled

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def short_waits(ctx):
    """Waits of about a tenth of a millisecond."""
    old = ctx.get_option(spt.OPT_WAIT_LIMIT)
    ctx.set_option(spt.OPT_WAIT_LIMIT, 18)
    try:
        yield
    finally:
        ctx.set_option(spt.OPT_WAIT_LIMIT, old)
        ctx.set_option(spt.OPT_FAULT_STAGE, -1)


def reported(ctx):
    with pytest.raises(spt.SptError) as e:
        ctx.sync()
    assert e.value.status == spt.ERR_TIMEOUT and "attention" in str(e.value)


@pytest.mark.parametrize("step", [0, 1, 2])
@pytest.mark.parametrize("dim,counts", [(64, None), (128, None), (64, [2, 1, 1])], ids=str)
def test_a_step_that_never_comes(ctx, dim, counts, step):
    """Single tokens: a warp that waits in vain takes its remaining copies in and leaves with the others; the
    counters of the shares end at zero, so the next calls are right."""
    import torch
    lengths = [400000, 40, 5000]  # of which the first warp has three steps at least
    cache, table, held = filled(ctx, 21, lengths, 1, dim, 64)
    n = 3 if counts is None else sum(counts)
    q, out = torch.randn(n, 8, dim, device="cuda"), torch.zeros(n, 8, dim, device="cuda")
    dev = Device(table, lengths, counts)
    torch.cuda.synchronize()
    with short_waits(ctx):
        ctx.set_option(spt.OPT_FAULT_STAGE, step)
        cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 8, scale=0.125)
        reported(ctx)
    for _ in range(2):
        check(ctx, cache, table, held, lengths, counts, 8, scale=0.125, q=q)
    cache.close()


def test_single_tokens_behind_a_call_that_gave_up(ctx):
    """The error that an earlier call left for the next synchronisation does not end this one's waits."""
    import torch
    lengths = [30000, 700]
    cache, table, held = filled(ctx, 22, lengths, 2, 64, 16)
    q, out = torch.randn(364, 16, 64, device="cuda"), torch.zeros(364, 16, 64, device="cuda")
    many, one = Device(table, lengths, [300, 64]), Device(table, lengths)
    want = check(ctx, cache, table, held, lengths, None, 16, scale=0.125, q=q[:2].contiguous())
    got = torch.zeros_like(want)
    torch.cuda.synchronize()
    with short_waits(ctx):
        ctx.set_option(spt.OPT_FAULT_STAGE, 2)
        cache.attention_device(many.batch, q.data_ptr(), out.data_ptr(), 16, scale=0.125)
        ctx.set_option(spt.OPT_FAULT_STAGE, -1)
        cache.attention_device(one.batch, q.data_ptr(), got.data_ptr(), 16, scale=0.125)
        reported(ctx)
    assert bool((got == want).all())
    cache.close()


def test_many_rows_behind_a_call_that_gave_up(ctx):
    """The same for chunks of rows, of which every CTA waits for copies and for its other warps."""
    import torch
    lengths, counts = [3000, 700], [300, 64]
    cache, table, held = filled(ctx, 23, lengths, 2, 64, 16)
    q, out = torch.randn(364, 16, 64, device="cuda"), torch.zeros(364, 16, 64, device="cuda")
    dev = Device(table, lengths, counts)
    want = check(ctx, cache, table, held, lengths, counts, 16, scale=0.125, q=q)
    got = torch.zeros_like(want)
    torch.cuda.synchronize()
    with short_waits(ctx):
        ctx.set_option(spt.OPT_FAULT_STAGE, 2)
        cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 16, scale=0.125)
        ctx.set_option(spt.OPT_FAULT_STAGE, -1)
        cache.attention_device(dev.batch, q.data_ptr(), got.data_ptr(), 16, scale=0.125)
        reported(ctx)
    assert bool((got == want).all())
    cache.close()
