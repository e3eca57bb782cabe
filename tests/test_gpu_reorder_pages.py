"""The beam reorder of tables whose last pages lie outside the pool, or whose
spare pages do: which page each child has, and which spare pages stay free."""
import numpy as np
import pytest

from kv_plain import Device, held

pytestmark = pytest.mark.gpu


def reorder(ctx, cache, parents, table, lengths, spare):
    import torch
    batch, beams = np.asarray(parents).shape
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")  # noqa: E731
    par, tab, n, sp = i32(parents), i32(table), i32(lengths), i32(spare)
    tab2, n2 = torch.full_like(tab, 99), torch.full_like(n, 99)
    copied = torch.full((batch * beams,), 99, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    cache.reorder_device(batch, beams, tab.shape[1], par.data_ptr(), beams, tab.data_ptr(), n.data_ptr(), sp.data_ptr(),
                         tab2.data_ptr(), n2.data_ptr(), copied.data_ptr())
    ctx.sync()
    return tab2.tolist(), n2.tolist(), copied.tolist()


@pytest.mark.parametrize("bad", [-1, 8, 2 ** 31 - 1])
def test_last_pages_outside_the_pool(ctx, bad):
    """No spare page is handed out for them, so `copied` tells the free ones; the keys there stay left out."""
    import torch
    cache = ctx.kv_cache(kv_heads=1, head_dim=32, page_tokens=16, pages=8)
    x = torch.randn(16, 1, 32, device="cuda")
    junk = torch.full((16, 1, 32), 50.0, device="cuda")
    whole, spare = Device([[0]], [16], [16]), Device([[5]], [16], [16])
    torch.cuda.synchronize()
    cache.append_device(whole.batch, x.data_ptr(), x.data_ptr())
    cache.append_device(spare.batch, junk.data_ptr(), junk.data_ptr())
    table, lengths, copied = reorder(ctx, cache, [[0, 0, 0]], [[0, bad], [1, 2], [3, 4]], [20, 20, 20], [4, 5, 6])
    assert table == [[0, bad]] * 3 and lengths == [20] * 3 and copied == [0] * 3
    q, out = torch.randn(3, 1, 32, device="cuda"), torch.zeros(3, 1, 32, device="cuda")
    q[1:] = q[0]
    dev = Device(table, lengths)
    torch.cuda.synchronize()
    cache.attention_device(dev.batch, q.data_ptr(), out.data_ptr(), 1)
    ctx.sync()
    assert bool((out[0] == out[1]).all()) and bool((out[0] == out[2]).all())
    cache.close()


def test_spare_pages_outside_the_pool(ctx):
    """Two parents, one with a good spare page for its second child and one without."""
    import torch
    cache = ctx.kv_cache(kv_heads=1, head_dim=32, page_tokens=16, pages=8)
    x = torch.randn(40, 1, 32, device="cuda")
    dev = Device([[0, 1], [2, 3]], [20, 20], [20, 20])
    torch.cuda.synchronize()
    cache.append_device(dev.batch, x.data_ptr(), x.data_ptr())
    for spare, copied in ((6, 1), (-1, 0), (8, 0)):
        table, lengths, got = reorder(ctx, cache, [[1, 1]], [[0, 1], [2, 3]], [20, 20], [7, spare])
        assert table == [[2, 3], [2, spare]] and lengths == [20, 20] and got == [0, copied]
    read = Device([[2, 6]], [20], [20])
    out = torch.zeros(20, 1, 32, device="cuda")
    torch.cuda.synchronize()
    cache.read_device(read.batch, out.data_ptr(), 0)
    ctx.sync()
    assert np.array_equal(out.cpu().numpy(), held(x[20:].cpu().numpy()).astype(np.float32))
    cache.close()
