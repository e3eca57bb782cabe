"""4-bit KV cache on the GPU: appended rows read back equal the format's
definition exactly, whatever the types, strides, pages and lengths; refusals."""
import numpy as np
import pytest

from kv_plain import TYPES, Device, held, random_table, spt, torch_type

pytestmark = pytest.mark.gpu


def rows(seed, n, heads, dim, type):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=gen, device="cuda")
    return (x * torch.exp(2.0 * torch.randn(n, heads, 1, generator=gen, device="cuda"))).to(torch_type(type))


def same(a, b):
    import torch
    return bool(torch.equal(torch.nan_to_num(a.float(), nan=1e30), torch.nan_to_num(b.float(), nan=1e30)))


def expected(x):
    import torch
    return torch.tensor(held(x.float().cpu().numpy()), device="cuda").to(x.dtype)


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("head_dim", [32, 64, 96, 128])
@pytest.mark.parametrize("page,heads,lengths,counts", [
    (16, 1, [1], None),
    (16, 3, [17, 1, 40], [17, 0, 9]),
    (48, 2, [49, 100, 16], [1, 100, 2]),
    (128, 8, [5, 129, 300], None),
], ids=str)
def test_append_reads_back_exactly(ctx, type, head_dim, page, heads, lengths, counts):
    import torch
    rng = np.random.default_rng(head_dim + page)
    table, _, pages = random_table(rng, lengths, page)
    n = len(lengths) if counts is None else sum(counts)
    k, v = rows(1, n, heads, head_dim, type), rows(2, n, heads, head_dim, type)
    dev = Device(table, lengths, counts)
    cache = ctx.kv_cache(kv_heads=heads, head_dim=head_dim, page_tokens=page, pages=pages, layers=2)
    ko, vo = torch.full_like(k, 7), torch.full_like(v, 7)
    torch.cuda.synchronize()
    cache.append_device(dev.batch, k.data_ptr(), v.data_ptr(), TYPES[type], layer=1)
    cache.read_device(dev.batch, ko.data_ptr(), vo.data_ptr(), TYPES[type], layer=1)
    ctx.sync()
    assert same(ko, expected(k)) and same(vo, expected(v))
    cache.read_device(dev.batch, ko.data_ptr(), 0, TYPES[type], layer=0)  # the other layer is still zero
    ctx.sync()
    assert not ko.any() and same(vo, expected(v))
    cache.close()


def test_special_values(ctx):
    """Zeros, subnormals, halfway quotients, equal magnitudes of both signs, infinities, NaN."""
    import torch
    rng = np.random.default_rng(3)
    x = np.zeros((12, 1, 64), np.float32)
    x[1] = 1e-42
    x[2] = rng.standard_normal(64) * 1e-7
    x[3, 0] = np.tile([8.0, -8.0, 0.5, -0.5, 1.5, 2.5, -3.5, 7.5], 8)
    x[4, 0] = np.tile([-8.0, 8.0, 0.5, -0.5, 1.5, 2.5, -3.5, 7.5], 8)
    x[5] = rng.standard_normal(64) * 1e30
    x[6], x[6, 0, 5] = 1.0, np.inf
    x[7], x[7, 0, 40] = 1.0, -np.inf
    x[8], x[8, 0, 33] = 1.0, np.nan
    x[9] = 6.2e-5 * rng.standard_normal(64)
    x[10] = -3.0
    x[11] = 65504.0 * 8
    t = torch.tensor(x, device="cuda")
    dev = Device([[0]], [12], [12])
    cache = ctx.kv_cache(kv_heads=1, head_dim=64, page_tokens=16, pages=1)
    ko, vo = torch.empty_like(t), torch.empty_like(t)
    torch.cuda.synchronize()
    cache.append_device(dev.batch, t.data_ptr(), t.data_ptr())
    cache.read_device(dev.batch, ko.data_ptr(), vo.data_ptr())
    ctx.sync()
    want = expected(t)
    assert same(ko, want) and same(vo, want)
    cache.close()


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("gap,shift", [(8, 0), (3, 0), (1, 5)])
def test_strides_and_alignment(ctx, type, gap, shift):
    """Rows of one wider array (a fused projection), starting anywhere; the gaps stay as they were."""
    import torch
    heads, dim, n = 2, 64, 21
    width = heads * dim
    wide = rows(5, n, 1, 2 * width + gap + 8, type).reshape(n, -1).contiguous()
    stride = wide.shape[1]
    size = wide.element_size()
    dev = Device([[1, 0]], [n], [n])
    cache = ctx.kv_cache(kv_heads=heads, head_dim=dim, page_tokens=16, pages=2)
    out = torch.full_like(wide, 7)
    torch.cuda.synchronize()
    cache.append_device(dev.batch, wide.data_ptr() + shift * size, wide.data_ptr() + (shift + width) * size,
                        TYPES[type], k_stride=stride, v_stride=stride)
    cache.read_device(dev.batch, out.data_ptr() + shift * size, out.data_ptr() + (shift + width) * size, TYPES[type],
                      k_stride=stride, v_stride=stride)
    ctx.sync()
    want = torch.full_like(wide, 7)
    want[:, shift:shift + 2 * width] = expected(wide[:, shift:shift + 2 * width].contiguous())
    assert same(out, want)
    cache.close()


def test_rows_outside_are_left_alone(ctx):
    """A padded batch's tail, rows before position 0, rows behind the table, and pages outside
    the pool are skipped by the device calls: nothing else in the cache or the output changes."""
    import torch
    n = 40
    k = rows(6, n, 2, 32, "f32")
    cache = ctx.kv_cache(kv_heads=2, head_dim=32, page_tokens=16, pages=4)
    # sequence 0: 20 rows but a length of 12; 1: pages -1, 9 and 2; 2: longer than its table
    table, lengths, counts = [[0, -1, -1], [-1, 9, 2], [3, -1, -1]], [12, 40, 64], [20, 12, 5]
    dev = Device(table, lengths, counts, tokens=n)
    out = torch.full_like(k, 7)
    torch.cuda.synchronize()
    cache.append_device(dev.batch, k.data_ptr(), k.data_ptr())
    cache.read_device(dev.batch, out.data_ptr(), 0)
    ctx.sync()
    want = torch.full_like(k, 7)
    want[8:20] = expected(k[8:20])    # positions 0 .. 11
    want[24:32] = expected(k[24:32])  # positions 32 .. 39 of sequence 1, on page 2
    assert same(out, want)
    # all of the pool: pages 0 and 2 hold those rows, the rest is zero
    every = Device([[0], [1], [2], [3]], [16] * 4, [16] * 4)
    pool = torch.empty(64, 2, 32, device="cuda")
    cache.read_device(every.batch, pool.data_ptr(), 0)
    ctx.sync()
    full = torch.zeros_like(pool)
    full[:12], full[32:40] = want[8:20], want[24:32]
    assert same(pool, full)
    cache.close()


def test_host_calls(ctx):
    rng = np.random.default_rng(11)
    lengths, counts = [20, 3], [4, 3]
    table, _, pages = random_table(rng, lengths, 16)
    cache = ctx.kv_cache(kv_heads=2, head_dim=64, page_tokens=16, pages=pages)
    batch = spt.KvBatch(2, 9, table.shape[1], table, lengths, np.concatenate([[0], np.cumsum(counts)]))
    k, v = (rng.standard_normal((9, 2, 64)).astype(np.float32) for _ in range(2))
    cache.append(batch, k, v)
    ko, vo = cache.read(batch)
    assert np.array_equal(ko[:7], held(k[:7]).astype(np.float32)) and not ko[7:].any()
    assert np.array_equal(vo[:7], held(v[:7]).astype(np.float32))
    cancel = np.ones(1, np.int32)
    with pytest.raises(spt.CanceledError):
        cache.append(batch, k, v, cancel=cancel)
    cache.close()


def test_limits_and_overlaps(ctx):
    """Counts beyond what a launch numbers, strides beyond 64 bits, outputs on top of one another; a
    buffer whose rows are keys and values in turn is none of these."""
    import torch
    cache = ctx.kv_cache(kv_heads=2, head_dim=64, page_tokens=16, pages=3)
    table, lengths = np.array([[0, 1]], np.int32), np.array([17], np.int32)
    rng = np.random.default_rng(3)
    x = rng.normal(size=(17, 2, 64)).astype(np.float32)
    cache.append(spt.KvBatch(1, 17, 2, table, lengths, [0, 17]), x, -x)
    dev = Device(table, [17], [17])
    p = torch.zeros(17, 256, device="cuda")

    def refused(status, call):
        with pytest.raises(spt.SptError) as e:
            call()
        assert e.value.status == status, e.value

    d, n = p.data_ptr(), 2 ** 31 - 1
    big = lambda **c: spt.KvBatch(**{**dict(sequences=1, tokens=17, max_pages=2, table=d, lengths=d, offsets=d), **c})  # noqa: E731
    for call in (cache.append_device, cache.read_device):
        refused(spt.ERR_UNSUPPORTED, lambda: call(big(sequences=n), d, d))
        refused(spt.ERR_UNSUPPORTED, lambda: call(big(sequences=2 ** 21, max_pages=2 ** 20), d, d))
        refused(spt.ERR_DIMENSIONS, lambda: call(big(), d, d, k_stride=2 ** 60))
        refused(spt.ERR_DIMENSIONS, lambda: call(big(tokens=n), d, d, v_stride=2 ** 40))
    refused(spt.ERR_UNSUPPORTED, lambda: cache.attention_device(big(tokens=n), d, d, heads=4))
    refused(spt.ERR_OVERLAP, lambda: cache.read_device(dev.batch, d, d))
    refused(spt.ERR_OVERLAP, lambda: cache.read_device(dev.batch, d, d + 4 * 64, k_stride=256, v_stride=256))
    refused(spt.ERR_OVERLAP, lambda: cache.read_device(dev.batch, d, d + 4 * 256, k_stride=128, v_stride=256))
    refused(spt.ERR_UNSUPPORTED, lambda: ctx.validate_kv(kv_heads=64, head_dim=128, page_tokens=65536, pages=2, layers=128))
    torch.cuda.synchronize()
    cache.read_device(dev.batch, d, d + 4 * 128, k_stride=256, v_stride=256)
    ctx.sync()
    got = p.cpu().numpy().reshape(17, 2, 2, 64)
    assert np.array_equal(got[:, 0], held(x).astype(np.float32)) and np.array_equal(got[:, 1], held(-x).astype(np.float32))
    cache.close()


def test_calls_refused(ctx):
    import torch
    cache = ctx.kv_cache(kv_heads=2, head_dim=64, page_tokens=16, pages=3)
    x = np.zeros((2, 2, 64), np.float32)
    d = torch.zeros(1024, device="cuda")
    table, lengths = np.array([[0, 1], [2, -1]], np.int32), np.array([20, 3], np.int32)
    good = lambda **c: spt.KvBatch(**{**dict(sequences=2, tokens=2, max_pages=2, table=table, lengths=lengths), **c})  # noqa: E731
    cache.append(good(), x, x)

    def refused(status, call):
        with pytest.raises(spt.SptError) as e:
            call()
        assert e.value.status == status, e.value

    dim, null, unsup = spt.ERR_DIMENSIONS, spt.ERR_NULL_ARG, spt.ERR_UNSUPPORTED
    refused(dim, lambda: cache.append(good(), x, x, layer=1))
    refused(dim, lambda: cache.append(good(), x, x, layer=-1))
    refused(dim, lambda: cache.append(good(), x[:1], x))
    refused(dim, lambda: cache.append(good(tokens=-1), x, x))
    refused(dim, lambda: cache.append(good(lengths=[33, 3]), x, x))        # beyond its table
    refused(dim, lambda: cache.append(good(lengths=[20, 17]), x, x))       # page -1
    refused(dim, lambda: cache.append(good(lengths=[20, 0]), x, x))        # a new row, no length
    refused(dim, lambda: cache.append(good(table=[[0, 3], [2, -1]]), x, x))
    refused(dim, lambda: cache.append(good(offsets=[0, 2, 1]), x, x))
    refused(dim, lambda: cache.append(good(offsets=[0, 1, 3]), x, x))
    refused(dim, lambda: cache.append(good(offsets=[-1, 1, 2]), x, x))
    refused(null, lambda: cache.append(good(lengths=None), x, x))
    refused(unsup, lambda: cache.append_device(good(table=d.data_ptr(), lengths=d.data_ptr()), d.data_ptr(),
                                               d.data_ptr(), type=2))
    refused(dim, lambda: cache.append_device(good(table=d.data_ptr(), lengths=d.data_ptr()), d.data_ptr(),
                                             d.data_ptr(), k_stride=100))
    refused(dim, lambda: cache.append_device(good(table=d.data_ptr(), lengths=d.data_ptr()), d.data_ptr() + 2,
                                             d.data_ptr()))
    refused(dim, lambda: cache.append_device(good(table=d.data_ptr() + 2, lengths=d.data_ptr()), d.data_ptr(),
                                             d.data_ptr()))
    refused(null, lambda: cache.append_device(good(table=d.data_ptr(), lengths=d.data_ptr()), 0, d.data_ptr()))
    other = spt.Context(0)
    cache.ctx, mine = other, cache.ctx
    refused(dim, lambda: cache.append(good(), x, x))
    cache.ctx = mine
    other.close()
    cache.close()
