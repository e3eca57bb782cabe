"""The Python mirror's host arrays without a GPU: what does not fit is refused
before an address of it is taken."""
import numpy as np
import pytest

from kv_plain import spt


@pytest.fixture
def cache(host_ctx):
    """A cache without a handle: a call that gets past the mirror's own checks is refused as a null argument."""
    c = spt.KvCache.__new__(spt.KvCache)
    c.ctx, c.kv_heads, c.head_dim, c.page_tokens, c.pages, c.layers, c._h = host_ctx, 2, 64, 16, 4, 1, None
    return c


def refused(call, status=None):
    with pytest.raises(spt.SptError) as e:
        call()
    assert e.value.status == (spt.ERR_DIMENSIONS if status is None else status), e.value


TABLE, LENGTHS = np.array([[0, 1], [2, 3]], np.int32), np.array([20, 3], np.int32)


@pytest.mark.parametrize("change", [dict(table=TABLE[:1]), dict(table=[[0], [1]]), dict(lengths=[20]), dict(offsets=[0, 1]),
                                    dict(sequences=3), dict(max_pages=3), dict(lengths=[])], ids=str)
def test_batches_of_too_small_arrays(change):
    good = dict(sequences=2, tokens=2, max_pages=2, table=TABLE, lengths=LENGTHS, offsets=[0, 1, 2])
    spt.KvBatch(**good)
    refused(lambda: spt.KvBatch(**{**good, **change}))


def test_host_arrays_and_device_addresses(cache):
    """Neither kind of call takes the other's."""
    x, n = np.zeros((2, 2, 64), np.float32), spt.ERR_NULL_ARG
    host = spt.KvBatch(2, 2, 2, TABLE, LENGTHS)
    refused(lambda: cache.append(host, x, x), n)
    refused(lambda: cache.read(host), n)
    refused(lambda: cache.attention(host, x, 2), n)
    refused(lambda: cache.append_device(host, 4096, 8192))
    refused(lambda: cache.read_device(host, 4096, 8192))
    refused(lambda: cache.attention_device(host, 4096, 8192, 2))
    for address in (4096, np.int64(4096)):
        device = spt.KvBatch(2, 2, 2, address, address)
        refused(lambda: cache.append(device, x, x))
        refused(lambda: cache.read(device))
        refused(lambda: cache.attention(device, x, 2))
        refused(lambda: cache.append_device(device, 4096, 8192), n)
    mixed = spt.KvBatch(2, 2, 2, TABLE, 4096)
    refused(lambda: cache.append(mixed, x, x))
    refused(lambda: cache.append_device(mixed, 4096, 8192))


def test_attention_outputs_and_sinks(cache):
    q, batch = np.zeros((2, 4, 64), np.float32), spt.KvBatch(2, 2, 2, TABLE, LENGTHS)
    locked = np.zeros_like(q)
    locked.flags.writeable = False
    for out in (np.zeros((2, 4, 64)), np.zeros((64, 4, 2), np.float32).T, locked, q.tolist()):
        refused(lambda: cache.attention(batch, q, 4, out=out))
    for sinks in (np.zeros(3), np.zeros(5), np.zeros(0)):
        refused(lambda: cache.attention(batch, q, 4, sinks=sinks))
    refused(lambda: cache.attention(batch, q, 4, sinks=np.zeros(4), out=np.zeros_like(q)), spt.ERR_NULL_ARG)


def test_reorder_arrays(cache):
    good = dict(parents=np.array([[1, 1]]), table=TABLE, lengths=LENGTHS, spare=np.array([1, 2]))
    refused(lambda: cache.reorder(**good), spt.ERR_NULL_ARG)
    for change in (dict(table=TABLE[:1]), dict(table=TABLE.ravel()), dict(lengths=LENGTHS[:1]), dict(spare=[1]),
                   dict(parents=np.array([[0, 0, 1]])), dict(parents=np.array([[0, 1], [0, 1]]))):
        refused(lambda: cache.reorder(**{**good, **change}))
