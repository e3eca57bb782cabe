"""4-bit KV cache, attention and beam search without a GPU: what the calls
refuse, and the cache's layout as arithmetic."""
import numpy as np
import pytest

from kv_plain import held, spt


@pytest.mark.parametrize("change,status", [
    (dict(layers=0), spt.ERR_DIMENSIONS),
    (dict(kv_heads=0), spt.ERR_DIMENSIONS),
    (dict(pages=0), spt.ERR_DIMENSIONS),
    (dict(head_dim=-64), spt.ERR_DIMENSIONS),
    (dict(page_tokens=-16), spt.ERR_DIMENSIONS),
    (dict(head_dim=80), spt.ERR_UNSUPPORTED),
    (dict(head_dim=160), spt.ERR_UNSUPPORTED),
    (dict(page_tokens=24), spt.ERR_UNSUPPORTED),
    (dict(page_tokens=1 << 17), spt.ERR_UNSUPPORTED),
    (dict(pages=1 << 31), spt.ERR_UNSUPPORTED),
    (dict(kv_heads=5000), spt.ERR_UNSUPPORTED),
    (dict(pages=(1 << 31) - 1, layers=65536, kv_heads=4096, page_tokens=65536), spt.ERR_DIMENSIONS),
], ids=str)
def test_cache_configurations_refused(host_ctx, change, status):
    good = dict(kv_heads=8, head_dim=64, page_tokens=64, pages=16, layers=1)
    host_ctx.validate_kv(**good)
    with pytest.raises(spt.SptError) as e:
        host_ctx.validate_kv(**{**good, **change})
    assert e.value.status == status


@pytest.mark.parametrize("change,status", [
    (dict(batch=0), spt.ERR_DIMENSIONS),
    (dict(beams=0), spt.ERR_DIMENSIONS),
    (dict(vocab=0), spt.ERR_DIMENSIONS),
    (dict(keep=0), spt.ERR_DIMENSIONS),
    (dict(beams=65), spt.ERR_UNSUPPORTED),
    (dict(keep=65), spt.ERR_UNSUPPORTED),
    (dict(batch=20000), spt.ERR_UNSUPPORTED),
    (dict(vocab=1 << 31), spt.ERR_UNSUPPORTED),
], ids=str)
def test_beam_configurations_refused(host_ctx, change, status):
    good = dict(batch=2, beams=4, vocab=1000, keep=8)
    host_ctx.validate_beam(**good)
    with pytest.raises(spt.SptError) as e:
        host_ctx.validate_beam(**{**good, **change})
    assert e.value.status == status


def test_no_device_no_cache(host_ctx):
    for make in (lambda: host_ctx.kv_cache(kv_heads=1, head_dim=32, page_tokens=16, pages=1),
                 lambda: host_ctx.beam(1, 1, 10, 1)):
        with pytest.raises(spt.SptError) as e:
            make()
        assert e.value.status == spt.ERR_NO_DEVICE


def word(nb, b, lane, h):
    return b // 2 * 512 + (lane * 16 + ((b & 1) * 2 + h) * 4 if (b | 1) < nb else lane * 8 + h * 4)


def scale(nb, b, token):
    return (token % 8) // 2 * nb * 8 + b * 8 + (token // 8 * 2 + token % 2) * 2


@pytest.mark.parametrize("nb", [1, 2, 3, 4])
def test_layout_covers_a_tile_once(nb):
    """Every code and scale of a 16-token tile has bytes of its own inside the
    tile's nb * 576, and a token's codes share no byte with another's."""
    owner = {}

    def own(at, who):
        assert 0 <= at < nb * 576 and owner.setdefault(at, who) == who

    for token in range(16):
        g, h = token % 8, token // 8
        for b in range(nb):
            for quarter in range(4):
                for byte in range(4):
                    own(word(nb, b, g * 4 + quarter, h) + byte, (token, "k", b, quarter, byte))
            for g4 in range(8):  # dims 4 g4 .. + 3
                at = nb * 256 + word(nb, b, g4 * 4 + (token % 8) // 2, h) + 2 * (token % 2)
                for byte in range(2):
                    own(at + byte, (token, "v", b, g4, byte))
            for byte in range(2):
                own(nb * 512 + scale(nb, b, token) + byte, (token, "ks", b, byte))
                own(nb * 544 + scale(nb, b, token) + byte, (token, "vs", b, byte))
    assert len(owner) == nb * 576


def test_quotient_rounding_needs_no_wide_division():
    """rint(fl32(x / d)) is the exact quotient's rounding for float16 d, next to
    every halfway point too."""
    rng = np.random.default_rng(0)
    d = rng.integers(1, 0x7c00, 20000).astype(np.uint16).view(np.float16)
    half = rng.integers(-8, 8, d.size) + 0.5
    at = (half * d.astype(np.float64)).astype(np.float32)
    for step in (-2, -1, 0, 1, 2):
        x = (at.view(np.int32) + step).view(np.float32)
        want = np.rint(x.astype(np.float64) / d.astype(np.float64))  # 53 bits tell x / d from a half: 24 + 11 bits
        got = np.rint(x / d.astype(np.float32))
        assert np.array_equal(want, got)


def test_plain_format():
    x = np.zeros(32, np.float32)
    assert (held(x) == 0).all()
    x[3], x[7] = 8.0, -8.0  # equal magnitudes: the first sets the sign of the scale
    h = held(x)
    assert h[3] == 8.0 and h[7] == -7.0
    x[0] = np.inf
    h = held(x)
    assert h[0] == 8 * 65504.0 and h[3] == 0.0
    x[1] = np.nan
    assert np.isnan(held(x)).all()
