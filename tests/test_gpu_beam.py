"""Beam search's selection and the reordering of the caches it implies, against
plain 64-bit arithmetic: parents and tokens equal, scores within a rounding."""
import numpy as np
import pytest

from kv_plain import TYPES, Device, beam_select, held, random_table, spt, torch_type

pytestmark = pytest.mark.gpu


def check(ctx, logits, scores, keep, finished=None, end_token=0):
    """logits [batch, beams, vocab] tensor, scores [batch, beams] array."""
    import torch
    type = {v: k for k, v in (("f32", torch.float32), ("f16", torch.float16), ("bf16", torch.bfloat16))}[logits.dtype]
    batch, beams, vocab = logits.shape
    plan = ctx.beam(batch, beams, vocab, keep)
    s = torch.tensor(np.asarray(scores, np.float32), device="cuda")
    f = None if finished is None else torch.tensor(np.asarray(finished, np.uint8), device="cuda")
    out = torch.empty(batch, keep, device="cuda")
    parents, tokens = (torch.empty(batch, keep, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    plan.select_device(logits.data_ptr(), s.data_ptr(), out.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                       TYPES[type], row_stride=logits.stride(1) if beams > 1 else logits.stride(0),
                       finished_ptr=0 if f is None else f.data_ptr(), end_token=end_token)
    ctx.sync()
    x = logits.double().cpu().numpy()
    for b in range(batch):
        want = beam_select(x[b], s[b].cpu().numpy(), keep, None if finished is None else finished[b], end_token)
        assert np.array_equal(parents[b].cpu().numpy(), want[1]), b
        assert np.array_equal(tokens[b].cpu().numpy(), want[2]), b
        got = out[b].double().cpu().numpy()
        live = want[1] >= 0
        assert (got[~live] == -np.inf).all()
        # sum of exponentials: each 2^-21 off, a chunk's sum of 8,192 in 32 bits (32 + 13 additions); then one rounding
        tol = 64 * 2.0 ** -24 + np.abs(want[0][live]) * 2.0 ** -24
        assert (np.abs(got[live] - want[0][live]) <= tol).all()
    plan.close()


@pytest.mark.parametrize("type", list(TYPES))
@pytest.mark.parametrize("batch,beams,vocab,keep", [(1, 1, 1, 1), (2, 1, 7, 4), (1, 4, 33, 8), (3, 2, 255, 64),
                                                    (2, 3, 8191, 6), (2, 8, 8192, 16), (1, 5, 8193, 10),
                                                    (2, 4, 50257, 8), (1, 2, 201088, 4), (1, 64, 300, 64)])
def test_selection(ctx, type, batch, beams, vocab, keep):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(vocab + keep)
    logits = (torch.randn(batch, beams, vocab, generator=gen, device="cuda") * 3).to(torch_type(type))
    scores = np.random.default_rng(keep).normal(size=(batch, beams)) * 2 - 4
    check(ctx, logits, scores, keep)


def test_ties_and_first_step(ctx):
    """Equal logits, equal rows, unused beams: the lowest beam, then the lowest token."""
    import torch
    check(ctx, torch.zeros(1, 2, 20000, device="cuda"), [[0.0, 0.0]], 12)            # every logit ties
    check(ctx, torch.zeros(1, 3, 50, device="cuda"), [[-1.0, -1.0, -1.0]], 64)       # beyond one beam's tokens
    x = torch.randn(1, 1, 9000, device="cuda").expand(1, 4, 9000).contiguous()
    check(ctx, x, [[0.0, 0.0, 0.0, 0.0]], 16)                                        # equal beams
    check(ctx, x, [[0.0, -np.inf, -np.inf, -np.inf]], 8)                             # a search's first step
    check(ctx, x.round().bfloat16(), [[0.0, -0.5, -0.25, -np.inf]], 32)              # few distinct logits
    check(ctx, torch.tensor([[[0.0, -0.0, 0.0, -0.0]]], device="cuda"), [[0.0]], 4)  # zeros of both signs


def test_masked_logits(ctx):
    """-inf, the type's lowest value, NaN, +inf; rows with nothing left."""
    import torch
    inf = float("inf")
    x = torch.randn(1, 4, 10000, device="cuda")
    x[0, 0, 5:] = -inf
    x[0, 1, :] = -inf
    x[0, 2, ::2] = torch.finfo(torch.float32).min
    x[0, 3, 1::3] = float("nan")
    check(ctx, x, [[0.0, 0.0, 0.0, 0.0]], 16)
    check(ctx, x[:, :2].contiguous(), [[0.0, 0.0]], 16)                   # fewer candidates than places
    check(ctx, x[:, 1:2].contiguous(), [[0.0]], 3)                        # none
    check(ctx, x, [[0.0, 0.0, float("nan"), -1.0]], 8)                    # a beam without a score
    x[0, 3, 77] = inf                                                     # its other tokens have probability 0
    check(ctx, x, [[0.0, 0.0, 0.0, 0.0]], 8)
    check(ctx, torch.full((1, 2, 9), float("nan"), device="cuda"), [[0.0, 0.0]], 2)


def test_finished_beams(ctx):
    import torch
    x = torch.randn(2, 4, 1000, device="cuda")
    x[0, 1] = float("nan")  # a finished beam's logits are not read
    check(ctx, x, [[-1.0, -0.5, -9.0, -1.0], [-1.0, -0.5, -0.5, -1.0]], 8,
          finished=[[0, 1, 1, 0], [1, 1, 1, 1]], end_token=999)
    check(ctx, x, [[-np.inf, -np.inf, 0.0, 0.0], [0.0, 0.0, 0.0, 0.0]], 3, finished=[[1, 0, 1, 0], [1, 0, 0, 1]])


def test_strided_rows(ctx):
    import torch
    for pad in (1, 4, 24):
        wide = torch.randn(1, 3, 9001 + pad, device="cuda")
        check(ctx, wide[:, :, :9001], [[0.0, -1.0, -2.0]], 6)
        check(ctx, wide.half()[:, :, :9001], [[0.0, -1.0, -2.0]], 6)


@pytest.mark.parametrize("pattern", ["rising", "falling", "ties", "few", "lowest", "masked", "late", "nan", "large", "inf"])
@pytest.mark.parametrize("type,keep,vocab", [("f32", 64, 30001), ("bf16", 7, 24576), ("f16", 16, 29999)])
def test_long_rows(ctx, pattern, type, keep, vocab):
    """Many rows of several pieces each: candidates that outrun the list, masks over whole pieces."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(keep)
    x = torch.randn(6, 64, vocab, generator=gen, device="cuda") * 2
    inf = float("inf")
    if pattern in ("rising", "falling"):
        x = x.sort(-1, descending=pattern == "falling").values
    elif pattern == "ties":
        x = torch.zeros_like(x)
    elif pattern == "few":
        x = x.round()
    elif pattern == "lowest":  # rows of nothing but the type's lowest value, and rows that end with it
        x[:, ::2] = x[:, 1::2, 9000:] = torch.finfo(torch_type(type)).min
    elif pattern == "masked":
        x[:, :, 100:20000] = -inf
        x[:, 5] = -inf
    elif pattern == "late":  # everything that counts in the last piece
        x[:, :, :-70] = -inf
    elif pattern == "nan":
        x[:, :, 1::2] = float("nan")
        x[:, 3, :20000] = float("nan")
    elif pattern == "large":
        x = x * (1e30 if type != "f16" else 1e4)
    elif pattern == "inf":
        x[:, ::3, 20000] = inf
    scores = np.random.default_rng(keep).normal(size=(6, 64)) - 4
    check(ctx, x.to(torch_type(type)), scores, keep)


def test_host_call_and_refusals(ctx):
    rng = np.random.default_rng(1)
    plan = ctx.beam(2, 3, 500, 6)
    x, s = rng.normal(size=(6, 500)).astype(np.float32), rng.normal(size=(2, 3)).astype(np.float32)
    fin = np.array([[0, 1, 0], [0, 0, 0]], np.uint8)
    scores, parents, tokens = plan.select(x, s, fin, 7)
    for b in range(2):
        want = beam_select(x[3 * b:3 * b + 3], s[b], 6, fin[b], 7)
        assert np.array_equal(parents[b], want[1]) and np.array_equal(tokens[b], want[2])

    def refused(status, call):
        with pytest.raises(spt.SptError) as e:
            call()
        assert e.value.status == status, e.value

    import torch
    d = torch.zeros(4096, device="cuda")
    p = d.data_ptr()
    dim = spt.ERR_DIMENSIONS
    refused(dim, lambda: plan.select(x[:5], s))
    refused(dim, lambda: plan.select(x, s[:1]))
    refused(dim, lambda: plan.select(x, s, fin, 500))
    refused(dim, lambda: plan.select_device(p, p, p, p, p, row_stride=499))
    refused(dim, lambda: plan.select_device(p + 2, p, p, p, p))
    refused(dim, lambda: plan.select_device(p, p + 1, p, p, p))
    refused(dim, lambda: plan.select_device(p, p, p, p, p, finished_ptr=p, end_token=-1))
    refused(spt.ERR_NULL_ARG, lambda: plan.select_device(0, p, p, p, p))
    o = [torch.zeros(64, device="cuda").data_ptr() for _ in range(3)]
    refused(spt.ERR_OVERLAP, lambda: plan.select_device(p, p, p, o[1], o[2]))           # scores in place
    refused(spt.ERR_OVERLAP, lambda: plan.select_device(p, p, o[0], p + 4 * 2999, o[2]))  # the last logit
    refused(spt.ERR_OVERLAP, lambda: plan.select_device(p, p, o[0], o[1], o[1] + 44))
    refused(spt.ERR_UNSUPPORTED, lambda: plan.select_device(p, p, p, p, p, type=8))
    plan.close()


@pytest.mark.parametrize("lengths", [[5] * 6, [16] * 6, [40] * 6, [33, 1, 48, 20, 31, 64], [0, 3, 0, 16, 17, 2]])
@pytest.mark.parametrize("parents", [[[0, 1, 2], [0, 1, 2]], [[0, 0, 0], [2, 2, 1]], [[2, 1, 2], [1, 0, 0]],
                                     [[1, -1, 1], [7, 2, 0]]])
def test_reorder(ctx, lengths, parents):
    """Each child reads its parent's tokens on every layer; what it appends next stays its own."""
    import torch
    rng = np.random.default_rng(2)
    page, heads, dim, layers = 16, 2, 64, 2
    table, spare, pages = random_table(rng, [max(n, 1) for n in lengths], page, spare=6)
    cache = ctx.kv_cache(kv_heads=heads, head_dim=dim, page_tokens=page, pages=pages, layers=layers)
    total = sum(lengths)
    at = np.concatenate([[0], np.cumsum(lengths)])
    data = torch.randn(layers, max(total, 1), heads, dim, device="cuda")
    dev = Device(table, lengths, lengths)
    torch.cuda.synchronize()
    for i in range(layers):
        cache.append_device(dev.batch, data[i].data_ptr(), data[i].data_ptr(), layer=i)
    par = torch.tensor(parents, dtype=torch.int32, device="cuda")
    sp = torch.tensor(spare[:6], dtype=torch.int32, device="cuda")
    new_table, new_lengths = torch.full_like(dev.table, 99), torch.full_like(dev.lengths, 99)
    copied = torch.full((6,), 99, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    cache.reorder_device(2, 3, table.shape[1], par.data_ptr(), 3, dev.table.data_ptr(), dev.lengths.data_ptr(),
                         sp.data_ptr(), new_table.data_ptr(), new_lengths.data_ptr(), copied.data_ptr())
    ctx.sync()
    want_lengths, want_copied = [], []
    for s in range(6):
        p = parents[s // 3][s % 3]
        ok = 0 <= p < 3
        want_lengths.append(lengths[s // 3 * 3 + p] if ok else 0)
        want_copied.append(int(ok and p in parents[s // 3][:s % 3] and want_lengths[-1] % page != 0))
    assert new_lengths.tolist() == want_lengths and copied.tolist() == want_copied
    n = sum(want_lengths)
    got = torch.zeros(max(n, 1), heads, dim, device="cuda")
    after = Device(new_table.cpu().numpy(), want_lengths, want_lengths)
    torch.cuda.synchronize()
    for i in range(layers):
        cache.read_device(after.batch, got.data_ptr(), 0, layer=i)
        ctx.sync()
        where = 0
        for s in range(6):
            if not want_lengths[s]:
                assert (new_table[s] == -1).all()
                continue
            src = s // 3 * 3 + parents[s // 3][s % 3]
            want = held(data[i, at[src]:at[src + 1]].cpu().numpy()).astype(np.float32)
            assert np.array_equal(got[where:where + want_lengths[s]].cpu().numpy(), want), (i, s)
            where += want_lengths[s]
    # places behind a partial last page belong to one sequence each
    partial = [int(new_table[s, want_lengths[s] // page]) for s in range(6) if want_lengths[s] % page]
    assert len(set(partial)) == len(partial)
    cache.close()


def test_step_captured_and_replayed(ctx):
    """Selection, reorder and the read-back in a graph: replayed on other logits it does what the calls do."""
    import torch
    page, heads, dim, beams, keep, vocab = 16, 2, 64, 3, 6, 20011
    lengths = [21, 40, 5, 33, 16, 50]
    table, spare, pages = random_table(np.random.default_rng(7), lengths, page, spare=6)
    cache = ctx.kv_cache(kv_heads=heads, head_dim=dim, page_tokens=page, pages=pages)
    plan = ctx.beam(2, beams, vocab, keep)
    dev = Device(table, lengths, lengths)
    data = torch.randn(sum(lengths), heads, dim, device="cuda")
    torch.cuda.synchronize()
    cache.append_device(dev.batch, data.data_ptr(), data.data_ptr())
    x, scores = torch.empty(6, vocab, device="cuda"), torch.full((6,), -1.0, device="cuda")
    sp = torch.tensor(spare[:6], dtype=torch.int32, device="cuda")

    def outputs():
        i32 = lambda *n: torch.full(n, 99, dtype=torch.int32, device="cuda")  # noqa: E731
        return dict(scores=torch.empty(2, keep, device="cuda"), parents=i32(2, keep), tokens=i32(2, keep),
                    table=i32(*dev.table.shape), lengths=i32(6), rows=torch.zeros(6, heads, dim, device="cuda"))

    def step(o):
        p = {k: v.data_ptr() for k, v in o.items()}
        plan.select_device(x.data_ptr(), scores.data_ptr(), p["scores"], p["parents"], p["tokens"])
        cache.reorder_device(2, beams, table.shape[1], p["parents"], keep, dev.table.data_ptr(), dev.lengths.data_ptr(),
                             sp.data_ptr(), p["table"], p["lengths"], 0)
        cache.read_device(spt.KvBatch(6, 6, table.shape[1], p["table"], p["lengths"]), p["rows"], 0)

    eager, held_out, stream = outputs(), outputs(), torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(held_out)
        for seed in range(3):
            x.copy_(torch.randn(6, vocab, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            step(eager)
            ctx.sync()
            for name in eager:
                assert torch.equal(eager[name], held_out[name]), (seed, name)
            assert int((eager["lengths"] > 0).sum()) == 6 and bool((eager["rows"] != 0).any())
    finally:
        ctx.set_stream(0)
    plan.close()
    cache.close()


def test_reorder_host_and_refusals(ctx):
    cache = ctx.kv_cache(kv_heads=1, head_dim=32, page_tokens=16, pages=8)
    rng = np.random.default_rng(0)
    table, lengths = np.array([[0, 1], [2, 3]], np.int32), np.array([20, 17], np.int32)
    x = rng.standard_normal((37, 1, 32)).astype(np.float32)
    cache.append(spt.KvBatch(2, 37, 2, table, lengths, [0, 20, 37]), x, x)
    spare = np.array([4, 5], np.int32)
    t, n, c = cache.reorder(np.array([[1, 1]]), table, lengths, spare)
    assert t.tolist() == [[2, 3], [2, 5]] and n.tolist() == [17, 17] and c.tolist() == [0, 1]
    k, _ = cache.read(spt.KvBatch(2, 34, 2, t, n, [0, 17, 34]))
    assert np.array_equal(k[:17], k[17:]) and np.array_equal(k[:17], held(x[20:]).astype(np.float32))

    def refused(status, call):
        with pytest.raises(spt.SptError) as e:
            call()
        assert e.value.status == status, e.value

    dim = spt.ERR_DIMENSIONS
    refused(dim, lambda: cache.reorder(np.array([[2, 0]]), table, lengths, spare))
    refused(dim, lambda: cache.reorder(np.array([[0, 0]]), table, lengths, np.array([-1, -1], np.int32)))
    refused(dim, lambda: cache.reorder(np.array([[0, 0]]), table, np.array([33, 1], np.int32), spare))
    refused(dim, lambda: cache.reorder(np.array([[0, 0]]), np.array([[0, 8], [2, 3]], np.int32), lengths, spare))
    p = __import__("torch").zeros(64, dtype=__import__("torch").int32, device="cuda").data_ptr()
    refused(spt.ERR_OVERLAP, lambda: cache.reorder_device(1, 2, 2, p, 2, p + 32, p + 64, p + 96, p + 32, p + 160))
    refused(spt.ERR_NULL_ARG, lambda: cache.reorder_device(1, 2, 2, 0, 2, p, p, p, p + 128, p + 160))
    refused(dim, lambda: cache.reorder_device(1, 2, 2, p, 1, p, p, p, p + 128, p + 160))
    cache.close()


def test_a_search_step(ctx):
    """The operators as a search uses them: write a token, attend, select, reorder, twice over."""
    import torch
    from kv_plain import attention, attention_tolerance
    rng = np.random.default_rng(4)
    beams, heads, kv, dim, page, vocab = 3, 8, 2, 64, 16, 700
    cache = ctx.kv_cache(kv_heads=kv, head_dim=dim, page_tokens=page, pages=32)
    prompt = rng.standard_normal((30, kv, dim)).astype(np.float32)
    free = list(range(32))
    first = [free.pop(), free.pop()]
    table = np.full((beams, 4), -1, np.int32)
    table[:, :1] = first[0]
    pages = [first[1], free.pop(), free.pop()]
    table[:, 1] = pages
    for b in range(beams):  # the beams share the prompt's whole page and have the rest of their own
        cache.append(spt.KvBatch(1, 30, 4, table[b:b + 1], [30], [0, 30]), prompt, prompt)
    history = [list(prompt) for _ in range(beams)]
    lengths, scores = np.full(beams, 30, np.int32), np.zeros((1, beams), np.float32)
    plan = ctx.beam(1, beams, vocab, beams)
    for step in range(5):
        new = rng.standard_normal((beams, kv, dim)).astype(np.float32)
        lengths = lengths + 1
        for b in range(beams):
            if table[b, (lengths[b] - 1) // page] < 0:
                table[b, (lengths[b] - 1) // page] = free.pop()
            history[b].append(new[b])
        batch = spt.KvBatch(beams, beams, 4, table, lengths)
        cache.append(batch, new, new)
        q = rng.standard_normal((beams, heads, dim)).astype(np.float32)
        out = cache.attention(batch, q, heads, scale=0.125)
        for b in range(beams):
            kv64 = torch.tensor(held(np.stack(history[b])))
            want = attention(torch.tensor(q[b:b + 1]).double(), kv64, kv64, lengths[b] - 1, 0.125)
            tol = attention_tolerance(*want, int(lengths[b]), "f32")
            assert bool(((torch.tensor(out[b:b + 1]).double() - want[0]).abs() <= tol).all()), (step, b)
        logits = rng.normal(size=(beams, vocab)).astype(np.float32)
        want = beam_select(logits, scores[0], beams)
        scores, parents, tokens = plan.select(logits, scores)
        assert np.array_equal(parents[0], want[1]) and np.array_equal(tokens[0], want[2])
        spare = np.array([free.pop() for _ in range(beams)], np.int32)
        table, lengths, copied = cache.reorder(parents, table, lengths, spare)
        free += [int(p) for p, c in zip(spare, copied) if not c]
        history = [list(history[p]) for p in parents[0]]
    plan.close()
    cache.close()
