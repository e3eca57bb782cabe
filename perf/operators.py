"""Cases of the 4-bit KV cache, the attention over it, and beam search's
selection and reordering: inputs, plain forms in elementary torch operations,
the framework's calls, and results in 64 bits.

A case's sizes are plain values; the lengths of its sequences follow from them
alone, the contents and the order of the pages from the seed.
"""
import importlib
import math
from types import SimpleNamespace

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
BLOCK = 32  # values that share one 4-bit scale
VOCAB = 201088

_context = None


def context():
    """The framework's context on this GPU, one for the process."""
    global _context
    if _context is None:
        _context = importlib.import_module("stream-pt_b200").Context(0)
    return _context


# ---- cases ------------------------------------------------------------------
def listed():
    def cache(name, sequences, context, new, type, page, kv_heads=8, head_dim=64):
        return dict(name=name, op="cache", sequences=sequences, context=context, new=new, kv_heads=kv_heads,
                    head_dim=head_dim, type=type, page=page)

    def attention(name, sequences, context, new, type, page, heads=64, kv_heads=8, head_dim=64, window=0, sinks=True):
        return dict(name=name, op="attention", sequences=sequences, context=context, new=new, heads=heads,
                    kv_heads=kv_heads, head_dim=head_dim, window=window, sinks=sinks, type=type, page=page)

    def beam(name, batch, beams, keep, type, context, page, layers, first=False):
        return dict(name=name, op="beam", batch=batch, beams=beams, keep=keep, vocab=VOCAB, type=type, context=context,
                    page=page, layers=layers, kv_heads=8, head_dim=64, first=first)

    return [
        # one decoded token of one sequence: a single layer's write, and the rows read back
        cache("cache-decode-1", 1, 700, 1, "f32", 64),
        # a batch of prompts of ragged lengths, as a prefill writes them
        cache("cache-prompts", 24, 2048, 2048, "f32", 64),
        # wide heads, 16-bit activations, pages that end inside the prompts
        cache("cache-bf16-wide", 7, 1111, 1111, "bf16", 16, head_dim=128),
        # one user's decode step at the end of a 2,048-token context, full-attention layer
        attention("decode-1x2047", 1, 2047, 1, "f32", 64),
        # a serving batch on a sliding-window layer: only 128 keys of each long sequence count
        attention("decode-48-window", 48, 6000, 1, "f32", 64, window=128),
        # a large serving batch of ragged long contexts: the cache's bytes bound it
        attention("decode-64x8k", 64, 8192, 1, "f32", 64),
        # one very long context in 16 bits, wide heads shared by four queries
        attention("decode-128k-bf16", 1, 131000, 1, "bf16", 128, heads=32, kv_heads=8, head_dim=128, sinks=False),
        # a 32-token prefill chunk late in a context
        attention("chunk-32", 1, 2048, 32, "f32", 64),
        # a whole 2,000-token prompt
        attention("prompt-2000", 1, 2000, 2000, "f32", 64),
        # chunked prefill beside decoding sequences, 16 bits, small pages
        attention("mixed-f16", 12, 3001, 500, "f16", 16),
        # one user's beam search, four beams on the whole vocabulary
        beam("beam-1x4", 1, 4, 4, "f32", 403, 16, 2),
        # sixteen searches of eight beams, twice as many candidates as beams
        beam("beam-16x8", 16, 8, 16, "f32", 1003, 64, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cache", "attention", "attention", "attention", "beam"])
    type = rng.choice(["f32", "f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8])
        batch = _log(rng, 1, 128 // beams)
        return dict(op=op, batch=batch, beams=beams, keep=beams * rng.choice([1, 2]), vocab=_log(rng, 500, VOCAB),
                    type=type, context=_log(rng, 1, 1000), page=page, layers=rng.choice([1, 2, 3]), kv_heads=8,
                    head_dim=64, first=rng.random() < 0.2)
    head_dim = rng.choice([64, 64, 128, 32, 96])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    if op == "cache":
        sequences = _log(rng, 1, 32)
        context = _log(rng, 1, 2048 if sequences <= 20 else 1024)
        new = 1 if rng.random() < 0.3 else max(1, int(context * rng.random()))
        return dict(op=op, sequences=sequences, context=context, new=new, kv_heads=kv_heads, head_dim=head_dim,
                    type=type, page=page)
    heads = kv_heads * rng.choice([1, 3, 4, 6, 8])
    kind = rng.choice(["decode", "decode", "chunk"])
    if kind == "decode":
        sequences = _log(rng, 1, 64)
        context = _log(rng, 1, 400000 // sequences if sequences > 8 else 50000)
        new = rng.choice([1, 1, 1, 2, 4])
    else:
        sequences = _log(rng, 1, 8)
        context = _log(rng, 32, 3000)
        new = min(context, _log(rng, 8, 1500 // sequences))
    context = max(context, new)
    return dict(op=op, sequences=sequences, context=context, new=new, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, window=rng.choice([0, 0, 128, 97]), sinks=rng.random() < 0.7, type=type, page=page)


def lengths_of(case):
    """(cached tokens, new tokens among them) of each sequence: the first has
    the case's own, the others spread below them."""
    out = []
    for b in range(case["sequences"]):
        u = 1.0 if b == 0 else math.modf((b + 1) * 0.6180339887498949)[0]
        length = 1 + int((case["context"] - 1) * (0.2 + 0.8 * u))
        new = case["new"] if b == 0 else 1 + int((case["new"] - 1) * math.modf((b + 1) * 0.7548776662466927)[0])
        if case["op"] == "attention" and case["new"] > 8 and b % 2 == 1:
            new = 1  # a decoding sequence beside the chunks
        out.append((length, min(new, length)))
    return out


# ---- inputs -----------------------------------------------------------------
def rows_of(gen, n, heads, dim, type):
    """Rows of projected activations: unit variance, some channels much larger, as keys have them."""
    x = torch.randn(n, heads, dim, generator=gen, device="cuda")
    channel = torch.exp(0.7 * torch.randn(heads, dim, generator=gen, device="cuda"))
    return (x * channel).to(TYPES[type])


def quantise(x):
    """4-bit blocks of [..., dim]: codes (one a byte) and 16-bit scales."""
    x = x.float()
    blocks = x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    at = blocks.abs().argmax(-1, keepdim=True)
    scale = (blocks.gather(-1, at) * -0.125).clamp(-65504.0, 65504.0).to(torch.float16)
    wide = scale.double()
    steps = torch.where(wide == 0, 0.0, blocks.double() / torch.where(wide == 0, 1.0, wide))
    codes = (torch.round(steps) + 8).clamp(0, 15).to(torch.uint8)
    return codes.reshape(x.shape), scale[..., 0]


def pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def decode(packed, scale):
    """The values that packed codes [..., dim/2] and scales [..., dim/32] stand for."""
    codes = torch.stack([packed & 15, packed >> 4], -1).flatten(-2).float() - 8.0
    blocks = codes.reshape(*scale.shape, BLOCK) * scale.float()[..., None]
    return blocks.flatten(-2)


def page_tables(gen, counts, page, extra=0):
    """A table of distinct pages for sequences of `counts` tokens, and the pages used and spare."""
    need = [-(-c // page) for c in counts]
    order = torch.randperm(sum(need) + extra, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(counts), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order[at:], sum(need) + extra


def device_ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def slots(table, lengths, counts, page):
    """Page and place of each sequence's last `counts` tokens, in row order."""
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), torch.tensor(counts, device="cuda"))
    first = torch.tensor([n - c for n, c in zip(lengths, counts)], device="cuda")
    start = torch.tensor(starts(counts)[:-1], device="cuda")
    position = torch.arange(sum(counts), device="cuda") - start[seq] + first[seq]
    return table[seq, position // page].long(), position % page


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = SimpleNamespace(case=case, **{k: v for k, v in case.items() if k not in ("name", "op")})
    {"cache": prepare_cache, "attention": prepare_attention, "beam": prepare_beam}[case["op"]](s, gen)
    torch.cuda.synchronize()
    return s


def prepare_cache(s, gen):
    pairs = lengths_of(s.case)
    s.seq_lengths, s.counts = [p[0] for p in pairs], [p[1] for p in pairs]
    s.rows = sum(s.counts)
    s.table, _, s.pages = page_tables(gen, s.seq_lengths, s.page)
    s.k = rows_of(gen, s.rows, s.kv_heads, s.head_dim, s.type)
    s.v = rows_of(gen, s.rows, s.kv_heads, s.head_dim, s.type)
    s.lengths, s.offsets = device_ints(s.seq_lengths), device_ints(starts(s.counts))
    if own:
        spt = importlib.import_module("stream-pt_b200")
        s.cache = context().kv_cache(kv_heads=s.kv_heads, head_dim=s.head_dim, page_tokens=s.page, pages=s.pages)
        s.batch = spt.KvBatch(len(s.counts), s.rows, s.table.shape[1], s.table.data_ptr(), s.lengths.data_ptr(),
                              s.offsets.data_ptr())
        s.k_out, s.v_out = torch.empty_like(s.k), torch.empty_like(s.v)
    else:
        s.page_of, s.place = slots(s.table, s.seq_lengths, s.counts, s.page)
        shape = (s.pages, s.page, s.kv_heads)
        s.k_codes = torch.zeros(*shape, s.head_dim // 2, dtype=torch.uint8, device="cuda")
        s.v_codes = torch.zeros_like(s.k_codes)
        s.k_scale = torch.zeros(*shape, s.head_dim // BLOCK, dtype=torch.float16, device="cuda")
        s.v_scale = torch.zeros_like(s.k_scale)


def fill(s, k, v, lengths, layer=0):
    """Puts every cached token's k and v rows in place, in this side's form of the cache."""
    if own:
        spt = importlib.import_module("stream-pt_b200")
        all_lengths, all_offsets = device_ints(lengths), device_ints(starts(lengths))
        torch.cuda.synchronize()
        batch = spt.KvBatch(len(lengths), k.shape[0], s.table.shape[1], s.table.data_ptr(), all_lengths.data_ptr(),
                            all_offsets.data_ptr())
        s.cache.append_device(batch, k.data_ptr(), v.data_ptr(), GGML["f32"], layer=layer)
        context().sync()
        return
    page_of, place = slots(s.table, lengths, lengths, s.page)
    for x, codes, scale in ((k, s.k_codes[layer], s.k_scale[layer]), (v, s.v_codes[layer], s.v_scale[layer])):
        for at in range(0, x.shape[0], 1 << 15):  # in parts: the 64-bit quotients take room
            c, d = quantise(x[at:at + (1 << 15)])
            codes[page_of[at:at + (1 << 15)], place[at:at + (1 << 15)]] = pack(c)
            scale[page_of[at:at + (1 << 15)], place[at:at + (1 << 15)]] = d


def empty_cache(s, layers):
    if own:
        s.cache = context().kv_cache(kv_heads=s.kv_heads, head_dim=s.head_dim, page_tokens=s.page, pages=s.pages,
                                     layers=layers)
        return
    shape = (layers, s.pages, s.page, s.kv_heads)
    s.k_codes = torch.zeros(*shape, s.head_dim // 2, dtype=torch.uint8, device="cuda")
    s.v_codes = torch.zeros_like(s.k_codes)
    s.k_scale = torch.zeros(*shape, s.head_dim // BLOCK, dtype=torch.float16, device="cuda")
    s.v_scale = torch.zeros_like(s.k_scale)


def attention_inputs(s, gen):
    """Cached keys and values in 32 bits, queries, sinks: the same whatever computes them."""
    pairs = lengths_of(s.case)
    s.seq_lengths, s.counts = [p[0] for p in pairs], [p[1] for p in pairs]
    s.rows, total = sum(s.counts), sum(s.seq_lengths)
    s.table, _, s.pages = page_tables(gen, s.seq_lengths, s.page)
    k = rows_of(gen, total, s.kv_heads, s.head_dim, "f32")
    v = rows_of(gen, total, s.kv_heads, s.head_dim, "f32")
    s.q = torch.randn(s.rows, s.heads, s.head_dim, generator=gen, device="cuda").to(TYPES[s.type])
    s.sink = torch.randn(s.heads, generator=gen, device="cuda") if s.sinks else None
    s.scale = s.head_dim ** -0.5
    return k, v


def prepare_attention(s, gen):
    k, v = attention_inputs(s, gen)
    empty_cache(s, 1)
    fill(s, k, v, s.seq_lengths)
    s.lengths, s.offsets = device_ints(s.seq_lengths), device_ints(starts(s.counts))
    if own:
        spt = importlib.import_module("stream-pt_b200")
        s.batch = spt.KvBatch(len(s.counts), s.rows, s.table.shape[1], s.table.data_ptr(), s.lengths.data_ptr(),
                              s.offsets.data_ptr() if max(s.counts) > 1 else 0)
        s.out = torch.empty_like(s.q)
    else:
        most = max(s.counts)
        place = torch.arange(most, device="cuda")[None, :]
        count = torch.tensor(s.counts, device="cuda")[:, None]
        s.row_of = (s.offsets[:-1, None].long() + place).clamp(max=s.rows - 1)  # [sequences, most]
        s.position = s.lengths[:, None].long() - count + place
        seq = torch.repeat_interleave(torch.arange(len(s.counts), device="cuda"), count[:, 0])
        s.flat = seq * most + torch.arange(s.rows, device="cuda") - s.offsets[seq].long()


def beam_inputs(s, gen):
    rows = s.batch * s.beams
    s.logits = torch.randn(rows, s.vocab, generator=gen, device="cuda") * 2.0
    peak = torch.randint(0, s.vocab, (rows, 24), generator=gen, device="cuda")
    s.logits.scatter_add_(1, peak, 8.0 * torch.rand(rows, 24, generator=gen, device="cuda"))
    s.logits = s.logits.to(TYPES[s.type])
    s.scores = -3.0 * torch.rand(s.batch, s.beams, generator=gen, device="cuda") - 5.0
    s.finished = torch.zeros(s.batch, s.beams, dtype=torch.uint8, device="cuda")
    s.finished[:, 1::4] = (torch.rand(s.batch, s.finished[:, 1::4].shape[1], generator=gen, device="cuda") < 0.5).to(torch.uint8)
    if s.first:  # a search's first step: only its first beam counts
        s.scores[:, 1:] = -math.inf
        s.finished.zero_()
    s.end_token = s.vocab - 1
    s.lengths_list = [s.context] * rows
    s.table, spare, s.pages = page_tables(gen, s.lengths_list, s.page, extra=rows)
    s.spare = spare.contiguous()
    s.part = s.context % s.page or s.page  # tokens in each sequence's last page
    total = rows * s.context
    return [(rows_of(gen, total, s.kv_heads, s.head_dim, "f32"), rows_of(gen, total, s.kv_heads, s.head_dim, "f32"))
            for _ in range(s.layers)]


def prepare_beam(s, gen):
    layers = beam_inputs(s, gen)
    rows = s.batch * s.beams
    empty_cache(s, s.layers)
    for i, (k, v) in enumerate(layers):
        fill(s, k, v, s.lengths_list, layer=i)
    s.lengths = device_ints(s.lengths_list)
    if own:
        spt = importlib.import_module("stream-pt_b200")
        s.plan = context().beam(batch=s.batch, beams=s.beams, vocab=s.vocab, keep=s.keep)
        s.out_scores = torch.empty(s.batch, s.keep, device="cuda")
        s.out_parents = torch.empty(s.batch, s.keep, dtype=torch.int32, device="cuda")
        s.out_tokens = torch.empty_like(s.out_parents)
        s.new_table, s.new_lengths = torch.empty_like(s.table), torch.empty_like(s.lengths)
        s.copied = torch.empty(rows, dtype=torch.uint8, device="cuda")
        s.offsets = device_ints(starts([s.part] * rows))
        s.moved = spt.KvBatch(rows, rows * s.part, s.table.shape[1], s.new_table.data_ptr(), s.new_lengths.data_ptr(),
                              s.offsets.data_ptr())
        shape = (s.layers, rows * s.part, s.kv_heads, s.head_dim)
        s.k_out, s.v_out = torch.empty(shape, device="cuda"), torch.empty(shape, device="cuda")


# ---- one pass -----------------------------------------------------------------
def run(s):
    return {"cache": run_cache, "attention": run_attention, "beam": run_beam}[s.case["op"]](s)


def run_cache(s):
    """New tokens' k and v into the cache, and the rows as the cache now holds them."""
    if own:
        t = GGML[s.type]
        s.cache.append_device(s.batch, s.k.data_ptr(), s.v.data_ptr(), t)
        s.cache.read_device(s.batch, s.k_out.data_ptr(), s.v_out.data_ptr(), t)
        return {"k": s.k_out, "v": s.v_out}
    out = {}
    for name, x, codes, scale in (("k", s.k, s.k_codes, s.k_scale), ("v", s.v, s.v_codes, s.v_scale)):
        c, d = quantise(x)
        codes[s.page_of, s.place], scale[s.page_of, s.place] = pack(c), d
        out[name] = decode(codes[s.page_of, s.place], scale[s.page_of, s.place]).to(TYPES[s.type])
    return out


def run_attention(s):
    if own:
        s.cache.attention_device(s.batch, s.q.data_ptr(), s.out.data_ptr(), s.heads, GGML[s.type], scale=s.scale,
                                 window=s.window, sinks_ptr=s.sink.data_ptr() if s.sinks else 0)
        return s.out
    group, (sequences, most) = s.heads // s.kv_heads, s.row_of.shape
    wide = s.table.shape[1]
    if s.window:  # only the pages that hold the rows' windows
        first = (s.position[:, :1] - s.window + 1).clamp(min=0) // s.page
        page = first + torch.arange(min(wide, (s.window + most) // s.page + 2), device="cuda")
    else:
        page = torch.arange(wide, device="cuda").expand(sequences, wide)
    pages = s.table.gather(1, page.clamp(max=wide - 1)).clamp(min=0).long()

    def cached(codes, scale):  # [sequences, kv_heads, tokens, head_dim]
        x = decode(codes[0, pages], scale[0, pages])
        return x.flatten(1, 2).transpose(1, 2)

    q = s.q.float()[s.row_of].reshape(sequences, most, s.kv_heads, group, s.head_dim)
    q = q.transpose(1, 2).reshape(sequences, s.kv_heads, most * group, s.head_dim)
    score = torch.matmul(q, cached(s.k_codes, s.k_scale).transpose(2, 3)) * s.scale
    score = score.reshape(sequences, s.kv_heads, most, group, -1)
    key = (page[:, :, None] * s.page + torch.arange(s.page, device="cuda")).flatten(1)[:, None, :]
    seen = key <= s.position[..., None]
    if s.window:
        seen &= key > s.position[..., None] - s.window
    score = score.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    if s.sinks:
        sink = s.sink.reshape(1, s.kv_heads, 1, group, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    if s.sinks:
        total = total + torch.exp(sink - top)
    weight = weight.reshape(sequences, s.kv_heads, most * group, -1)
    out = torch.matmul(weight, cached(s.v_codes, s.v_scale)).reshape(sequences, s.kv_heads, most, group, s.head_dim)
    out = (out / total).transpose(1, 2).reshape(sequences * most, s.heads, s.head_dim)
    return out[s.flat].to(TYPES[s.type])


def best_of(x, k):
    """The k largest of each row, in order, the lowest index first among equals: (values, indices)."""
    last = torch.topk(x, k, dim=-1).values[..., -1:]
    tie = x == last
    room = k - (x > last).sum(-1, keepdim=True)
    taken = (x > last) | (tie & (torch.cumsum(tie, -1, dtype=torch.int32) <= room))
    place = torch.arange(x.shape[-1], device=x.device)
    index = torch.topk(torch.where(taken, -place, -x.shape[-1]), k, dim=-1).values.neg()
    value, order = torch.sort(x.gather(-1, index), dim=-1, descending=True, stable=True)
    return value, index.gather(-1, order)


def run_beam(s):
    """Selection over beams and vocabulary, then the caches of the first `beams` survivors put in
    their order: scores, parents, tokens, the new tables, and the last page of each as it now reads."""
    if own:
        s.plan.select_device(s.logits.data_ptr(), s.scores.data_ptr(), s.out_scores.data_ptr(),
                             s.out_parents.data_ptr(), s.out_tokens.data_ptr(), GGML[s.type],
                             finished_ptr=s.finished.data_ptr(), end_token=s.end_token)
        s.cache.reorder_device(s.batch, s.beams, s.table.shape[1], s.out_parents.data_ptr(), s.keep,
                               s.table.data_ptr(), s.lengths.data_ptr(), s.spare.data_ptr(), s.new_table.data_ptr(),
                               s.new_lengths.data_ptr(), s.copied.data_ptr())
        for i in range(s.layers):
            s.cache.read_device(s.moved, s.k_out[i].data_ptr(), s.v_out[i].data_ptr(), GGML["f32"], layer=i)
        return {"scores": s.out_scores, "parents": s.out_parents, "tokens": s.out_tokens, "table": s.new_table,
                "copied": s.copied, "k": s.k_out, "v": s.v_out}
    rows = s.batch * s.beams
    x = s.logits.double()
    top = x.amax(-1, keepdim=True)
    norm = top + torch.exp(x - top).sum(-1, keepdim=True).log()
    done = s.finished.reshape(rows, 1) != 0
    only = torch.full((1, s.vocab), -math.inf, dtype=torch.float64, device="cuda")
    only[0, s.end_token] = 0.0
    total = torch.where(done, only, x - norm) + s.scores.double().reshape(rows, 1)
    value, token = best_of(total, min(s.keep, s.vocab))
    value, at = torch.sort(value.reshape(s.batch, -1), dim=-1, descending=True, stable=True)
    value, at = value[:, :s.keep], at[:, :s.keep]
    parents = (at // token.shape[-1]).to(torch.int32)
    tokens = token.reshape(s.batch, -1).gather(1, at).to(torch.int32)
    pick = parents[:, :s.beams].long()
    earlier = torch.ones(s.beams, s.beams, dtype=torch.bool, device="cuda").tril(-1)
    repeated = ((pick[:, :, None] == pick[:, None, :]) & earlier).any(-1).reshape(rows)
    source = (pick + torch.arange(s.batch, device="cuda")[:, None] * s.beams).reshape(rows)
    table = s.table[source]
    last = (s.context - 1) // s.page
    copied = repeated & (s.context % s.page != 0)
    old = table[:, last].long()
    new = torch.where(copied, s.spare.long(), old)
    table[:, last] = new.to(torch.int32)
    for pool in (s.k_codes, s.k_scale, s.v_codes, s.v_scale):
        pool[:, new] = pool[:, old]
    k = decode(s.k_codes[:, new, :s.part], s.k_scale[:, new, :s.part]).flatten(1, 2)
    v = decode(s.v_codes[:, new, :s.part], s.v_scale[:, new, :s.part]).flatten(1, 2)
    return {"scores": value.float(), "parents": parents, "tokens": tokens, "table": table,
            "copied": copied.to(torch.uint8), "k": k, "v": v}


# ---- what a pass cannot do without ----------------------------------------------
def seen_keys(case, length, new):
    """Keys that the last `new` positions of a sequence attend to, in all, and those any of them reads."""
    w = case["window"] or length
    each = sum(min(w, p + 1) for p in range(length - new, length))
    return each, length - max(0, length - new + 1 - w)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    token = 2 * case["kv_heads"] * case["head_dim"]  # values of k and v
    if case["op"] == "cache":
        rows = sum(n for _, n in lengths_of(case))
        # input read, cache written and read, rows written
        return {"bytes": rows * token * (2 * size + 2 * 4.5 / 8), "flops": rows * token * 4}
    if case["op"] == "attention":
        pairs = lengths_of(case)
        each, held = (sum(v) for v in zip(*(seen_keys(case, length, n) for length, n in pairs)))
        rows = sum(n for _, n in pairs)
        return {"bytes": held * token * 4.5 / 8 + 2 * rows * case["heads"] * case["head_dim"] * size,
                "flops": 4 * each * case["heads"] * case["head_dim"]}
    rows = case["batch"] * case["beams"]
    part = case["context"] % case["page"] or case["page"]
    moved = rows * part * token * case["layers"]
    return {"bytes": rows * case["vocab"] * size + moved * (4.5 / 8 + 4), "flops": rows * case["vocab"] * 4}


# ---- the definitions in 64 bits ---------------------------------------------------
def held(x):
    """What the cache holds of x [rows, heads, dim], in 64 bits: each block of 32 in steps of a 16-bit scale."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for b in range(x.shape[-1] // BLOCK):
        part = x[..., b * BLOCK:(b + 1) * BLOCK].double()
        high, low = part.amax(-1), part.amin(-1)
        first_high = (part == high[..., None]).to(torch.uint8).argmax(-1)
        first_low = (part == low[..., None]).to(torch.uint8).argmax(-1)
        use_high = (high > -low) | ((high == -low) & (first_high < first_low))
        scale = (torch.where(use_high, high, low) / -8.0).clamp(-65504, 65504).half().double()[..., None]
        n = torch.round(part / torch.where(scale == 0, 1.0, scale)).clamp(-8, 7)
        out[..., b * BLOCK:(b + 1) * BLOCK] = n * scale
    return out


def exact(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = SimpleNamespace(case=case, **{k: v for k, v in case.items() if k not in ("name", "op")})
    if case["op"] == "cache":
        pairs = lengths_of(case)
        rows = sum(n for _, n in pairs)
        page_tables(gen, [n for n, _ in pairs], s.page)
        k = rows_of(gen, rows, s.kv_heads, s.head_dim, s.type)
        v = rows_of(gen, rows, s.kv_heads, s.head_dim, s.type)
        return {"k": held(k), "v": held(v)}
    if case["op"] == "attention":
        return exact_attention(s, gen)
    layers = beam_inputs(s, gen)
    scores = []
    for b in range(s.batch):
        found = []
        for j in range(s.beams):
            before = float(s.scores[b, j])
            if int(s.finished[b, j]):
                found.append(torch.tensor([before], dtype=torch.float64, device="cuda"))
                continue
            x = s.logits[b * s.beams + j].double()
            found.append(torch.topk(torch.log_softmax(x, 0) + before, min(s.keep, s.vocab)).values)
        found = torch.sort(torch.cat(found), descending=True).values[:s.keep]
        scores.append(torch.nn.functional.pad(found, (0, s.keep - found.numel()), value=-math.inf))
    del layers  # the pages that move depend on the choice: whole numbers are compared for themselves
    return {"scores": torch.stack(scores), "parents": None, "tokens": None, "table": None, "copied": None, "k": None,
            "v": None}


def exact_attention(s, gen):
    k, v = attention_inputs(s, gen)
    if s.rows * s.heads * max(s.seq_lengths) > 1 << 30:
        return None
    group, at, row, outs = s.heads // s.kv_heads, 0, 0, []
    for length, n in zip(s.seq_lengths, s.counts):
        kb, vb = held(k[at:at + length]), held(v[at:at + length])
        qb = s.q[row:row + n].double()
        at, row = at + length, row + n
        position = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None, :]
        hidden = (key > position) | ((key <= position - s.window) if s.window else False)
        heads = []
        for h in range(s.heads):
            logit = (qb[:, h] @ kb[:, h // group].T) * s.scale
            logit = logit.masked_fill(hidden, -math.inf)
            if s.sinks:
                logit = torch.cat([logit, s.sink[h].double().expand(n, 1)], 1)
            heads.append(torch.softmax(logit, 1)[:, :length] @ vb[:, h // group])
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)
