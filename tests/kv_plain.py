"""The 4-bit cache, the attention over it and beam selection in plain 64-bit
arithmetic, with what the tests of the kernels need around them."""
import importlib
import math
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

spt = importlib.import_module("stream-pt_b200")

TYPES = {"f32": 0, "f16": 1, "bf16": 30}


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def held(x):
    """What the cache holds of float32 x [..., dim]: blocks of 32, float64."""
    x = np.asarray(x, np.float32)
    out = np.empty(x.shape, np.float64)
    flat, res = x.reshape(-1, 32), out.reshape(-1, 32)
    for block, to in zip(flat, res):
        if np.isnan(block).any():
            to[:] = np.nan
            continue
        top = block[int(np.argmax(np.abs(block)))]  # the first among equals
        d = float(np.float16(np.clip(np.float64(top) / -8.0, -65504.0, 65504.0)))
        if d == 0.0:
            to[:] = 0.0
            continue
        with np.errstate(over="ignore"):
            n = np.clip(np.rint(block.astype(np.float64) / d), -8, 7)  # rint: half to even
        to[:] = n * d
    return out


def random_table(rng, lengths, page, spare=0):
    """A table of distinct pages in random order (-1 behind the last), the spare pages, the pool's size."""
    need = [-(-int(n) // page) for n in lengths]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    table = np.full((len(need), max(need + [1])), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order[at:], max(1, sum(need) + spare)


class Device:
    """A table, lengths and offsets on the GPU, as a KvBatch."""

    def __init__(self, table, lengths, counts=None, tokens=None):
        import torch
        self.table = torch.tensor(np.asarray(table), dtype=torch.int32, device="cuda")
        self.lengths = torch.tensor(np.asarray(lengths), dtype=torch.int32, device="cuda")
        self.offsets = None
        if counts is not None:
            at = np.concatenate([[0], np.cumsum(counts)])
            self.offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
        rows = len(lengths) if counts is None else int(sum(counts))
        self.batch = spt.KvBatch(len(lengths), rows if tokens is None else tokens, self.table.shape[1],
                                 self.table.data_ptr(), self.lengths.data_ptr(),
                                 0 if self.offsets is None else self.offsets.data_ptr())


def attention(q, keys, values, position, scale, window=0, sinks=None):
    """One sequence: q [n, heads, dim], keys / values [length, kv_heads, dim] float64
    tensors, position of q's first row.  (out, and for the tolerance per row and
    head: sum of weight * |v| [n, heads, dim], largest |scale| sum |q||k|, largest |s|, largest |v|)."""
    import torch
    n, heads, dim = q.shape
    group = heads // keys.shape[1]
    k, v = (x.repeat_interleave(group, 1) for x in (keys, values))
    s = torch.einsum("nhd,lhd->nhl", q, k) * scale
    bound = torch.einsum("nhd,lhd->nhl", q.abs(), k.abs()) * scale
    p = torch.arange(position, position + n, device=q.device)[:, None, None]
    j = torch.arange(keys.shape[0], device=q.device)
    seen = (j <= p) & ((j > p - window) if window else True)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if keys.shape[0] else torch.full((n, heads, 1), -math.inf, dtype=q.dtype, device=q.device)
    sink = None if sinks is None else sinks.double()[None, :, None]
    if sink is not None:
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    w = torch.where(total > 0, w / total, 0.0)
    # a masked key's value counts for nothing, whatever it is
    v = torch.where(seen.any(0).any(0)[:, None, None], v, 0.0) if keys.shape[0] else v
    out = torch.einsum("nhl,lhd->nhd", w, v)
    size = torch.einsum("nhl,lhd->nhd", w, v.abs())
    live = seen.expand(n, heads, -1)
    worst = torch.where(live, bound, 0.0).amax(-1) if keys.shape[0] else torch.zeros(n, heads, device=q.device)
    far = torch.where(live, s.abs(), 0.0).amax(-1) if keys.shape[0] else torch.zeros(n, heads, device=q.device)
    largest = torch.where(live[..., None], v.abs().transpose(0, 1), 0.0).amax((-2, -1)) if keys.shape[0] else far
    return out, size, worst, far, largest


def attention_tolerance(out, size, worst, far, largest, length, type):
    """How far a row may be off, from the roundings the kernel makes.

    Scores: q as two f16 terms (2^-22 of each product), sums of at most 128
    products in 32 bits whose additions may truncate (2^-23 each, counted as 32
    additions of the largest partial sum): 2^-18 of sum |q||k|.  The scaled
    score, its difference to the running maximum (at most twice the largest
    score in 32 bits, a few roundings, base-2: factor 1.45): 2^-21 of the
    largest |s|; the exponential 2^-21.  A weight's relative error w then
    gives 2 w of sum weight |v| (numerator and denominator).  Values: the
    scaled weight 2^-24, its two f16 terms 2^-21, sums over a step of 64 keys
    and over the steps: 64 + length / 64 + 64 additions of 2^-23.  16-bit rows:
    q is one exact term, the weights one f16 term (half a step of f16, eps / 2 =
    2^-11 of each weight; the denominator sums the unrounded ones), the sum over all steps stays in the tensor cores
    (length / 16 additions), and the result is rounded once.

    A weight times its value's scale is an f16 with steps of 2^-24 at least, so
    2^-25 off whatever its size, while the largest weight is held as 2^(7 - e)
    or more and the scales are at most 2^e <= 2 max |v| / 8.  With codes up to 8
    that is 8 * 2^-25 / 2^(7 - e) <= 2^-31 max |v| a key, of which there are
    `length`: keys whose weight is that small count where the others' codes
    are 0."""
    import torch
    w = 2.0 ** -18 * worst + 2.0 ** -21 * far + 2.0 ** -21
    relative = 2 * w[..., None] + 2.0 ** -21 + (128 + length / 64) * 2.0 ** -23
    if type != "f32":
        relative = relative + 2.0 ** -11 + (length / 16) * 2.0 ** -23
    tol = size * relative + length * 2.0 ** -31 * largest[..., None] + 1e-30
    if type != "f32":
        eps = torch.finfo(torch_type(type)).eps / 2
        tol = tol + (out.abs() + tol) * eps + (2.0 ** -25 if type == "f16" else 0.0)
    return tol


def beam_select(logits, scores, keep, finished=None, end_token=0):
    """(scores, parents, tokens) of one search: logits [beams, vocab], scores [beams]; float64."""
    found = []
    for j, (x, before) in enumerate(zip(np.asarray(logits, np.float64), np.asarray(scores, np.float64))):
        if finished is not None and finished[j]:
            if before > -math.inf:
                found.append((-before, j, end_token))
            continue
        live = x[~np.isnan(x)]
        if not live.size or live.max() == -math.inf or np.isnan(before):
            continue
        with np.errstate(invalid="ignore"):
            norm = live.max() + math.log(np.exp(live - live.max()).sum()) if np.isfinite(live.max()) else math.nan
            total = (x - norm) + before
        order = np.lexsort((np.arange(total.size), -np.where(np.isnan(total), -math.inf, total)))[:keep]
        found += [(-total[t], j, int(t)) for t in order if total[t] > -math.inf]
    found = sorted(found)[:keep]
    out = np.full(keep, -math.inf), np.full(keep, -1, np.int64), np.full(keep, -1, np.int64)
    for i, (s, j, t) in enumerate(found):
        out[0][i], out[1][i], out[2][i] = -s, j, t
    return out
