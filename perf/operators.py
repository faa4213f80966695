"""What a decode step does between its matmuls, and behind the last one: performance cases of the attention over an 8-bit cache, of the
append that fills it, and of the logits' penalties, biases and grammar masks.

Three paths:

  attend   softmax(rules(scale q K^T)) V of a ragged batch over a paged cache of 8-bit keys and values
  append   the rows' new keys (rotated) and values go into the cache, the queries are rotated, and the cache's newest tokens are read
           back as the values that they stand for (`oxhip_dev_kv_append`, then `oxhip_dev_kv_read`)
  logits   repetition / frequency / presence penalties, biases and grammar masks on rows of logits, and the best token of each row

The cache (`oxhip_kv_cache`): k and v are bytes [page][head][block of 32 tokens][32 d], a byte u standing for (u - 128) times the f32 scale of
its block and head ([page][head][block]). Inside a block the bytes lie as the matrix instructions take them. Keys: [d / 32][4][16][2][8] =
[c / 32][c % 32 / 8][token % 16][token / 16][c % 8]; values: [d / 32][4][16][2][2][4] = [c / 32][token % 16 / 4][c % 16][c % 32 / 16][token / 16][token % 4].
"""
import math
import zlib

import numpy as np
import torch

own = False
DEV = "cuda"
FLOOR, CEIL = 2.0**-60, 2.0**60  # of a block's scale


def listed():
    return [
        # single-stream chat, a few hundred tokens in: a handful of microseconds, where latency counts
        dict(name="attend_one_short", op="attend", seqs=1, rows=1, length=397, n_kv=8, g=4, d=128, page=64, dtype="f32", cap=0.0, window=0, alibi=False, prefix=0, docs=False),
        # one token over a very long document
        dict(name="attend_one_long", op="attend", seqs=1, rows=1, length=131072, n_kv=8, g=4, d=128, page=256, dtype="f32", cap=0.0, window=0, alibi=False, prefix=0, docs=False),
        # a server's decode step: 64 sequences of very different lengths
        dict(name="attend_batch", op="attend", seqs=64, rows=1, length=8192, n_kv=8, g=4, d=128, page=64, dtype="f32", cap=0.0, window=0, alibi=False, prefix=0, docs=False),
        # five drafted tokens of 16 sequences verified at once; capped scores and a sliding window over wide heads
        dict(name="attend_verify", op="attend", seqs=16, rows=5, length=5003, n_kv=4, g=2, d=256, page=128, dtype="bf16", cap=50.0, window=4096, alibi=False, prefix=0, docs=False),
        # an ordinary prompt
        dict(name="attend_prompt", op="attend", seqs=1, rows=4096, length=4096, n_kv=8, g=4, d=128, page=64, dtype="bf16", cap=0.0, window=0, alibi=False, prefix=0, docs=False),
        # chunks of five prompts behind what the cache holds of them: f32 rows, narrow heads, distance bias, a prefix that all see, packed documents
        dict(name="attend_chunks", op="attend", seqs=5, rows=777, length=3001, n_kv=4, g=3, d=64, page=32, dtype="f32", cap=0.0, window=0, alibi=True, prefix=37, docs=True),
        # the same server's step: one new token of each of 64 sequences
        dict(name="append_step", op="append", seqs=64, rows=1, length=8192, n_kv=8, g=4, d=128, page=64, dtype="f32", rot=128, pairs=False),
        # two prompts
        dict(name="append_prompts", op="append", seqs=2, rows=4096, length=4096, n_kv=8, g=4, d=128, page=64, dtype="bf16", rot=128, pairs=False),
        # ragged chunks that begin and end inside blocks, partly rotated heads in adjacent pairs
        dict(name="append_chunks", op="append", seqs=7, rows=301, length=2999, n_kv=2, g=5, d=96, page=32, dtype="f32", rot=64, pairs=True),
        # single-stream chat's token
        dict(name="logits_one", op="logits", rows=1, vocab=128256, history=1000, dtype="f32", penalties=True, biases=0, mask=False),
        # a server's step, grammar masks on every other row
        dict(name="logits_batch", op="logits", rows=64, vocab=151936, history=2000, dtype="bf16", penalties=True, biases=20, mask=True),
        # a small odd vocabulary, long histories and many biases
        dict(name="logits_odd", op="logits", rows=9, vocab=32003, history=9001, dtype="f32", penalties=True, biases=300, mask=True),
    ]


def _spread(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "logits"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "logits":
        rows = _spread(rng, 1, 96)
        return dict(op=op, rows=rows, vocab=_spread(rng, 1000, 160000), history=_spread(rng, 1, 10000), dtype=dtype, penalties=rng.random() < 0.8,
                    biases=rng.choice([0, 1, _spread(rng, 2, 400)]), mask=rng.random() < 0.5)
    n_kv, g, d, page = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([64, 64, 96, 128, 128, 128, 256]), rng.choice([32, 64, 128, 256])
    heads = dict(n_kv=n_kv, g=g, d=d, page=page, dtype=dtype)
    if op == "append":
        seqs, rows = (_spread(rng, 1, 96), 1) if rng.random() < 0.5 else (_spread(rng, 1, 8), _spread(rng, 2, 2048))
        return dict(op=op, seqs=seqs, rows=rows, length=rows + _spread(rng, 1, 4096), **heads, rot=rng.choice([0, d // 2, d, d]), pairs=rng.random() < 0.3)
    kind = rng.choice(["step", "step", "few", "prompt"])
    if kind == "prompt":
        seqs, rows = _spread(rng, 1, 6), _spread(rng, 17, 2048)
        length = rows + rng.choice([0, _spread(rng, 1, 4096)])
    else:
        seqs, rows = _spread(rng, 1, 96), 1 if kind == "step" else rng.randint(2, 16)
        length = rows + _spread(rng, 1, 60000)
    length = max(rows, min(length, int(2.5e8 / (seqs * n_kv * d)), int(4e8 / (seqs * rows * n_kv * g))))
    rule = rng.choice(["", "", "cap", "window", "alibi", "prefix", "docs", "all"])
    every = rule == "all"
    return dict(op=op, seqs=seqs, rows=rows, length=length, **heads, cap=rng.choice([20.0, 50.0]) if every or rule == "cap" else 0.0,
                window=_spread(rng, 16, 4096) if every or rule == "window" else 0, alibi=every or rule == "alibi",
                prefix=_spread(rng, 1, max(2, length // 2)) if every or rule == "prefix" else 0, docs=every or rule == "docs")


# ---- a case's shapes (they go by the case alone) and its data (by the seed) ---------------------------------------------------------------


def _shapes(c):
    """(rows of each sequence, tokens it then holds, first key that each row sees): ragged, one sequence as long as the case says."""
    r = np.random.RandomState(zlib.crc32(repr([c[k] for k in ("op", "seqs", "rows", "length", "n_kv", "d")]).encode()))
    n = r.randint(1, c["rows"] + 1, c["seqs"])
    n[0] = c["rows"]
    if c["seqs"] > 4 and c["rows"] > 1:
        n[2] = 0  # a sequence that has no part in this call
    lens = np.exp(r.uniform(math.log(max(1, c["length"] / 16)), math.log(c["length"] + 0.5), c["seqs"])).astype(np.int64)
    lens[0] = c["length"]
    lens = np.maximum(np.maximum(lens, n), 1)
    first = np.concatenate([(lens[s] - n[s] + np.arange(n[s])) * r.randint(0, 3) // 3 for s in range(c["seqs"])]) if c["op"] == "attend" else None
    return n, lens, first


def _dtype(c):
    return torch.bfloat16 if c["dtype"] == "bf16" else torch.float32


def _ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    def uniform(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(shape, generator=gen, device=DEV)

    st = dict(case=c)
    if c["op"] == "logits":
        t, vocab, h = c["rows"], c["vocab"], c["history"]
        st["logits"] = (3 * normal(t, vocab)).to(_dtype(c))
        # words that come again and again: ids spread over the logarithm of the vocabulary
        ids = torch.exp(uniform(0, math.log(vocab), t, h)).to(torch.int32).clamp_(0, vocab - 1)
        lens = (h * uniform(0.5, 1.0, t)).to(torch.int32).clamp_(min=1)
        st.update(history=ids, history_len=lens, prompt_len=(lens * uniform(0.2, 0.8, t)).to(torch.int32))
        if c["penalties"]:
            st.update(repetition=uniform(1.0, 1.3, t), presence=uniform(0.0, 0.6, t), frequency=uniform(0.0, 0.4, t))
        if c["biases"]:
            st["bias_start"] = _ints(np.arange(t + 1) * c["biases"])
            st["bias_id"] = torch.randint(0, vocab, (t * c["biases"],), generator=gen, device=DEV).to(torch.int32)
            st["bias"] = 4 * normal(t * c["biases"])
        if c["mask"]:
            words = (vocab + 31) // 32
            st["allowed"] = torch.randint(-2**31, 2**31, (t, words), generator=gen, device=DEV).to(torch.int32)
            st["allowed_row"] = _ints([i if i % 2 else -1 for i in range(t)])
        return st

    n, lens, first = _shapes(c)
    n_kv, d, page, dtype = c["n_kv"], c["d"], c["page"], _dtype(c)
    per = page // 32
    need = -(-lens // page)
    n_pages, width = int(need.sum()) + 3, int(need.max()) + 1
    order = torch.randperm(n_pages, generator=gen, device=DEV)[: int(need.sum())]
    seq = torch.tensor(np.repeat(np.arange(c["seqs"]), need), device=DEV)
    at = torch.tensor(np.concatenate([np.arange(k) for k in need]), device=DEV)
    pages = torch.zeros((c["seqs"], width), dtype=torch.int32, device=DEV)
    pages[seq, at] = order.to(torch.int32)

    def codes():
        out = torch.empty((n_pages, n_kv, per, 32 * d), dtype=torch.uint8, device=DEV)
        for i in range(0, n_pages, 512):
            part = out[i : i + 512]
            part.copy_((40 * normal(*part.shape)).round_().clamp_(-127, 127).add_(128))
        return out

    st.update(k=codes(), v=codes(), pages=pages, kv_len=_ints(lens), rows=int(n.sum()), row_start=None if c["rows"] == 1 else _ints(np.concatenate([[0], np.cumsum(n)])),
              k_scale=0.025 * torch.exp(0.2 * normal(n_pages, n_kv, per)), v_scale=0.025 * torch.exp(0.5 * normal(n_pages, n_kv, per)))
    total = st["rows"]
    st["q"] = (1.5 * normal(total, n_kv * c["g"] * d)).to(dtype)
    if c["op"] == "attend":
        n_q = n_kv * c["g"]
        st["scale"] = 1 / math.sqrt(d)
        st["slopes"] = torch.exp2(-8 * torch.arange(1, n_q + 1, device=DEV) / n_q).to(torch.float32) if c["alibi"] else None
        st["prefix"] = _ints([c["prefix"]] * c["seqs"]) if c["prefix"] else None
        st["first"] = _ints(first) if c["docs"] else None
        return st
    st["new_k"] = (normal(total, n_kv * d) * torch.exp(0.5 * normal(n_kv * d))).to(dtype)  # (keys have loud channels)
    st["new_v"] = normal(total, n_kv * d).to(dtype)
    st["table"] = None
    if c["rot"]:
        angle = torch.arange(int(lens.max()), dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-2 * torch.arange(c["rot"] // 2, dtype=torch.float64, device=DEV) / c["rot"])
        st["table"] = torch.stack([angle.cos(), angle.sin()], 2).to(torch.float32)
    return st


def _count(c):
    """Tokens of each sequence that an append's pass reads back: the new ones and what shares a block with them."""
    return min(c["length"], c["rows"] + 31)


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------------

def _rows_of(which, blocks, d):
    """Codes [..., n_kv, 32 d] of blocks as they lie in the cache -> [..., 32 tokens, n_kv, d]."""
    lead, n_kv = blocks.shape[:-2], blocks.shape[-2]
    if which == "k":  # [n, n_kv, c / 32, c % 32 / 8, token % 16, token / 16, c % 8]
        x = blocks.reshape(-1, n_kv, d // 32, 4, 16, 2, 8).permute(0, 5, 4, 1, 2, 3, 6)
    else:  # [n, n_kv, c / 32, token % 16 / 4, c % 16, c % 32 / 16, token / 16, token % 4]
        x = blocks.reshape(-1, n_kv, d // 32, 4, 16, 2, 2, 4).permute(0, 6, 3, 7, 1, 2, 5, 4)
    return x.reshape(*lead, 32, n_kv, d)


def _blocks_of(which, rows):
    """The inverse: [n, 32, n_kv, d] -> [n, n_kv, 32 d]."""
    n, _, n_kv, d = rows.shape
    if which == "k":
        x = rows.reshape(n, 2, 16, n_kv, d // 32, 4, 8).permute(0, 3, 4, 5, 2, 1, 6)
    else:
        x = rows.reshape(n, 2, 4, 4, n_kv, d // 32, 2, 16).permute(0, 4, 5, 2, 7, 6, 1, 3)
    return x.reshape(n, n_kv, 32 * d)


def _held(st, which, page, block):
    """The f32 values [..., 32, n_kv, d] of blocks (page, block in the page) of the cache."""
    codes = _rows_of(which, st[which][page, :, block], st["case"]["d"]).float() - 128
    return codes * st[which + "_scale"][page, :, block][..., None, :, None]


def _places(st):
    """(sequence, number in it, position) of each row."""
    kv_len = st["kv_len"].long()
    if st["row_start"] is None:
        seq = torch.arange(st["rows"], device=DEV)
        return seq, torch.zeros_like(seq), kv_len - 1
    start = st["row_start"].long()
    row = torch.arange(st["rows"], device=DEV)
    seq = torch.searchsorted(start, row, right=True) - 1
    return seq, row - start[seq], kv_len[seq] - start[seq + 1] + row


def _attend_plain(st):
    c = st["case"]
    n_kv, g, d, most, per = c["n_kv"], c["g"], c["d"], c["rows"], c["page"] // 32
    blocks = -(-c["length"] // 32)
    b = torch.arange(blocks, device=DEV)
    page = st["pages"].long()[:, b // per]
    k, v = (_held(st, w, page, (b % per).expand_as(page)).reshape(c["seqs"], blocks * 32, n_kv, d) for w in "kv")
    seq, i, pos = _places(st)
    q = torch.zeros((c["seqs"], most, n_kv, g, d), device=DEV)
    q[seq, i] = st["q"].float().reshape(-1, n_kv, g, d)
    at, first = (torch.zeros((c["seqs"], most), dtype=torch.long, device=DEV) for _ in range(2))
    at[seq, i] = pos
    if st["first"] is not None:
        first[seq, i] = st["first"].long()
    j = torch.arange(blocks * 32, device=DEV)
    p, lo = at[:, :, None], first[:, :, None]
    sees = (j <= p) & (j >= lo)
    if c["window"]:
        sees &= j > p - c["window"]
    if st["prefix"] is not None:
        sees |= j < st["prefix"][:, None, None]
    sees &= j < st["kv_len"][:, None, None]
    s = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(c["seqs"], n_kv, g * most, d), k.permute(0, 2, 3, 1).contiguous()) * st["scale"]
    s = s.reshape(c["seqs"], n_kv, g, most, blocks * 32)
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    if st["slopes"] is not None:
        s = s - st["slopes"].reshape(n_kv, g, 1, 1) * (p - j).abs().float()[:, None, None]
    s = torch.where(sees[:, None, None], s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top > float("-inf"), top, 0.0))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(c["seqs"], n_kv, g * most, -1), v.permute(0, 2, 1, 3).contiguous()).reshape(c["seqs"], n_kv, g, most, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4)
    return o[seq, i].reshape(-1, n_kv * g * d).to(_dtype(c))


def _turned(st, x, pos):
    """x [rows, heads, d] rotated by the table's angles of the rows' positions: in 64 bits, since what is quantized lies next to a border now and then."""
    c, half, x = st["case"], st["case"]["rot"] // 2, x.double()
    if not half:
        return x
    cos, sin = st["table"].double()[pos][:, None, :, 0], st["table"].double()[pos][:, None, :, 1]
    if c["pairs"]:
        a, b = x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., 2 * half :]], -1)
    a, b = x[..., :half], x[..., half : 2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half :]], -1)


def _append_plain(st):
    c = st["case"]
    n_kv, d, per = c["n_kv"], c["d"], c["page"] // 32
    seq, i, pos = _places(st)
    kv_len = st["kv_len"].long()
    before = torch.zeros_like(kv_len).scatter_add_(0, seq, torch.ones_like(seq)).neg_().add_(kv_len)  # tokens held before this call
    # every sequence's run of blocks, from the one that holds its first new token
    run = (c["rows"] + 30) // 32 + 1
    b = (before // 32)[:, None] + torch.arange(run, device=DEV)
    token = (b * 32)[..., None] + torch.arange(32, device=DEV)
    page = st["pages"].long().gather(1, (b // per).clamp_(max=st["pages"].shape[1] - 1))
    new, old = (token >= before[:, None, None]) & (token < kv_len[:, None, None]), token < before[:, None, None]
    touched = new.any(-1)
    for which, x in (("k", _turned(st, st["new_k"].reshape(-1, n_kv, d), pos)), ("v", st["new_v"].double().reshape(-1, n_kv, d))):
        x = x.clamp(-127 * CEIL, 127 * CEIL)
        rows = torch.zeros((c["seqs"], run * 32, n_kv, d), dtype=torch.float64, device=DEV)
        rows[seq, pos - (before // 32 * 32)[seq]] = x
        rows = rows.reshape(c["seqs"], run, 32, n_kv, d)
        need = (rows.abs().amax((2, 4)) / 127).clamp_(min=FLOOR).float()
        was = torch.where(old.any(-1)[..., None], st[which + "_scale"][page, :, b % per], FLOOR)
        (m1, e1), (m0, e0) = torch.frexp(need), torch.frexp(was)
        grown = torch.ldexp(was, (e1 - e0 + (m1 > m0).int()).clamp_(min=0))
        scale = torch.where(was > FLOOR, grown, need)
        held = (_rows_of(which, st[which][page, :, b % per], d).float() - 128) * (was / scale)[:, :, None, :, None]
        put = (rows / scale.double()[:, :, None, :, None]).round_().clamp_(-127, 127)
        codes = torch.where(new[..., None, None], put.float(), held.round_()) + 128
        at = page[touched], (b % per)[touched]
        st[which][at[0], :, at[1]] = _blocks_of(which, codes[touched]).to(torch.uint8)
        st[which + "_scale"][at[0], :, at[1]] = scale[touched]
    q = _turned(st, st["q"].reshape(st["rows"], -1, d), pos).reshape(st["rows"], -1).to(_dtype(c))
    last = kv_len[:, None] - _count(c) + torch.arange(_count(c), device=DEV)
    at = last.clamp(min=0)
    page = st["pages"].long().gather(1, at // c["page"])
    out = [q]
    for which in "kv":
        b = at // 32 % per
        off = torch.arange(32 * d, device=DEV).reshape(1, 1, 32 * d)
        off = _rows_of(which, off, d)[0, :, 0]  # where a token's values lie in its block
        codes = st[which][page[..., None, None], torch.arange(n_kv, device=DEV)[:, None], b[..., None, None], off[at % 32][:, :, None]].float() - 128
        out.append(torch.where((last >= 0)[..., None, None], codes * st[which + "_scale"][page, :, b][..., None], 0.0))
    return out


def _logits_plain(st):
    c = st["case"]
    t, vocab = c["rows"], c["vocab"]
    x = st["logits"].float()
    if c["penalties"]:
        at = torch.arange(c["history"], device=DEV)
        used, said = at < st["history_len"][:, None], at >= st["prompt_len"][:, None]
        ids = torch.where(used, st["history"], vocab).long()
        count = torch.zeros((t, vocab + 1), dtype=torch.int32, device=DEV).scatter_add_(1, ids, said.int())[:, :vocab]
        seen = torch.zeros((t, vocab + 1), dtype=torch.int32, device=DEV).scatter_add_(1, ids, used.int())[:, :vocab] > 0
        rep = st["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = torch.where(count > 0, (x - st["frequency"][:, None] * count) - st["presence"][:, None], x)
    if c["biases"]:
        entry = torch.arange(st["bias"].numel(), device=DEV)
        place = (torch.searchsorted(st["bias_start"].long(), entry, right=True) - 1) * vocab + st["bias_id"]
        last = torch.full((t * vocab,), -1, dtype=torch.long, device=DEV).scatter_reduce_(0, place, entry, "amax").reshape(t, vocab)
        x = torch.where(last >= 0, x + st["bias"][last.clamp(min=0)], x)
    if c["mask"]:
        word = torch.arange(vocab, device=DEV)
        ok = (st["allowed"][:, word // 32] >> (word % 32)) & 1
        x = torch.where((ok == 1) | (st["allowed_row"] < 0)[:, None], x, float("-inf"))
    out = x.to(_dtype(c))
    top = out.amax(-1, keepdim=True)
    best = torch.where(out == top, torch.arange(vocab, device=DEV), vocab).amin(-1)
    return [out, torch.where(top[:, 0] > float("-inf"), best, -1).to(torch.int32)]


# ---- the framework's kernels --------------------------------------------------------------------------------------------------------------

_kept = {}


def _backend():
    """One backend per process, as a program keeps it."""
    if "be" not in _kept:
        from oxinfer_amd import HipBackend
        _kept["be"] = HipBackend(0)
    return _kept["be"]


def _handles(st):
    """The cache, batch and table of a state as the binding's own objects, made once, as a program keeps them."""
    if "cache" not in st:
        from oxinfer_amd import hip
        st["cache"] = hip.KvCache(st["k"], st["v"], st["k_scale"], st["v_scale"], st["case"]["page"], st["case"]["d"])
        st["batch"] = hip.KvBatch(st["kv_len"], st["pages"], rows=st["rows"], row_start=st["row_start"])
        st["rope"] = hip.Rope(st["table"], interleaved=st["case"]["pairs"]) if st.get("table") is not None else None
    return st["cache"], st["batch"], st["rope"]


def _attend_own(st):
    cache, batch, _ = _handles(st)
    c = st["case"]
    return _backend().attend(cache, batch, st["q"], scale=st["scale"], cap=c["cap"], slopes=st["slopes"], window=c["window"], prefix=st["prefix"], first=st["first"])


def _append_own(st):
    cache, batch, rope = _handles(st)
    q = _backend().kv_append(cache, batch, st["new_k"], st["new_v"], q=st["q"], rope=rope)
    return [q, *_backend().kv_read(cache, batch, _count(st["case"]))]


def _logits_own(st):
    rules = {k: st[k] for k in ("bias_start", "bias_id", "bias", "allowed", "allowed_row") if k in st}
    if st["case"]["penalties"]:
        rules.update({k: st[k] for k in ("history", "history_len", "prompt_len", "repetition", "presence", "frequency")})
    return list(_backend().adjust_logits(st["logits"], **rules))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _attend_own, "append": _append_own, "logits": _logits_own}[op](state)
    return {"attend": _attend_plain, "append": _append_plain, "logits": _logits_plain}[op](state)


def _pairs(c):
    """Query rows x keys that they see, over all sequences."""
    n, lens, first = _shapes(c)
    total, row = 0, 0
    for s in range(c["seqs"]):
        pos = np.arange(lens[s] - n[s], lens[s])
        lo = first[row : row + n[s]] if c["docs"] else np.zeros_like(pos)
        if c["window"]:
            lo = np.maximum(lo, pos - c["window"] + 1)
        row += n[s]
        pre = min(c["prefix"], lens[s])
        total += int((np.maximum(pos + 1 - np.maximum(lo, pre), 0) + pre).sum())
    return total


def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "logits":
        t = c["rows"]
        extra = (0.75 * 4 * c["history"] + 20 if c["penalties"] else 0) + 8 * c["biases"] + (c["vocab"] / 16 if c["mask"] else 0)
        return {"bytes": t * (2 * size * c["vocab"] + extra + 4), "flops": 4 * t * c["vocab"]}
    n, lens, first = _shapes(c)
    heads, d = c["n_kv"] * c["g"], c["d"]
    if c["op"] == "append":
        rows, kept = int(n.sum()), int(np.minimum(_count(c), lens).sum())
        values = c["n_kv"] * d
        return {"bytes": rows * (size * (2 * heads * d + 2 * values) + 4 * c["rot"] + 2 * values) + 2 * values * (kept + 4 * c["seqs"] * _count(c)), "flops": 3 * rows * d * (heads + 2 * c["n_kv"])}
    live = lens[n > 0]  # of a window's or a document's sequence: what its rows see
    if not c["prefix"] and (c["window"] or c["docs"]):
        row, live = 0, []
        for s in range(c["seqs"]):
            if n[s]:
                lo = first[row] if c["docs"] else 0
                live.append(lens[s] - max(lo, lens[s] - n[s] - c["window"] + 1 if c["window"] else 0))
            row += n[s]
    return {"bytes": float(np.sum(live)) * c["n_kv"] * (2 * d + 0.25) + 2 * size * int(n.sum()) * heads * d, "flops": 4 * d * heads * _pairs(c)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------------------


def _addresses(d):
    """Where (token, channel) lies in a block of keys and of values."""
    t, ch = np.meshgrid(np.arange(32), np.arange(d), indexing="ij")
    k = ch // 32 * 1024 + ch % 32 // 8 * 256 + t % 16 * 16 + t // 16 * 8 + ch % 8
    v = ch // 32 * 1024 + t % 16 // 4 * 256 + ch % 16 * 16 + ch % 32 // 16 * 8 + t // 16 * 4 + t % 4
    return {"k": torch.tensor(k, device=DEV), "v": torch.tensor(v, device=DEV)}


def _sequence(st, which, s, length, address):
    """(codes less 128 [length, n_kv, d], their scales [length, n_kv, 1]) of the first tokens of sequence s, f64."""
    per = st["case"]["page"] // 32
    b = torch.arange(-(-length // 32), device=DEV)
    page = st["pages"][s].long()[b // per]
    codes = st[which][page, :, b % per][:, :, address].double() - 128
    scale = st[which + "_scale"][page, :, b % per].double()
    return codes.transpose(1, 2).flatten(0, 1)[:length], scale.repeat_interleave(32, 0)[:length, :, None]


def _attend_exact(st):
    c, out, row = st["case"], [], 0
    n, lens, _ = _shapes(c)
    address = _addresses(c["d"])
    for s in range(c["seqs"]):
        if not n[s]:
            continue
        count, length = int(n[s]), int(lens[s])
        (kc, ks), (vc, vs) = (_sequence(st, w, s, length, address[w]) for w in "kv")
        q = st["q"][row : row + count].double().reshape(count, c["n_kv"], c["g"], c["d"])
        pos, key = torch.arange(length - count, length, device=DEV)[:, None], torch.arange(length, device=DEV)[None]
        hidden = key > pos
        if c["docs"]:
            hidden = hidden | (key < st["first"][row : row + count, None])
        if c["window"]:
            hidden = hidden | (pos - key >= c["window"])
        hidden = hidden & (key >= c["prefix"])
        for h in range(c["n_kv"]):
            score = (q[:, h].reshape(-1, c["d"]) @ (kc[:, h] * ks[:, h]).T).reshape(count, c["g"], length) * st["scale"]
            if c["cap"]:
                score = torch.tanh(score / c["cap"]) * c["cap"]
            if c["alibi"]:
                score = score - st["slopes"][h * c["g"] : (h + 1) * c["g"], None].double() * (pos - key).abs().double()[:, None]
            weight = torch.softmax(score.masked_fill(hidden[:, None], float("-inf")), -1).nan_to_num_(0.0)
            out.append((row, h, (weight.reshape(-1, length) @ (vc[:, h] * vs[:, h])).reshape(count, c["g"], c["d"])))
        row += count
    whole = torch.zeros((row, c["n_kv"], c["g"], c["d"]), dtype=torch.float64, device=DEV)
    for at, h, o in out:
        whole[at : at + len(o), h] = o
    return whole.reshape(row, -1)


def _append_exact(st):
    c, row = st["case"], 0
    n, lens, _ = _shapes(c)
    d, n_kv, count = c["d"], c["n_kv"], _count(c)
    address = _addresses(d)
    rotated = {}
    pos = torch.cat([torch.arange(int(lens[s] - n[s]), int(lens[s]), device=DEV) for s in range(c["seqs"])])
    for name, heads in (("q", n_kv * c["g"]), ("new_k", n_kv)):
        x = st[name].double().reshape(-1, heads, d).clone()
        if c["rot"]:
            half = c["rot"] // 2
            i = torch.arange(half, device=DEV)
            a, b = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + half)
            turn = torch.view_as_complex(st["table"].double())[pos][:, None] * torch.complex(x[..., a], x[..., b])
            x[..., a], x[..., b] = turn.real, turn.imag
        rotated[name] = x
    outs = {w: torch.zeros((c["seqs"], count, n_kv, d), dtype=torch.float64, device=DEV) for w in "kv"}
    for s in range(c["seqs"]):
        have, length = int(lens[s] - n[s]), int(lens[s])
        for w, source in (("k", rotated["new_k"]), ("v", st["new_v"].double().reshape(-1, n_kv, d))):
            codes, scales = _sequence(st, w, s, length, address[w])
            scales = scales.expand(-1, -1, d).clone()
            new = source[row : row + int(n[s])]
            for b in range(have // 32 * 32, length, 32):
                lo, hi = max(b, have), min(b + 32, length)
                if hi <= lo:
                    continue
                need = (new[lo - have : hi - have].abs().amax((0, 2)) / 127).clamp_(min=FLOOR).float().double()  # (held in 32 bits)
                scale = need
                if lo > b:
                    was = scales[b, :, 0]
                    scale = torch.where(was > FLOOR, was * torch.exp2(torch.ceil(torch.log2(need / was)).clamp_(min=0)), need)
                    codes[b:lo] = torch.round(codes[b:lo] * (was / scale)[:, None])
                codes[lo:hi] = torch.round(new[lo - have : hi - have] / scale[:, None])
                scales[b:hi] = scale[:, None]
            take = min(count, length)
            outs[w][s, count - take :] = (codes * scales)[length - take :]
        row += int(n[s])
    return [rotated["q"].reshape(row, -1), outs["k"], outs["v"]]


def _logits_exact(st):
    c = st["case"]
    x = st["logits"].double()
    for r in range(c["rows"]):
        if c["penalties"]:
            said = st["history"][r, : int(st["history_len"][r])].long()
            for ids, which in ((said, "seen"), (said[int(st["prompt_len"][r]) :], "count")):
                many = torch.bincount(ids, minlength=c["vocab"])
                if which == "seen":
                    p = st["repetition"][r].double()
                    x[r] = torch.where(many > 0, torch.where(x[r] > 0, x[r] / p, x[r] * p), x[r])
                else:
                    x[r] -= many * st["frequency"][r].double() + (many > 0) * st["presence"][r].double()
        if c["biases"]:
            part = slice(int(st["bias_start"][r]), int(st["bias_start"][r + 1]))
            last = dict(zip(st["bias_id"][part].tolist(), st["bias"][part].tolist()))
            x[r, list(last)] += torch.tensor(list(last.values()), dtype=torch.float64, device=DEV)
        if c["mask"] and int(st["allowed_row"][r]) >= 0:
            bits = np.unpackbits(st["allowed"][r].cpu().numpy().view(np.uint8), bitorder="little")[: c["vocab"]]
            x[r, torch.tensor(bits == 0, device=DEV)] = float("-inf")
    return [x, None]


def exact(case, seed):
    state = prepare(case, seed)
    return {"attend": _attend_exact, "append": _append_exact, "logits": _logits_exact}[case["op"]](state)
