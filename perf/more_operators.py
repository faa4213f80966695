"""What a server with many or long sequences does beside plain attention, and behind the logits: performance cases of attention over a shared
prefix, of sparse attention over chosen blocks of an 8-bit cache, and of the draw of the next tokens.

Four paths:

  shared    softmax(rules(scale q K^T)) V of a batch whose sequences begin, group by group, with the same tokens
  select    the mean keys of the spans that the rows' tokens touch are made anew and read back as the values that they stand for, then each
            row's best spans are chosen by an 8-bit score (`oxhip_dev_kv_summarize`, `oxhip_dev_kv_summary_read`, `oxhip_dev_kv_select`)
  selected  the attention of rows over the spans that were chosen for them
  sample    temperature, top-k, top-p and min-p on rows of logits, and the token that a given random number draws

The cache (`oxhip_kv_cache`): k and v are bytes [page][head][block of 32 tokens][32 d], a byte u standing for (u - 128) times the f32 scale of
its block and head ([page][head][block]). Inside a block the bytes lie as the matrix instructions take them. Keys: [d / 32][4][16][2][8] =
[c / 32][c % 32 / 8][token % 16][token / 16][c % 8]; values: [d / 32][4][16][2][2][4] = [c / 32][token % 16 / 4][c % 16][c % 32 / 16][token / 16][token % 4].
Summaries: signed bytes [page][head][span of the page][d], and an f32 scale for each.
"""
import math
import zlib

import numpy as np
import torch

own = False
DEV = "cuda"
LEAST = 2.0**-60  # a block's scale below this counts as 0


def listed():
    return [
        # four answers to one question: a handful of microseconds, where latency counts
        dict(name="shared_four", op="shared", groups=1, seqs=4, rows=1, common=700, length=100, n_kv=8, g=4, d=128, page=64, dtype="f32", cap=0.0, window=0, alibi=False),
        # a server's decode step: 64 conversations behind one long system prompt
        dict(name="shared_server", op="shared", groups=1, seqs=64, rows=1, common=8192, length=1024, n_kv=8, g=4, d=128, page=64, dtype="bf16", cap=0.0, window=0, alibi=False),
        # drafted tokens of several groups' sequences: wide heads, capped scores, a window, prefixes that end inside pages and blocks
        dict(name="shared_verify", op="shared", groups=3, seqs=24, rows=4, common=5001, length=777, n_kv=4, g=2, d=256, page=128, dtype="bf16", cap=50.0, window=4096, alibi=False),
        # 128 samples over one very long document, f32 rows
        dict(name="shared_long", op="shared", groups=1, seqs=128, rows=1, common=32768, length=512, n_kv=8, g=4, d=128, page=256, dtype="f32", cap=0.0, window=0, alibi=False),
        # one token over a very long document: 64 of 2048 spans
        dict(name="select_one", op="select", seqs=1, rows=1, length=131072, n_kv=8, g=4, d=128, page=256, dtype="f32", span=64, count=64, first=1, last=2),
        # a server's step over long sequences
        dict(name="select_batch", op="select", seqs=64, rows=1, length=32768, n_kv=8, g=4, d=128, page=64, dtype="bf16", span=64, count=64, first=1, last=2),
        # a chunk of a long prompt, odd heads
        dict(name="select_chunk", op="select", seqs=2, rows=509, length=20001, n_kv=4, g=3, d=96, page=128, dtype="f32", span=32, count=48, first=2, last=3),
        # what the three choices above are for
        dict(name="selected_one", op="selected", seqs=1, rows=1, length=131072, n_kv=8, g=4, d=128, page=256, dtype="f32", span=64, count=64, cap=0.0, window=0, alibi=False),
        dict(name="selected_batch", op="selected", seqs=64, rows=1, length=32768, n_kv=8, g=4, d=128, page=64, dtype="bf16", span=64, count=64, cap=0.0, window=0, alibi=False),
        dict(name="selected_chunk", op="selected", seqs=2, rows=509, length=20001, n_kv=4, g=3, d=96, page=128, dtype="f32", span=32, count=48, cap=30.0, window=0, alibi=True),
        # single-stream chat's token
        dict(name="sample_one", op="sample", rows=1, vocab=128256, dtype="f32", top_k=50, top_p=0.9, min_p=0.0, greedy=False, peaks=12),
        # a server's step: nucleus sampling without a limit on the number, every eighth row greedy
        dict(name="sample_batch", op="sample", rows=64, vocab=151936, dtype="bf16", top_k=0, top_p=0.95, min_p=0.02, greedy=True, peaks=40),
    ]


def _spread(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["shared", "shared", "select", "selected", "sample"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "sample":
        return dict(op=op, rows=_spread(rng, 1, 96), vocab=_spread(rng, 1000, 160000), dtype=dtype, top_k=rng.choice([0, 0, 1, 40, _spread(rng, 2, 1000)]),
                    top_p=rng.choice([1.0, 0.9, 0.95, rng.uniform(0.1, 0.999)]), min_p=rng.choice([0.0, 0.0, 0.05, rng.uniform(0.001, 0.3)]), greedy=rng.random() < 0.3,
                    peaks=rng.choice([0, 1, _spread(rng, 2, 200)]))
    n_kv, g, d, page = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([64, 64, 96, 128, 128, 128, 256]), rng.choice([32, 64, 128, 256])
    heads = dict(n_kv=n_kv, g=g, d=d, page=page, dtype=dtype)
    rule = rng.choice(["", "", "cap", "window", "alibi", "all"])
    rules = dict(cap=rng.choice([20.0, 50.0]) if rule in ("cap", "all") else 0.0, window=_spread(rng, 16, 4096) if rule in ("window", "all") else 0, alibi=rule in ("alibi", "all"))
    if op == "shared":
        seqs, rows = _spread(rng, 1, 128), rng.choice([1, 1, rng.randint(2, 8)])
        most = int(min(4e8 / (seqs * n_kv * d), 2e8 / (seqs * rows * n_kv * g)))
        common = min(_spread(rng, 32, 32768), most)
        return dict(op=op, groups=rng.choice([1, 1, rng.randint(1, 6)]), seqs=seqs, rows=rows, common=common, length=rows + min(_spread(rng, 1, 4096), most), **heads, **rules)
    span = page if page == 32 else rng.choice([32, 64]) if page == 64 else rng.choice([32, 64, 128])
    count = _spread(rng, 4, 96)
    if rng.random() < 0.7:
        seqs, rows = _spread(rng, 1, 96), rng.choice([1, 1, rng.randint(2, 8)])
    else:
        seqs, rows = _spread(rng, 1, 3), _spread(rng, 9, 600)
    length = rows + _spread(rng, 1, 100000)
    length = max(rows, min(length, int(2.5e8 / (seqs * n_kv * d))))
    if op == "select":
        return dict(op=op, seqs=seqs, rows=rows, length=length, **heads, span=span, count=count, first=rng.randint(0, 2), last=rng.randint(1, 2))
    return dict(op=op, seqs=seqs, rows=rows, length=length, **heads, span=span, count=count, **rules)


# ---- a case's shapes (they go by the case alone) and its data (by the seed) ---------------------------------------------------------------


def _random(c):
    return np.random.RandomState(zlib.crc32(repr([c[k] for k in ("op", "seqs", "rows", "length", "n_kv", "d")]).encode()))


def _shapes(c):
    """(rows of each sequence, tokens it then holds, where groups begin and end, the tokens that each shares): ragged, one sequence and one group as long
    as the case says."""
    r = _random(c)
    n = r.randint(1, c["rows"] + 1, c["seqs"])
    n[0] = c["rows"]
    lens = np.exp(r.uniform(math.log(max(1, c["length"] / 16)), math.log(c["length"] + 0.5), c["seqs"])).astype(np.int64)
    lens[0] = c["length"]
    lens = np.maximum(np.maximum(lens, n), 1)
    if c["op"] != "shared":
        return n, lens, None, None
    groups = min(c["groups"], c["seqs"])
    end = c["seqs"] - (1 if c["seqs"] > groups > 1 else 0)  # (with several groups, the last sequence is in none)
    start = np.concatenate([[0], np.sort(r.permutation(end - 1)[: groups - 1]) + 1, [end]]) if end > 1 else np.array([0, end])
    groups = len(start) - 1
    common = np.exp(r.uniform(math.log(max(1, c["common"] / 8)), math.log(c["common"] + 0.5), groups)).astype(np.int64)
    common[0] = c["common"]
    for i in range(groups):
        lens[start[i] : start[i + 1]] += common[i]
    return n, lens, start, common


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
    if c["op"] == "sample":
        t, vocab = c["rows"], c["vocab"]
        x = 2.2 * normal(t, vocab)
        if c["peaks"]:  # some words that the context asks for
            x.scatter_add_(1, torch.randint(0, vocab, (t, c["peaks"]), generator=gen, device=DEV), 8 + 2 * normal(t, c["peaks"]))
        st.update(logits=x.to(_dtype(c)), u=uniform(0, 1, t).clamp_(max=1 - 2.0**-24), temperature=uniform(0.5, 1.2, t))
        if c["greedy"]:
            st["temperature"][7::8] = 0.0
        if c["top_k"]:
            st["top_k"] = torch.full((t,), c["top_k"], dtype=torch.int32, device=DEV)
        if c["top_p"] < 1:
            st["top_p"] = torch.full((t,), c["top_p"], device=DEV)
        if c["min_p"]:
            st["min_p"] = torch.full((t,), c["min_p"], device=DEV)
        return st

    n, lens, start, common = _shapes(c)
    n_kv, d, page, dtype = c["n_kv"], c["d"], c["page"], _dtype(c)
    per = page // 32
    need = -(-lens // page)
    skip = np.zeros_like(need)  # whole pages of a prefix that another sequence names
    if c["op"] == "shared":
        for i in range(len(common)):
            skip[start[i] + 1 : start[i + 1]] = common[i] // page
    n_pages, width = int((need - skip).sum()) + 3, int(need.max()) + 1
    order = torch.randperm(n_pages, generator=gen, device=DEV)[: int((need - skip).sum())]
    seq = torch.tensor(np.repeat(np.arange(c["seqs"]), need - skip), device=DEV)
    at = torch.tensor(np.concatenate([np.arange(b, k) for b, k in zip(skip, need)]), device=DEV)
    pages = torch.zeros((c["seqs"], width), dtype=torch.int32, device=DEV)
    pages[seq, at] = order.to(torch.int32)
    if c["op"] == "shared":
        for i in range(len(common)):
            pages[start[i] + 1 : start[i + 1], : common[i] // page] = pages[start[i], : common[i] // page]
        st.update(group_start=_ints(start), common=_ints(common))

    def codes():
        out = torch.empty((n_pages, n_kv, per, 32 * d), dtype=torch.uint8, device=DEV)
        for i in range(0, n_pages, 512):
            part = out[i : i + 512]
            part.copy_((40 * normal(*part.shape)).round_().clamp_(-127, 127).add_(128))
        return out

    total = int(n.sum())
    st.update(k=codes(), pages=pages, kv_len=_ints(lens), rows=total, row_start=None if c["rows"] == 1 else _ints(np.concatenate([[0], np.cumsum(n)])),
              k_scale=0.025 * torch.exp(0.2 * normal(n_pages, n_kv, per)))
    st["v"] = codes() if c["op"] != "select" else torch.empty_like(st["k"])
    st["v_scale"] = 0.025 * torch.exp(0.5 * normal(n_pages, n_kv, per))
    n_q = n_kv * c["g"]
    st["q"] = (1.5 * normal(total, n_q * d)).to(dtype)
    if c["op"] == "select":  # the summaries as the steps before have left them
        st["means"] = torch.empty((n_pages, n_kv, page // c["span"], d), dtype=torch.int8, device=DEV)
        st["mean_scale"] = torch.empty((n_pages, n_kv, page // c["span"]), device=DEV)
        for i in range(0, n_pages, 512):
            spans = _rows_of("k", st["k"][i : i + 512].transpose(1, 2), d).float().sub_(128) * st["k_scale"][i : i + 512].transpose(1, 2)[:, :, None, :, None]
            mean = spans.reshape(-1, page // c["span"], c["span"], n_kv, d).mean(2)  # [pages, spans, n_kv, d]
            scale = mean.abs().amax(-1) / 127
            st["means"][i : i + 512] = (mean / scale[..., None]).round_().transpose(1, 2).to(torch.int8)
            st["mean_scale"][i : i + 512] = scale.transpose(1, 2)
        return st
    st["scale"] = 1 / math.sqrt(d)
    st["slopes"] = torch.exp2(-8 * torch.arange(1, n_q + 1, device=DEV) / n_q).to(torch.float32) if c["alibi"] else None
    if c["op"] == "selected":  # the first span, the row's own, and others
        seqs, i, pos = _places(st)
        last = (pos // c["span"])[:, None]
        spans = int(lens.max() - 1) // c["span"] + 1
        liking = uniform(0, 1, total, n_kv, spans)
        where = torch.arange(spans, device=DEV)
        liking = torch.where((where == 0) | (where == last[:, :, None]), 2.0, liking)
        liking = torch.where(where > last[:, :, None], -1.0, liking)
        top = liking.topk(min(c["count"], spans), -1)
        pick = torch.where(top.values >= 0, top.indices, spans).sort(-1).values
        chosen = torch.full((total, n_kv, c["count"]), -1, dtype=torch.int32, device=DEV)
        chosen[..., : pick.shape[-1]] = torch.where(pick < spans, pick, -1)
        st["chosen"] = chosen
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------------------------------


def _rows_of(which, blocks, d):
    """Codes [..., n_kv, 32 d] of blocks as they lie in the cache -> [..., 32 tokens, n_kv, d]."""
    lead, n_kv = blocks.shape[:-2], blocks.shape[-2]
    if which == "k":  # [n, n_kv, c / 32, c % 32 / 8, token % 16, token / 16, c % 8]
        x = blocks.reshape(-1, n_kv, d // 32, 4, 16, 2, 8).permute(0, 5, 4, 1, 2, 3, 6)
    else:  # [n, n_kv, c / 32, token % 16 / 4, c % 16, c % 32 / 16, token / 16, token % 4]
        x = blocks.reshape(-1, n_kv, d // 32, 4, 16, 2, 2, 4).permute(0, 6, 3, 7, 1, 2, 5, 4)
    return x.reshape(*lead, 32, n_kv, d)


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


def _weighed(c, s, v, sees):
    """Scores [..., keys] as they are, values [..., keys, d], what is seen -> the rows' results."""
    s = torch.where(sees, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top > float("-inf"), top, 0.0))
    total = e.sum(-1, keepdim=True)
    lead = e.shape[: v.dim() - 2]
    o = torch.matmul(e.reshape(*lead, -1, e.shape[-1]), v).reshape(*e.shape[:-1], v.shape[-1])
    return torch.where(total > 0, o / total, 0.0)


def _ruled(st, s, far):
    """The rules on scaled scores [..., n_kv, g, (rows,) keys], `far` (broadcast) the distance of each key from the row."""
    c = st["case"]
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    if st["slopes"] is not None:
        s = s - st["slopes"].reshape(c["n_kv"], c["g"], *[1] * (s.dim() - 3 if s.dim() == 5 else 1)) * far.abs().float()
    return s


def _shared_plain(st):
    c = st["case"]
    n_kv, g, d, most, page = c["n_kv"], c["g"], c["d"], c["rows"], c["page"]
    per = page // 32
    n, lens, start, common = _shapes(c)
    blocks = -(-int(lens.max()) // 32)
    b = torch.arange(blocks, device=DEV)
    seq, i, pos = _places(st)
    q = torch.zeros((c["seqs"], most, n_kv, g, d), device=DEV)
    q[seq, i] = st["q"].float().reshape(-1, n_kv, g, d)
    at = torch.zeros((c["seqs"], most), dtype=torch.long, device=DEV)
    at[seq, i] = pos
    # a group's first sequence says where the tokens lie that its sequences share
    leader, shares = torch.arange(c["seqs"], device=DEV), torch.zeros(c["seqs"], dtype=torch.long, device=DEV)
    where, length = st["group_start"].long(), st["common"].long()
    group = torch.searchsorted(where, leader, right=True) - 1
    within = group < len(length)
    group = group.clamp(max=len(length) - 1)
    leader, shares = torch.where(within, where[group], leader), torch.where(within, length[group], shares)
    j = torch.arange(blocks * 32, device=DEV)
    table = st["pages"].long()
    parts = []
    step = max(1, int(2e9 // (blocks * 32 * n_kv * d * 4)))
    for lo in range(0, c["seqs"], step):
        part = slice(lo, lo + step)
        mine, theirs = table[part][:, b // per], table[leader[part]][:, b // per]
        whole = torch.where((b * 32 + 32)[None] <= shares[part, None], theirs, mine)
        kv = []
        for w in "kv":
            x = _held(st, w, whole, (b % per).expand_as(whole))  # [seqs, blocks, 32, n_kv, d]
            edge = (shares[part] // 32).clamp(max=blocks - 1)  # the block that holds both kinds
            row = torch.arange(len(edge), device=DEV)
            mixed = torch.where((edge[:, None] * 32 + torch.arange(32, device=DEV) < shares[part, None])[..., None, None], _held(st, w, theirs[row, edge], edge % per), x[row, edge])
            x[row, edge] = mixed
            kv.append(x.reshape(len(edge), blocks * 32, n_kv, d))
        p = at[part][:, :, None]
        sees = (j <= p) & (j < st["kv_len"][part, None, None])
        if c["window"]:
            sees &= j > p - c["window"]
        rows = q[part].permute(0, 2, 3, 1, 4)  # [seqs, n_kv, g, rows, d]
        s = torch.matmul(rows.reshape(-1, n_kv, g * most, d), kv[0].permute(0, 2, 3, 1).contiguous()).reshape(-1, n_kv, g, most, blocks * 32) * st["scale"]
        s = _ruled(st, s, (p - j)[:, None, None])
        parts.append(_weighed(c, s, kv[1].permute(0, 2, 1, 3).contiguous(), sees[:, None, None]).permute(0, 3, 1, 2, 4))
    return torch.cat(parts)[seq, i].reshape(-1, n_kv * g * d).to(_dtype(c))


def _last_spans(st):
    """(whether there is such a span, its first token) of the spans that a select pass reads back of each sequence: [seqs, count]."""
    c = st["case"]
    last = (st["kv_len"].long() - 1)[:, None] // c["span"]
    span = last - _count(c) + 1 + torch.arange(_count(c), device=DEV)
    return span >= 0, span.clamp(min=0) * c["span"]


def _count(c):
    """Spans of each sequence that a pass reads back: what its rows may have touched."""
    return (c["rows"] + 2 * c["span"] - 2) // c["span"]


def _select_plain(st):
    c = st["case"]
    n_kv, g, d, span, page = c["n_kv"], c["g"], c["d"], c["span"], c["page"]
    per, kv_len = span // 32, st["kv_len"].long()
    seq, i, pos = _places(st)
    n = torch.zeros_like(kv_len).scatter_add_(0, seq, torch.ones_like(seq))
    # the mean keys of the spans that the rows touch, in 64 bits, since what is quantized lies next to a border now and then
    have, first = _last_spans(st)
    touched = have & (first + span > (kv_len - n)[:, None])
    who, t0 = touched.nonzero()[:, 0], first[touched]
    at = t0[:, None] + 32 * torch.arange(per, device=DEV)
    table = st["pages"].long()
    where = table[who[:, None], (at // page).clamp(max=table.shape[1] - 1)]
    codes = (_rows_of("k", st["k"][where, :, at % page // 32], d).double() - 128).reshape(-1, per, 32, n_kv, d)
    scale = st["k_scale"][where, :, at % page // 32].double()
    held = (at[..., None] + torch.arange(32, device=DEV) < kv_len[who, None, None])[..., None, None]
    mean = (torch.where(held, codes, 0.0).sum(2) * torch.where(scale < LEAST, 0.0, scale)[..., None]).sum(1) / (kv_len[who] - t0).clamp(max=span)[:, None, None]
    size = (mean.abs().amax(-1) / 127).float()
    put = torch.where(size[..., None] > 0, (mean / size.double()[..., None]).round_().clamp_(-127, 127), 0.0)
    page0 = table[who, t0 // page]
    st["means"][page0, :, t0 % page // span] = put.to(torch.int8)
    st["mean_scale"][page0, :, t0 % page // span] = size
    # read back
    where = table.gather(1, (first // page).clamp(max=table.shape[1] - 1))
    back = torch.where(have[..., None, None], st["means"][where, :, first % page // span].float() * st["mean_scale"][where, :, first % page // span][..., None], 0.0)
    # the choice: integer products of codes are exact in 32 bits, what they are multiplied with is held in 64
    spans = (int(c["length"]) - 1) // span + 1
    b = torch.arange(spans, device=DEV)
    q = st["q"].float().reshape(-1, n_kv, g, d)
    q_scale = q.abs().amax(-1) / 127
    q_code = torch.where(q_scale[..., None] > 0, (q.double() / q_scale.double()[..., None]).round_().clamp_(-127, 127), 0.0).float()
    where = table[:, (b * span // page).clamp(max=table.shape[1] - 1)]
    key = st["means"][where, :, b * span % page // span]  # [seqs, spans, n_kv, d]
    key_scale = st["mean_scale"][where, :, b * span % page // span].double()
    chosen = torch.full((st["rows"], n_kv, c["count"]), -1, dtype=torch.int32, device=DEV)
    take = min(c["count"], spans)
    step = max(1, int(1e9 // (spans * n_kv * (d + 6 * g) * 4)))
    for lo in range(0, st["rows"], step):
        part = slice(lo, lo + step)
        who, p = seq[part], pos[part]
        if c["rows"] == 1:
            dot = torch.matmul(key[who].permute(0, 2, 1, 3).float(), q_code[part].transpose(2, 3).contiguous())  # [rows, n_kv, spans, g]
        else:
            dot = torch.cat([torch.matmul(q_code[part][who == s].permute(1, 0, 2, 3).reshape(n_kv, -1, d), key[s].permute(1, 2, 0).float().contiguous())
                             .reshape(n_kv, -1, g, spans).permute(1, 0, 3, 2) for s in who.unique_consecutive().tolist()])
        score = (dot.double() * key_scale[who].transpose(1, 2)[..., None] * q_scale[part].double()[:, :, None]).amax(-1)  # [rows, n_kv, spans]
        own_span = (p // span)[:, None, None]
        score = torch.where((b < c["first"]) | (b > own_span - c["last"]), float("inf"), score)
        score = torch.where(b <= own_span, score, float("-inf"))
        best = torch.sort(score, dim=-1, descending=True, stable=True)
        pick = torch.where(best.values[..., :take] > float("-inf"), best.indices[..., :take], spans).sort(-1).values
        chosen[part, :, :take] = torch.where(pick < spans, pick, -1).to(torch.int32)
    return [back, chosen]


def _selected_plain(st):
    c = st["case"]
    n_kv, g, d, span, page = c["n_kv"], c["g"], c["d"], c["span"], c["page"]
    per, table = span // 32, st["pages"].long()
    seq, i, pos = _places(st)
    q = st["q"].float().reshape(-1, n_kv, g, d)
    head = torch.arange(n_kv, device=DEV)[:, None]
    inside = torch.arange(32 * d, device=DEV).reshape(1, 1, 32 * d)
    out = torch.empty_like(q)
    step = max(1, int(1e9 // (c["count"] * span * n_kv * d * 4)))
    for lo in range(0, st["rows"], step):
        part = slice(lo, lo + step)
        p, chosen = pos[part], st["chosen"][part].long()
        first = chosen.clamp(min=0)[..., None] * span + 32 * torch.arange(per, device=DEV)
        first = first.flatten(2)  # [rows, n_kv, blocks]
        where = table[seq[part, None, None], (first // page).clamp(max=table.shape[1] - 1)]
        kv = []
        for w in "kv":
            off = _rows_of(w, inside, d)[0, :, 0]  # where a token's values lie in its block
            x = st[w][where, head, first % page // 32][..., off.flatten()].reshape(*first.shape, 32, d).float() - 128
            kv.append((x * st[w + "_scale"][where, head, first % page // 32][..., None, None]).flatten(2, 3))
        j = (first[..., None] + torch.arange(32, device=DEV)).flatten(2)[:, :, None]  # [rows, n_kv, 1, keys]
        at = p[:, None, None, None]
        sees = (j <= at) & (chosen >= 0).repeat_interleave(span, -1)[:, :, None]
        if c["window"]:
            sees &= j > at - c["window"]
        s = torch.matmul(q[part], kv[0].transpose(2, 3).contiguous()) * st["scale"]
        out[part] = _weighed(c, _ruled(st, s, at - j), kv[1], sees)
    return out.reshape(st["rows"], -1).to(_dtype(c))


def _sample_plain(st):
    c = st["case"]
    x = st["logits"].float()
    best = torch.sort(x, dim=-1, descending=True, stable=True)  # of equal logits the lower id first
    heat = st["temperature"].double()[:, None]
    y = (best.values.double() - best.values[:, :1].double()) / torch.where(heat > 0, heat, 1.0)
    w = torch.exp(y)  # (sums of many weights, and what lies next to a border: in 64 bits)
    rank = torch.arange(c["vocab"], device=DEV)
    keep = w > 0
    if c["top_k"]:
        keep &= rank < st["top_k"][:, None]
    if c["top_p"] < 1:
        kept = torch.where(keep, w, 0.0)
        before = kept.cumsum(-1) - kept
        keep &= before < st["top_p"].double()[:, None] * kept.sum(-1, keepdim=True)
    if c["min_p"]:
        keep &= w >= st["min_p"].double()[:, None]
    keep &= (heat > 0) | (rank == 0)
    weight = torch.zeros_like(w).scatter_(1, best.indices, torch.where(keep, w, 0.0))
    upto = weight.cumsum(-1)
    total = upto[:, -1:]
    over = (upto > st["u"].double()[:, None] * total) & (weight > 0)
    ids = torch.arange(c["vocab"], device=DEV)
    token = torch.where(over, ids, c["vocab"]).amin(-1)
    token = torch.where(token < c["vocab"], token, torch.where(weight > 0, ids, -1).amax(-1))
    return [token.to(torch.int32), torch.log(weight.gather(1, token[:, None]) / total)[:, 0].float()]


# ---- the framework's kernels --------------------------------------------------------------------------------------------------------------

_kept = {}


def _backend():
    """One backend per process, as a program keeps it."""
    if "be" not in _kept:
        from oxinfer_amd import HipBackend
        _kept["be"] = HipBackend(0)
    return _kept["be"]


def _handles(st):
    """The cache, batch and what belongs to them of a state as the binding's own objects, made once, as a program keeps them."""
    if "cache" not in st:
        from oxinfer_amd import hip
        c = st["case"]
        st["cache"] = hip.KvCache(st["k"], st["v"], st["k_scale"], st["v_scale"], c["page"], c["d"])
        st["batch"] = hip.KvBatch(st["kv_len"], st["pages"], rows=st["rows"], row_start=st["row_start"])
        st["more"] = None
        if c["op"] == "shared":
            st["more"] = hip.KvShared(st["group_start"], st["common"])
        if c["op"] == "select":
            st["more"] = hip.KvSummary(st["means"], st["mean_scale"], c["span"])
    return st["cache"], st["batch"], st["more"]


def _shared_own(st):
    cache, batch, shared = _handles(st)
    c = st["case"]
    return _backend().attend_shared(cache, batch, shared, st["q"], scale=st["scale"], cap=c["cap"], slopes=st["slopes"], window=c["window"])


def _select_own(st):
    cache, batch, summary = _handles(st)
    c, be = st["case"], _backend()
    be.kv_summarize(cache, batch, summary)
    return [be.kv_summary_read(cache, batch, summary, _count(c)), be.kv_select(cache, batch, summary, st["q"], c["count"], first=c["first"], last=c["last"])]


def _selected_own(st):
    cache, batch, _ = _handles(st)
    c = st["case"]
    return _backend().attend_selected(cache, batch, st["q"], st["chosen"], c["span"], scale=st["scale"], cap=c["cap"], slopes=st["slopes"], window=c["window"])


def _sample_own(st):
    return list(_backend().sample(st["logits"], st["u"], **{k: st[k] for k in ("temperature", "top_k", "top_p", "min_p") if k in st}))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"shared": _shared_own, "select": _select_own, "selected": _selected_own, "sample": _sample_own}[op](state)
    return {"shared": _shared_plain, "select": _select_plain, "selected": _selected_plain, "sample": _sample_plain}[op](state)


def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "sample":
        return {"bytes": c["rows"] * (size * c["vocab"] + 24), "flops": 4 * c["rows"] * c["vocab"]}
    n, lens, start, common = _shapes(c)
    rows, heads, d = int(n.sum()), c["n_kv"] * c["g"], c["d"]
    row = np.repeat(lens - n, n) + np.arange(rows) - np.repeat(np.cumsum(n) - n, n)  # its position
    token = c["n_kv"] * (2 * d + 0.25)
    if c["op"] == "shared":
        seen = row + 1 if not c["window"] else np.minimum(row + 1, c["window"])
        lo = np.maximum(lens - n - c["window"] + 1, 0) if c["window"] else np.zeros_like(lens)  # the first token that a sequence's rows see
        tokens, grouped = 0, np.zeros(c["seqs"], dtype=np.int64)
        for i in range(len(common)):
            part = slice(start[i], start[i + 1])
            grouped[part] = common[i]
            tokens += max(0, common[i] - int(lo[part].min()))
        tokens += int((lens - np.maximum(lo, grouped)).sum())
        return {"bytes": float(tokens) * token + 2 * size * rows * heads * d, "flops": 4.0 * d * heads * int(seen.sum())}
    spans = row // c["span"] + 1
    if c["op"] == "select":
        read = int(((lens - 1) // c["span"] + 1).sum()) * c["n_kv"] * (d + 4)
        touched = int((lens - (lens - n) // c["span"] * c["span"]).sum()) * c["n_kv"] * d
        return {"bytes": read + touched + 4 * c["seqs"] * _count(c) * c["n_kv"] * d + size * rows * heads * d + 4 * rows * c["n_kv"] * c["count"],
                "flops": 2.0 * d * heads * int(spans.sum())}
    keys = np.minimum(spans, c["count"]) * c["span"] - (spans * c["span"] - row - 1)
    if c["window"]:
        keys = np.minimum(keys, c["window"])
    once = float(np.minimum(keys, row + 1).sum())
    per_seq = np.minimum(np.add.reduceat(keys, np.cumsum(n) - n), lens).sum()  # (rows of a sequence share what they have in common)
    return {"bytes": float(per_seq) * token + 2 * size * rows * heads * d + 4 * rows * c["n_kv"] * c["count"], "flops": 4.0 * d * heads * once}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------------------


def _addresses(d):
    """Where (token, channel) lies in a block of keys and of values."""
    t, ch = np.meshgrid(np.arange(32), np.arange(d), indexing="ij")
    k = ch // 32 * 1024 + ch % 32 // 8 * 256 + t % 16 * 16 + t // 16 * 8 + ch % 8
    v = ch // 32 * 1024 + t % 16 // 4 * 256 + ch % 16 * 16 + ch % 32 // 16 * 8 + t // 16 * 4 + t % 4
    return {"k": torch.tensor(k, device=DEV), "v": torch.tensor(v, device=DEV)}


def _sequence(st, which, s, lo, hi, address):
    """The values [hi - lo, n_kv, d] of the tokens lo .. hi - 1 that sequence s's table names, f64."""
    per = st["case"]["page"] // 32
    b = torch.arange(lo // 32, -(-hi // 32), device=DEV)
    page = st["pages"][s].long()[b // per]
    x = (st[which][page, :, b % per][:, :, address].double() - 128) * st[which + "_scale"][page, :, b % per].double()[..., None, None]
    return x.transpose(1, 2).flatten(0, 1)[lo - lo // 32 * 32 :][: hi - lo]


def _softmax_exact(st, q, k, v, pos, key, hidden, h):
    """Queries [rows, g, d] over keys [keys, d]: f64."""
    c = st["case"]
    score = (q.flatten(0, 1) @ k.T).reshape(len(q), c["g"], -1) * st["scale"]
    if c["cap"]:
        score = torch.tanh(score / c["cap"]) * c["cap"]
    if c["alibi"]:
        score = score - st["slopes"][h * c["g"] : (h + 1) * c["g"], None].double() * (pos - key).abs().double()[:, None]
    weight = torch.softmax(score.masked_fill(hidden[:, None], float("-inf")), -1).nan_to_num_(0.0)
    return (weight.flatten(0, 1) @ v).reshape(len(q), c["g"], -1)


def _shared_exact(st):
    c, row = st["case"], 0
    n, lens, start, common = _shapes(c)
    address = _addresses(c["d"])
    whole = torch.zeros((int(n.sum()), c["n_kv"], c["g"], c["d"]), dtype=torch.float64, device=DEV)
    held, group = None, -1
    for s in range(c["seqs"]):
        i = int(np.searchsorted(start, s, side="right")) - 1
        shares = int(common[i]) if i < len(common) else 0
        if i != group:
            held, group = {w: _sequence(st, w, s, 0, shares, address[w]) for w in "kv"} if shares else None, i
        kv = {w: _sequence(st, w, s, shares, int(lens[s]), address[w]) for w in "kv"}
        if shares:
            kv = {w: torch.cat([held[w], kv[w]]) for w in "kv"}
        count, length = int(n[s]), int(lens[s])
        pos, key = torch.arange(length - count, length, device=DEV)[:, None], torch.arange(length, device=DEV)[None]
        hidden = key > pos
        if c["window"]:
            hidden = hidden | (pos - key >= c["window"])
        q = st["q"][row : row + count].double().reshape(count, c["n_kv"], c["g"], c["d"])
        for h in range(c["n_kv"]):
            whole[row : row + count, h] = _softmax_exact(st, q[:, h], kv["k"][:, h], kv["v"][:, h], pos, key, hidden, h)
        row += count
    return whole.reshape(row, -1)


def _selected_exact(st):
    c, row = st["case"], 0
    n, lens, _, _ = _shapes(c)
    address = _addresses(c["d"])
    whole = torch.zeros((int(n.sum()), c["n_kv"], c["g"], c["d"]), dtype=torch.float64, device=DEV)
    for s in range(c["seqs"]):
        count, length = int(n[s]), int(lens[s])
        kv = {w: _sequence(st, w, s, 0, length, address[w]) for w in "kv"}
        key = torch.arange(length, device=DEV)[None]
        for lo in range(0, count, 128):
            rows = slice(row + lo, row + min(lo + 128, count))
            pos = torch.arange(length - count + lo, length - count + min(lo + 128, count), device=DEV)[:, None]
            q = st["q"][rows].double().reshape(-1, c["n_kv"], c["g"], c["d"])
            for h in range(c["n_kv"]):
                named = torch.zeros((len(q), (length - 1) // c["span"] + 2), dtype=torch.bool, device=DEV)
                named.scatter_(1, torch.where(st["chosen"][rows, h] >= 0, st["chosen"][rows, h], named.shape[1] - 1).long(), True)
                hidden = (key > pos) | ~named[:, :-1].repeat_interleave(c["span"], 1)[:, :length]
                if c["window"]:
                    hidden = hidden | (pos - key >= c["window"])
                whole[rows, h] = _softmax_exact(st, q[:, h], kv["k"][:, h], kv["v"][:, h], pos, key, hidden, h)
        row += count
    return whole.reshape(row, -1)


def _select_exact(st):
    c = st["case"]
    n, lens, _, _ = _shapes(c)
    address, count, span = _addresses(c["d"]), _count(c), c["span"]
    back = torch.zeros((c["seqs"], count, c["n_kv"], c["d"]), dtype=torch.float64, device=DEV)
    for s in range(c["seqs"]):
        last = (int(lens[s]) - 1) // span
        for x in range(max(0, last - count + 1), last + 1):
            page = int(st["pages"][s, x * span // c["page"]])
            if (x + 1) * span > int(lens[s] - n[s]):
                mean = _sequence(st, "k", s, x * span, min((x + 1) * span, int(lens[s])), address["k"]).mean(0)
                size = (mean.abs().amax(-1, keepdim=True) / 127).float().double()  # (held in 32 bits)
                value = torch.round(mean / size) * size
            else:
                at = x * span % c["page"] // span
                value = st["means"][page, :, at].double() * st["mean_scale"][page, :, at, None].double()
            back[s, x - last + count - 1] = value
    return [back, None]


def _sample_exact(st):
    c = st["case"]
    out = []
    for r in range(c["rows"]):
        x = st["logits"][r].cpu().double().numpy()
        heat = float(st["temperature"][r])
        order = np.argsort(-x, kind="stable")
        if heat <= 0:
            out.append(0.0)
            continue
        w = np.exp((x[order] - x[order[0]]) / heat)
        if c["top_k"]:
            w = w[: c["top_k"]]
        if c["top_p"] < 1:
            share = np.cumsum(w) / w.sum()
            w = w[: int(np.searchsorted(share, float(st["top_p"][r]))) + 1]
        if c["min_p"]:
            w = w[: max(1, int((w >= float(st["min_p"][r])).sum()))]
        ids = order[: len(w)]
        by_id = np.argsort(ids)
        upto = np.cumsum(w[by_id])
        at = min(int(np.searchsorted(upto, float(st["u"][r]) * upto[-1], side="right")), len(w) - 1)
        out.append(math.log(w[by_id][at] / upto[-1]))
    return [None, torch.tensor(out, dtype=torch.float64, device=DEV)]


def exact(case, seed):
    state = prepare(case, seed)
    return {"shared": _shared_exact, "select": _select_exact, "selected": _selected_exact, "sample": _sample_exact}[case["op"]](state)
