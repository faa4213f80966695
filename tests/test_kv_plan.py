"""The index arithmetic of the key / value cache (csrc/kv_plan.hpp) compiled for the CPU, and what its entry points refuse (no device needed)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from tests import kv_ref

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oxinfer_amd", "csrc")

PROGRAM = r"""
#include "kv_plan.hpp"
#include <cstdio>
#include <cstring>
#include <vector>
using namespace oxhip;
int main() {
    char what[16];
    while (std::scanf("%15s", what) == 1) {
        if (!std::strcmp(what, "offsets")) {
            unsigned d;
            if (std::scanf("%u", &d) != 1) return 1;
            for (unsigned t = 0; t < KV_BLOCK; t++)
                for (unsigned c = 0; c < d; c++) std::printf("%u %u\n", kv_key_offset(t, c), kv_value_offset(t, c));
        } else if (!std::strcmp(what, "place")) {
            unsigned long long start, s;
            unsigned unit, more;
            if (std::scanf("%llu %llu %u %u", &start, &s, &unit, &more) != 4) return 1;
            std::printf("%llu %llu\n", (unsigned long long)kv_first_place(start, s, unit, more), (unsigned long long)kv_places(start, s, unit, more));
        } else if (!std::strcmp(what, "span")) {
            long long pre, lo, hi;
            if (std::scanf("%lld %lld %lld", &pre, &lo, &hi) != 3) return 1;
            const KvSpan s = kv_span(pre, lo, hi);
            for (unsigned i = 0; i < s.count; i++) std::printf("%u ", kv_span_block(s, i));
            std::printf("\n");
        } else if (!std::strcmp(what, "part")) {
            int s, r0, r1, len;
            unsigned rows, pages, shift;
            if (std::scanf("%d %d %d %d %u %u %u", &s, &r0, &r1, &len, &rows, &pages, &shift) != 7) return 1;
            const KvSeq q = kv_part(s, r0, r1, len, rows, pages, shift);
            std::printf("%d %d %d %d\n", q.s, q.row0, q.n, q.len);
        } else if (!std::strcmp(what, "weight")) {
            int n, len, prefix;
            unsigned window, quantum, g;
            if (std::scanf("%d %d %u %d %u %u", &n, &len, &window, &prefix, &quantum, &g) != 6) return 1;
            const KvSeq q{0, 0, n, len};
            std::printf("%u %u\n", kv_weight(q, window, prefix, quantum), kv_tiles(q, g));
        } else if (!std::strcmp(what, "quantum")) {
            unsigned long long tiles, blocks;
            if (std::scanf("%llu %llu", &tiles, &blocks) != 2) return 1;
            std::printf("%u\n", kv_quantum(tiles, blocks));
        } else {
            int id;
            unsigned most, n_pages, block, shift;
            if (std::scanf("%d %u %u %u %u", &id, &most, &n_pages, &block, &shift) != 5) return 1;
            std::vector<int32_t> table(most, id);
            std::printf("%d\n", kv_page_of(table.data(), most, n_pages, block, shift));
        }
    }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_plan")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(d / "main.cpp"), "-o", str(d / "main")], check=True)

    def ask(lines):
        r = subprocess.run([str(d / "main")], input="\n".join(lines), capture_output=True, text=True, check=True)
        return [list(map(int, line.split())) for line in r.stdout.splitlines()]
    return ask


@pytest.mark.parametrize("d", range(32, 257, 32))
def test_a_blocks_bytes(ask, d):
    """Every token's channel has a byte of its own, where the reference layout has it."""
    got = np.array(ask([f"offsets {d}"])).reshape(32, d, 2)
    for i, want in enumerate(kv_ref.offsets(d)):
        assert np.array_equal(got[..., i], want)
        assert np.array_equal(np.sort(got[..., i].reshape(-1)), np.arange(32 * d))


def test_places_of_ragged_sequences(ask):
    """Every sequence has room for its tiles (of 16 entries, g to a row) and for the blocks that its tokens touch, and the launch covers all."""
    rng = np.random.default_rng(1)
    for _ in range(30):
        n = rng.integers(0, rng.choice([2, 5, 40, 300]), rng.integers(1, 70))
        start = np.concatenate([[0], np.cumsum(n)])
        for g in (1, 3, 16, 17):
            got = np.array(ask([f"place {v * g} {s} 16 1" for s, v in enumerate(start)]))
            assert (np.diff(got[:, 0]) >= -(-(n * g) // 16)).all() and got[-1, 1] >= got[-1, 0]
        got = np.array(ask([f"place {v} {s} 32 2" for s, v in enumerate(start)]))
        for at in range(32):  # wherever the first token lies in its block
            assert (np.diff(got[:, 0]) >= np.where(n > 0, (at + n + 31) // 32, 0)).all()
        assert (np.diff(got[:, 0]) > 0).all()


def test_spans_of_blocks(ask):
    """The blocks of [0, prefix) and [lo, hi), each once, in order."""
    rng = np.random.default_rng(2)
    cases = [(0, 0, 0), (0, 5, 5), (0, 2**31 - 1, 0), (0, 0, 1), (32, 0, 32), (33, 40, 70), (7, 100, 101), (200, 10, 90), (1, 31, 33), (64, 64, 65)]
    cases += [tuple(int(v) for v in rng.integers(0, 400, 3)) for _ in range(200)]
    for (pre, lo, hi), got in zip(cases, ask([f"span {p} {a} {b}" for p, a, b in cases])):
        want = set(range(-(-pre // 32))) | (set(range(lo // 32, -(-hi // 32))) if hi > lo else set())
        assert got == sorted(want), (pre, lo, hi)


def test_weights_of_tiles(ask):
    """A sequence's weight is no less than the blocks that any of its rows sees (window and prefix as the launch has them), and no
    more than all of its blocks; its tiles hold its entries. Lengths below the rows (rows at negative positions) count all blocks."""
    rng = np.random.default_rng(3)
    cases = [(1, 0, 0, 0), (1, 1, 0, 0), (1, 33, 1, 0), (5, 3, 2, 0), (1, 2**31 - 64, 0, 0), (1, 2**31 - 64, 2**31 - 2, 2**31 - 1), (4, 1000, 100, 2**31 - 1), (4, 1000, 100, -7), (300, 64, 10, 5)]
    cases += [(int(rng.integers(1, 400)), int(rng.integers(0, 5000)), int(rng.integers(0, 700)), int(rng.integers(-50, 5000))) for _ in range(400)]
    gs = [int(rng.choice([1, 3, 8, 17])) for _ in cases]
    quanta = [int(2 ** rng.integers(0, 4)) for _ in cases]
    got = ask([f"weight {n} {ln} {w} {p} {q} {g}" for (n, ln, w, p), q, g in zip(cases, quanta, gs)])
    for (n, ln, w, p), q, g, (weight, tiles) in zip(cases, quanta, gs, got):
        everything = -(-ln // 32)
        lo = max(ln - n - w + 1, 0) // 32 if w else 0
        seen = everything - lo + min(-(-max(min(p, ln), 0) // 32), lo)  # of all its rows together
        assert max(1, -(-seen // q)) <= weight <= max(1, -(-everything // q)), (n, ln, w, p, q)
        assert tiles == -(-n * g // 16)


def test_quanta_of_launches(ask):
    """32 bits hold the sum of all tiles' weights, in the smallest power of two of blocks that does it; none for a launch that is too large."""
    cases = [(1, 1), (1, 2**26), (31, 2**26), (32, 2**26), (2**20, 2**26), (2**30 - 1, 2**26), (2**30, 1), (2**40, 2**26)]
    for (tiles, blocks), (q,) in zip(cases, ask([f"quantum {t} {b}" for t, b in cases])):
        if tiles >= 2**30:
            assert q == 0
        else:
            assert q & (q - 1) == 0 and q and tiles * -(-blocks // q) < 2**31 and (q == 1 or tiles * -(-blocks // (q // 2)) >= 2**31)


def test_unsound_sequences_and_pages(ask):
    """Rows outside the batch, lengths outside the table and pages outside the cache are cut off before anything is read with them."""
    parts = [("0 0 4 7 4 2 0", [0, 0, 4, 7]), ("1 -5 3 7 4 2 0", [1, 0, 3, 7]), ("1 2 9 7 4 2 0", [1, 2, 2, 7]), ("1 9 2 7 4 2 0", [1, 9, 0, 7]), ("2 5 9 7 4 2 0", [2, 5, 0, 7]),
             ("0 0 1 -3 4 2 0", [0, 0, 1, 0]), ("0 0 1 65 4 2 0", [0, 0, 1, 64]), ("0 0 1 2147483647 4 2 3", [0, 0, 1, 512]), ("0 0 1 2147483647 1 67108862 0", [0, 0, 1, 2147483584])]
    assert ask([f"part {p}" for p, _ in parts]) == [w for _, w in parts]
    pages = [("3 2 4 0 0", 3), ("4 2 4 0 0", -1), ("-1 2 4 0 0", -1), ("-2147483648 2 4 0 0", -1), ("2147483647 2 4 0 0", -1), ("3 2 4 2 0", -1), ("3 2 4 15 3", 3), ("3 2 4 16 3", -1)]
    assert ask([f"page {p}" for p, _ in pages]) == [[w] for _, w in pages]


# ---- refusals: every check comes before the context is looked at, so that valid arguments without one are told from invalid ones ----------

P = 4096  # stands for a device pointer: nothing on this side reads it


@pytest.fixture(scope="module")
def lib():
    from oxinfer_amd import build, hip
    if not os.path.exists(hip.library_path()):
        build.build()
    return hip.load_library()


def structs(hip, kv=(), b=()):
    c = dict(k=P, v=P, k_scale=P, v_scale=P, n_pages=9, page_tokens=64, n_kv=2, d=64, **{})
    bb = dict(n_seqs=3, rows=3, row_start=None, kv_len=P, pages=P, max_pages=4)
    c.update(kv)
    bb.update(b)
    return hip.KvCacheC(**c), hip.KvBatchC(**bb)


def said(lib, ok):
    assert ok == 0
    return lib.oxhip_last_error().decode()


BAD_KV = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=P + 8), dict(v=P + 1), dict(k_scale=P + 2), dict(d=0), dict(d=48), dict(d=288), dict(page_tokens=16), dict(page_tokens=0),
          dict(page_tokens=96), dict(page_tokens=2**31), dict(n_kv=0), dict(n_kv=20000), dict(n_pages=0), dict(n_pages=2**31), dict(n_pages=2**29, n_kv=2), dict(n_pages=2**31 // 256 + 1, n_kv=4, page_tokens=2048)]
BAD_B = [dict(kv_len=None), dict(pages=None), dict(kv_len=P + 1), dict(row_start=P + 2), dict(n_seqs=0), dict(n_seqs=2**25, rows=2**25), dict(max_pages=0), dict(max_pages=2**31), dict(max_pages=2**26), dict(rows=4),
         dict(rows=2**29, row_start=P)]
OF_KV = [(a, ()) for a in BAD_KV] + [((), a) for a in BAD_B]


@pytest.mark.parametrize("kv,b", OF_KV)
def test_caches_and_batches_that_are_refused(lib, kv, b):
    from oxinfer_amd import hip
    good, bad = structs(hip), structs(hip, kv, b)
    for cache, batch, null in ((*good, True), (*bad, False)):
        for ok in (lambda: lib.oxhip_dev_attend(None, C.byref(cache), C.byref(batch), P, 0, 4, 0, 1.0, None, 2 * P, 0, None),
                   lambda: lib.oxhip_dev_kv_append(None, C.byref(cache), C.byref(batch), P, 0, P, 0, None, 0, None, 0, 0, 0, None, None),
                   lambda: lib.oxhip_dev_kv_read(None, C.byref(cache), C.byref(batch), 5, P, P, 0, None)):
            assert ("null context" in said(lib, ok())) == null


def test_rows_and_rules_that_are_refused(lib):
    from oxinfer_amd import hip
    cache, batch = (C.byref(s) for s in structs(hip))

    def attend(q=P, qs=0, n_q=4, dtype=0, scale=0.5, rules=None, out=2 * P, os=0):
        return said(lib, lib.oxhip_dev_attend(None, cache, batch, q, qs, n_q, dtype, scale, C.byref(hip.AttendRulesC(**rules)) if rules is not None else None, out, os, None))

    for good in (dict(), dict(dtype=1, q=P + 2, out=2 * P + 2), dict(qs=256, os=300), dict(scale=-2.0), dict(scale=0.0), dict(rules=dict(cap=30.0, slopes=P, window=2**40, prefix=P, first=P))):
        assert "null context" in attend(**good), good
    for bad in (dict(q=None), dict(out=None), dict(q=P + 2), dict(out=P + 1, dtype=1), dict(n_q=0), dict(n_q=3), dict(n_q=2**17), dict(dtype=2), dict(dtype=-1), dict(scale=float("inf")), dict(scale=float("nan")),
                dict(qs=255), dict(os=1), dict(rules=dict(cap=-1.0)), dict(rules=dict(cap=float("nan"))), dict(rules=dict(cap=float("inf"))), dict(rules=dict(cap=1e30)), dict(rules=dict(cap=1e-30)), dict(scale=1.4e36), dict(scale=-1e38), dict(out=P, q=P),  dict(rules=dict(slopes=P + 1)), dict(rules=dict(first=P + 2))):
        assert "null context" not in attend(**bad), bad

    def append(k=P, ks=0, v=P, vs=0, q=P, qs=0, out=P, os=0, n_q=4, dtype=0, rope=None):
        return said(lib, lib.oxhip_dev_kv_append(None, cache, batch, k, ks, v, vs, q, qs, out, os, n_q, dtype, C.byref(hip.RopeC(*rope)) if rope else None, None))

    for good in (dict(), dict(q=None, out=None, n_q=0), dict(rope=(P, 9, 64, 0)), dict(rope=(P, 1, 2, 1)), dict(qs=300, os=300), dict(qs=300, out=2 * P, os=301)):
        assert "null context" in append(**good), good
    for bad in (dict(k=None), dict(v=None), dict(q=None), dict(out=None), dict(n_q=0), dict(n_q=40000), dict(k=P + 2), dict(dtype=5), dict(ks=127), dict(vs=1), dict(qs=255), dict(os=255), dict(qs=256, os=300),
                dict(rope=(None, 9, 64, 0)), dict(rope=(P + 4, 9, 64, 0)), dict(rope=(P, 0, 64, 0)), dict(rope=(P, 9, 63, 0)), dict(rope=(P, 9, 0, 0)), dict(rope=(P, 9, 66, 0))):
        assert "null context" not in append(**bad), bad
    read = lambda *a: said(lib, lib.oxhip_dev_kv_read(None, cache, batch, *a, None))  # noqa: E731
    assert "null context" in read(5, P, None, 1)
    for bad in ((5, None, None, 0), (5, P, P, 2), (5, P + 2, P, 0), (2**31, P, P, 0)):
        assert "null context" not in read(*bad), bad


def test_logits_rules_that_are_refused(lib):
    from oxinfer_amd import hip

    def logits(x=P, s=0, out=P, os=0, rows=3, vocab=1000, dtype=0, next=P, **rules):
        return said(lib, lib.oxhip_dev_logits(None, x, s, out, os, rows, vocab, dtype, C.byref(hip.LogitRulesC(**rules)) if rules else None, next, None))

    hist = dict(history=P, history_stride=7, history_len=P)
    bias = dict(bias_start=P, bias_id=P, bias=P, n_bias=4)
    mask = dict(allowed=P, allowed_stride=32, n_allowed=3)
    for good in (dict(), dict(out=None), dict(next=None), dict(s=1001, os=1001), dict(s=1001, out=2 * P, os=1000), hist, dict(hist, repetition=P, prompt_len=P), bias, mask, dict(mask, n_allowed=1, allowed_row=P)):
        assert "null context" in logits(**good), good
    for bad in (dict(x=None), dict(out=None, next=None), dict(dtype=3), dict(vocab=0), dict(vocab=2**31), dict(rows=2**25), dict(x=P + 2), dict(next=P + 2), dict(s=999), dict(os=999), dict(s=1001),
                dict(history=P), dict(hist, history_stride=0), dict(hist, history_len=None), dict(repetition=P), dict(prompt_len=P), dict(bias, bias=None), dict(bias, bias_start=None), dict(bias, n_bias=2**31),
                dict(mask, allowed_stride=31), dict(mask, n_allowed=0), dict(mask, n_allowed=2), dict(allowed_row=P), dict(mask, allowed=P + 2)):
        assert "null context" not in logits(**bad), bad


def test_the_bindings_own_checks():
    """What the binding tells from shapes, types and devices before the library is called."""
    import torch
    from oxinfer_amd import hip
    z = lambda *s, t=torch.uint8: torch.zeros(s, dtype=t)  # noqa: E731
    with pytest.raises(ValueError, match="wanted .* on cuda"):
        hip.KvCache(z(3, 2, 2, 2048), z(3, 2, 2, 2048), z(3, 2, 2, t=torch.float32), z(3, 2, 2, t=torch.float32), 64, 64)
    with pytest.raises(ValueError, match="int8"):
        hip.KvCache(z(3, 2, 2, 2048, t=torch.int8), z(3, 2, 2, 2048), z(3, 2, 2, t=torch.float32), z(3, 2, 2, t=torch.float32), 64, 64)
    with pytest.raises(ValueError, match="wanted"):
        hip.KvBatch(z(3), z(3, 4, t=torch.int32))
    with pytest.raises(ValueError, match="wanted"):
        hip.Rope(z(3, 4, 2, t=torch.float64))


def test_how_many_rows_have_a_best_token(lib):
    """With `next`, rows and their slices of 4096 logits have to fit the stream's scratch; the refusal names both bounds."""
    def logits(rows, vocab, next=P):
        return said(lib, lib.oxhip_dev_logits(None, P, 0, P, 0, rows, vocab, 0, None, next, None))

    for rows, vocab in ((16384, 1), (16384, 524288), (8192, 2**20), (4, 2**31 - 4096)):
        assert "null context" in logits(rows, vocab), (rows, vocab)
    for rows, vocab in ((16385, 1), (16384, 524289), (8193, 2**20), (5, 2**31 - 4096)):
        assert "16384 rows" in logits(rows, vocab) and "2^21 slices" in logits(rows, vocab), (rows, vocab)
    assert "2^31 - 4096" in logits(1, 2**31 - 4095) and "null context" in logits(16385, 5, next=None)


def test_calls_of_more_than_one_launch_takes(lib):
    """A launch has fewer than 2^32 threads, and 65535 workgroups at most in its second direction: the calls on either side of that."""
    from oxinfer_amd import hip

    def batch(n_seqs, rows=None, ragged=False, **kv):
        return structs(hip, kv, dict(n_seqs=n_seqs, rows=n_seqs if rows is None else rows, row_start=P if ragged else None))

    def append(s, n_q=4):
        return said(lib, lib.oxhip_dev_kv_append(None, C.byref(s[0]), C.byref(s[1]), P, 0, P, 0, P, 0, P, 0, n_q, 0, None, None))

    def read(s, count):
        return said(lib, lib.oxhip_dev_kv_read(None, C.byref(s[0]), C.byref(s[1]), count, P, P, 0, None))

    def attend(s, n_q=4):
        return said(lib, lib.oxhip_dev_attend(None, C.byref(s[0]), C.byref(s[1]), P, 0, n_q, 0, 1.0, None, 2 * P, 0, None))

    def logits(rows, vocab):
        return said(lib, lib.oxhip_dev_logits(None, P, 0, P, 0, rows, vocab, 0, None, None, None))

    m = 2**20
    wide = dict(n_kv=16384, n_pages=9)
    for good, bad in ((append(batch(8 * m - 1)), append(batch(8 * m))), (append(batch(8 * m - 1, 5, True)), append(batch(8 * m, 5, True))), (append(batch(1, 9, True, **wide), 32766), append(batch(1, 9, True, **wide), 32768)),
                      (read(batch(8 * m - 1), 33), read(batch(8 * m - 1), 65)), (attend(batch(4 * m - 1)), attend(batch(4 * m))), (attend(batch(m, 2 * m, True), 2 * 16), attend(batch(m, 4 * m, True), 2 * 16)),
                      (attend(batch(1, 2**28, True), 2 * 3), attend(batch(1, 2**28, True), 2 * 4)), (logits(8 * m - 1, 4096), logits(8 * m, 4096)), (logits(4 * m - 1, 4097), logits(4 * m, 4097))):
        assert "null context" in good and "one launch" in bad, (good, bad)
