"""What the entry points of shared prefixes, chosen spans and the draw refuse, and the index arithmetic behind them (no device needed)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from tests.test_kv_plan import BAD_B, BAD_KV, CSRC, OF_KV, P, lib, said, structs  # noqa: F401

PROGRAM = r"""
#include "kv_plan.hpp"
#include <cstdio>
using namespace oxhip;
int main() {
    long long base, pre, lo, hi;
    while (std::scanf("%lld %lld %lld %lld", &base, &pre, &lo, &hi) == 4) {
        const KvSpan s = kv_span_from((uint32_t)base, pre, lo, hi);
        for (unsigned i = 0; i < s.count; i++) std::printf("%lld ", i < s.pre ? base + i : (long long)s.lo + (i - s.pre));
        std::printf("\n");
    }
    std::printf("%llu %llu %llu %llu\n", (unsigned long long)kv_row_tiles(100, 5, true), (unsigned long long)kv_row_tiles(100, 5, false), (unsigned long long)kv_row_tiles(100, 16, true),
                (unsigned long long)kv_row_tiles(100, 33, true));
}
"""


def test_spans_from_a_block_on(tmp_path):
    """The blocks of [0, prefix) and [lo, hi) from `base` on, each once, in order; tiles of rows."""
    rng = np.random.default_rng(2)
    cases = [(0, 0, 0, 0), (3, 0, 100, 101), (3, 200, 96, 300), (3, 90, 96, 97), (2, 65, 64, 64), (5, 400, 160, 161), (0, 40, 10, 90)]
    cases += [(int(b), *(int(v) for v in rng.integers(0, 400, 3))) for b in rng.integers(0, 9, 300)]
    (tmp_path / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", CSRC, str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")], check=True)
    r = subprocess.run([str(tmp_path / "main")], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True, check=True)
    *got, tiles = [list(map(int, line.split())) for line in r.stdout.splitlines()]
    for (base, pre, lo, hi), blocks in zip(cases, got):
        want = set(range(-(-pre // 32))) | (set(range(lo // 32, -(-hi // 32))) if hi > lo else set())
        assert blocks == sorted(b for b in want if b >= base), (base, pre, lo, hi)
    assert tiles == [34, 100, 100, 300]


def calls(lib, hip, cache, batch):  # noqa: F811
    shared, held = hip.KvSharedC(P, P, 1), hip.KvSummaryC(P, P, 32)
    c, b = C.byref(cache), C.byref(batch)
    return (lambda: lib.oxhip_dev_attend_shared(None, c, b, C.byref(shared), P, 0, 4, 0, 1.0, None, 2 * P, 0, None),
            lambda: lib.oxhip_dev_kv_summarize(None, c, b, C.byref(held), None),
            lambda: lib.oxhip_dev_kv_summary_read(None, c, b, C.byref(held), 5, P, None),
            lambda: lib.oxhip_dev_kv_select(None, c, b, C.byref(held), P, 0, 4, 0, 5, 1, 1, P, None),
            lambda: lib.oxhip_dev_attend_selected(None, c, b, P, 5, 32, P, 0, 4, 0, 1.0, None, 2 * P, 0, None))


@pytest.mark.parametrize("kv,b", OF_KV)
def test_caches_and_batches_that_are_refused(lib, kv, b):  # noqa: F811
    from oxinfer_amd import hip
    good, bad = structs(hip), structs(hip, kv, b)
    for (cache, batch), null in ((good, True), (bad, False)):
        for call in calls(lib, hip, cache, batch):
            assert ("null context" in said(lib, call())) == null


def test_arguments_that_are_refused(lib):  # noqa: F811
    from oxinfer_amd import hip
    cache, batch = structs(hip)
    c, b = C.byref(cache), C.byref(batch)

    def shared(of=(P, P, 2), q=P, qs=0, n_q=4, dtype=0, scale=0.5, rules=None, out=2 * P, os=0):
        return said(lib, lib.oxhip_dev_attend_shared(None, c, b, C.byref(hip.KvSharedC(*of)) if of else None, q, qs, n_q, dtype, scale, C.byref(hip.AttendRulesC(**rules)) if rules else None, out, os, None))

    def selected(chosen=P, count=7, span=64, q=P, qs=0, n_q=4, dtype=0, scale=0.5, rules=None, out=2 * P, os=0):
        return said(lib, lib.oxhip_dev_attend_selected(None, c, b, chosen, count, span, q, qs, n_q, dtype, scale, C.byref(hip.AttendRulesC(**rules)) if rules else None, out, os, None))

    for good in (dict(), dict(dtype=1, q=P + 2, out=2 * P + 2), dict(qs=256, os=300), dict(scale=-2.0), dict(rules=dict(cap=30.0, slopes=P, window=2**40, prefix=P, first=P))):
        assert "null context" in shared(**good) and "null context" in selected(**good), good
    for bad in (dict(q=None), dict(out=None), dict(q=P + 2), dict(out=P + 1, dtype=1), dict(n_q=0), dict(n_q=3), dict(n_q=2**17), dict(dtype=2), dict(scale=float("nan")), dict(scale=1e38), dict(qs=255), dict(os=1),
                dict(rules=dict(cap=-1.0)), dict(rules=dict(cap=1e30)), dict(out=P, q=P), dict(rules=dict(slopes=P + 1)), dict(rules=dict(first=P + 2))):
        assert "null context" not in shared(**bad) and "null context" not in selected(**bad), bad
    for bad in ((None, P, 2), (P, None, 2), (P, P, 0), (P, P, 2**25), (P + 2, P, 2), (P, P + 1, 2), None):
        assert "null context" not in shared(of=bad), bad
    for bad in (dict(chosen=None), dict(chosen=P + 2), dict(count=0), dict(count=2**26), dict(span=16), dict(span=0), dict(span=48), dict(span=128)):
        assert "null context" not in selected(**bad), bad

    def select(of=(P, P, 32), q=P, qs=0, n_q=4, dtype=0, count=6, first=1, last=2, chosen=P, batch=b):
        return said(lib, lib.oxhip_dev_kv_select(None, c, batch, C.byref(hip.KvSummaryC(*of)) if of else None, q, qs, n_q, dtype, count, first, last, chosen, None))

    for good in (dict(), dict(of=(P, P, 64)), dict(dtype=1, q=P + 2), dict(qs=257), dict(first=0, last=0), dict(first=4, last=2), dict(count=16384)):
        assert "null context" in select(**good), good
    for bad in (dict(of=None), dict(of=(None, P, 32)), dict(of=(P, None, 32)), dict(of=(P + 8, P, 32)), dict(of=(P, P + 2, 32)), dict(of=(P, P, 16)), dict(of=(P, P, 48)), dict(of=(P, P, 128)), dict(q=None), dict(q=P + 2), dict(n_q=3),
                dict(n_q=0), dict(dtype=4), dict(qs=255), dict(count=0), dict(count=16385), dict(first=7), dict(first=5, last=2), dict(last=2**63), dict(first=2**64 - 1, last=2), dict(chosen=None), dict(chosen=P + 1)):
        assert "null context" not in select(**bad), bad
    wide = structs(hip, b=dict(max_pages=8192))[1]
    assert "null context" in select(batch=C.byref(wide))
    wide = structs(hip, b=dict(max_pages=8193))[1]
    assert "16384" in select(batch=C.byref(wide)) and "null context" in select(batch=C.byref(wide), of=(P, P, 64))
    read = lambda count, out: said(lib, lib.oxhip_dev_kv_summary_read(None, c, b, C.byref(hip.KvSummaryC(P, P, 32)), count, out, None))  # noqa: E731
    assert "null context" in read(5, P)
    for bad in ((5, None), (5, P + 8), (2**31, P), (2**27, P)):
        assert "null context" not in read(*bad), bad


def test_draws_that_are_refused(lib):  # noqa: F811
    from oxinfer_amd import hip

    def draw(x=P, s=0, rows=3, vocab=1000, dtype=0, u=P, next=P, logp=P, **rules):
        return said(lib, lib.oxhip_dev_sample(None, x, s, rows, vocab, dtype, C.byref(hip.SampleRulesC(**rules)) if rules else None, u, next, logp, None))

    for good in (dict(), dict(logp=None), dict(s=1001), dict(dtype=1, x=P + 2), dict(temperature=P), dict(top_k=P, top_p=P, min_p=P), dict(vocab=2**31 - 4096), dict(vocab=1)):
        assert "null context" in draw(**good), good
    for bad in (dict(x=None), dict(u=None), dict(next=None), dict(dtype=2), dict(vocab=0), dict(vocab=2**31 - 4095), dict(rows=2**25), dict(x=P + 2), dict(u=P + 1), dict(next=P + 2), dict(logp=P + 2), dict(s=999), dict(temperature=P + 1),
                dict(top_k=P + 2), dict(top_p=P + 3), dict(min_p=P + 1)):
        assert "null context" not in draw(**bad), bad


def test_calls_of_more_than_one_launch_takes(lib):  # noqa: F811
    from oxinfer_amd import hip
    m = 2**20

    def batch(n_seqs, rows=None, ragged=False, **kv):
        return structs(hip, kv, dict(n_seqs=n_seqs, rows=n_seqs if rows is None else rows, row_start=P if ragged else None))

    def ask(s, which):
        return said(lib, calls(lib, hip, *s)[which]())

    for good, bad in ((ask(batch(8 * m, 32 * m - 8, True), 0), ask(batch(8 * m, 32 * m, True), 0)), (ask(batch(8 * m - 1), 1), ask(batch(8 * m), 1)), (ask(batch(m, 32 * m, True), 1), ask(batch(8 * m, 5, True), 1)),
                      (ask(batch(16 * m), 2), ask(batch(16 * m, d=128), 2)), (ask(batch(2 * m - 1), 3), ask(batch(2 * m), 3)), (ask(batch(m, m - 1, True), 3), ask(batch(m, m, True), 3)), (ask(batch(4 * m - 1), 4), ask(batch(4 * m), 4))):
        assert "null context" in good and "one launch" in bad, (good, bad)


def test_the_bindings_own_checks():
    import torch
    from oxinfer_amd import hip
    z = lambda *s, t=torch.int32: torch.zeros(s, dtype=t)  # noqa: E731
    with pytest.raises(ValueError, match="wanted"):
        hip.KvShared(z(3), z(2))
    with pytest.raises(ValueError, match="wanted"):
        hip.KvSummary(z(3, 2, 2, 64, t=torch.int8), z(3, 2, 2, t=torch.float32), 32)
    with pytest.raises(ValueError, match="wanted"):
        hip.KvSummary(z(3, 2, 64, t=torch.int8), z(3, 2, t=torch.float32), 32)
    assert os.path.exists(hip.library_path())


def test_appends_behind_shared_tokens_that_are_refused(lib):  # noqa: F811
    """What oxhip_dev_kv_append refuses, and groups that are none."""
    from oxinfer_amd import hip

    def append(s, of=(P, P, 2), k=P, ks=0, q=P, n_q=4, dtype=0, rope=None, null=False):
        r = C.byref(hip.RopeC(*rope)) if rope else None
        return said(lib, lib.oxhip_dev_kv_append_shared(None, C.byref(s[0]), C.byref(s[1]), None if null else C.byref(hip.KvSharedC(*of)), k, ks, P, 0, q, 0, q, 0, n_q, dtype, r, None))

    good = structs(hip)
    for kw in (dict(), dict(q=None, n_q=0), dict(dtype=1, k=P + 2), dict(ks=130), dict(rope=(P, 100, 32, 0))):
        assert "null context" in append(good, **kw), kw
    for kw in (dict(null=True), dict(of=(None, P, 2)), dict(of=(P, None, 2)), dict(of=(P, P, 0)), dict(of=(P, P, 2**25)), dict(of=(P + 2, P, 2)), dict(of=(P, P + 1, 2)), dict(k=None), dict(k=P + 2), dict(ks=1), dict(q=None),
               dict(n_q=0), dict(dtype=2), dict(rope=(P, 0, 32, 0)), dict(rope=(None, 4, 32, 0))):
        assert "null context" not in append(good, **kw), kw
        assert lib.oxhip_last_error().decode().startswith("kv_append_shared: ")
    for kv, b in OF_KV:
        assert "null context" not in append(structs(hip, kv, b))
    m = 2**20
    ragged = lambda rows: append(structs(hip, {}, dict(n_seqs=7 * m, rows=rows, row_start=P)), q=None, n_q=0)  # noqa: E731
    assert "null context" in ragged(5) and "one launch" in ragged(2**28)
