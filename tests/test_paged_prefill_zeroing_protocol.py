"""CPU model check of the V tiles that the paged prefill kernel zeroes in part
(paged_prefill.cu): a tile with rows that none of the CTA's queries sees is
copied on a barrier of its own (V_RAW), its rows are zeroed by the producer,
and a plain arrival hands it to the MMA on V_FULL. V_RAW's phases are counted
over the segments of a share. The rest of the protocol is that of
test_paged_prefill_protocol.py; planted mistakes must be caught. (An arrival
is modelled like a copy: the others may see it late.)"""

import itertools
import random

import pytest

import test_paged_prefill_protocol as P
import test_prefill_protocol as T


def _programs(nts, rnd, flaw=None):
    raw = {(g, j) for g, n in enumerate(nts) for j in range(n)
           if rnd.random() < (0.7 if j in (0, n - 1) else 0.3)}
    progs = P._programs(nts, rnd)
    d = [(sum((n + 1) // 2 for n in nts[:g]), sum(n // 2 for n in nts[:g])) for g in range(len(nts))]

    def par(g, s, k):
        return (k + d[g][s]) & 1

    def vp():
        raws = 0
        for g, n in enumerate(nts):
            if flaw == "phases restart":
                raws = 0
            if g > 0:
                yield ("wait", "MMA_DONE", (g - 1) & 1)
            last = False
            for j in range(n):
                if j >= 2:
                    yield ("wait", ("DONE", j & 1), par(g, j & 1, (j >> 1) - 1))
                    yield ("check", lambda s, g=g, j=j: ("PV", g, j - 2) in s, f"V{g}.{j} over a stage that is read")
                last = (g, j) in raw
                if not last:
                    yield ("tma", ("VF", j & 1), ("V", g, j))
                    continue
                yield ("tma", "VR", ("VR", g, j))
                if flaw != "zeroed unseen":
                    yield ("wait", "VR", raws & 1)
                raws += 1
                yield ("check", lambda s, g=g, j=j: ("VR", g, j) in s, f"V{g}.{j} zeroed before it landed")
                if flaw == "handed over first":
                    yield ("tma", ("VF", j & 1), ("V", g, j))
                yield ("done", ("Z", g, j))
                if flaw != "handed over first":
                    yield ("tma", ("VF", j & 1), ("V", g, j))
            # The drain: the last tile where it was copied, the one before on V_FULL.
            for j in range(max(0, n - 2), n):
                if last and j == n - 1:
                    yield ("wait", "VR", (raws - 1) & 1)
                else:
                    yield ("wait", ("VF", j & 1), par(g, j & 1, j >> 1))

    def mma(steps):
        for op in steps:
            if op[0] == "mma" and op[1][0] == "PV" and op[1][1:] in raw:
                yield ("check", lambda s, at=op[1][1:]: ("Z",) + at in s, f"PV{op[1][1:]} before its rows are zeroed")
            yield op

    progs["vp"], progs["mma"] = vp(), mma(progs["mma"])
    return progs


def _results(monkeypatch, shapes, seeds, flaw=None):
    monkeypatch.setattr(T, "_programs", lambda n, rnd, flawed: _programs(n, rnd, flaw))
    return {(nts, seed): T._run(nts, seed) for nts in shapes for seed in range(seeds)}


@pytest.mark.parametrize("first", [1, 2, 3, 4, 7])
def test_zeroed_tiles_never_deadlock_or_reorder(monkeypatch, first):
    shapes = [(first, b, c) for b, c in itertools.product([1, 2, 3, 6], [1, 2, 5])] + [(first, 1, 1, 2, 1, 3, 8)]
    bad = {k: r for k, r in _results(monkeypatch, shapes, 25).items() if r != "ok"}
    assert not bad, list(bad.items())[:3]


@pytest.mark.parametrize("flaw,what", [("phases restart", ("violation", "deadlock")), ("zeroed unseen", ("violation",)),
                                       ("handed over first", ("violation",))])
def test_a_planted_mistake_is_caught(monkeypatch, flaw, what):
    rnd = random.Random(0)
    shapes = [tuple(rnd.randint(1, 5) for _ in range(3)) for _ in range(20)]
    results = set(_results(monkeypatch, shapes, 25, flaw).values())
    assert any(r.startswith(what) for r in results), results
