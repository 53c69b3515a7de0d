"""CPU model check of the paged prefill kernel's mbarrier protocol over several
segments of a share (paged_prefill.cu): the roles go from one segment to the
next without a barrier of the CTA, and the phases run on. The scheduler and the
rules are those of test_prefill_protocol.py; a planted mistake (the producers
do not wait for the segment before) must be caught."""

import itertools
import random

import pytest

import test_prefill_protocol as T


def _programs(nts, rnd, flawed=False, rescale_prob=0.3):
    # Completions before each segment: of stage 0 and 1 tiles, of PRO[1].
    d = [(sum((n + 1) // 2 for n in nts[:g]), sum(n // 2 for n in nts[:g])) for g in range(len(nts))]
    twos = [sum(n >= 2 for n in nts[:g]) for g in range(len(nts))]

    def par(g, s, k):
        return (k + d[g][s]) & 1

    def last(kind, g):
        return lambda s: g == 0 or (kind, g - 1, nts[g - 1] - 1) in s

    def producer(is_k):
        def prog():
            for g, n in enumerate(nts):
                if g > 0 and not flawed:
                    yield ("wait", "MMA_DONE", (g - 1) & 1)
                yield ("check", last("S", g), "Q or K over what an S reads") if is_k else (
                    "check", last("PV", g), "V over what a P.V reads")
                if is_k:
                    yield ("tma", "Q", ("Q", g))
                for j in range(n):
                    if j >= 2:
                        if is_k and j < 4:
                            yield ("wait", ("PRO", j - 2), (g if j == 2 else twos[g]) & 1)
                        else:
                            yield ("wait", ("DONE", j & 1), par(g, j & 1, (j >> 1) - (2 if is_k else 1)))
                        need = ("S" if is_k else "PV", g, j - 2)
                        yield ("check", lambda s, need=need: need in s, f"a stage overwritten before {need}")
                    yield ("tma", ("KF" if is_k else "VF", j & 1), ("K" if is_k else "V", g, j))
                # The copies land before the producer goes on.
                if is_k:
                    yield ("wait", "Q", g & 1)
                for j in range(max(0, n - 2), n):
                    yield ("wait", ("KF" if is_k else "VF", j & 1), par(g, j & 1, j >> 1))
        return prog()

    def mma():
        for g, n in enumerate(nts):
            def s_(j):
                yield ("wait", ("KF", j & 1), par(g, j & 1, j >> 1))
                yield ("check", lambda s: ("K", g, j) in s and ("Q", g) in s, f"S{g}.{j} before its operands")
                yield ("mma", ("S", g, j))

            yield ("wait", "Q", g & 1)
            for j in range(min(2, n)):
                yield from s_(j)
                yield ("commit", ("PRO", j))
            for j in range(n):
                yield ("wait", ("VF", j & 1), par(g, j & 1, j >> 1))
                yield ("wait", ("PF", j & 1), par(g, j & 1, j >> 1))
                yield ("check", lambda s, j=j: ("V", g, j) in s and all(("P", g, j, w) in s for w in range(T.WARPS)),
                       f"PV{g}.{j} before P / V")
                yield ("check", lambda s, j=j: j > 0 or g == 0 or all(("O", g - 1, w) in s for w in range(T.WARPS)),
                       "O overwritten before it is read out")
                yield ("mma", ("PV", g, j))
                if j + 2 < n:
                    yield from s_(j + 2)
                yield ("commit", ("DONE", j & 1))
            for x in (0, 1):
                if n > x:
                    yield ("wait", ("DONE", x), par(g, x, (n - x - 1) >> 1))
            yield ("commit", "MMA_DONE")
            yield ("wait", "MMA_DONE", g & 1)

    def softmax(w):
        for g, n in enumerate(nts):
            for j in range(n):
                if j < 2:
                    yield ("wait", ("PRO", j), (g if j == 0 else twos[g]) & 1)
                else:
                    yield ("wait", ("DONE", j & 1), par(g, j & 1, (j >> 1) - 1))
                yield ("check", lambda s, j=j: ("S", g, j) in s, f"S{g}.{j} read before it is computed")
                if j >= 1 and rnd.random() < rescale_prob:
                    yield ("wait", ("DONE", (j - 1) & 1), par(g, (j - 1) & 1, (j - 1) >> 1))
                    yield ("check", lambda s, j=j: ("PV", g, j - 1) in s, f"O rescaled under PV{g}.{j - 1}")
                yield ("done", ("P", g, j, w))
                yield ("arrive", ("PF", j & 1), (g, j))
            yield ("wait", ("DONE", (n - 1) & 1), par(g, (n - 1) & 1, (n - 1) >> 1))
            yield ("check", lambda s: ("PV", g, n - 1) in s, "O read out under the last P.V")
            yield ("done", ("O", g, w))

    progs = {"kp": producer(True), "vp": producer(False), "mma": mma()}
    for w in range(T.WARPS):
        progs[f"softmax{w}"] = softmax(w)
    return progs


@pytest.mark.parametrize("first", [1, 2, 3, 4, 5, 9])
def test_segments_never_deadlock_or_reorder(monkeypatch, first):
    monkeypatch.setattr(T, "_programs", _programs)
    shapes = [(first, b, c) for b, c in itertools.product([1, 2, 3, 4, 7], [1, 2, 5])] + [(first, 1, 1, 2, 1, 3, 8)]
    bad = [(nts, seed, r) for nts in shapes for seed in range(25) for r in [T._run(nts, seed)] if r != "ok"]
    assert not bad, bad[:3]


def test_the_checker_catches_a_producer_that_does_not_wait_for_the_segment(monkeypatch):
    monkeypatch.setattr(T, "_programs", lambda n, rnd, flawed: _programs(n, rnd, flawed=True))
    rnd = random.Random(0)
    shapes = [(rnd.randint(1, 5), rnd.randint(1, 5), rnd.randint(1, 5)) for _ in range(20)]
    results = {T._run(nts, seed) for nts in shapes for seed in range(25)}
    assert any(r.startswith("violation") for r in results), results
