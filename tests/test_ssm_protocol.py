"""The barriers of the chunked scan's output kernel (csrc/ssm_prefill_chunked.cu) as a model on the
CPU: every role as the sequence of its waits, arrivals and accesses, run under schedules that let
any role fall behind as far as the barriers allow.

A wait by parity passes when its barrier's current phase has the other parity, so it is sound only
while that barrier is in the awaited phase or the one after. The model checks this at every poll,
and that every access finds the chunk that it is meant for.
"""
import random
import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parents[1] / "flashinfer_bench_tma_thrust_b200" / "csrc" / \
    "ssm_prefill_chunked.cu"

X_STAGES, PLACES, GATE_STAGES, WARPS = 3, 2, 4, 2  # WARPS: of each role, the barriers' counts


class Unsound(Exception):
    """A wait whose barrier is behind or ahead of it, or an access to the wrong chunk's data."""


class Bar:
    def __init__(self, name, count):
        self.name, self.count, self.pending, self.phase = name, count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def passed(self, k):
        """The test of phase k's parity."""
        if self.phase not in (k, k + 1):
            raise Unsound(f"{self.name}: a wait for phase {k} meets phase {self.phase}")
        return self.phase % 2 != k % 2


class Model:
    def __init__(self, chunks, ragged, x_read=0, free_by_quarter=True, checked_late=False):
        """As the kernel has it; or with "x read" as barriers of its own (``x_read`` of them), with
        one barrier per place of f x, or with "checked" waited for behind the hand-over of Y."""
        self.n, self.ragged, self.slots = chunks, ragged, x_read
        self.by_quarter, self.late = free_by_quarter, checked_late
        b = lambda name, count, k=None: (  # noqa: E731
            Bar(name, count) if k is None else [Bar(f"{name}[{i}]", count) for i in range(k)])
        self.full_x, self.full_b, self.full_c = b("full_x", 1, X_STAGES), b("full_b", 1), b("full_c", 1)
        self.gates_full, self.gates_free = b("gates_full", 1, GATE_STAGES), \
            b("gates_free", 2 * WARPS, GATE_STAGES)
        self.cb, self.ds, self.ym = b("cb", 1), b("ds", 1), b("ym", 1)
        self.fx, self.fx_free = b("fx", WARPS, PLACES), b("fx_free", 1, 4)
        self.my, self.state, self.y_free = b("my", WARPS), b("state", WARPS), b("y_free", WARPS)
        self.staged, self.zeroed = b("staged", WARPS, X_STAGES), b("zeroed", WARPS)
        self.checked, self.together = b("checked", WARPS), b("together", WARPS)
        self.x_read = b("x_read", WARPS, self.slots)
        # what each place holds, by the warp whose part it is
        self.X = [[None] * WARPS for _ in range(X_STAGES)]
        self.F = [[None] * WARPS for _ in range(PLACES)]
        self.G, self.Y, self.S = [None] * WARPS, [None] * WARPS, [None] * WARPS
        self.B = self.C = self.D = None
        self.clean = [0] * chunks  # warps that have taken what is not finite out of x
        self.pipe, self.loads = [], []  # products and commits, bulk loads: each in order
        self.done = False

    def expect(self, got, want, what):
        if any(g != want for g in (got if isinstance(got, list) else [got])):
            raise Unsound(f"{what}: found {got}, wanted {want}")

    def is_ragged(self, c):
        return self.ragged and c == self.n - 1

    # Roles: generators that yield what they wait for (None: nothing, another may go first).

    def write_fx(self, w, c, t):
        place, last = (4 * c + t) % PLACES, 4 * c + t - PLACES
        self.expect(self.X[c % X_STAGES], ("x", c), "x read for f x")
        if last >= 0:
            if self.by_quarter:
                yield lambda: self.fx_free[last % 4].passed(last // 4)
            else:
                yield lambda: self.fx_free[place].passed(last // PLACES)
        self.F[place][w] = (c, t)
        yield None
        self.fx[place].arrive()
        if t == 3 and self.slots:
            self.x_read[c % self.slots].arrive()

    def first_fx(self, w, c):
        yield lambda: self.full_x[c % X_STAGES].passed(c // X_STAGES)
        if self.is_ragged(c):
            yield lambda: self.zeroed.passed(0)
        yield lambda: self.gates_full[c % GATE_STAGES].passed(c // GATE_STAGES)
        yield from self.write_fx(w, c, 0)

    def output(self, w):
        yield from self.first_fx(w, 0)
        for c in range(self.n):
            yield lambda: self.gates_full[c % GATE_STAGES].passed(c // GATE_STAGES)
            yield lambda: self.cb.passed(c)
            self.expect([self.G[w], self.Y[w]], ("cb", c), "C B^T and C S^T")
            yield None
            self.G[w] = self.Y[w] = ("m", c)
            self.my.arrive()
            self.gates_free[c % GATE_STAGES].arrive()
            yield None
            if c + 1 < self.n:
                yield from self.first_fx(w, c + 1)
            yield lambda: self.ym.passed(c)
            if not self.late:
                yield lambda: self.checked.passed(c)
            self.expect(self.Y[w], ("y", c), "Y read out")
            yield None
            self.y_free.arrive()
            if self.late:
                yield lambda: self.checked.passed(c)
            if self.slots:
                yield lambda: self.x_read[c % self.slots].passed(c // self.slots)
            self.X[c % X_STAGES][w] = ("out", c)
            yield None
            if not self.is_ragged(c):
                self.staged[c % X_STAGES].arrive()

    def states(self, w):
        def hand_over(c):
            self.S[w] = c
            self.state.arrive()

        hand_over(0)
        for c in range(self.n + 1):
            if c < self.n:
                yield lambda: self.full_x[c % X_STAGES].passed(c // X_STAGES)
                if self.is_ragged(c):
                    yield lambda: self.full_b.passed(c)
                    self.expect(self.B, c, "B, to be cut")
                    self.together.arrive()
                    yield lambda: self.together.phase > 0
                    self.zeroed.arrive()
                yield lambda: self.gates_full[c % GATE_STAGES].passed(c // GATE_STAGES)
            if c > 0:
                yield lambda: self.ds.passed(c - 1)
                self.expect(self.D, (c - 1, 3), "dS")
                self.expect(self.X[(c - 1) % X_STAGES], ("x", c - 1), "x to be checked")
                yield None
                self.clean[c - 1] += 1
                self.checked.arrive()
                yield None
                self.gates_free[(c - 1) % GATE_STAGES].arrive()
                if c < self.n:
                    hand_over(c)
            for t in (1, 2, 3) if c < self.n else ():
                yield from self.write_fx(w, c, t)

    def issue(self):
        for c in range(self.n):
            has = dict(b=False, s=False, cb=False, ym=False, t=0)

            def look(act, c=c, has=has):
                """One turn of the issuing loop (act: False only says whether it would act)."""
                has["b"] = has["b"] or self.full_b.passed(c)
                has["s"] = has["s"] or self.state.passed(c)
                t, acted = has["t"], False
                if has["b"] and has["s"] and t < (4 if has["cb"] else 3) and \
                        self.fx[(4 * c + t) % PLACES].passed((4 * c + t) // PLACES):
                    if not act:
                        return True
                    free = self.fx_free[t if self.by_quarter else (4 * c + t) % PLACES]
                    self.pipe += [("ds", c, t), ("arrive", free)]
                    self.pipe += [("arrive", self.ds)] if t == 3 else []
                    has["t"], acted = t + 1, True
                if not has["cb"]:
                    if has["b"] and has["s"] and self.full_c.passed(c) \
                            and (not self.is_ragged(c) or self.zeroed.passed(0)) \
                            and (c == 0 or self.y_free.passed(c - 1)):
                        if not act:
                            return True
                        self.pipe += [("cb", c), ("arrive", self.cb)]
                        has["cb"] = acted = True
                elif not has["ym"] and self.my.passed(c) and self.checked.passed(c):
                    if not act:
                        return True
                    self.pipe += [("ym", c), ("arrive", self.ym)]
                    has["ym"] = acted = True
                return acted

            while not has["ym"] or has["t"] < 4:
                yield lambda: look(False)
                look(True)

    def products(self):
        while True:
            yield lambda: bool(self.pipe)
            kind, *op = self.pipe[0]
            if kind == "arrive":
                op[0].arrive()
                self.pipe.pop(0)
                continue
            c = op[0]

            def inputs():
                if kind == "ds":
                    self.expect(self.F[(4 * c + op[1]) % PLACES], (c, op[1]), "f x as an operand")
                    self.expect(self.B, c, "B of dS")
                elif kind == "cb":
                    self.expect([self.B, self.C] + self.S, c, "B, C and S")
                else:
                    self.expect(self.G, ("m", c), "M")
                    self.expect(self.X[c % X_STAGES], ("x", c), "x of M x")
                    self.expect(self.clean[c], WARPS, "x without what is not finite")

            inputs()
            yield None
            inputs()  # and still so at its end
            if kind == "ds":
                self.D = (c, op[1])
            elif kind == "cb":
                self.G, self.Y = [("cb", c)] * WARPS, [("cb", c)] * WARPS
            else:
                self.expect(self.Y, ("m", c), "Y to add to")
                self.Y = [("y", c)] * WARPS
            self.pipe.pop(0)

    def copies(self):
        def load(what, c):
            self.loads.append((what, c))

        load("b", 0), load("c", 0)
        for c in range(min(X_STAGES, self.n)):
            load("x", c)
        for c in range(self.n):
            if c + 1 < self.n:
                yield lambda: self.cb.passed(c)
                load("c", c + 1)
                yield lambda: self.ds.passed(c)
                load("b", c + 1)
            if not self.is_ragged(c):
                yield lambda: self.staged[c % X_STAGES].passed(c // X_STAGES)
                self.expect(self.X[c % X_STAGES], ("out", c), "y to be stored")
                if c + X_STAGES < self.n:
                    load("x", c + X_STAGES)

    def arrivals(self):
        while True:
            yield lambda: bool(self.loads)
            what, c = self.loads.pop(0)
            if what == "x":
                self.X[c % X_STAGES] = [("x", c)] * WARPS
                self.full_x[c % X_STAGES].arrive()
            else:
                setattr(self, what.upper(), c)
                getattr(self, "full_" + what).arrive()

    def gates(self):
        for c in range(self.n):
            if c >= GATE_STAGES:
                yield lambda: self.gates_free[c % GATE_STAGES].passed(c // GATE_STAGES - 1)
            yield None
            self.gates_full[c % GATE_STAGES].arrive()

    def run(self, rng):
        """Strict priorities, redrawn for one role now and then: whoever is last falls behind as
        far as it can."""
        roles = [self.output(w) for w in range(WARPS)] + [self.states(w) for w in range(WARPS)]
        roles += [self.issue(), self.copies(), self.gates()]
        service = [self.products(), self.arrivals()]
        waits = {r: (lambda: True) for r in roles + service}
        order = roles + service
        rng.shuffle(order)
        while any(r in waits for r in roles):
            # every pending wait is polled, as on the machine, so that an unsound one is seen
            able = [r for r in order if r in waits and waits[r]()]
            if not able:
                raise Unsound("nobody can go on")
            if rng.random() < 0.03:
                order.remove(able[0])
                order.append(able[0])
            try:
                waits[able[0]] = next(able[0]) or (lambda: True)
            except StopIteration:
                del waits[able[0]]


def schedules(count, **kw):
    for seed in range(count):
        rng = random.Random(seed)
        Model(rng.randint(1, 9), rng.random() < 0.5, **kw).run(rng)


def test_every_wait_meets_its_phase():
    schedules(600)


def test_the_model_sees_a_barrier_that_runs_ahead():
    """One barrier for all chunks' "x read" let the state's warps go two chunks ahead of an output
    warp that had yet to look at it: the block then stood still. So would one for "checked" that is
    looked at behind the hand-over of Y. Two, by the chunk's parity, do not."""
    with pytest.raises(Unsound, match="x_read"):
        schedules(600, x_read=1)
    with pytest.raises(Unsound, match="checked"):
        schedules(600, checked_late=True)
    schedules(200, x_read=2)


def test_the_model_sees_a_phase_that_is_skipped():
    """One barrier per place of f x has two phases per chunk. The output's warps, which write one
    quarter of four, looked at every other, and could write over a quarter still to be read."""
    with pytest.raises(Unsound, match="fx_free"):
        schedules(600, free_by_quarter=False)


def test_tmem_accesses_are_fenced_behind_the_products():
    """Each wait on a barrier that a product's commit completes is followed by the fence that orders
    this thread's tensor memory accesses behind it, before the next such access. (The issuing
    warp's and the copies' waits precede none.)"""
    code = re.sub(r"//[^\n]*", "", SOURCE.read_text())
    events = re.findall(
        r"\bwait\(bars_u \+ 8 \* \(?(kCB|kYM|kDS|kFxFree)\b|\b(tc_fence_after)\(\)"
        r"|\b(tmem_ld|tmem_st)(?:\d+|_frag)\(", code)
    pending, seen = None, set()
    for bar, fence, access in events:
        if bar:
            pending = bar
            seen.add(bar)
        elif fence:
            pending = None
        else:
            assert pending is None, f"{access} behind a wait for {pending} without a fence"
    assert seen == {"kCB", "kYM", "kDS", "kFxFree"}
