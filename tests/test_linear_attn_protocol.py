"""The barriers of the tensor-core linear attention kernels, on the CPU.

A wait names the parity of the phase that it wants.  If the phase after that one
can complete before the waiter has looked, the wait sees the other parity and
stays until its limit.  The roles of the two kernels are restated here as
programs of waits and arrivals, with the barriers' array sizes read from the
kernels' source, and run under many schedules: priorities that starve one role
after another, and random ones.  No schedule may complete two phases past a
wait, or leave a role waiting for good.
"""

import itertools
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gateddeltanet-2_b200", "csrc",
                      "linear_attn_tc.cu")


def declared(struct):
    """{barrier: array size as written, or None} of a shared-memory struct."""
    text = open(SOURCE).read()
    body = text[text.index("struct alignas(1024) " + struct):]
    body = body[:body.index("\n};")]
    out = {}
    for line in re.findall(r"uint64_t ([^;]+);", body):
        for item in line.split(","):
            name, size = re.match(r"\s*(\w+)(?:\[(\w+)\])?", item).groups()
            out[name] = size
    return out


class Machine:
    def __init__(self):
        self.need, self.left, self.done = {}, {}, {}
        self.roles, self.queues, self.loads = {}, {}, []

    def bar(self, name, n, count):
        for i in range(n):
            self.need[name, i] = self.left[name, i] = count
            self.done[name, i] = 0

    def arrive(self, b, count):
        while count:
            step = min(count, self.left[b])
            self.left[b] -= step
            count -= step
            if self.left[b] == 0:
                self.left[b] = self.need[b]
                self.done[b] += 1

    def step(self, r):
        """One operation of role r; whether it could."""
        if r in self.queues:
            if not self.queues[r]:
                return False
            self.arrive(self.queues[r].pop(0), 1)
            return True
        if r == "tma":
            if not self.loads:
                return False
            self.arrive(self.loads.pop(), 1)
            return True
        op = self.roles[r][0]
        if op is None:
            return False
        kind, b, x = op
        if kind == "wait":
            assert self.done[b] <= x + 1, f"{r} missed phase {x} of {b}: {self.done[b]} are complete"
            if self.done[b] != x + 1:
                return False
        elif kind == "arrive":
            self.arrive(b, x)
        elif kind == "load":
            self.loads.append(b)
        else:  # an MMA issuer's commit: in its order, some time later
            self.queues[x].append(b)
        self.roles[r][0] = next(self.roles[r][1], None)
        return True

    def run(self, programs, pick):
        self.roles = {r: [next(p, None), p] for r, p in programs.items()}
        agents = [*self.roles, *self.queues, "tma"]
        while True:
            for r in pick(agents):
                if self.step(r):
                    break
            else:
                break
        stuck = {r: s[0] for r, s in self.roles.items() if s[0] is not None}
        assert not stuck, f"waiting for good: {stuck}"


def schedules():
    """Fixed priorities, then random ones, then mixtures."""
    def fixed(order):
        return lambda agents: sorted(agents, key=lambda r: order[r])

    for seed in range(400):
        rng = random.Random(seed)
        if seed % 3 == 0:
            order = {}
            yield fixed(type("Order", (dict,), {"__missing__": lambda s, k, g=rng: s.setdefault(k, g.random())})(order))
        elif seed % 3 == 1:
            yield lambda agents, g=rng: g.sample(agents, len(agents))
        else:  # one role last, the others at random
            who = rng.random()

            def pick(agents, g=rng, w=who):
                last = agents[int(w * len(agents))]
                return [r for r in g.sample(agents, len(agents)) if r != last] + [last]
            yield pick


def scan(total, heads, out, store, clear, pick):
    """la_scan_kernel: `total` chunks, `heads`: the first chunks of its tasks."""
    sizes = declared("ScanSmem")
    m = Machine()
    NX, NY, NB = (2, 3, 1) if out else (3, 3, 2)
    number = lambda name: {None: 1, "NX": NX, "NY": NY, "NB": NB, "2": 2}[sizes[name]]  # noqa: E731
    counts = dict(full_x=1, empty_x=2 if out else 1, full_y=1, empty_y=1 if out else 128, y_ready=128, f_full=32,
                  f_empty=16 if out else 4, qk_full=1, p_full=256, o_full=2, yw_full=128, ds_full=1, ds_free=128,
                  s_full=128, s_free=1, o_free=128, drained=2 if out else 1)
    assert set(counts) == set(sizes)
    for name, c in counts.items():
        m.bar(name, number(name), c)
    m.queues = {"pipe1": [], "pipe3": []}

    def at(name, i):  # the barrier and phase of the i-th use
        n = number(name)
        return (name, i % n), i // n

    def wait(name, i):
        b, phase = at(name, i)
        return "wait", b, phase

    def arrive(name, i, count):
        return "arrive", at(name, i)[0], count

    def commit(name, i, queue):
        return "commit", at(name, i)[0], queue

    def loads():
        for it in range(total):
            if it >= NY:
                yield wait("empty_y", it - NY)
            yield "load", at("full_y", it)[0], 0
            if it >= NX:
                yield wait("empty_x", it - NX)
            yield "load", at("full_x", it)[0], 0

    def stored(d):
        yield wait("s_full", d)
        yield arrive("s_free", d, 1)

    def sums():
        for it in range(total):
            if out and store and it >= 2:
                yield from stored(it - 2)
            if it >= 2:
                yield wait("f_empty", it - 2)
            yield arrive("f_full", it, 32)
        if out and store:
            for d in range(max(total - 2, 0), total):
                yield from stored(d)

    def issuer1():
        if not out:
            for it in range(total if store else 0):
                yield from stored(it)
            return
        for it in range(total + (total > 0)):
            if it < total:
                yield wait("full_x", it)
                yield commit("qk_full", it, "pipe1")
                yield commit("empty_x", it, "pipe1")
            if it > 0:
                j = it - 1
                if j > 0:
                    yield wait("o_free", j - 1)
                yield wait("y_ready", j)
                yield wait("p_full", j)
                yield commit("o_full", j, "pipe1")
                yield commit("empty_y", j, "pipe1")
        yield commit("drained", 0, "pipe1")
        yield wait("drained", 0)

    def issuer3():
        for it in range(total):
            yield wait("full_x", it)
            yield wait("yw_full", it)
            if out and it > 0:
                yield wait("ds_free", it - 1)
            yield commit("ds_full", it, "pipe3")
            if out:
                if it >= 2:
                    yield wait("o_free", it - 2)
                yield wait("s_full", it)
                yield commit("o_full", it, "pipe3")
            yield commit("empty_x", it, "pipe3")
        yield commit("drained", 0, "pipe3")
        yield wait("drained", 0)

    def scores():  # half of the warps
        for it in range(total):
            yield wait("f_full", it)
            yield arrive("f_empty", it, 4)
            yield wait("qk_full", it)
            yield arrive("p_full", it, 128)

    def made(it, half):  # w v of a chunk, by half of its warps
        yield wait("f_full", it)
        yield arrive("f_empty", it, 2)
        yield wait("full_y", it)
        if clear:
            yield wait("full_x", it)
        if it >= NB:
            yield wait("ds_full", it - NB)
        yield arrive("yw_full", it, half)
        yield arrive("y_ready" if out else "empty_y", it, half)

    def taken(d, half):
        yield wait("ds_full", d)
        if out:
            yield arrive("ds_free", d, half)

    def state():
        for it in range(total):
            if it > 0 and it in heads:
                yield from taken(it - 1, 64)
            if out:
                yield wait("f_full", it)
                yield arrive("f_empty", it, 2)
            else:
                yield from made(it, 64)
            if it > 0 and it not in heads:
                yield from taken(it - 1, 64)
            if out or store:
                if store and it > 0:
                    yield wait("s_free", it - 1)
                if out and it > 0:
                    yield wait("empty_x", it - 1)
                yield arrive("s_full", it, 64)
        if total:
            yield from taken(total - 1, 64)

    def output():
        def one(d):
            yield wait("o_full", d)
            yield arrive("o_free", d, 64)
        for it in range(total):
            yield from made(it, 64)
            if it > 1:
                yield from one(it - 2)
        for d in range(max(total - 2, 0), total):
            yield from one(d)

    programs = dict(loads=loads(), sums=sums(), issuer1=issuer1(), issuer3=issuer3(), state_a=state(), state_b=state())
    if out:
        programs.update(scores_a=scores(), scores_b=scores(), output_a=output(), output_b=output())
    m.run(programs, pick)


def backward(total, clear, dg, pick):
    """la_bwd_tc_kernel: `total` pairs of a chunk and a value head."""
    sizes = declared("BwdSmem")
    m = Machine()
    counts = dict(full=1, empty=17, f_full=32, f_empty=16, clean=512, g1=1, g2_=1, pe=512, rmw1=512, g3=1, rmw2=512,
                  g4a=1, g4b=1, qk_free=512, dv_free=512, xy_full=512, xy_free=32, aborted=1)
    assert set(counts) == set(sizes)
    for name, c in counts.items():
        m.bar(name, int(sizes[name] or 1), c)
    m.queues = {"pipe": []}
    Q, K, DO, V, S, DS = range(6)
    slot = lambda x, n: (0x201534 >> (4 * x)) & 7 if n & 1 else x  # noqa: E731
    wait = lambda name, n, i=0: ("wait", (name, i), n)  # noqa: E731
    arrive = lambda name, c, i=0: ("arrive", (name, i), c)  # noqa: E731
    commit = lambda name, i=0: ("commit", (name, i), "pipe")  # noqa: E731

    def loads():
        for n, x in itertools.product(range(total), range(6)):
            if n > 0:
                yield wait("empty", n - 1, slot(x, n))
            yield "load", ("full", slot(x, n)), 0

    def issuer():
        for n in range(total):
            def full(x, n=n):
                return wait("full", n, slot(x, n))
            yield full(Q)
            yield full(K)
            yield wait("clean", n)
            yield full(DO)
            yield full(V)
            if n > 0:
                yield wait("dv_free", n - 1)
            yield commit("g1")
            yield full(S)
            if n > 0:
                yield wait("qk_free", n - 1)
            yield full(DS)
            yield commit("g2_")
            yield commit("empty", slot(V, n))
            yield commit("empty", slot(S, n))
            yield wait("pe", n)
            yield commit("g3")
            yield commit("empty", slot(DS, n))
            yield wait("rmw1", n)
            yield commit("g4a")
            yield commit("empty", slot(Q, n))
            yield commit("empty", slot(K, n))
            yield wait("rmw2", n)
            yield commit("g4b")
            yield commit("empty", slot(DO, n))
        yield commit("aborted")
        yield wait("aborted", 0)

    def sums():
        for n in range(total):
            if n > 0:
                yield wait("f_empty", n - 1)
            yield arrive("f_full", 32)

    def decays():
        for n in range(total if dg else 0):
            yield wait("xy_full", n)
            yield arrive("xy_free", 32)

    def rows():  # a quarter of the warps
        for n in range(total):
            if clear:
                for x in (Q, K, DO, V):
                    yield wait("full", n, slot(x, n))
            yield arrive("clean", 128)
            yield wait("f_full", n)
            yield wait("g1", n)
            yield arrive("pe", 128)
            yield arrive("f_empty", 4)
            yield wait("g2_", n)
            yield arrive("rmw1", 128)
            for x in (S, DS, V, DO, K):
                yield arrive("empty", 4, slot(x, n))
            yield wait("g3", n)
            yield arrive("rmw2", 128)
            yield wait("g4a", n)
            yield arrive("empty", 4, slot(Q, n))
            yield arrive("qk_free", 128)
            if dg:
                if n > 0:
                    yield wait("xy_free", n - 1)
                yield arrive("xy_full", 128)
            yield wait("g4b", n)
            yield arrive("dv_free", 128)

    programs = dict(loads=loads(), issuer=issuer(), sums=sums(), decays=decays())
    programs.update({f"rows_{i}": rows() for i in range(4)})
    m.run(programs, pick)


@pytest.mark.parametrize("out,store", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("total,heads", [(1, (0,)), (2, (0, 1)), (3, (0,)), (5, (0, 2, 3)), (8, (0,)), (9, (0, 4))])
def test_scan(out, store, total, heads):
    for i, pick in enumerate(schedules()):
        scan(total, heads, out, store, i % 2 == 0, pick)


@pytest.mark.parametrize("dg", [False, True])
@pytest.mark.parametrize("total", [1, 2, 5])
def test_backward(total, dg):
    for i, pick in enumerate(schedules()):
        backward(total, i % 2 == 0, dg, pick)
