"""A model of the tensor-core kernel's barriers (csrc/linear_sm100.cu, lin_tc_kernel), run in random orders.

Every role of the kernel is a list of waits, arrivals and asynchronous completions, as in the source: the TMA warp, three MMA warps
(completions of one warp in order, after a random time), the state warps and the output warps.  A wait names the phase it means, and goes by parity, as
mbarrier.try_wait.parity does: it must not return before that phase is complete (but for the one wait whose early return only
changes an order), must not miss it, and every role must end.  The first form of the kernel missed phases in two places when one role
fell behind, which showed on the GPU only as a rare wait that gave up."""
import heapq
import random

import pytest


class Bar:
    def __init__(self, count):
        self.count = self.left = count
        self.done = 0

    def arrive(self):
        self.left -= 1
        if not self.left:
            self.left, self.done = self.count, self.done + 1


def roles(wide, swap, na, nb, chunks):
    """{name: generator}; ("wait", barrier, phase[, "hint"]), ("arrive", barrier), ("load", barrier), ("mma", steps, barriers)."""
    groups, two = max(na, nb), 2
    items = chunks * groups
    stages = {"A": 1 if wide else two, "B": 1 if wide and swap else two, "C": 1 if wide and not swap else two}
    at = lambda n, i: ((n, i % stages[n]), i // stages[n])
    full = lambda n, i: ("wait", ("full",) + at(n, i)[0], at(n, i)[1])
    empty = lambda n, i: ("empty",) + at(n, i)[0]

    def tma():
        used = {"A": 0, "B": 0, "C": 0}
        for _ in range(chunks):
            for g in range(groups):
                new_b = g == 0 or nb > 1
                order = (["C"] if swap else ["B"]) * new_b + ["A"] * (g == 0 or na > 1) + (["B"] if swap else ["C"]) * new_b
                for n in order:
                    i = used[n]
                    if i >= stages[n]:
                        yield ("wait", empty(n, i), i // stages[n] - 1)
                    yield ("load", ("full",) + at(n, i)[0])
                    used[n] += 1

    def steps():
        ca = cb = -1
        for t in range(items):
            c, g = divmod(t, groups)
            first, last, end = g == 0, g == groups - 1, c == chunks - 1
            new_b, do_i = first or nb > 1, first or na > 1
            ca, cb = ca + do_i, cb + new_b
            yield t, c, first, last, end, new_b, do_i, ca, cb

    def mma1():
        noi = 0
        for t, c, first, last, end, new_b, do_i, ca, cb in steps():
            if new_b:
                yield full("B", cb)
            if do_i:
                yield full("A", ca)
            if t:
                yield ("wait", "PV", t - 1)
            yield ("mma", 8, ["P"] + [empty("A", ca)] * (last or na > 1) + [empty("B", cb)] * (last or nb > 1))
            if new_b:
                yield full("C", cb)
            yield ("wait", "P_READY", t)
            if do_i:
                yield ("wait", "OI_READ", noi)
                noi += 1
            yield ("mma", 16, ["PV"] + [empty("C", cb)] * (last or nb > 1))

    def mma2():
        nx = nor = 0
        for t, c, first, last, end, new_b, do_i, ca, cb in steps():
            if first:
                yield ("wait", "XS", nx)
                nx += 1
            if do_i:
                if t:
                    yield ("wait", "O_READ", nor)
                    nor += 1
                yield full("A", ca)
                yield ("wait", "P", t, "hint")
                yield ("mma", 16, ["OI"] + ["X_READ"] * (na == 1 or last))
            if last or na > 1:
                yield ("mma", 0, [empty("A", ca)])

    def mma3():
        nx = nbt = 0
        for t, c, first, last, end, new_b, do_i, ca, cb in steps():
            do_b = new_b and not end
            if first and not end:
                yield ("wait", "XS", nx)
                nx += 1
            if do_b:
                yield ("wait", "BT", nbt)
                nbt += 1
            if new_b and (swap or not do_b):
                yield full("B", cb)
            if not swap and (last or nb > 1):
                yield ("arrive", empty("B", cb))
            if new_b and (not swap or not do_b):
                yield full("C", cb)
            if do_b:
                yield ("mma", 16, ["X_DONE"])
            if last or nb > 1:
                yield ("mma", 0, [empty("B", cb)] * swap + [empty("C", cb)])

    def state():
        nbt = 0
        for t, c, first, last, end, new_b, do_i, ca, cb in steps():
            do_b = new_b and not end
            if first and t:
                yield ("wait", "X_READ", c - 1)
            if nbt and (first or do_b):
                yield ("wait", "X_DONE", nbt - 1)
            if first:
                yield ("arrive", "XS")
            if do_b:
                yield full("C" if swap else "B", cb)
                yield ("arrive", "BT")
                nbt += 1

    def out():
        noi = 0
        for t in range(items + 1):
            if t:
                yield ("wait", "PV", t - 1)
                if nb == 1 or (t - 1) % groups == groups - 1:
                    yield ("arrive", "O_READ")
            if t == items:
                return
            yield ("wait", "P", t)
            yield ("arrive", "P_READY")
            if nb == 1 or t % groups == 0:
                yield ("wait", "OI", noi)
                noi += 1
                yield ("arrive", "OI_READ")

    warps = 3
    made = {"tma": tma(), "mma1": mma1(), "mma2": mma2(), "mma3": mma3()}
    made.update({f"state{i}": state() for i in range(warps)})
    made.update({f"out{i}": out() for i in range(warps)})
    bars = {n: Bar(1) for n in ("P", "PV", "X_DONE", "OI", "X_READ")}
    bars.update({n: Bar(warps) for n in ("P_READY", "XS", "BT", "OI_READ", "O_READ")})
    for n in "ABC":
        for s in range(2):
            bars[("full", n, s)], bars[("empty", n, s)] = Bar(1), Bar(2)
    return made, bars


def play(seed, wide, swap, na, nb, chunks):
    rng = random.Random(seed)
    made, bars = roles(wide, swap, na, nb, chunks)
    slow = {n: rng.choice([1, 1, 5, 30]) for n in made}
    now, op, free, ended, pipe, later, count = 0.0, {}, dict.fromkeys(made, 0.0), set(), dict.fromkeys(made, 0.0), [], 0
    while len(ended) < len(made):
        moved = False
        while later and later[0][0] <= now:
            for b in heapq.heappop(later)[2]:
                bars[b].arrive()
            moved = True
        for n in rng.sample(sorted(made), len(made)):
            if n in ended or free[n] > now:
                continue
            if n not in op:
                op[n] = next(made[n], None)
                if op[n] is None:
                    ended.add(n)
                    moved = True
                    continue
            what, b, *rest = op[n]
            if what == "wait":
                bar, phase = bars[b], rest[0]
                if (bar.done & 1) == (phase & 1):
                    assert bar.done <= phase, f"{n} misses phase {phase} of {b}, which is at {bar.done}"
                    continue
                assert bar.done > phase or rest[1:] == ["hint"], f"{n} passes phase {phase} of {b}, which is at {bar.done}"
            elif what == "arrive":
                bars[b].arrive()
            elif what == "load":
                heapq.heappush(later, (now + 5 + 20 * rng.expovariate(1), count, [b]))
            else:
                pipe[n] = max(pipe[n], now) + b * 2 * rng.random()
                heapq.heappush(later, (pipe[n], count, rest[0]))
            count += 1
            del op[n]
            free[n] = now + slow[n] * rng.expovariate(1)
            moved = True
        if not moved:
            ahead = [free[n] for n in made if n not in ended and free[n] > now] + [e[0] for e in later[:1]]
            assert ahead, f"nobody moves: { {n: op[n] for n in made if n not in ended} }"
            now = min(ahead)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("swap,na,nb", [(False, 1, 1), (False, 2, 1), (False, 4, 1), (False, 1, 2), (False, 1, 4), (True, 1, 1), (True, 1, 2), (True, 1, 3)])
def test_roles_keep_in_step(wide, swap, na, nb):
    for seed in range(60):
        play(seed, wide, swap, na, nb, (1, 2, 3, 4, 6)[seed % 5])
