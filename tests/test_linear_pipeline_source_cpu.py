"""The model of the tensor-core kernel's barriers (test_linear_pipeline_cpu) against the kernel's source: who waits for what, who arrives
where, in which order, and how many arrivals complete a phase.  A change of lin_tc_kernel's barriers fails here until the model follows."""
import os
import re

import pytest

import fa_abi as A
from test_linear_pipeline_cpu import roles

SOURCE = os.path.join(A.ROOT, "flash-attention-rdna2_b200", "csrc", "linear_sm100.cu")
# the model's names of the kernel's barriers
NAMES = {"P": "P_FULL", "PV": "PV_DONE", "XS": "XS_READY", "BT": "BT_READY", "OI": "OI_FULL", "X_DONE": "X_DONE", "X_READ": "X_READ",
         "P_READY": "P_READY", "OI_READ": "OI_READ", "O_READ": "O_READ"}
# where each role begins in the source, in its order
MARKS = [("tma", "if (warp == WARP_TMA && lane == 0) {"), ("mma1", "// ------------------------------------------------------------ P = a b^T, O = P c"),
         ("mma2", "// ------------------------------------------------------------ O = a X"),
         ("mma3", "// ------------------------------------------------------------ X += "), ("drain", "const uint32_t drain = bar"),
         ("state", "// ---------------------------------------------------------- state"), ("out", "// ---------------------------------------------------------- outputs"),
         ("end", "// states: what a segment adds to the state")]
# what a role does in the order of its text; a load is a wait for the buffer, then the copy
ORDER = {
    "tma": "load C, load B, load A, load B, load C, wait A_FULL, wait B_FULL, wait C_FULL",
    "mma1": "wait B_FULL, wait A_FULL, wait PV_DONE, commit P_FULL, commit A_EMPTY, commit B_EMPTY, wait C_FULL, wait P_READY, wait OI_READ, "
            "commit PV_DONE, commit C_EMPTY",
    "mma2": "wait XS_READY, wait O_READ, wait A_FULL, wait P_FULL, commit OI_FULL, commit X_READ, commit A_EMPTY",
    "mma3": "wait XS_READY, wait BT_READY, wait B_FULL, arrive B_EMPTY, wait C_FULL, commit X_DONE, commit B_EMPTY, commit C_EMPTY",
    "state": "wait X_READ, wait X_DONE, arrive XS_READY, wait C_FULL/B_FULL, arrive BT_READY",
    "out": "wait PV_DONE, arrive O_READ, wait P_FULL, arrive P_READY, wait OI_FULL, arrive OI_READ",
}


@pytest.fixture(scope="module")
def kernel():
    text = open(SOURCE).read()
    return text[text.index("lin_tc_kernel(const __grid_constant__"):text.index(MARKS[-1][1]) + len(MARKS[-1][1])]


def steps(text):
    """The barrier operations of a piece of source, in order."""
    found = []
    pattern = (r"load\(&t(?P<load>[abc]),|mma_commit\(bar \+ Bz::(?P<commit>\w+)|mbar_arrive\(bar \+ Bz::(?P<arrive>\w+)|"
               r"(?:mbar_wait|wait_warp)\(bar \+ Bz::(?P<w1>\w+)|\bwait\(Bz::(?P<w2>\w+)|\bwait\(\(SWAP \? Bz::(?P<w3>\w+) : Bz::(?P<w4>\w+)\)")
    for m in re.finditer(pattern, text):
        g = m.groupdict()
        if g["load"]:
            found.append("load " + g["load"].upper())
        elif g["w3"]:
            found.append(f"wait {g['w3']}/{g['w4']}")
        else:
            found += [f"{kind} {g[k]}" for kind, k in (("commit", "commit"), ("arrive", "arrive"), ("wait", "w1"), ("wait", "w2")) if g[k]]
    return found


def test_source_has_the_steps_that_the_model_was_made_of(kernel):
    places = [kernel.index(mark) for _, mark in MARKS]
    assert places == sorted(places)
    for (name, _), start, stop in zip(MARKS, places, places[1:]):
        if name in ORDER:
            assert ", ".join(steps(kernel[start:stop])) == ORDER[name], name


def test_model_has_each_role_step_of_the_source():
    """Over all forms together a role of the model waits for, arrives at and completes what the source's role does."""
    flat = lambda b: {"full": f"{b[1]}_FULL", "empty": f"{b[1]}_EMPTY"}[b[0]] if isinstance(b, tuple) else NAMES[b]
    did = {}
    for wide in (False, True):
        for swap, na, nb in ((False, 1, 1), (False, 3, 1), (False, 1, 3), (True, 1, 1), (True, 1, 3)):
            for name, role in roles(wide, swap, na, nb, 4)[0].items():
                mine = did.setdefault(name.rstrip("0123456789") if name.startswith(("state", "out")) else name, set())
                for op in role:
                    if op[0] == "mma":
                        mine.update("commit " + flat(b) for b in op[2])
                    elif op[0] == "load":
                        mine.add("load " + op[1][1])
                    else:
                        mine.add(f"{op[0]} {flat(op[1])}")
    for name, order in ORDER.items():
        want = set()
        for step in order.split(", "):
            kind, _, bars = step.partition(" ")
            want |= {f"{kind} {b}" for b in bars.split("/")}
        if name == "tma":      # the waits before a load are in the loader; those for the last copies end the role and hold nobody up
            want = {s for s in want if s.startswith("load")} | {f"wait {n}_EMPTY" for n in "ABC"}
        assert did[name] == want, name


def test_phases_complete_after_as_many_arrivals(kernel):
    bars = roles(False, False, 1, 1, 1)[1]
    counts = {m[0]: m[1] for m in re.findall(r"mbar_init\(bar \+ Bz::(\w+)(?: \+ 8 \* s)?, (\w+)\)", kernel)}
    assert counts.pop("DRAIN") == "1"      # one commit each, of the MMA warps' last
    every = {"1": 1, "2": 2, "NOUT": bars["P_READY"].count, "NSTATE": bars["XS"].count}      # the model has three warps of the eight
    assert {NAMES[n] for n in bars if not isinstance(n, tuple)} | {f"{n}_{k}" for n in "ABC" for k in ("FULL", "EMPTY")} == set(counts)
    for n, bar in bars.items():
        source = counts[f"{n[1]}_{n[0].upper()}" if isinstance(n, tuple) else NAMES[n]]
        assert bar.count == every[source], n
    assert {counts[n] for n in ("P_READY", "OI_READ", "O_READ")} == {"NOUT"} and {counts[n] for n in ("XS_READY", "BT_READY")} == {"NSTATE"}
