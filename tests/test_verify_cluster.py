"""CPU: in the kernels' source, no CTA of a cluster stores to another before a cluster-wide
barrier has said that all of them run (which no run can show: they usually start together)."""
from __future__ import annotations

import re

from conftest import ROOT

SOURCE = (ROOT / "kernels_b200" / "csrc" / "verify.cu").read_text()


def body(name: str) -> str:
    """A kernel's text, from its name to the brace that closes it."""
    at = SOURCE.index("{", SOURCE.index(name + "("))
    depth = 0
    for i in range(at, len(SOURCE)):
        depth += {"{": 1, "}": -1}.get(SOURCE[i], 0)
        if depth == 0:
            return SOURCE[at:i]
    raise AssertionError(name)


def test_the_walk_waits_for_its_cluster_before_it_stores_to_it():
    text = re.sub(r"//[^\n]*", "", body("verify_walk_kernel"))
    # the lambdas that store remotely are defined first and called from the walk's loop on
    loop = text.index("for (;;)")
    arrive = [m.start() for m in re.finditer(r"cluster_here\(\)", text)]
    wait = [m.start() for m in re.finditer(r"cluster_all_here\(\)", text)]
    assert len(arrive) == len(wait) == 1
    # one arrival and one wait of every thread: both under the same condition, outside loops and
    # behind the only return, which the whole cluster takes
    assert text.rindex("return;", 0, arrive[0]) < arrive[0] < wait[0] < loop
    for at in (arrive[0], wait[0]):
        assert text[:at].rstrip().endswith("if (ctas > 1)")
    for call in re.finditer(r"\b(sums|mass_of|without)\(", text):   # (what stores remotely)
        assert call.start() > loop


def test_only_the_walk_stores_to_other_ctas():
    stores = [m.start() for m in re.finditer(r"store_remote\(", SOURCE)]
    walk = SOURCE.index("verify_walk_kernel")
    inside = body("verify_walk_kernel")
    assert len(stores) == 2            # its definition and the one use
    assert stores[0] < walk < stores[1] < walk + SOURCE[walk:].index(inside) + len(inside)
