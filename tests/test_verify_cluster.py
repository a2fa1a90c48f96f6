"""CPU: what the kernels' source has to say and no run can show (a fault of this kind comes or stays
away with how the compiler lays out the code, or with how CTAs start): no CTA of a cluster stores to
another before a cluster-wide barrier has said that all of them run; assembly that reads memory is
volatile; every exponential knows its table."""
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


def test_assembly_that_loads_is_volatile():
    """The compiler may run other assembly ahead of the branch that guards its address."""
    for path in sorted((ROOT / "kernels_b200" / "csrc").glob("*.cu*")):
        for m in re.finditer(r'\basm\s*\(\s*((?:"[^"]*"\s*(?://[^\n]*\n\s*)?)+)', path.read_text()):
            assert not re.search(r"\b(ld|ldmatrix|ldu|atom|red)\.", m.group(1)), (path.name, m.group(1))


def test_every_exponential_has_its_table():
    """Of the kernels that never set it too: its address is read whatever the compiler makes of it."""
    assert "explicit Expo(const double* powers)" in SOURCE
    assert not re.search(r"\bExpo \w+\s*[;,]", SOURCE)
