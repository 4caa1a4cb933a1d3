"""Which copies a CTA waits for before it leaves behind a wait that ran out (csrc/copy_ring.h, compiled here), against
barriers whose phases are counted: a wait for a parity returns once the barrier is no longer in the phase of that parity."""
import itertools
import os
import re
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "nncp-metal_b200", "csrc")


@pytest.fixture(scope="module")
def ring(tmp_path_factory):
    d = tmp_path_factory.mktemp("copy_ring")
    (d / "ring.cc").write_text("""#include <cstdio>
#include "copy_ring.h"
int main() { int places, asked; while (scanf("%d %d", &places, &asked) == 2) {
 CopyRing r(places); r.asked = asked;
 for (int j = 0; j < asked; j++) printf("%d %d ", r.place(j), r.parity(j));
 printf("|"); r.each_open([](int place, int parity) { printf(" %d %d", place, parity); }); printf("\\n"); } }
""")
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, "-o", str(d / "ring"), str(d / "ring.cc")], check=True)

    def ask(places, asked):
        line = subprocess.run([str(d / "ring")], input="%d %d\n" % (places, asked), capture_output=True, text=True, check=True).stdout
        pairs = lambda x: list(zip(*[iter(map(int, x.split()))] * 2))  # noqa: E731
        return [pairs(x) for x in line.split("|")]

    return ask


@pytest.mark.parametrize("places", [1, 2, 3, 4])
@pytest.mark.parametrize("asked", [0, 1, 2, 3, 4, 5, 7, 8, 9, 13])
def test_every_copy_in_flight_is_waited_for(ring, places, asked):
    copies, waits = ring(places, asked)
    last = {}
    for j, (place, parity) in enumerate(copies):
        assert place == j % places and parity == sum(p == place for p, _ in copies[:j]) % 2  # a barrier's n-th phase has parity n % 2
        last[place] = j
    # a place is filled again when the copy before has landed, so only the last one of each can be on its way
    for n in range(len(last) + 1):
        for flying in itertools.combinations(last, n):
            phase = {p: sum(q == p for q, _ in copies) - (p in flying) for p in last}  # completed phases of each barrier
            blocked = {p for p, parity in waits if phase[p] % 2 == parity}             # still in the phase of that parity
            assert blocked == set(flying), (places, asked, flying, waits)


def test_kernels_take_their_parities_from_the_ring():
    """No wait of a kernel with such a ring counts phases of its own"""
    for name in ("linear_attention.cuh", "distill.cuh"):
        text = open(os.path.join(CSRC, name)).read()
        waits = re.findall(r"mbar_wait\(([^;]*)\);", text)
        assert waits and all("parity" in w for w in waits), (name, waits)
