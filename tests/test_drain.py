"""How two thread blocks that gave up settle what their copies still owe the barriers (csrc/drain.h), on a model of such a barrier."""
import ctypes
import itertools
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

STAGES, BYTES = 3, 65536


class Owed(ctypes.Structure):
    _fields_ = [("expect", ctypes.c_uint), ("complete", ctypes.c_uint), ("arrivals", ctypes.c_int)]


@pytest.fixture(scope="module")
def owed(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler here")
    folder = tmp_path_factory.mktemp("drain")
    src, lib = str(folder / "drain.cpp"), str(folder / "drain.so")
    with open(src, "w") as fh:
        fh.write('#include "drain.h"\nextern "C" pe::Owed owed(int i, int mine, int theirs, int fed, unsigned bytes) {\n'
                 "  return pe::owed_to_stage(i, mine, theirs, fed, bytes);\n}\n")
    subprocess.run([cxx, "-shared", "-fPIC", "-I", os.path.join(ROOT, "pytorch-engine_b200", "csrc"), src, "-o", lib], check=True)
    fn = ctypes.CDLL(lib).owed
    fn.restype = Owed
    return fn


class Barrier:
    """Two arrivals a phase, and a balance of bytes announced and arrived; a phase is complete when both are used up."""

    def __init__(self):
        self.phase, self.pending, self.bytes = 0, 2, 0

    def _settle(self):
        assert self.pending >= 0
        if self.pending == 0 and self.bytes == 0:
            self.phase, self.pending = self.phase + 1, 2

    def expect(self, n):
        self.bytes += n
        self._settle()

    def complete(self, n):
        self.bytes -= n
        self._settle()

    def arrive(self, expect=0):
        self.bytes += expect
        self.pending -= 1
        self._settle()


@pytest.mark.parametrize("done", [0, 1, 2, 3, 7])
def test_every_way_to_stop(owed, done):
    """``done`` stages were used; each block may have started up to three more, scales may have been handed over for as many; copies
    land before or after the blocks settle.  Each stage's phase is complete exactly when the copies that were started have landed."""
    ahead = range(STAGES + 1)
    for mine, theirs, fed in itertools.product(ahead, ahead, ahead):
        mine, theirs, fed = done + mine, done + theirs, done + fed
        for late in itertools.product((False, True), repeat=2):
            bars = [Barrier() for _ in range(STAGES)]
            for i in range(done):
                bars[i % STAGES].arrive(2 * BYTES)
                bars[i % STAGES].arrive()
                bars[i % STAGES].complete(2 * BYTES)
            for i in range(done, done + STAGES):
                bar = bars[i % STAGES]
                if i < theirs and not late[1]:
                    bar.complete(BYTES)          # the other block's copies may land before the bytes are announced
                if i < mine:
                    bar.arrive(2 * BYTES)
                if i < mine and not late[0]:
                    bar.complete(BYTES)
                if i < fed:
                    bar.arrive()
            last = max(mine, theirs)
            for i in range(max(0, last - STAGES), last):
                bar, o = bars[i % STAGES], owed(i, mine, theirs, fed, BYTES)
                if o.expect:
                    bar.expect(o.expect)
                if o.complete:
                    bar.complete(o.complete)
                for _ in range(o.arrivals):
                    bar.arrive()
                on_their_way = (late[0] and done <= i < mine) + (late[1] and done <= i < theirs)
                assert (bar.phase > i // STAGES) == (on_their_way == 0), (i, mine, theirs, fed, late)
                for _ in range(on_their_way):
                    bar.complete(BYTES)
                assert bar.phase == i // STAGES + 1
