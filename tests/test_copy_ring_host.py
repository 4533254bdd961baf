"""The ring that attention over a 4-bit cache copies through: where a copy lies, and that one which did not arrive in time leaves no
copy behind.  Barriers are modelled by the phases that they have completed."""
import ctypes
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm_singularity_b200", "csrc")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("ring")
    text = '#include "copy_ring.h"\n' + "".join(
        f'extern "C" int stage{s}(unsigned u, int k) {{ return CopyRing<{s}>{{u}}.stage(k); }}\n'
        f'extern "C" int parity{s}(unsigned u, int k) {{ return (int)CopyRing<{s}>{{u}}.parity(k); }}\n'
        f'extern "C" int issued{s}(int k, int n) {{ return CopyRing<{s}>::issued(k, n); }}\n' for s in (2, 4))
    (d / "ring.cpp").write_text(text)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", str(d / "ring.so"), str(d / "ring.cpp")], check=True)
    return ctypes.CDLL(str(d / "ring.so"))


class Stage:
    def __init__(self):
        self.phase, self.busy = 0, None

    def waits(self, parity):
        """Whether a wait for the phase of this parity has to wait now (a barrier's wait returns at once if that phase is over)."""
        return self.phase % 2 == parity


@pytest.mark.parametrize("stages", [2, 4])
@pytest.mark.parametrize("used", [0, 1, 3, 6, 2 ** 32 - 8])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 9, 100])
def test_every_copy_under_way_is_waited_for(lib, stages, used, n):
    stage, parity, issued = (getattr(lib, f"{name}{stages}") for name in ("stage", "parity", "issued"))
    for broken in range(n + 1):                                 # the piece that does not come (n: all do)
        ring = [Stage() for _ in range(stages)]
        for i in range(used if used < 100 else used % (2 * stages)):          # (the phases that the walks before have left)
            ring[i % stages].phase += 1

        def issue(k):
            if k < n:
                s = ring[stage(used, k)]
                assert s.busy is None, "a copy lands where another is read or under way"
                s.busy = k

        for k in range(stages - 1):
            issue(k)
        for k in range(n):
            issue(k + stages - 1)
            s = ring[stage(used, k)]
            assert s.busy == k and s.waits(parity(used, k))
            if k == broken:
                break
            s.phase, s.busy = s.phase + 1, None
        if broken < n:
            left = {k for k in (s.busy for s in ring) if k is not None}
            assert left == set(range(broken, issued(broken, n)))
            for k in left:
                s = ring[stage(used, k)]
                assert s.busy == k and s.waits(parity(used, k)), "the wait would return while the copy is under way"
        else:
            assert all(s.busy is None for s in ring)
