"""CPU tests of the per-pixel heads at the ends of their ranges: sizes that only the host side meets
(the scratch queries of the C ABI, which plan a whole call), and calls that are refused."""
import subprocess
import sys

import pytest
import torch

# The queries in a process of their own: a division by zero there would end this one.
QUERIES = """
import ctypes, sys
sys.path.insert(0, "tests")
import heads_abi as ha
lib = ha.load()
m = lambda r, c: ctypes.byref(ha.Matrix(256, r, c, c, 1))
for dt, M, K, V in eval(sys.argv[1]):
    for dx in (None, m(M, K)):
        print(dt, M, K, V, lib.vi_linear_ce_backward_scratch_bytes(dt, m(M, K), m(V, K), None, dx, m(V, K), None), flush=True)
"""


def test_many_rows_of_many_features():
    # so many rows that a piece of the vocabulary is 256 columns, and more columns of dweight's
    # tiles than run at a time: a piece stays at least one tile wide
    cases = [(dt, M, K, V) for dt in (0, 1, 2)
             for M, K, V in ((655361, 18944, 300), (655361, 18945, 256), (655361, 19200, 300), (700000, 20000, 1000),
                             (2 ** 30, 2 ** 30, 2 ** 30))]
    r = subprocess.run([sys.executable, "-c", QUERIES, repr(cases)], capture_output=True, text=True)
    lines = [[int(v) for v in line.split()] for line in r.stdout.splitlines()]
    assert r.returncode == 0, (r.returncode, lines[-1:], r.stderr)
    assert len(lines) == 2 * len(cases)
    for dt, M, K, V, got in lines:  # the masked copy of x, and one piece of G
        assert got >= (M * K + M * min(V, 256)) * 2 * (3 if dt == 0 else 1)


def test_tangents_are_refused():
    # before anything else is looked at, so that no device is needed to see it
    import torch.autograd.forward_ad as fwad
    from volume_integration import _C
    x, w, b, r = torch.randn(6, 4), torch.randn(5, 4), torch.randn(5), torch.randn(6, 5)
    t = torch.zeros(6, dtype=torch.int64)
    with fwad.dual_level():
        for i in range(4):
            v = [x, w, b, r]
            v[i] = fwad.make_dual(v[i], torch.ones_like(v[i]))
            with pytest.raises(RuntimeError, match="linear_act: forward-mode"):
                _C.linear_act(v[0], v[1], v[2], v[3], 0)
            if i < 3:
                with pytest.raises(RuntimeError, match="linear_cross_entropy: forward-mode"):
                    _C.linear_cross_entropy(v[0], v[1], v[2], t, -100, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        _C.linear_act(x, w, None, None, 0)
