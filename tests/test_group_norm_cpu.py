"""What group norm refuses: no GPU needed."""
import ctypes

import pytest
import torch

import neuronspark_b200 as nsb
from neuronspark_b200 import _lib, build
from neuronspark_b200 import group_norm as gn


@pytest.fixture(scope="module", autouse=True)
def _built():
    build.build()


def test_shapes_and_types_are_checked():
    x = torch.zeros(3, 8)
    bad = [(x[0], 2, {}), (x, 0, {}), (x, 3, {}), (x, 16, {}), (x, 2, {"weight": torch.ones(4)}), (x, 2, {"bias": torch.ones(1, 8)}),
           (x, 2, {"activation": "gelu"}), (x.double(), 2, {}), (x.int(), 2, {})]
    for t, G, k in bad:
        with pytest.raises(nsb.NSBError):
            gn.group_norm_act(t, G, **k)
    with pytest.raises(nsb.NSBError, match="CUDA"):
        gn.group_norm_act(x, 2)
    with pytest.raises(nsb.NSBError, match="CUDA"):
        gn.GroupNorm(2, 8)(x)


def test_abi_refusals():
    L, z, p, odd = _lib.lib(), ctypes.c_void_p(0), ctypes.c_void_p(64), ctypes.c_void_p(66)
    fwd = lambda N=2, l=5, C=8, G=2, act=1, dt=0, x=p, y=p, w=z, mean=z, sc=p: L.nsb_group_norm_fwd(  # noqa: E731
        x, w, z, y, mean, z, sc, N, l, C, G, 1e-5, act, dt, z)
    for k in (dict(N=-1), dict(l=-1), dict(C=-8), dict(G=0), dict(G=3), dict(act=2), dict(dt=3), dict(x=z), dict(y=z), dict(w=odd),
              dict(x=odd), dict(mean=p), dict(sc=z), dict(sc=odd)):
        assert fwd(**k) == 1, k
    assert fwd(C=(1 << 24) + 2) == 5 and fwd(N=0) == 0 and fwd(C=0) == 0
    bwd = lambda dy=p, mean=p, sc=p, dw=p, G=2: L.nsb_group_norm_bwd(  # noqa: E731
        dy, p, z, z, mean, p, p, dw, z, sc, 2, 5, 8, G, 1, 0, z)
    for k in (dict(dy=z), dict(mean=z), dict(sc=z), dict(dw=odd), dict(G=3)):
        assert bwd(**k) == 1, k


def test_scratch():
    size = _lib.lib().nsb_group_norm_scratch_floats
    assert size(0, 1, 8, 2, 0) == 0 and size(4, 1, 8, 2, 0) == 0 and size(4, 1, 8, 3, 1) == 0
    assert size(4, 1, 8, 2, 1) >= 2 * 8
    assert size(4, 100, 8, 2, 0) >= 3 * 4 * 2 and size(4, 100, 8, 2, 1) >= 2 * 4 * 8 + 2 * 4 * 2
