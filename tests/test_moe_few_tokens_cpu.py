"""What the expert layer for a few tokens refuses: no GPU needed."""
import ctypes

import pytest
import torch

import neuronspark_b200 as nsb
from neuronspark_b200 import _lib, build
from neuronspark_b200 import moe_kernels as mk


@pytest.fixture(scope="module", autouse=True)
def _built():
    build.build()


def args(N=3, E=4, D=8, F=16, dt=torch.float32):
    return [torch.zeros(N, D, dtype=dt), torch.zeros(E, D, dtype=dt), torch.zeros(E, 2 * F, D, dtype=dt),
            torch.zeros(E, D, F, dtype=dt)]


def test_shapes_and_types_are_checked():
    ok = args()
    bad = [(args(N=65), 2, {}), (ok, 0, {}), (ok, 5, {}), (args(E=20), 17, {}), (args(E=1025, D=1, F=1), 1, {}),
           (ok, 2, {"shared": torch.zeros(3, 4)}), (args(dt=torch.float64), 2, {}), (ok, 2, {"shared": torch.zeros(3, 8).half()})]
    for i in range(4):
        bad.append((ok[:i] + [ok[i][..., :-1]] + ok[i + 1:], 2, {}))
        bad.append((ok[:i] + [ok[i][0]] + ok[i + 1:], 2, {}))
    bad.append((ok[:2] + [torch.zeros(4, 8, 32).transpose(1, 2), ok[3]], 2, {}))
    bad.append((ok[:3] + [ok[3].clone().requires_grad_()], 2, {}))
    for a, k, more in bad:
        with pytest.raises(nsb.NSBError):
            mk.moe_few_tokens(*a, k, **more)
    with pytest.raises(nsb.NSBError, match="CUDA"):
        mk.moe_few_tokens(*ok, 2)


def test_abi_refusals():
    L, z, p = _lib.lib(), ctypes.c_void_p(0), ctypes.c_void_p(64)
    call = lambda N=2, E=4, K=2, D=8, F=8, dt=0, x=p, out=p, ids=p, scratch=p, wi=p: L.nsb_moe_few_tokens(  # noqa: E731
        x, 8, p, wi, p, z, out, ids, p, scratch, N, E, K, D, F, dt, z)
    odd = ctypes.c_void_p(66)
    for k in (dict(N=-1), dict(K=0), dict(K=5), dict(E=0), dict(D=-1), dict(F=-1), dict(dt=4), dict(x=z), dict(out=z),
              dict(ids=z), dict(scratch=z), dict(wi=z), dict(x=odd), dict(scratch=ctypes.c_void_p(72)), dict(ids=odd)):
        assert call(**k) == 1, k
    for k in (dict(N=65), dict(E=1025), dict(E=20, K=17), dict(D=(1 << 20) + 1), dict(F=(1 << 20) + 1)):
        assert call(**k) == 5, k
    assert call(N=0) == 0


def test_scratch():
    L = _lib.lib()
    size = lambda *a: L.nsb_moe_few_tokens_scratch_bytes(*a)  # noqa: E731
    assert size(65, 4, 2, 8, 8) == 0 and size(4, 4, 5, 8, 8) == 0
    for a in ((1, 1, 1, 1, 1), (64, 1024, 16, 4096, 2048), (3, 7, 2, 37, 19)):
        N, E, K, D, F = a
        assert size(*a) >= 4 * (N * E + N * K * (D + F + 1) + D / 16 + 3 * min(E, N * K) + 1)
