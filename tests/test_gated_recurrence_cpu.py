"""What the gated linear recurrence refuses, and the sizes of its buffers: no GPU needed."""
import ctypes

import pytest
import torch

import neuronspark_b200 as nsb
from neuronspark_b200 import _lib, build
from neuronspark_b200 import gated_recurrence as gr


@pytest.fixture(scope="module", autouse=True)
def _built():
    build.build()


def test_shapes_and_types_are_checked():
    x = torch.zeros(4, 2, 8)
    bad = [(x, x[:3], {}), (x[0, 0], x[0, 0], {}), (x, x, {"h0": torch.zeros(8)}), (x, x, {"bias": torch.zeros(2, 8)}),
           (x, x, {"cu_seqlens": torch.tensor([0, 4])}), (x[:, 0], x[:, 0], {"cu_seqlens": torch.tensor([0.0, 4.0])}),
           (x[:, 0], x[:, 0], {"cu_seqlens": torch.tensor([[0, 4]])}), (x[:, 0], x[:, 0], {"h0": torch.zeros(2, 8), "cu_seqlens": torch.tensor([0, 4])})]
    for raw, v, k in bad:
        with pytest.raises(nsb.NSBError):
            gr.gated_linear_recurrence(raw, v, **k)
    with pytest.raises(nsb.NSBError, match="CUDA"):
        gr.gated_linear_recurrence(x, x)
    h = torch.zeros(2, 8)
    for args in ((x[0], x[0], h[:1]), (x[0], x[0], h.bfloat16()), (x[0], x[0], torch.zeros(8, 2).T), (x, x, x),
                 (x[0].clone().requires_grad_(), x[0], h)):
        with pytest.raises(nsb.NSBError):
            gr.gated_linear_recurrence_step(*args)
    with torch.no_grad(), pytest.raises(nsb.NSBError, match="CUDA"):
        gr.gated_linear_recurrence_step(x[0], x[0], h)


def test_abi_refusals():
    L, z, p = _lib.lib(), ctypes.c_void_p(0), ctypes.c_void_p(64)
    fwd = lambda T=4, B=2, D=8, dt=0, raw=p, cu=z, seqs=0, y=p, hl=p, h0=z: L.nsb_gated_recurrence_fwd(  # noqa: E731
        raw, 16, 8, p, 16, 8, z, h0, cu, seqs, y, hl, z, z, T, B, D, dt, z)
    for k in (dict(T=-1), dict(D=-1), dict(dt=5), dict(raw=z), dict(y=z), dict(hl=z), dict(seqs=1), dict(cu=p, seqs=2),
              dict(raw=ctypes.c_void_p(65)), dict(h0=ctypes.c_void_p(66)), dict(cu=ctypes.c_void_p(66), B=1, seqs=1)):
        assert fwd(**k) == 1, k
    assert fwd(T=1 << 31) == 5
    assert fwd(B=0) == 0 and fwd(D=0) == 0
    bwd = lambda T=4, dy=p, db=z, part=z, ckpt=z, dt=0: L.nsb_gated_recurrence_bwd(  # noqa: E731
        p, 16, 8, p, 16, 8, z, z, z, 0, ckpt, dy, z, p, p, db, z, part, z, T, 2, 8, dt, z)
    for k in (dict(T=-1), dict(dy=z), dict(db=p), dict(T=4000), dict(dt=3)):
        assert bwd(**k) == 1, k
    step = lambda B=2, D=8, h=p, dt=0: L.nsb_gated_recurrence_step(p, 8, p, 8, z, h, p, B, D, dt, z)  # noqa: E731
    assert step(B=-1) == 1 and step(h=z) == 1 and step(dt=9) == 1 and step(B=0) == 0


def test_buffer_sizes():
    L = _lib.lib()
    assert L.nsb_gated_chunks(0) == 0 and L.nsb_gated_scratch_words(0, 5) == 0
    chunks = [L.nsb_gated_chunks(T) for T in range(1, 3000)]
    assert chunks[0] == 1 and all(b - a in (0, 1) for a, b in zip(chunks, chunks[1:]))
    for T in (1, 8, 64, 65, 1000, 65536):
        n, words = L.nsb_gated_chunks(T), L.nsb_gated_scratch_words(T, 100)
        assert (words == 0) == (n == 1)
        # all chunks' maps and one state in 32, or all chunks' states, behind the ticket
        assert n == 1 or words >= 4 + max(2 * n * 100 + n // 32 * 100, n * 100)
