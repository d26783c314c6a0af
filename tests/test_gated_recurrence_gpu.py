"""The gated linear recurrence against a step-by-step evaluation in 64 bits, values and gradients.

Tolerances are running error bounds, evaluated beside the reference. Every rounded operation of the kernel is
off by at most u = 2^-24 relative. A gate takes an addition, an exponential (2 units in the last place, and
its argument's rounding, which counts |a| times), an addition, a division (2 units) and a product: at most
(8 + |a|) u relative, in f and in 1 - f. A step adds two roundings, and every composition of steps, of warps
and of chunks two more on quantities that the scan of absolute values bounds; a term passes at most
8 + 8 + 32 + 8 compositions beside its own steps. So with A_t = f A_{t-1} + (1-f)|x| the error of a state obeys
e_t <= f e_{t-1} + (c + |a|) u A_t, c = 16, plus 128 u A_t for the compositions. Stored outputs add half a
step of their type."""
import pytest
import torch

import neuronspark_b200 as nsb
from neuronspark_b200 import _lib
from neuronspark_b200 import gated_recurrence as gr

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _no_timeouts():
    yield
    assert nsb.device_error_word() == 0


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def reference(raw, x, h0, bias, cu=None, dy=None, dh=None):
    """Values and error bounds, one step after the other, all in 64 bits. Rows of ``raw``: [T, ...]."""
    a = raw.double() + (0 if bias is None else bias.double())
    x = x.double()
    T = x.shape[0]
    f, m = torch.sigmoid(a), torch.sigmoid(-a)
    state = (len(cu) - 1,) + x.shape[1:] if cu is not None else x.shape[1:]
    h0 = torch.zeros(state, dtype=torch.float64, device=x.device) if h0 is None else h0.double()
    c = (16 + a.abs().clamp(max=100).nan_to_num(0)) * U
    seqs = [(s, cu[s], cu[s + 1]) for s in range(len(cu) - 1)] if cu is not None else [(Ellipsis, 0, T)]
    y, prev, A, err, perr = (torch.zeros_like(x) for _ in range(5))
    h_last, e_last = h0.clone(), torch.zeros_like(h0)
    for s, b, e in seqs:
        h, ab, er = h0[s], h0[s].abs(), torch.zeros_like(h0[s])
        for t in range(b, e):
            prev[t], perr[t] = h, er + 128 * U * ab
            h = f[t] * h + m[t] * x[t]
            ab = f[t] * ab + m[t] * x[t].abs()
            er = f[t] * er + c[t] * ab
            y[t], A[t], err[t] = h, ab, er + 128 * U * ab
        h_last[s] = h
        e_last[s] = er + 128 * U * ab
    out = {"y": (y, err), "h_last": (h_last, e_last)}
    if dy is None:
        return out
    dy = dy.double()
    dh = torch.zeros_like(h0) if dh is None else dh.double()
    G, AG, eG = (torch.zeros_like(x) for _ in range(3))
    d_h0, e_h0 = dh.clone(), torch.zeros_like(dh)
    for s, b, e in seqs:
        K, aK, eK = dh[s], dh[s].abs(), torch.zeros_like(dh[s])
        for t in range(e - 1, b - 1, -1):
            G[t], AG[t], eG[t] = dy[t] + K, dy[t].abs() + aK, eK + (128 + 1) * U * (dy[t].abs() + aK)
            K, aK = f[t] * G[t], f[t] * AG[t]
            eK = f[t] * eK + c[t] * aK
        d_h0[s], e_h0[s] = K, eK + 129 * U * aK
    d = prev - x
    d_raw = G * d * f * m
    e_raw = (eG * d.abs() + AG * (perr + 2 * U * d.abs()) + 4 * c * AG * d.abs()) * f * m
    lead = tuple(range(x.dim() - 1))
    n = d_raw.numel() / x.shape[-1]
    out.update(d_raw=(d_raw, e_raw), d_x=(m * G, m * (eG + 2 * c * AG)), d_h0=(d_h0, e_h0),
               # 64 rows are added one after the other before the sum goes on in 64 bits
               d_bias=(d_raw.sum(lead), e_raw.sum(lead) + min(n, 72) * U * d_raw.abs().sum(lead)))
    return out


def check(got, want, what):
    value, err = want
    got = got.double()
    assert got.shape == value.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN in other places"
    return got, value, err


def close(got, want, dtype, what):
    g, value, err = check(got, want, what)
    tiny = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126}[dtype]
    bound = err * (1 + half_step(dtype)) + half_step(dtype) * value.abs() + tiny
    bad = (g - value).abs() > bound
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off; worst "
                           f"{float(((g - value).abs() / bound)[bad].max()):.2f} times the bound")


def make(shape, dtype, seed, seqs=None, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    D = shape[-1]
    state = (seqs, D) if seqs is not None else shape[1:]
    return dict(raw=(spread * rn(*shape) + 1).to(dtype), x=rn(*shape).to(dtype), h0=rn(*state), bias=rn(D),
                dy=rn(*shape).to(dtype), dh=rn(*state))


def run(v, cu=None, use_h0=True, use_bias=True, use_dh=True):
    leaves = {n: v[n].clone().requires_grad_() for n in ("raw", "x", "h0", "bias")}
    y, h_last = gr.gated_linear_recurrence(leaves["raw"], leaves["x"], leaves["h0"] if use_h0 else None,
                                           leaves["bias"] if use_bias else None, cu_seqlens=cu)
    names = ["raw", "x"] + ["h0"] * use_h0 + ["bias"] * use_bias
    outs, grads = ((y, h_last), (v["dy"], v["dh"])) if use_dh else ((y,), (v["dy"],))
    d = torch.autograd.grad(outs, [leaves[n] for n in names], grads, allow_unused=True)
    return {"y": y.detach(), "h_last": h_last.detach(), **{"d_" + n: t for n, t in zip(names, d)}}


def compare(got, want, dtype):
    for n, t in got.items():
        assert t.dtype == (dtype if n in ("y", "d_raw", "d_x") else torch.float32), n
        close(t, want[n], t.dtype, n)


SHAPES = [(1, 1, 1), (1, 5, 33), (2, 3, 64), (7, 2, 31), (8, 1, 128), (9, 4, 66), (16, 1, 1), (33, 2, 99), (64, 3, 40),
          (65, 1, 65), (129, 2, 130), (500, 1, 3), (2051, 1, 37), (640, 40, 770)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_time_major(shape, dtype):
    v = make(shape, dtype, 1000 + shape[0])
    compare(run(v), reference(v["raw"], v["x"], v["h0"], v["bias"], None, v["dy"], v["dh"]), dtype)


@pytest.mark.parametrize("h0,bias,dh", [(False, True, True), (True, False, True), (False, False, False)])
def test_optional_arguments(h0, bias, dh):
    v = make((150, 2, 34), torch.bfloat16, 3)
    want = reference(v["raw"], v["x"], v["h0"] if h0 else None, v["bias"] if bias else None, None, v["dy"],
                     v["dh"] if dh else None)
    compare(run(v, None, h0, bias, dh), want, torch.bfloat16)


CUTS = [[0, 0], [0, 1], [0, 200], [0, 0, 0, 7, 7, 8, 200], [0, 64, 128, 192, 200], [3, 63, 65, 66, 66, 150],
        [0, 8, 16, 17, 24, 24, 100, 199], list(range(201)), [0, 90, 200, 200, 200], [0]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cu", CUTS, ids=lambda c: f"{len(c)}-{c[-1]}")
def test_packed(cu, dtype):
    for D in (1, 33, 128):
        v = make((200, D), dtype, 7 + len(cu), seqs=len(cu) - 1)
        got = run(v, torch.tensor(cu, device=DEV))
        compare(got, reference(v["raw"], v["x"], v["h0"], v["bias"], cu, v["dy"], v["dh"]), dtype)
        outside = torch.ones(200, dtype=torch.bool, device=DEV)
        outside[cu[0]:cu[-1]] = False
        for n in ("y", "d_raw", "d_x"):
            assert (got[n][outside] == 0).all()


def test_packed_long_and_int32():
    cu = [0, 1000, 1001, 1001, 5000, 9000]
    v = make((9100, 48), torch.bfloat16, 11, seqs=5)
    got = run(v, torch.tensor(cu, device=DEV, dtype=torch.int32))
    compare(got, reference(v["raw"], v["x"], v["h0"], v["bias"], cu, v["dy"], v["dh"]), torch.bfloat16)


# 42 to 77 MB of inputs: the forward goes over them twice, in three launches (by 4, 2 and 1 columns of 16 bits, 2 and 1 of 32)
@pytest.mark.parametrize("packed,dtype,T,D", [(True, torch.bfloat16, 14001, 800), (True, torch.float16, 11003, 998),
                                              (True, torch.float16, 11003, 1001), (True, torch.float32, 8100, 650),
                                              (False, torch.bfloat16, 24000, 800), (False, torch.float16, 20011, 1001),
                                              (False, torch.float32, 13000, 651)])
def test_long_forwards(packed, dtype, T, D):
    cu = [0, 1, 3000, 3000, 7001, T - 70, T - 70, T - 10] if packed else None  # (empty ones, and rows behind the last)
    v = make((T, D), dtype, 59, seqs=len(cu) - 1 if packed else None)
    if packed:
        v["x"][5000, 1] = v["raw"][5000, 2] = float("nan")  # one sequence's own
    cut = torch.tensor(cu, device=DEV) if packed else None
    with torch.no_grad():
        y, h_last = gr.gated_linear_recurrence(v["raw"], v["x"], v["h0"], v["bias"], cu_seqlens=cut)
        again = gr.gated_linear_recurrence(v["raw"], v["x"], v["h0"], v["bias"], cu_seqlens=cut)
        bare, _ = gr.gated_linear_recurrence(v["raw"], v["x"], cu_seqlens=cut)
    want = reference(v["raw"], v["x"], v["h0"], v["bias"], cu)
    close(y, want["y"], dtype, "y")
    close(h_last, want["h_last"], torch.float32, "h_last")
    assert torch.equal(y.nan_to_num(7.0), again[0].nan_to_num(7.0)) and torch.equal(h_last.nan_to_num(7.0), again[1].nan_to_num(7.0))
    close(bare, reference(v["raw"], v["x"], None, None, cu)["y"], dtype, "y without a state or bias")


def test_gradients_of_a_long_forward():
    """The backward starts its chunks from the states that the forward's second launch found; batch-major inputs."""
    T, B, D = 24000, 2, 400
    v = make((T, B, D), torch.bfloat16, 61)
    v = {n: t.transpose(0, 1).contiguous().transpose(0, 1) if n in ("raw", "x", "dy") else t for n, t in v.items()}
    compare(run(v), reference(v["raw"], v["x"], v["h0"], v["bias"], None, v["dy"], v["dh"]), torch.bfloat16)


def test_packed_rows_are_the_sequences_alone():
    """Bit for bit where the chunks lie alike; the state of a sequence never reaches its neighbour."""
    v = make((128, 64), torch.float32, 13, seqs=2)
    v["x"][:64] = float("nan")
    y, h_last = gr.gated_linear_recurrence(v["raw"], v["x"], v["h0"], v["bias"], torch.tensor([0, 64, 128], device=DEV))
    alone, last = gr.gated_linear_recurrence(v["raw"][64:], v["x"][64:], v["h0"][1], v["bias"])
    assert torch.isnan(y[:64]).all() and torch.isnan(h_last[0]).all()
    close(y[64:], reference(v["raw"][64:], v["x"][64:], v["h0"][1], v["bias"])["y"], torch.float32, "y")
    assert torch.equal(h_last[1], last) and torch.equal(y[64:], alone)


def test_cu_seqlens_out_of_order_touch_nothing_else():
    """Values that are not allowed: the results mean nothing, but only the tensors given are touched."""
    v = make((100, 32), torch.float32, 17, seqs=4)
    for cu in ([0, 90, 10, 400, 100], [-5, 20, 2000000000, 50, 60], [50, 40, 30, 20, 10]):
        y, h_last = gr.gated_linear_recurrence(v["raw"], v["x"], v["h0"], v["bias"], torch.tensor(cu, device=DEV))
        torch.cuda.synchronize()
        assert y.shape == (100, 32) and h_last.shape == (4, 32)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_of_one_projection(dtype):
    T, B, D = 140, 3, 66
    g = torch.Generator(device=DEV).manual_seed(5)
    both = torch.randn(T, B, 2 * D + 1, generator=g, device=DEV).to(dtype)
    for at in (0, 1):  # the second starts on an odd element
        raw, x = both[..., at:at + D], both[..., at + D:at + 2 * D]
        y, h = gr.gated_linear_recurrence(raw, x)
        y2, h2 = gr.gated_linear_recurrence(raw.contiguous(), x.contiguous())
        assert torch.equal(y, y2) and torch.equal(h, h2)
        leaf = both.clone().requires_grad_()
        (gr.gated_linear_recurrence(leaf[..., at:at + D], leaf[..., at + D:at + 2 * D])[0].float()).sum().backward()
        want = reference(raw, x, None, None, None, torch.ones_like(raw))
        close(leaf.grad[..., at:at + D], want["d_raw"], dtype, "d_raw")
        close(leaf.grad[..., at + D:at + 2 * D], want["d_x"], dtype, "d_x")
    t = torch.randn(D, B, T, generator=g, device=DEV).to(dtype).permute(2, 1, 0)  # no unit stride anywhere useful
    assert torch.equal(gr.gated_linear_recurrence(t, t)[0], gr.gated_linear_recurrence(t.contiguous(), t.contiguous())[0])


def test_mixed_types_and_broadcast_state():
    v = make((70, 2, 40), torch.bfloat16, 19)
    raw = v["raw"].float().requires_grad_()
    h0 = torch.randn(40, device=DEV).half().requires_grad_()
    y, h = gr.gated_linear_recurrence(raw, v["x"], h0.expand(2, 40), v["bias"].bfloat16())
    want = reference(raw.detach(), v["x"], h0.detach().expand(2, 40), v["bias"].bfloat16(), None, v["dy"].float())
    close(y, want["y"], torch.bfloat16, "y")
    d = torch.autograd.grad(y, (raw, h0), v["dy"])
    assert d[0].dtype == torch.float32 and d[1].dtype == torch.float16
    close(d[0], want["d_raw"], torch.float32, "d_raw")
    value, err = want["d_h0"]  # two rows' gradients, each rounded to half precision, then added
    total = value.sum(0)
    assert ((d[1].double() - total).abs() <= err.sum(0) + 3 * 2.0 ** -11 * value.abs().sum(0) + 2.0 ** -24).all()


@pytest.mark.parametrize("T", [40, 400])
def test_extreme_gates(T):
    """Gates of +-inf keep and replace the state; a NaN stays in its own column."""
    v = make((T, 1, 32), torch.float32, 23)
    raw = v["raw"].clone()
    raw[T // 4:T // 2] = float("inf")
    raw[T // 2 + 3, :, 8:16] = float("-inf")
    raw[:, :, 5] = 300.0
    raw[:, :, 6] = -300.0
    y, h = gr.gated_linear_recurrence(raw, v["x"], v["h0"])
    close(y, reference(raw, v["x"], v["h0"], None)["y"], torch.float32, "y")
    assert torch.equal(y[T // 2 + 3, :, 8:16], v["x"][T // 2 + 3, :, 8:16])
    assert torch.equal(y[:, 0, 5], v["h0"][0, 5].expand(T)) and torch.equal(y[:T // 4, 0, 6], v["x"][:T // 4, 0, 6])
    raw[T // 2, 0, 9] = float("nan")
    y2, h2 = gr.gated_linear_recurrence(raw, v["x"], v["h0"])
    assert torch.isnan(y2[T // 2:, 0, 9]).all() and torch.isnan(h2[0, 9]) and not torch.isnan(y2[:T // 2]).any()
    keep = torch.arange(32, device=DEV) != 9
    assert torch.equal(y2[..., keep], y[..., keep])


def test_gradients_against_differences():
    v = make((90, 1, 16), torch.float32, 29)
    got = run(v)
    loss = lambda **k: sum((o.double() * w.double()).sum() for o, w in zip(  # noqa: E731
        (lambda r: (r["y"][0], r["h_last"][0]))(reference(k["raw"], k["x"], k["h0"], k["bias"])), (v["dy"], v["dh"])))
    base = {n: v[n].double() for n in ("raw", "x", "h0", "bias")}
    g = torch.Generator(device=DEV).manual_seed(31)
    for n in base:
        step = torch.randn(base[n].shape, generator=g, device=DEV, dtype=torch.float64)
        # a central difference of a smooth function: off by step^2 times its third derivative, and by rounding
        diff = (loss(**{**base, n: base[n] + 1e-5 * step}) - loss(**{**base, n: base[n] - 1e-5 * step})) / 2e-5
        dot = (got["d_" + n].double() * step).sum()
        assert abs(float(dot - diff)) <= 1e-6 * float((got["d_" + n].double() * step).abs().sum()), n


def test_runs_are_identical():
    """Many chunks race for their turns; the results do not depend on who wins."""
    for shape in ((6000, 1, 70), (700, 16, 4000)):
        v = make(shape, torch.bfloat16, 37)
        first = run(v)
        for _ in range(5):
            for n, t in run(v).items():
                assert torch.equal(t, first[n]), n


def test_streams_and_graphs():
    v = make((300, 2, 130), torch.bfloat16, 41)
    want = run(v)
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    other = make((5000, 1, 64), torch.bfloat16, 43)
    want_other = run(other)
    torch.cuda.synchronize()
    for _ in range(3):  # two chains in flight at once
        with torch.cuda.stream(side):
            a = run(other)
        b = run(v)
        torch.cuda.synchronize()
        assert all(torch.equal(a[n], want_other[n]) for n in a) and all(torch.equal(b[n], want[n]) for n in b)
    leaves = {n: v[n].clone().requires_grad_() for n in ("raw", "x", "h0", "bias")}
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y, h = gr.gated_linear_recurrence(leaves["raw"], leaves["x"], leaves["h0"], leaves["bias"])
            d = torch.autograd.grad((y, h), list(leaves.values()), (v["dy"], v["dh"]))
    for k in range(2):
        with torch.no_grad():
            for n in leaves:
                leaves[n].copy_(v[n] if k == 0 else v[n].flip(0))
        graph.replay()
        torch.cuda.synchronize()
        w = want if k == 0 else run({**v, **{n: v[n].flip(0) for n in leaves}})
        assert torch.equal(y.detach(), w["y"]) and torch.equal(h.detach(), w["h_last"])
        assert all(torch.equal(t, w["d_" + n]) for n, t in zip(leaves, d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 67), (64, 768), (5, 130)])
def test_step_follows_the_scan(shape, dtype):
    B, D = shape
    v = make((6, B, D), dtype, 47)
    y, h_last = gr.gated_linear_recurrence(v["raw"], v["x"], v["h0"], v["bias"])
    h = v["h0"].clone()
    want = reference(v["raw"], v["x"], v["h0"], v["bias"])
    for t in range(6):
        out = gr.gated_linear_recurrence_step(v["raw"][t], v["x"][t], h, v["bias"])
        assert out.dtype == dtype and torch.equal(out, h.to(dtype))
        assert torch.equal(out, y[t])  # the same operations in the same order within one warp
    assert torch.equal(h, h_last)
    close(h, want["h_last"], torch.float32, "h")
    both = torch.randn(B, 2 * D + 1, device=DEV).to(dtype)
    h1, h2 = v["h0"].clone(), v["h0"].clone()
    a = gr.gated_linear_recurrence_step(both[:, 1:D + 1], both[:, D + 1:], h1)
    b = gr.gated_linear_recurrence_step(both[:, 1:D + 1].contiguous(), both[:, D + 1:].contiguous(), h2)
    assert torch.equal(a, b) and torch.equal(h1, h2)


def test_empty():
    for shape in ((0, 2, 8), (5, 0, 8), (5, 2, 0)):
        raw, x = (torch.zeros(shape, device=DEV, requires_grad=True) for _ in range(2))
        h0 = torch.randn(shape[1:], device=DEV, requires_grad=True)
        bias = torch.zeros(shape[2], device=DEV, requires_grad=True)
        y, h = gr.gated_linear_recurrence(raw, x, h0, bias)
        assert y.shape == shape and h.shape == shape[1:]
        if shape[0] == 0:
            assert torch.equal(h, h0)
        d = torch.autograd.grad((y, h), (raw, x, h0, bias), (torch.ones_like(y), torch.ones_like(h)))
        assert (d[3] == 0).all() and (shape[0] or torch.equal(d[2], torch.ones_like(h0)))
    x = torch.zeros(0, 8, device=DEV)
    y, h = gr.gated_linear_recurrence(x, x, torch.ones(2, 8, device=DEV), None, torch.tensor([0, 0, 0], device=DEV))
    assert y.shape == (0, 8) and (h == 1).all()
    assert gr.gated_linear_recurrence_step(x, x, torch.zeros(0, 8, device=DEV)).shape == (0, 8)


def test_offsets_beyond_32_bits():
    """Two projections of 2.3 G elements each (views of one row repeated would not reach the far addresses)."""
    T, D = 36000, 65536
    raw = torch.zeros(T, 1, D, dtype=torch.bfloat16, device=DEV)
    x = torch.zeros(T, 1, D, dtype=torch.bfloat16, device=DEV)
    x[-1], raw[-1, :, ::2] = 1.0, 100.0
    y, h = gr.gated_linear_recurrence(raw, x)
    # an open gate of 100 lets in exp(-100) = 3.7e-44, below the least normal number 2^-126
    assert (y[:-1] == 0).all() and (h[0, ::2] < 2.0 ** -126).all() and (h[0, 1::2] == 0.5).all()
    assert torch.equal(y[-1], h.bfloat16())


def test_a_call_after_a_timeout_is_refused():
    _lib.lib()
    v = make((300, 1, 32), torch.float32, 53)
    nsb.set_wait_limit_ns(1_000_000)
    try:
        _lib.check(_lib.lib().nsb_selftest_wait_timeout(_lib.stream_ptr(DEV)), "selftest")
        torch.cuda.synchronize()
        with pytest.raises(nsb.NSBError):
            gr.gated_linear_recurrence(v["raw"], v["x"])
    finally:
        nsb.set_wait_limit_ns()
        assert nsb.device_error_word() != 0
    gr.gated_linear_recurrence(v["raw"], v["x"])


def test_second_derivatives_are_refused():
    x = torch.randn(4, 6, device=DEV, requires_grad=True)
    y = gr.gated_linear_recurrence(x, x)[0]
    with pytest.raises(nsb.NSBError, match="second derivatives"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    torch.autograd.grad(y.sum(), x)


# one chunk; several that pass maps; several whose columns fill the GPU, so that states pass one by one
@pytest.mark.parametrize("dtype,rows,D", [(torch.float32, 64, 8), (torch.bfloat16, 64, 64), (torch.float32, 1500, 40),
                                          (torch.bfloat16, 1500, 66), (torch.float32, 200, 14300)])
def test_a_nan_gate_does_not_reach_the_sequence_before(dtype, rows, D):
    """Gradients of a packed batch: a NaN gate some rows behind a border, and a run without it."""
    for border, behind in ((20, 2), (16, 5), (23, 1), (rows - 30, 3), (rows // 2 + 3, 4)):
        v = make((rows, D), dtype, 67 + border, seqs=3)
        cu = torch.tensor([0, border, rows - 9, rows], device=DEV)
        clean = run(v, cu)
        v["raw"][border + behind] = float("nan")
        got = run(v, cu)
        for n in ("y", "d_raw", "d_x"):
            assert torch.equal(got[n][:border], clean[n][:border]), (n, border)
            assert torch.equal(got[n][rows - 9:], clean[n][rows - 9:]), (n, border)
        for n in ("h_last", "d_h0"):
            assert torch.equal(got[n][::2], clean[n][::2]) and torch.isnan(got[n][1]).all(), (n, border)
        assert torch.isnan(got["d_x"][border:border + behind]).all()


def test_gates_that_nearly_cancel():
    """raw + bias is a small exact difference of two large numbers: the gate goes by it, not by their sizes."""
    T, B, D = 300, 2, 40
    v = make((T, B, D), torch.float32, 71)
    a = torch.randint(-2048, 2049, (T, B, D), device=DEV) * 2.0 ** -9
    # (biases that a power of two does not divide much further: log2(e) times them is not exact)
    v["bias"] = (12345.0 + torch.arange(D, device=DEV) * 7.125) * torch.where(torch.arange(D, device=DEV) % 2 == 0, 1.0, -1.0)
    v["raw"] = a - v["bias"]
    assert torch.equal(v["raw"].double() + v["bias"].double(), a.double())
    want = reference(v["raw"], v["x"], v["h0"], v["bias"], None, v["dy"], v["dh"])
    compare(run(v), want, torch.float32)
    h = v["h0"].clone()
    for t in range(6):
        y = gr.gated_linear_recurrence_step(v["raw"][t], v["x"][t], h, v["bias"])
        close(y, tuple(w[t] for w in want["y"]), torch.float32, "step")
    T = 24000  # long enough for three launches
    v = make((T, 1, 700), torch.float32, 73)
    v["bias"] = torch.full((700,), 12345.0, device=DEV)
    v["raw"] = torch.randint(-2048, 2049, (T, 1, 700), device=DEV) * 2.0 ** -9 - 12345.0
    with torch.no_grad():
        y, _ = gr.gated_linear_recurrence(v["raw"], v["x"], v["h0"], v["bias"])
    close(y, reference(v["raw"], v["x"], v["h0"], v["bias"])["y"], torch.float32, "y")


def test_a_step_counts_as_a_change_of_the_state():
    """A state that a graph has saved and that is stepped afterwards: the backward pass is refused, as after any change in place."""
    v = make((5, 3, 16), torch.float32, 79)
    h = v["h0"].clone().requires_grad_()
    raw = v["raw"].clone().requires_grad_()
    y, _ = gr.gated_linear_recurrence(raw, v["x"], h)
    before = h._version
    with torch.no_grad():
        gr.gated_linear_recurrence_step(v["raw"][0], v["x"][0], h)
    assert h._version > before
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y.sum(), raw)
    with torch.inference_mode():
        state = v["h0"].clone()  # has no version to count
        out = gr.gated_linear_recurrence_step(v["raw"][0], v["x"][0], state)
        assert torch.equal(out, state)


def test_nothing_is_kept_for_a_backward_that_cannot_come():
    """A bias that is a parameter, as a module has it, costs no saved states without gradients."""
    v = make((400, 2, 64), torch.bfloat16, 83)
    cu = torch.tensor([0, 150, 400], device=DEV)

    def allocations(bias):
        def count():
            return torch.cuda.memory_stats(DEV)["allocation.all.allocated"]
        before = count()
        gr.gated_linear_recurrence(v["raw"], v["x"], v["h0"], bias)
        gr.gated_linear_recurrence(v["raw"][:, 0].contiguous(), v["x"][:, 0].contiguous(), v["h0"], bias, cu)
        return count() - before
    parameter = torch.nn.Parameter(v["bias"].clone())
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            assert allocations(parameter) == allocations(v["bias"])
    assert allocations(parameter) > allocations(v["bias"])  # (with gradients there are some to keep)


EMPTY = {"middle": lambda n: [0, 5] + [5] * n + [9, 200], "end": lambda n: [0, 100, 200] + [200] * n, "start": lambda n: [0] * (n + 1) + [200],
         "twice": lambda n: [0, 3] + [3] * n + [11] * n + [14, 14, 70, 200], "before the last row": lambda n: [0, 199] + [199] * n + [200]}


@pytest.mark.parametrize("n", [29, 30, 31, 32, 33, 70])
@pytest.mark.parametrize("where", EMPTY)
def test_many_empty_sequences_in_a_row(where, n):
    """Rows of one warp that dozens of sequences end in."""
    cu = EMPTY[where](n)
    for dtype, D in ((torch.float32, 5), (torch.bfloat16, 64)):
        v = make((200, D), dtype, 89 + n, seqs=len(cu) - 1)
        compare(run(v, torch.tensor(cu, device=DEV)), reference(v["raw"], v["x"], v["h0"], v["bias"], cu, v["dy"], v["dh"]), dtype)


@pytest.mark.parametrize("seqs", [1025, 5000])
def test_thousands_of_sequences(seqs):
    """Most of them empty: the search goes over more than 1024."""
    g = torch.Generator().manual_seed(seqs)
    cu = [0] + sorted(torch.randint(0, 391, (seqs - 1,), generator=g).tolist()) + [390]
    v = make((400, 34), torch.bfloat16, 97, seqs=seqs)
    compare(run(v, torch.tensor(cu, device=DEV)), reference(v["raw"], v["x"], v["h0"], v["bias"], cu, v["dy"], v["dh"]), torch.bfloat16)


@pytest.mark.parametrize("seqs", [7, 2000])
def test_gradients_of_a_long_packed_forward(seqs):
    """45 MB of inputs, so that the forward takes three launches and the backward starts from the states of the second."""
    rows, D = 14001, 800
    g = torch.Generator().manual_seed(seqs)
    cu = [0] + sorted(torch.randint(0, rows - 20, (seqs - 1,), generator=g).tolist()) + [rows - 20]
    v = make((rows, D), torch.bfloat16, 101, seqs=seqs)
    compare(run(v, torch.tensor(cu, device=DEV)), reference(v["raw"], v["x"], v["h0"], v["bias"], cu, v["dy"], v["dh"]), torch.bfloat16)


@pytest.mark.parametrize("dtype,T,D", [(torch.float32, 20000, 48), (torch.bfloat16, 9000, 130), (torch.bfloat16, 300, 28500)])
def test_slow_gates(dtype, T, D):
    """Gates around 0.995: states and their gradients live for hundreds of steps, over many chunks."""
    v = make((T, 1, D), dtype, 103, spread=0.5)
    v["raw"] = (v["raw"].float() + 4.3).to(dtype)
    compare(run(v), reference(v["raw"], v["x"], v["h0"], v["bias"], None, v["dy"], v["dh"]), dtype)


def test_captured_steps():
    """One token's step in a graph: every replay goes on from the state that the last one left."""
    v = make((6, 20, 96), torch.bfloat16, 107)
    raw, x, h = v["raw"][0].clone(), v["x"][0].clone(), v["h0"].clone()
    gr.gated_linear_recurrence_step(raw, x, h.clone(), v["bias"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gr.gated_linear_recurrence_step(raw, x, h, v["bias"])
    h.copy_(v["h0"])
    eager = v["h0"].clone()
    for t in range(6):
        raw.copy_(v["raw"][t])
        x.copy_(v["x"][t])
        graph.replay()
        want = gr.gated_linear_recurrence_step(v["raw"][t], v["x"][t], eager, v["bias"])
        assert torch.equal(y, want) and torch.equal(h, eager)


def test_gates_are_as_good_as_rounded():
    """A state of one and an input of zero: y = f. An error of f counts 1 / (1 - f) times in a long run, so it has to be
    little more than that of a rounding, 2^-25 for f in 1/2 .. 1. The exponential is off by 2 units in the last place and its argument
    by 1.3 |a| 2^-24, together (4 + 1.3 |a|) 2^-24, of which f takes f (1 - f) parts; below 1/2 the residual 1 - f - e f has
    a rounding of 2^-25, and f one of its own, 2^-24 of it."""
    rows, D = 14001, 800
    g = torch.Generator(device=DEV).manual_seed(109)
    raw = 16 * torch.rand(rows, D, generator=g, device=DEV) - 6
    a = raw.double()
    f = torch.sigmoid(a)
    bound = torch.where(f >= 0.5, torch.full_like(f, 2.0 ** -25), 1.5 * U * f) + f * (1 - f) * (4 + 1.3 * a.abs()) * U
    ones, zeros = torch.ones(rows, D, device=DEV), torch.zeros(rows, D, device=DEV)
    own = torch.arange(rows + 1, device=DEV)  # a sequence for each row
    for what, y in (("step", gr.gated_linear_recurrence_step(raw, zeros, ones.clone())),
                    ("three launches", gr.gated_linear_recurrence(raw, zeros, ones, None, own)[0]),
                    ("one launch", gr.gated_linear_recurrence(raw[:3000], zeros[:3000], ones[:3000], None, own[:3001])[0]),
                    ("time-major", gr.gated_linear_recurrence(raw[None], zeros[None], ones)[0][0])):
        assert ((y.double() - f[:len(y)]).abs() <= bound[:len(y)]).all(), what
    h0 = ones.clone().requires_grad_()
    y, h = gr.gated_linear_recurrence(raw, zeros, h0, None, own)
    d = torch.autograd.grad(y, h0, ones)[0]
    assert ((d.double() - f).abs() <= bound).all(), "gradient"
