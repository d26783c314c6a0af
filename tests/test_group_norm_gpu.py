"""Group norm with an activation against the definition in 64 bits, values and gradients.

Bounds, with u = 2^-24: a mean or a sum is a chain of at most 64 additions per level of the reduction, three
levels, each within u of the sum of absolute values: 192 u. The mean is off by e_m = 192 u mean|x|; a sum of squares
about it by e_m^2 n and 192 u of itself, so rstd by half of (192 u + e_m^2 / (var + eps)) relative, and 4 u. The
exponential and the quotient of a sigmoid are off by 2 units each and its argument counts |z| times. silu's slope is
at most 1.1 and its second derivative 0.5. dw and db add up N L rows, at most N L / 64 + 256 in one chain. Everything else
is a rounding per operation, and half a step of the type at the end."""
import pytest
import torch

import neuronspark_b200 as nsb
from neuronspark_b200 import gated_recurrence as gr
from neuronspark_b200 import group_norm as gn
from neuronspark_b200 import moe_kernels as mk

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def reference(x, G, w, b, dy=None, eps=1e-5, act=True):
    N, C = x.shape[0], x.shape[-1]
    L = x.numel() // (N * C)
    four = lambda t: t.double().reshape(N, L, G, C // G)  # noqa: E731
    v = four(x)
    one = lambda t, d: (torch.full((C,), d, device=DEV, dtype=torch.float64) if t is None else t.double()).reshape(G, -1)  # noqa: E731
    W, B = one(w, 1.0), one(b, 0.0)
    mean_of = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    mu = mean_of(v)
    var = mean_of((v - mu) ** 2)
    rstd = (var + eps) ** -0.5
    xh = (v - mu) * rstd
    e_m = 192 * U * mean_of(v.abs())
    r = 0.5 * (192 * U + e_m ** 2 / (var + eps)) + 4 * U
    e_xh = rstd * (e_m + U * (v - mu).abs()) + xh.abs() * (r + 2 * U)
    z = W * xh + B
    e_z = W.abs() * e_xh + 2 * U * ((W * xh).abs() + B.abs())
    s = torch.sigmoid(z) if act else torch.ones_like(z)
    y = z * s
    out = {"y": (y.reshape(x.shape), (1.1 * e_z + (8 + z.abs()) * U * y.abs()).reshape(x.shape))}
    if dy is None:
        return out
    dy = four(dy)
    slope = s * (1 + z * (1 - s))
    d = dy * slope
    e_d = dy.abs() * ((0.5 * e_z + (16 + 2 * z.abs()) * U * (s + (z * s * (1 - s)).abs())) if act else U)
    g = d * W
    e_g = W.abs() * e_d + U * g.abs()
    m1, m2 = mean_of(g), mean_of(g * xh)
    e_1 = mean_of(e_g) + 200 * U * mean_of(g.abs())
    e_2 = mean_of(e_g * xh.abs() + g.abs() * e_xh) + 200 * U * mean_of((g * xh).abs())
    dx = rstd * (g - m1 - xh * m2)
    e_dx = rstd * (e_g + e_1 + xh.abs() * e_2 + m2.abs() * e_xh + 4 * U * (g.abs() + m1.abs() + (xh * m2).abs())) + dx.abs() * (r + 2 * U)
    chain = (N * L / 64 + 256) * U
    total = lambda t: t.sum((0, 1)).reshape(C)  # noqa: E731
    out.update(d_x=(dx.reshape(x.shape), e_dx.reshape(x.shape)), d_b=(total(d), total(e_d + chain * d.abs())),
               d_w=(total(d * xh), total(e_d * xh.abs() + d.abs() * e_xh + chain * (d * xh).abs())))
    return out


def close(got, want, what):
    value, err = want
    t = got.dtype
    assert got.shape == value.shape, what
    tiny = 2.0 ** -25 if t == torch.float16 else 2.0 ** -126
    bound = err * (1 + half_step(t)) + half_step(t) * value.abs() + tiny
    off = (got.double() - value).abs()
    assert (off <= bound).all(), f"{what}: {int((~(off <= bound)).sum())} of {off.numel()} off; worst {float((off / bound).max()):.2f}"


def make(shape, dtype, seed, mean=0.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    C = shape[-1]
    return (1.5 * rn(*shape) + mean).to(dtype), 1 + 0.3 * rn(C), 0.3 * rn(C), rn(*shape).to(dtype)


def run(x, G, w, b, dy, **k):
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = gn.group_norm_act(leaves[0], G, leaves[1], leaves[2], **k)
    return {"y": y.detach(), **dict(zip(("d_x", "d_w", "d_b"), torch.autograd.grad(y, leaves, dy)))}


ROWS = [((1, 1), 1), ((3, 64), 1), ((5, 768), 12), ((1300, 768), 12), ((7, 66), 2), ((9, 100), 1), ((33, 240), 10), ((700, 256), 1),
        ((4, 255), 1), ((3, 257), 1), ((5, 1024), 2), ((6, 2050), 1), ((10, 48), 48), ((2000, 8), 1), ((2, 6144), 48), ((1, 16384), 512)]
MAPS = [((2, 2, 8), 2), ((1, 1000, 96), 3), ((3, 65, 132), 4), ((2, 300, 1024), 2), ((1, 5, 600), 1), ((40, 7, 48), 6), ((2, 4097, 64), 32),
        ((1, 33, 99), 3), ((2, 9, 11, 40), 5), ((1, 20000, 8), 1), ((300, 3, 768), 32), ((8, 130, 7), 7), ((1, 2, 5000), 8)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,G", ROWS + MAPS, ids=str)
def test_values_and_gradients(shape, G, dtype):
    x, w, b, dy = make(shape, dtype, sum(shape) + G)
    want = reference(x, G, w, b, dy)
    for n, t in run(x, G, w, b, dy).items():
        assert t.dtype == (dtype if n in ("y", "d_x") else torch.float32)
        close(t, want[n], n)
    with torch.no_grad():
        close(gn.group_norm_act(x, G, w, b), want["y"], "y without gradients")


@pytest.mark.parametrize("shape,G", [((50, 96), 6), ((2, 70, 96), 6)], ids=str)
def test_options(shape, G):
    x, w, b, dy = make(shape, torch.bfloat16, 3)
    want = reference(x, G, w, b, dy, eps=0.1, act=False)
    for n, t in run(x, G, w, b, dy, eps=0.1, activation=None).items():
        close(t, want[n], n)
    want = reference(x, G, None, None, dy)
    leaf = x.clone().requires_grad_()
    y = gn.group_norm_act(leaf, G)
    close(y.detach(), want["y"], "y")
    close(torch.autograd.grad(y, leaf, dy)[0], want["d_x"], "d_x")
    leaf_w = w.bfloat16().requires_grad_()  # a parameter alone, of another type
    want = reference(x, G, leaf_w.detach(), b, dy)
    close(torch.autograd.grad(gn.group_norm_act(x, G, leaf_w, b), leaf_w, dy)[0], want["d_w"], "d_w")
    module = gn.GroupNorm(G, shape[-1]).to(DEV)
    close(module(x).detach(), reference(x, G, None, None)["y"], "module")


@pytest.mark.parametrize("shape,G", [((64, 64), 1), ((2, 500, 64), 2)], ids=str)
def test_large_mean_small_variance(shape, G):
    """A variance computed from sums of squares would lose all its digits here."""
    x, w, b, dy = make(shape, torch.float32, 5)
    x = 1000 + 0.01 * x
    want = reference(x, G, w, b, dy)
    got = run(x, G, w, b, dy)
    close(got["y"], want["y"], "y")
    close(got["d_x"], want["d_x"], "d_x")
    # far inside the bound, which has to allow for a mean that is off by 192 roundings
    assert (got["y"].double() - want["y"][0]).abs().max() < 0.05


@pytest.mark.parametrize("shape,G", [((6, 32), 4), ((6, 40, 32), 4), ((6, 513), 1)], ids=str)
def test_constant_groups_infinities_and_nan(shape, G):
    x, w, b, dy = make(shape, torch.float32, 7)
    x[0] = 3.0
    x[2, ..., 0], x[4, ..., 1] = float("nan"), float("inf")
    got = run(x, G, w, b, dy)
    Cg = shape[-1] // G
    z = b.expand(shape[1:])
    # a constant's mean may be off by its rounding, which sqrt(eps) bounds from above when it is divided by
    assert (got["y"][0] - z * torch.sigmoid(z)).abs().max() < 1e-3
    for n in (2, 4):
        assert torch.isnan(got["y"][n, ..., :Cg]).all()
        if G > 1:
            assert not torch.isnan(got["y"][n, ..., Cg:]).any() and not torch.isnan(got["d_x"][n, ..., Cg:]).any()
    for n in (1, 3, 5):
        assert torch.isfinite(got["y"][n]).all() and torch.isfinite(got["d_x"][n]).all()


def test_saturated_activation():
    x = torch.tensor([[-200.0, 200.0, -90.0, 90.0]], device=DEV)
    w = torch.full((4,), 100.0, device=DEV)
    got = run(x, 1, w, torch.zeros(4, device=DEV), torch.ones_like(x))
    assert torch.isfinite(got["y"]).all() and torch.isfinite(got["d_x"]).all()
    want = reference(x, 1, w, torch.zeros(4, device=DEV), torch.ones_like(x))
    close(got["y"], want["y"], "y")
    close(got["d_x"], want["d_x"], "d_x")


@pytest.mark.parametrize("dtype", TYPES)
def test_unaligned_and_strided(dtype):
    for shape, G in (((30, 64), 2), ((2, 50, 64), 2)):
        x, w, b, dy = make(shape, dtype, 11)
        flat = torch.empty(x.numel() + 1, dtype=dtype, device=DEV)[1:].view(shape)
        flat.copy_(x)
        want = reference(x, G, w, b, dy)
        for n, t in run(flat, G, w, b, dy).items():
            close(t, want[n], n)
        wide = torch.zeros(*shape[:-1], 2 * shape[-1], dtype=dtype, device=DEV)
        wide[..., 64:] = x
        y = gn.group_norm_act(wide[..., 64:], G, w, b)
        assert torch.equal(y, gn.group_norm_act(x, G, w, b))
        leaf = x.clone().requires_grad_()
        d = torch.autograd.grad(gn.group_norm_act(leaf, G, w, b), leaf, dy[..., :1].expand(shape))[0]
        close(d, reference(x, G, w, b, dy[..., :1].expand(shape))["d_x"], "d_x of a broadcast gradient")


def test_gradients_against_differences():
    for shape, G in (((6, 24), 3), ((2, 35, 24), 3)):
        x, w, b, dy = make(shape, torch.float32, 13)
        got = run(x, G, w, b, dy)
        base = {"x": x.double(), "w": w.double(), "b": b.double()}
        loss = lambda v: (reference(v["x"], G, v["w"], v["b"])["y"][0] * dy.double()).sum()  # noqa: E731
        g = torch.Generator(device=DEV).manual_seed(17)
        for n, t in base.items():
            step = torch.randn(t.shape, generator=g, device=DEV, dtype=torch.float64)
            # central difference: off by step^2 times a third derivative of order one, and rounding / step
            diff = (loss({**base, n: t + 1e-5 * step}) - loss({**base, n: t - 1e-5 * step})) / 2e-5
            prod = got["d_" + n].double() * step
            assert abs(float(prod.sum() - diff)) <= 2e-6 * float(prod.abs().sum()) + 1e-7, n


def test_runs_streams_and_graphs():
    cases = [make((900, 768), torch.bfloat16, 19) + (12,), make((3, 777, 96), torch.bfloat16, 23) + (4,)]
    side = torch.cuda.Stream(device=DEV)
    wants = [run(x, G, w, b, dy) for x, w, b, dy, G in cases]
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream(DEV))
    for _ in range(4):
        with torch.cuda.stream(side):
            a = run(cases[0][0], 12, *cases[0][1:4])
        c = run(cases[1][0], 4, *cases[1][1:4])
        torch.cuda.synchronize()
        assert all(torch.equal(a[n], wants[0][n]) and torch.equal(c[n], wants[1][n]) for n in a)
    for (x, w, b, dy, G), want in zip(cases, wants):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = gn.group_norm_act(leaves[0], G, leaves[1], leaves[2])
            d = torch.autograd.grad(y, leaves, dy)
        for k in range(2):
            with torch.no_grad():
                leaves[0].copy_(x.flip(0) if k else x)
            graph.replay()
            torch.cuda.synchronize()
            want_k = run(x.flip(0), G, w, b, dy) if k else want
            assert torch.equal(y.detach(), want_k["y"]) and all(torch.equal(t, want_k[n]) for t, n in zip(d, ("d_x", "d_w", "d_b")))


def test_empty():
    for shape in ((0, 8), (3, 0, 8), (0, 4, 8), (3, 0)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w = torch.ones(shape[-1], device=DEV, requires_grad=True)
        y = gn.group_norm_act(x, 1 if shape[-1] == 0 else 2, w, w)
        assert y.shape == shape
        d = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert d[0].shape == shape and (d[1] == 0).all()


def test_offsets_beyond_32_bits():
    n, C = 2 ** 25 + 3, 66
    x = torch.zeros(n, C, dtype=torch.float16, device=DEV)
    x[-1] = torch.randn(C, device=DEV).half()
    y = gn.group_norm_act(x, 3)
    close(y[-1:], reference(x[-1:], 3, None, None)["y"], "y")
    assert (y[:-1] == 0).all()
    del y
    x = x.view(1, n, C)
    x[0, :, :22] = 1.0
    y = gn.group_norm_act(x, 3, activation=None)
    assert (y[0, :, :22].abs() < 1e-2).all() and (y[0, -1, 22:] != 0).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_layer_of_all_three(dtype):
    """Recurrence over time, its heads normalised, experts for the last position; and the same token by token."""
    T, B, D, E, F, heads = 40, 6, 128, 8, 64, 4
    g = torch.Generator(device=DEV).manual_seed(29)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    proj, bias = rn(T, B, 2 * D).to(dtype), rn(D)
    w, b = 1 + 0.1 * rn(D), 0.1 * rn(D)
    wr, wi, wo = rn(E, D).to(dtype) * D ** -0.5, rn(E, 2 * F, D).to(dtype) * D ** -0.5, rn(E, D, F).to(dtype) * F ** -0.5
    with torch.no_grad():
        raw, x = proj.chunk(2, -1)
        y, h_last = gr.gated_linear_recurrence(raw, x, None, bias)
        z = gn.group_norm_act(y.reshape(T * B, D), heads, w, b).view(T, B, D)
        out = mk.moe_few_tokens(z[-1], wr, wi, wo, 2, shared=x[-1])
        h = torch.zeros(B, D, device=DEV)
        for t in range(T):
            y_t = gr.gated_linear_recurrence_step(proj[t, :, :D], proj[t, :, D:], h, bias)
            z_t = gn.group_norm_act(y_t, heads, w, b)
        out_t = mk.moe_few_tokens(z_t, wr, wi, wo, 2, shared=proj[-1, :, D:])
    want = torch.zeros(B, D, dtype=torch.float64, device=DEV)
    a = raw.double() + bias.double()
    for t in range(T):
        want = torch.sigmoid(a[t]) * want + torch.sigmoid(-a[t]) * x[t].double()
    # a state is a mean of inputs with weights that add up to one, so no rounding of it grows: 40 steps, (16 + |a|) roundings each
    assert (h_last.double() - want).abs().max() <= 40 * (16 + float(a.abs().max()) + 128) * U * float(x.abs().max())
    assert (h_last - h).abs().max() <= 2 * 40 * (16 + float(a.abs().max()) + 128) * U * float(x.abs().max())
    zw = reference(y.reshape(T * B, D), heads, w, b)["y"]
    close(z.reshape(T * B, D), zw, "z")
    # the recurrence's output is the same in both ways but for roundings that may tip over, one step of the type
    assert torch.isfinite(out).all() and torch.isfinite(out_t).all()
    if dtype == torch.float32:
        assert (out - out_t).abs().max() <= 1e-4 * out.abs().max()
    # and a training step through the first two
    leaves = [t.clone().requires_grad_() for t in (proj, bias, w, b)]
    y, _ = gr.gated_linear_recurrence(leaves[0][..., :D], leaves[0][..., D:], None, leaves[1])
    gn.group_norm_act(y.reshape(T * B, D), heads, leaves[2], leaves[3]).float().square().sum().backward()
    assert all(t.grad is not None and torch.isfinite(t.grad).all() and (t.grad != 0).any() for t in leaves)
    assert nsb.device_error_word() == 0


def test_second_derivatives_are_refused():
    x = torch.randn(4, 6, device=DEV, requires_grad=True)
    y = gn.group_norm_act(x, 2)
    with pytest.raises(nsb.NSBError, match="second derivatives"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("shape,G", [((7, 96), 3), ((2, 70, 96), 3), ((1, 1000, 40), 1), ((3, 600), 1), ((2, 33, 520), 2)], ids=str)
def test_means_whose_square_overflows(shape, G):
    """A finite variance about a mean of 1e20, in both layouts."""
    _, w, b, dy = make(shape, torch.float32, 31)
    g = torch.Generator(device=DEV).manual_seed(37)
    x = 1e20 * (1 + 1e-4 * torch.randn(shape, generator=g, device=DEV))
    assert torch.isinf(x.mean() ** 2) and torch.isfinite((x - x.mean()).square().sum())
    want = reference(x, G, w, b, dy)
    for n, t in run(x, G, w, b, dy).items():
        close(t, want[n], n)


def test_nothing_is_kept_for_a_backward_that_cannot_come():
    """A module's parameters cost no saved statistics without gradients."""
    norm = gn.GroupNorm(6, 96).to(DEV)
    w, b = norm.weight.detach().clone(), norm.bias.detach().clone()

    def allocations(call):
        before = torch.cuda.memory_stats(DEV)["allocation.all.allocated"]
        call()
        return torch.cuda.memory_stats(DEV)["allocation.all.allocated"] - before
    for shape in ((50, 96), (2, 70, 96)):
        x = torch.randn(shape, device=DEV)
        for mode in (torch.no_grad, torch.inference_mode):
            with mode():
                assert allocations(lambda: norm(x)) == allocations(lambda: gn.group_norm_act(x, 6, w, b))
                assert torch.equal(norm(x), gn.group_norm_act(x, 6, w, b))
        assert allocations(lambda: norm(x)) > allocations(lambda: gn.group_norm_act(x, 6, w, b))
