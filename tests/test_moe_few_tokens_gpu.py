"""The expert layer for a few tokens against the same layer in 64 bits.

Bounds. A tensor-core product adds 16 (fp32 operands: 8, three times) summands to its fp32 accumulator; taking
2^-22 of the sum of absolute values for each such addition covers truncation and the alignment inside it. A logit is
such sums of at most every eighth block each, added up in fp32, and fp32 operands lose 2^-20 of each product. Hidden
values keep 2^-16 with 16-bit weights, 2^-21 otherwise. p is off by twice the
logits' error, and silu's slope is at most 1.1. The output adds half a step of its type. Which experts are taken is
checked against the 64-bit logits up to their error, and the values with the experts that were taken."""
import pytest
import torch

import neuronspark_b200 as nsb
from neuronspark_b200 import moe_kernels as mk

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(N, E, k, D, F, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    return ((scale * rn(N, D)).to(dtype), (2 * rn(E, D) * max(D, 1) ** -0.5).to(dtype),
            (rn(E, 2 * F, D) * max(D, 1) ** -0.5).to(dtype), (rn(E, D, F) * max(F, 1) ** -0.5).to(dtype), rn(N, D).to(dtype))


def check(x, wr, wi, wo, k, shared, got):
    out, ids, p = got
    N, D = x.shape
    E, F, dt = wr.shape[0], wo.shape[2], x.dtype
    assert out.shape == (N, D) and out.dtype == dt and ids.dtype == torch.int32 and p.dtype == torch.float32
    X, WR = x.double(), wr.double()
    logits = X @ WR.T
    per = (2.0 ** -22 * 3 / 8, 2.0 ** -20) if dt == torch.float32 else (2.0 ** -22 / 16, 0.0)
    e_l = ((D / 8 * per[0] + per[1] + 16 * 2.0 ** -22) * (X.abs() @ WR.abs().T)).amax(1, keepdim=True)
    ids = ids.long()
    taken = torch.zeros(N, E, dtype=torch.bool, device=DEV).scatter_(1, ids, True)
    assert (taken.sum(1) == k).all()  # distinct
    mine = logits.gather(1, ids)
    assert (mine[:, 1:] <= mine[:, :-1] + 2 * e_l).all()
    assert (logits.masked_fill(taken, -float("inf")).amax(1, keepdim=True) <= mine[:, -1:] + 2 * e_l).all()
    P = torch.softmax(mine, 1)
    # below the least normal number, 2^-126, p has fewer digits or none: a logit 120 under the best gives 2^-173
    e_p = P * (2 * e_l + 16 * 2.0 ** -24) + 2.0 ** -126
    assert ((p.double() - P).abs() <= e_p).all()
    value = torch.zeros(N, D, dtype=torch.float64, device=DEV) if shared is None else shared.double()
    err = (k + 2) * 2.0 ** -24 * value.abs()
    add = 2.0 ** -22 * (3 / 8 if dt == torch.float32 else 1 / 16)
    # 16-bit weights: the hidden value in two bf16 terms, the second at most 2^-8 of it and itself rounded by 2^-8; fp16
    # weights are exact in two bf16 terms, the second (what lies behind 8 bits) below 2^-7, and the product of both second
    # terms, 2^-8 x 2^-7, is left out: 2^-16 + 2^-15
    left = {torch.bfloat16: 2.0 ** -16, torch.float16: 1.5 * 2.0 ** -15, torch.float32: 2.0 ** -20}[dt]
    add2 = 2.0 ** -22 * {torch.bfloat16: 2 / 16, torch.float16: 3 / 16, torch.float32: 3 / 8}[dt]
    for n in range(N):
        for j in range(k):
            W, O = wi[ids[n, j]].double(), wo[ids[n, j]].double()
            u, e_u = W @ X[n], ((D * add + 16 * 2.0 ** -22) + (2.0 ** -20 if dt == torch.float32 else 0)) * (W.abs() @ X[n].abs())
            gate, up, e_g, e_up = u[:F], u[F:], e_u[:F], e_u[F:]
            s = gate * torch.sigmoid(gate)
            h = P[n, j] * s * up
            e_h = P[n, j] * (1.1 * e_g * up.abs() + (s.abs() + 1.1 * e_g) * e_up) + e_p[n, j] * (s * up).abs() \
                + (left + 16 * 2.0 ** -24) * h.abs()
            value[n] += O @ h
            err[n] += O.abs() @ e_h + (F * add2 + 24 * 2.0 ** -22) * (O.abs() @ h.abs())
    half = torch.finfo(dt).eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126
    off = (out.double() - value).abs()
    bound = err * (1 + half) + half * value.abs() + tiny
    assert (off <= bound).all(), f"{float((off / bound).max()):.2f} times the bound"


SIZES = [(1, 1, 1, 8, 8), (1, 8, 2, 768, 2304), (2, 3, 2, 64, 40), (7, 16, 4, 328, 72), (16, 4, 1, 128, 136), (17, 5, 3, 264, 64),
         (33, 8, 2, 256, 128), (64, 2, 2, 72, 200), (64, 128, 8, 512, 96), (64, 33, 16, 40, 24), (3, 1024, 16, 64, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, dtype):
    N, E, k, D, F = size
    x, wr, wi, wo, shared = make(N, E, k, D, F, dtype, sum(size))
    for sh in (shared, None):
        check(x, wr, wi, wo, k, sh, mk.moe_few_tokens(x, wr, wi, wo, k, shared=sh, return_routing=True))
    assert torch.equal(mk.moe_few_tokens(x, wr, wi, wo, k, shared=shared),
                       mk.moe_few_tokens(x, wr, wi, wo, k, shared=shared, return_routing=True)[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(5, 4, 2, 1, 1), (3, 6, 2, 37, 19), (20, 4, 2, 131, 67), (1, 2, 1, 9, 130)], ids=str)
def test_odd_widths(size, dtype):
    N, E, k, D, F = size
    x, wr, wi, wo, shared = make(N, E, k, D, F, dtype, sum(size))
    check(x, wr, wi, wo, k, shared, mk.moe_few_tokens(x, wr, wi, wo, k, shared=shared, return_routing=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_unaligned_weights_and_strided_tokens(dtype):
    N, E, k, D, F = 6, 4, 2, 64, 32
    x, wr, wi, wo, shared = make(N, E, k, D, F, dtype, 3)
    want = mk.moe_few_tokens(x, wr, wi, wo, k, shared=shared)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=dtype, device=DEV)[1:]
        return flat.copy_(t.flatten()).view(t.shape)
    got = mk.moe_few_tokens(x, shifted(wr), shifted(wi), shifted(wo), k, shared=shared, return_routing=True)
    check(x, wr, wi, wo, k, shared, got)
    wide = torch.randn(N, 3 * D + 1, device=DEV).to(dtype)
    wide[:, D:2 * D] = x
    assert torch.equal(mk.moe_few_tokens(wide[:, D:2 * D], wr, wi, wo, k, shared=shared), want) or D % 8
    seq = torch.randn(9, N, D, device=DEV).to(dtype)  # the last position of a time-major batch
    seq[-1] = x
    assert torch.equal(mk.moe_few_tokens(seq[-1], wr, wi, wo, k, shared=shared), want)
    assert torch.equal(mk.moe_few_tokens(x.T.contiguous().T, wr, wi, wo, k, shared=shared), want)


def test_all_tokens_to_the_same_experts():
    N, E, k, D, F = 64, 16, 2, 256, 128
    x, wr, wi, wo, shared = make(N, E, k, D, F, torch.bfloat16, 5)
    x[:, 0] = 30.0
    wr[:, 0] = 0
    wr[3, 0], wr[11, 0] = 8, 4
    got = mk.moe_few_tokens(x, wr, wi, wo, k, shared=shared, return_routing=True)
    assert (got[1] == torch.tensor([3, 11], device=DEV, dtype=torch.int32)).all()
    check(x, wr, wi, wo, k, shared, got)


def test_ties_take_the_lowest_index():
    N, E, k, D, F = 4, 40, 5, 64, 32
    x, wr, wi, wo, shared = make(N, E, k, D, F, torch.float32, 7)
    wr[:] = wr[0]
    wr[35] = wr[0] * 0
    wr[36] = -wr[35]  # a negative zero is a zero
    _, ids, p = mk.moe_few_tokens(x, wr, wi, wo, k, return_routing=True)
    sign = (x @ wr[0]).sign()
    for n in range(N):
        rest = [e for e in range(E) if e not in (35, 36)]
        want = rest[:k] if sign[n] > 0 else [35, 36] + rest[:k - 2]
        assert ids[n].tolist() == want
    assert torch.allclose(p.sum(1), torch.ones(N, device=DEV))


def test_infinities_and_nan_stay_with_their_token():
    N, E, k, D, F = 6, 8, 3, 64, 32
    for dtype in TYPES:
        x, wr, wi, wo, shared = make(N, E, k, D, F, dtype, 9)
        want = mk.moe_few_tokens(x, wr, wi, wo, k, shared=shared)
        x[1, 5], x[4, 7] = float("nan"), float("inf")
        out, ids, p = mk.moe_few_tokens(x, wr, wi, wo, k, shared=shared, return_routing=True)
        for n in (0, 2, 3, 5):
            assert torch.equal(out[n], want[n])
        assert torch.isnan(out[1]).all() and not torch.isfinite(out[4].float()).any()
        for n in range(N):
            assert len(set(ids[n].tolist())) == k and 0 <= int(ids[n].min()) and int(ids[n].max()) < E
    # an expert that no token takes is not read
    x, wr, wi, wo, shared = make(N, E, k, D, F, torch.bfloat16, 9)
    out, ids, _ = mk.moe_few_tokens(x, wr, wi, wo, 1, shared=shared, return_routing=True)
    for e in set(range(E)) - set(ids.flatten().tolist()):
        wi[e], wo[e] = float("nan"), float("nan")
    assert torch.equal(mk.moe_few_tokens(x, wr, wi, wo, 1, shared=shared), out)


def test_hidden_values_beyond_half_precision():
    """fp16 weights and tokens whose hidden values exceed 65504, brought back by the second product."""
    N, E, k, D, F = 3, 2, 1, 64, 32
    x, wr, wi, wo, shared = make(N, E, k, D, F, torch.float16, 11, scale=40.0)
    wi, wo = wi * 12, wo * 2.0 ** -12
    got = mk.moe_few_tokens(x, wr, wi, wo, k, shared=shared, return_routing=True)
    hidden = torch.einsum("nd,efd->nef", x.double(), wi.double())
    assert float((torch.sigmoid(hidden[..., :F]) * hidden[..., :F] * hidden[..., F:]).abs().max()) > 65504
    check(x, wr, wi, wo, k, shared, got)


def test_runs_streams_and_graphs():
    N, E, k, D, F = 24, 16, 4, 512, 256
    args = make(N, E, k, D, F, torch.bfloat16, 13)
    other = make(5, 8, 2, 256, 512, torch.bfloat16, 14)
    call = lambda a, k: mk.moe_few_tokens(*a[:4], k, shared=a[4], return_routing=True)  # noqa: E731
    want, want_other = call(args, k), call(other, 2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    for _ in range(5):
        with torch.cuda.stream(side):
            a = call(other, 2)
        b = call(args, k)
        torch.cuda.synchronize()
        assert all(map(torch.equal, a, want_other)) and all(map(torch.equal, b, want))
    x, shared = args[0].clone(), args[4].clone()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        g1 = call((x, *args[1:4], shared), k)
    with torch.cuda.graph(second, stream=side):
        g2 = call((x, *args[1:4], shared), k)
    for r in range(3):
        x.copy_(args[0].roll(r, 0))
        shared.copy_(args[4].roll(r, 0))
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        for got in (g1, g2):
            assert all(torch.equal(t, w.roll(r, 0)) for t, w in zip(got, want))


def test_empty():
    x, wr, wi, wo, shared = make(0, 4, 2, 64, 32, torch.bfloat16, 1)
    assert mk.moe_few_tokens(x, wr, wi, wo, 2).shape == (0, 64)
    x, wr, wi, wo, shared = make(3, 4, 2, 64, 0, torch.bfloat16, 1)
    assert torch.equal(mk.moe_few_tokens(x, wr, wi, wo, 2, shared=shared), shared)
    x, wr, wi, wo, shared = make(3, 4, 2, 0, 8, torch.bfloat16, 1)
    out, ids, p = mk.moe_few_tokens(x, wr, wi, wo, 2, return_routing=True)
    assert out.shape == (3, 0) and (ids == torch.tensor([0, 1], device=DEV)).all() and (p == 0.5).all()


def test_offsets_beyond_32_bits():
    """The last expert's weights lie more than 2^31 elements into w_in."""
    E, D, F = 9, 8192, 16384
    wi = torch.empty(E, 2 * F, D, dtype=torch.bfloat16, device=DEV)
    wi[E - 1].normal_(0, D ** -0.5)
    wo = torch.empty(E, D, F, dtype=torch.bfloat16, device=DEV)
    wo[E - 1].normal_(0, F ** -0.5)
    x = torch.randn(2, D, device=DEV).bfloat16()
    wr = torch.zeros(E, D, dtype=torch.bfloat16, device=DEV)
    x[:, 0], wr[E - 1, 0] = 4.0, 4.0
    got = mk.moe_few_tokens(x, wr, wi, wo, 1, return_routing=True)
    assert (got[1] == E - 1).all()
    check(x, wr, wi, wo, 1, None, got)


def test_no_gradients():
    x, wr, wi, wo, shared = make(2, 4, 2, 64, 32, torch.bfloat16, 1)
    wi.requires_grad_()
    with pytest.raises(nsb.NSBError):
        mk.moe_few_tokens(x, wr, wi, wo, 2)
    with torch.no_grad():
        mk.moe_few_tokens(x, wr, wi, wo, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [1, 3, 40])
def test_hidden_values_keep_their_digits(N, dtype):
    """Hidden values that are whole numbers of 23 bits, and outputs that are small differences of two of them: everything on the
    way is exact in fp32 (silu(g) = g where exp(-g) is below 2^-24, p = 1), and so is the output in its type."""
    D, F = 16, 32
    r = torch.arange(1, 17, device=DEV)
    g = 2890 - 3 * r                                # h = g (g - 1 - r) < 2^23, beside it (g - 1) (g - r) = h + r
    gate, up = torch.cat([g, g - 1]), torch.cat([g - 1 - r, g - r])
    assert int((gate * up).max()) < 2 ** 23 and int((gate * up).min()) > 2 ** 22
    bits = 2 ** torch.arange(D, device=DEV)
    w_in = torch.cat([gate, up])[:, None].bitwise_and(bits).to(dtype)[None]
    w_out = torch.cat([-torch.eye(16, device=DEV), torch.eye(16, device=DEV)], 1).to(dtype)[None]
    x = torch.ones(N, D, device=DEV, dtype=dtype)
    out = mk.moe_few_tokens(x, torch.zeros(1, D, device=DEV, dtype=dtype), w_in, w_out, 1)
    assert torch.equal(out, r.to(dtype).expand(N, D))


def test_long_sums_of_one_sign():
    """fp32, 32768 positive products a sum: rounding toward zero would lose some 1e-4 of each. Four warps share a row, so a warp
    adds 32768 / 16 / 4 = 512 chunks, each to the nearest: 512 / 2 half units in the last place (the partial sum is half of
    the whole on average), 2^-20 of each product and 6 products of a chunk at 2^-22."""
    D, F = 32768, 8
    g = torch.Generator(device=DEV).manual_seed(15)
    x, w_in = (0.5 + torch.rand(s, generator=g, device=DEV) for s in ((2, D), (1, 2 * F, D)))
    w_in /= D
    w_out = torch.zeros(1, D, F, device=DEV)
    w_out[0, :F] = torch.eye(F, device=DEV)
    out = mk.moe_few_tokens(x, torch.zeros(1, D, device=DEV), w_in, w_out, 1)[:, :F]
    u = (x.double()[:, None] * w_in.double()).sum(-1)
    gate, up = u[:, :F], u[:, F:]
    e = 2.0 ** -20 + 6 * 2.0 ** -22 + (512 / 2 + 8) * 2.0 ** -24
    s = gate * torch.sigmoid(gate)
    # the down product: 2^-20 of its one summand, and the sigmoid's, the activation's and p's roundings
    bound = 1.1 * e * gate * up + (s + 1.1 * e * gate) * e * up + (2.0 ** -20 + 24 * 2.0 ** -24) * s * up
    assert ((out.double() - s * up).abs() <= bound).all()
