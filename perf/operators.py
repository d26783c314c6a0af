"""Cases for the operators of a continuous (non-spiking) layer: the gated linear recurrence (training, packed
prefill, one token), group norm with an activation (training, decoding) and the expert layer for a few tokens.

``run`` computes them from elementary torch operations in 32 bits (``own`` false) or calls this package's
operators (``own`` true). ``exact`` computes them again in 64 bits, step by step.
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_DEV = "cuda"


def listed():
    return [
        # a layer of the 768-wide model in training: 8 sequences of 512 tokens x 16 frames
        {"name": "recurrence-train-768", "kind": "recurrence", "dtype": "bf16", "T": 8192, "B": 8, "D": 768, "train": True},
        # its hidden neurons: 8 x 768 channels each; the largest case
        {"name": "recurrence-train-6144", "kind": "recurrence", "dtype": "bf16", "T": 8192, "B": 8, "D": 6144, "train": True},
        # one long document in fp32: few columns, all parallelism is along time
        {"name": "recurrence-train-long-f32", "kind": "recurrence", "dtype": "f32", "T": 65536, "B": 1, "D": 768, "train": True},
        # documents of different lengths packed into one batch without padding, training
        {"name": "recurrence-train-packed", "kind": "packed", "dtype": "bf16", "rows": 32768, "seqs": 24, "D": 768, "train": True},
        # prompts of different lengths read in before generation; an odd width
        {"name": "recurrence-prefill-odd-f16", "kind": "packed", "dtype": "f16", "rows": 20011, "seqs": 37, "D": 1001, "train": False},
        # one token for each of 1024 running sequences
        {"name": "recurrence-step-1024", "kind": "step", "dtype": "bf16", "B": 1024, "D": 768},
        # the heads of every token normalised by themselves (12 heads of 64), training
        {"name": "norm-train-tokens", "kind": "norm", "dtype": "bf16", "N": 65536, "L": 1, "C": 768, "G": 12, "train": True},
        # statistics over whole sequences of 4096 positions, 32 groups, training
        {"name": "norm-train-maps", "kind": "norm", "dtype": "bf16", "N": 8, "L": 4096, "C": 768, "G": 32, "train": True},
        # the heads of 64 running sequences' next tokens: latency
        {"name": "norm-decode-f32", "kind": "norm", "dtype": "f32", "N": 64, "L": 1, "C": 768, "G": 12, "train": False},
        # one token through a small expert layer of the 768-wide model: latency
        {"name": "experts-1", "kind": "experts", "dtype": "bf16", "N": 1, "E": 8, "k": 2, "D": 768, "F": 2304},
        # sixteen running sequences, many narrow experts
        {"name": "experts-16-f16", "kind": "experts", "dtype": "f16", "N": 16, "E": 64, "k": 6, "D": 2048, "F": 1024},
        # the most tokens that still count as few: every expert is in use
        {"name": "experts-64", "kind": "experts", "dtype": "bf16", "N": 64, "E": 32, "k": 4, "D": 4096, "F": 1792},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["recurrence", "recurrence", "packed", "packed", "step", "norm", "norm", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.6
    if kind == "recurrence":
        B, D = _log(rng, 1, 64), _log(rng, 1, 8192)
        T = max(1, min(32768, _log(rng, 1 << 12, 1 << 26) // (B * D)))
        return {"kind": kind, "dtype": dtype, "T": T, "B": B, "D": D, "train": train}
    if kind == "packed":
        D = _log(rng, 16, 4096)
        rows = max(8, min(32768, _log(rng, 1 << 14, 1 << 25) // D))
        return {"kind": kind, "dtype": dtype, "rows": rows, "seqs": max(1, min(rows, _log(rng, 1, 300))), "D": D, "train": train}
    if kind == "step":
        return {"kind": kind, "dtype": dtype, "B": _log(rng, 1, 4096), "D": _log(rng, 64, 8192)}
    if kind == "norm":
        G, width = _log(rng, 1, 48), rng.choice([8, 16, 24, 33, 40, 64, 96, 100, 128])
        L = 1 if rng.random() < 0.5 else _log(rng, 2, 16384)
        N = max(1, min(65536, _log(rng, 1 << 12, 1 << 25) // (L * G * width)))
        return {"kind": kind, "dtype": dtype, "N": N, "L": L, "C": G * width, "G": G, "train": train}
    E = _log(rng, 2, 128)
    D, F = 8 * _log(rng, 16, 512), 8 * _log(rng, 16, 256)
    while E * D * F > 32 * 4096 * 1792:
        E = max(2, E // 2)
        F = F // 16 * 8 if F > 256 else F
    return {"kind": kind, "dtype": dtype, "N": _log(rng, 1, 64), "E": E, "k": rng.randint(1, min(8, E)), "D": D, "F": F}


def _lengths(case, seed):
    """First rows of the sequences (and the end of the last), with an empty one and one of a single row among
    them where there is room, and a few rows behind the last sequence that belong to none."""
    rng = random.Random(seed * 7919 + case["rows"])
    end, S = case["rows"] - case["rows"] // 64, case["seqs"]
    cuts = sorted(rng.randint(0, end) for _ in range(S - 1))
    if S >= 5 and cuts[3] + 1 <= end:
        cuts[1] = cuts[0]
        cuts[2] = min(cuts[0] + 1, cuts[3])
    return [0] + cuts + [end]


def prepare(case, seed):
    dt = _TYPES[case["dtype"]]
    g = torch.Generator(device=_DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=_DEV)  # noqa: E731
    s, kind, train = {"case": case}, case["kind"], case.get("train", False)
    if kind in ("recurrence", "packed", "step"):
        D = case["D"]
        shape = {"recurrence": (case.get("T"), case.get("B"), D), "packed": (case.get("rows"), D),
                 "step": (case.get("B"), D)}[kind]
        state = {"recurrence": (case.get("B"), D), "packed": (case.get("seqs"), D), "step": (case.get("B"), D)}[kind]
        s["raw"], s["x"] = (rn(shape) + 1.5).to(dt), rn(shape).to(dt)  # most gates keep most of the state
        s["bias"], s["h0"] = 0.5 * rn(D) + 0.5, rn(state)
        if kind == "packed":
            s["cu"] = torch.tensor(_lengths(case, seed), dtype=torch.int32, device=_DEV)
        leaves, grads = ("raw", "x", "bias", "h0"), {"dy": (shape, dt), "dh": (state, torch.float32)}
    elif kind == "norm":
        shape = (case["N"], case["L"], case["C"]) if case["L"] > 1 else (case["N"], case["C"])
        s["x"] = (rn(shape) * 1.5 + 0.5).to(dt)
        s["w"], s["b"] = 1 + 0.2 * rn(case["C"]), 0.2 * rn(case["C"])
        leaves, grads = ("x", "w", "b"), {"dy": (shape, dt)}
    else:
        N, E, D, F = case["N"], case["E"], case["D"], case["F"]
        s["x"], s["shared"] = rn(N, D).to(dt), rn(N, D).to(dt)
        s["router"] = (rn(E, D) * D ** -0.5).to(dt)
        s["w_in"], s["w_out"] = torch.empty(E, 2 * F, D, dtype=dt, device=_DEV), torch.empty(E, D, F, dtype=dt, device=_DEV)
        s["w_in"].normal_(0, D ** -0.5, generator=g)
        s["w_out"].normal_(0, F ** -0.5, generator=g)
        leaves, grads = (), {}
    if train:
        for n in leaves:
            s[n].requires_grad_()
        for n, (shape, t) in grads.items():
            s[n] = rn(shape).to(t)
    return s


# ------------------------------------------------------------------------------------------ plain forms


def _scan(A, H):
    """H_t <- H_t + A_t H_{t-1}, along the first dimension, by doubling the reach of every element."""
    d = 1
    while d < H.shape[0]:
        H = torch.cat([H[:d], torch.addcmul(H[d:], A[d:], H[:-d])])
        A = torch.cat([A[:d], A[d:] * A[:-d]])
        d *= 2
    return H


def _rows(s):
    """Of every packed row: its sequence, whether it is in one, and whether it is the first or last row there."""
    cu = s["cu"].long()
    S, rows = cu.numel() - 1, torch.arange(s["x"].shape[0], device=cu.device)
    seq = (cu[1:, None] <= rows).sum(0)
    inside = (seq < S)
    seq = seq.clamp(max=S - 1)
    return cu, seq, inside, inside & (rows == cu[seq]), inside & (rows + 1 == cu[seq + 1])


def _plain_recurrence(s):
    raw, x, h0, bias = (s[n].detach().float() for n in ("raw", "x", "h0", "bias"))
    dt, packed = s["x"].dtype, "cu" in s
    f, m = torch.sigmoid(raw + bias), torch.sigmoid(-(raw + bias))
    H = m * x
    col = lambda v: v[:, None]  # noqa: E731
    if packed:
        cu, seq, inside, first, last = _rows(s)
        some = col(cu[1:] > cu[:-1])
        start, end = cu[:-1].clamp(max=x.shape[0] - 1), (cu[1:] - 1).clamp(min=0)
        before = col(first) * h0[seq]  # the state that a first row continues from
        H = _scan(f * col(~first), torch.addcmul(H, f, before))
        h_last = torch.where(some, H[end], h0)
        y = (H * col(inside)).to(dt)
    else:
        H[0] += f[0] * h0
        H = _scan(f, H)
        h_last = H[-1].clone()
        y = H.to(dt)
    if "dy" not in s:
        return {"y": y, "h_last": h_last}
    dy, dh = s["dy"].float(), s["dh"]
    back = torch.zeros_like(f)  # what a step hands to the one before it
    back[:-1] = f[1:]
    if packed:
        E = dy * col(inside) + col(last) * dh[seq]
        back = back * col(~last)
    else:
        E = torch.cat([dy[:-1], dy[-1:] + dh])
    G = _scan(back.flip(0), E.flip(0)).flip(0)
    if packed:
        prev = torch.cat([H[:1], H[:-1]])
        prev = torch.where(col(first), before, prev)
        d_h0 = torch.where(some, (f * G)[start], dh)
        G = G * col(inside)
    else:
        prev = torch.cat([h0[None], H[:-1]])
        d_h0 = f[0] * G[0]
    d_raw = G * (prev - x) * f * m
    d_bias = d_raw.double().reshape(-1, x.shape[-1]).sum(0).float()
    return {"y": y, "h_last": h_last, "d_raw": d_raw.to(dt), "d_x": (m * G).to(dt), "d_bias": d_bias, "d_h0": d_h0}


def _plain_step(s):
    a = s["raw"].float() + s["bias"]
    h = s["h0"]
    h.copy_(torch.sigmoid(a) * h + torch.sigmoid(-a) * s["x"].float())
    return {"y": h.to(s["x"].dtype), "h": h}


def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    N, C, G = c["N"], c["C"], c["G"]
    x = s["x"].detach().float().reshape(N, -1, G, C // G)
    w, b = (s[n].detach().float().reshape(G, C // G) for n in ("w", "b"))
    mu = x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((x - mu).square().mean((1, 3), keepdim=True) + 1e-5)
    xh = (x - mu) * rstd
    z = xh * w + b
    sg = torch.sigmoid(z)
    y = (z * sg).to(dt).reshape(s["x"].shape)
    if "dy" not in s:
        return {"y": y}
    d = s["dy"].float().reshape(x.shape) * (sg * (1 + z * (1 - sg)))
    g = d * w
    dx = rstd * (g - g.mean((1, 3), keepdim=True) - xh * (g * xh).mean((1, 3), keepdim=True))
    dw, db = (d.double() * xh).sum((0, 1)), d.double().sum((0, 1))
    return {"y": y, "d_x": dx.to(dt).reshape(s["x"].shape), "d_w": dw.float().reshape(C), "d_b": db.float().reshape(C)}


def _plain_experts(s):
    c, x = s["case"], s["x"].float()
    N, E, k, F = c["N"], c["E"], c["k"], c["F"]
    logits = s["x"].double() @ s["router"].double().T  # in 64 bits: which experts are taken hangs on it
    top, ids = (v[:, :k] for v in torch.sort(logits, dim=1, descending=True, stable=True))
    p = torch.softmax(top, 1).float()
    if N * k < E:  # fewer choices than experts: take the chosen ones' weights
        u = torch.einsum("nd,nkfd->nkf", x, s["w_in"][ids].float())
        act = torch.sigmoid(u[..., :F]) * u[..., :F] * u[..., F:] * p[..., None]
        out = torch.einsum("nkf,nkdf->nd", act, s["w_out"][ids].float())
    else:  # all experts for all tokens, weighed with zero where they are not taken
        u = torch.matmul(x, s["w_in"].float().mT)
        act = torch.sigmoid(u[..., :F]) * u[..., :F] * u[..., F:]
        full = torch.zeros(N, E, device=x.device).scatter_(1, ids, p)
        out = torch.matmul(act * full.T[..., None], s["w_out"].float().mT).sum(0)
    return {"out": (out + s["shared"].float()).to(s["x"].dtype), "ids": ids.int(), "p": p}


# ------------------------------------------------------------------------------------------ the framework's calls


def _own(s):
    kind = s["case"]["kind"]
    if kind in ("recurrence", "packed", "step"):
        from neuronspark_b200 import gated_recurrence as gr
        if kind == "step":
            return {"y": gr.gated_linear_recurrence_step(s["raw"], s["x"], s["h0"], s["bias"]), "h": s["h0"]}
        y, h_last = gr.gated_linear_recurrence(s["raw"], s["x"], s["h0"], s["bias"], cu_seqlens=s.get("cu"))
        if "dy" not in s:
            return {"y": y, "h_last": h_last}
        d = torch.autograd.grad((y, h_last), [s[n] for n in ("raw", "x", "bias", "h0")], (s["dy"], s["dh"]))
        return {"y": y, "h_last": h_last, **dict(zip(("d_raw", "d_x", "d_bias", "d_h0"), d))}
    if kind == "norm":
        from neuronspark_b200 import group_norm as gn
        y = gn.group_norm_act(s["x"], s["case"]["G"], s["w"], s["b"], eps=1e-5, activation="silu")
        if "dy" not in s:
            return {"y": y}
        return {"y": y, **dict(zip(("d_x", "d_w", "d_b"), torch.autograd.grad(y, [s[n] for n in "xwb"], s["dy"])))}
    from neuronspark_b200 import moe_kernels as mk
    out, ids, p = mk.moe_few_tokens(s["x"], s["router"], s["w_in"], s["w_out"], s["case"]["k"], shared=s["shared"],
                                    return_routing=True)
    return {"out": out, "ids": ids, "p": p}


def run(state):
    if own:
        return _own(state)
    return {"recurrence": _plain_recurrence, "packed": _plain_recurrence, "step": _plain_step, "norm": _plain_norm,
            "experts": _plain_experts}[state["case"]["kind"]](state)


def work(case):
    es, kind, train = 4 if case["dtype"] == "f32" else 2, case["kind"], case.get("train", False)
    if kind in ("recurrence", "packed", "step"):
        n = case["D"] * (case["T"] * case["B"] if kind == "recurrence" else case["rows"] if kind == "packed" else case["B"])
        state = 8 * case["D"] * (case["seqs"] if kind == "packed" else case["B"])
        # forward: two streams in, one out; backward, a call of its own: three in, two out
        return {"bytes": n * es * (8 if train else 3) + state * (2 if train else 1), "flops": n * (30 if train else 10)}
    if kind == "norm":
        n = case["N"] * case["L"] * case["C"]
        return {"bytes": n * es * (5 if train else 2), "flops": n * (35 if train else 12)}
    N, E, k, D, F = (case[n] for n in "NEkDF")
    used = E * (1 - (1 - k / E) ** N)  # experts that some token takes, on average
    return {"bytes": es * (used * 3 * F * D + E * D + 3 * N * D), "flops": N * (k * 6 * F * D + 2 * E * D)}


# ------------------------------------------------------------------------------------------ 64 bits, step by step


def _exact_recurrence(s):
    raw, x, h0, bias = (s[n].detach().double() for n in ("raw", "x", "h0", "bias"))
    T, e = x.shape[0], torch.exp(-(raw + bias))
    f, m = 1 / (1 + e), e / (1 + e)
    cu = s["cu"].tolist() if "cu" in s else [0, T]
    seqs = [(i, a, b) for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])) if b > a]
    state = (lambda t, i: t[i]) if "cu" in s else (lambda t, i: t)
    H, before, h_last = torch.zeros_like(x), torch.zeros_like(x), h0.clone()
    mx = m * x
    for i, a, b in seqs:
        h = state(h0, i)
        for t in range(a, b):
            torch.addcmul(mx[t], f[t], h, out=H[t])
            h = H[t]
        before[a] = state(h0, i)
        before[a + 1:b] = H[a:b - 1]
        state(h_last, i).copy_(h)
    if "dy" not in s:
        return {"y": H, "h_last": h_last}
    dy, G, d_h0 = s["dy"].double(), torch.zeros_like(x), s["dh"].double()
    for i, a, b in seqs:
        carry = state(d_h0, i).clone()
        for t in range(b - 1, a - 1, -1):
            torch.add(dy[t], carry, out=G[t])
            torch.mul(f[t], G[t], out=carry)
        state(d_h0, i).copy_(carry)
    d_raw = G * (before - x) * f * m
    return {"y": H, "h_last": h_last, "d_raw": d_raw, "d_x": m * G, "d_bias": d_raw.reshape(-1, x.shape[-1]).sum(0), "d_h0": d_h0}


def _exact_step(s):
    e = torch.exp(-(s["raw"].double() + s["bias"].double()))
    h = (s["h0"].double() + e * s["x"].double()) / (1 + e)
    return {"y": h, "h": h}


def _exact_norm(s):
    c = s["case"]
    x, w, b = (s[n].detach().double().requires_grad_("dy" in s) for n in "xwb")
    v = x.reshape(c["N"], c["L"], c["G"], -1).transpose(1, 2).flatten(2)  # a sample's group in one row
    v = (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5)
    v = v.reshape(c["N"], c["G"], c["L"], -1).transpose(1, 2).reshape(x.shape) * w + b
    y = v / (1 + torch.exp(-v))
    if "dy" not in s:
        return {"y": y}
    d = torch.autograd.grad(y, (x, w, b), s["dy"].double())
    return {"y": y.detach(), "d_x": d[0], "d_w": d[1], "d_b": d[2]}


def _exact_experts(s):
    c, x = s["case"], s["x"].double()
    logits = (x[:, None] * s["router"].double()).sum(-1).tolist()
    out, probs = s["shared"].double(), []
    for n, row in enumerate(logits):
        taken = sorted(range(c["E"]), key=lambda e: (-row[e], e))[:c["k"]]
        p = [math.exp(row[e] - row[taken[0]]) for e in taken]
        probs.append([v / sum(p) for v in p])
        for e, v in zip(taken, probs[-1]):
            u = s["w_in"][e].double() @ x[n]
            gate, up = u[:c["F"]], u[c["F"]:]
            out[n] += v * (s["w_out"][e].double() @ (gate / (1 + torch.exp(-gate)) * up))
    return {"out": out, "ids": None, "p": torch.tensor(probs, dtype=torch.float64, device=x.device)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"recurrence": _exact_recurrence, "packed": _exact_recurrence, "step": _exact_step, "norm": _exact_norm,
            "experts": _exact_experts}[case["kind"]](s)
