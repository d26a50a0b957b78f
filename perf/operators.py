"""Cases that measure the language-model training operators: the scaled
embedding lookup with its gradient, the gated linear recurrence (scan, its
backward, its one-token step) and the Newton-Schulz orthogonalisation of
weight updates.

``run`` computes a case in its plain form (elementary torch operations in 32
bits, rounded once at the end) or, where ``own`` is true, by the package's
kernels; ``exact`` computes it in 64 bits from the definition.

    embedding    y[n] = s W[id_n];  dW[v] = s sum over {n : id_n = v} of dy[n]
    recurrence   h_t = e^{g_t} h_{t-1} + x_t per channel (g = -inf starts a
                 new packed sequence)
    orthogonal   X_0 = G / (|G|_F + eps); X <- a X + (b A + c A A) X with
                 A = X X^T, five steps, on the smaller side of G
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
_EPS = 1e-7
_STEPS = 5


def listed():
    return [
        # One decode step of 64 sequences: the lookup alone, all latency.
        dict(name="embed decode 64", op="embed", train=False, N=64, V=32000, D=1024,
             dtype="bf16", scale=32.0, pad=-1),
        # Prefill of eight prompts of 8192 tokens.
        dict(name="embed prefill 64k", op="embed", train=False, N=65536, V=32000, D=1024,
             dtype="bf16", scale=32.0, pad=-1),
        # A ragged fp32 batch (padded tokens, odd width and vocabulary) of a small model's
        # training step: lookup and gradient.
        dict(name="embed train ragged", op="embed", train=True, N=9973, V=50257, D=321,
             dtype="f32", scale=17.9, pad=0),
        # A full training batch, 32 sequences of 4096 tokens: lookup and gradient.
        dict(name="embed train 128k", op="embed", train=True, N=131072, V=32000, D=1024,
             dtype="bf16", scale=32.0, pad=-1),
        # One decode token of 64 sequences through the recurrence.
        dict(name="scan step 64", op="step", B=64, D=1024, dtype="bf16", gdtype="f32"),
        # One long prompt.
        dict(name="scan prefill 64k", op="scan", train=False, B=1, T=65536, D=1024, dtype="bf16",
             gdtype="f32", init=False, packed=False),
        # An fp32 model on packed sequences of different lengths, odd sizes, forward and backward.
        dict(name="scan train packed", op="scan", train=True, B=3, T=1531, D=777, dtype="f32",
             gdtype="f32", init=True, packed=True),
        # A training batch, 8 sequences of 8192 tokens, forward and backward.
        dict(name="scan train 64k", op="scan", train=True, B=8, T=8192, D=1024, dtype="bf16",
             gdtype="f32", init=True, packed=False),
        # Updates of one promotion projection, [levels - 1, heads, 128, 128] of three levels and
        # eight heads.
        dict(name="orth 16x128x128", op="orth", batch=16, rows=128, cols=128, dtype="f32",
             out="bf16"),
        # An odd rectangular weight on its own, taller than wide.
        dict(name="orth 1001x345", op="orth", batch=1, rows=1001, cols=345, dtype="f32",
             out="bf16"),
        # One channel-mixer weight.
        dict(name="orth 1024x2816", op="orth", batch=1, rows=1024, cols=2816, dtype="bf16",
             out="bf16"),
        # The down projections of twelve layers, fp32 momenta.
        dict(name="orth 12x1024x2816", op="orth", batch=12, rows=1024, cols=2816, dtype="f32",
             out="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["embed", "embed", "scan", "scan", "scan", "step", "orth", "orth", "orth"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "embed":
        train = rng.random() < 0.6
        D, V = _log(rng, 24, 2048), _log(rng, 500, 64000)
        V = min(V, 32000 * 1024 // D)
        N = min(_log(rng, 1, 131072), 65536 * 1024 // D)
        return dict(op=op, train=train, N=N, V=V, D=D, dtype=dtype,
                    scale=round(math.sqrt(D), 3), pad=rng.choice([-1, 0, V // 2]))
    if op == "step":
        return dict(op=op, B=_log(rng, 1, 1024), D=_log(rng, 16, 4096), dtype=dtype,
                    gdtype=rng.choice(["f32", "f32", dtype]))
    if op == "scan":
        B, T, D = _log(rng, 1, 32), _log(rng, 1, 65536), _log(rng, 16, 2048)
        T = max(1, min(T, (1 << 26) // (B * D)))
        return dict(op=op, train=rng.random() < 0.6, B=B, T=T, D=D, dtype=dtype,
                    gdtype=rng.choice(["f32", "f32", dtype]), init=rng.random() < 0.5,
                    packed=rng.random() < 0.5)
    rows, cols, batch = _log(rng, 8, 4096), _log(rng, 8, 4096), _log(rng, 1, 64)
    small, large = min(rows, cols), max(rows, cols)
    batch = max(1, min(batch, (12 * 1024 * 1024 * 2816) // (small * small * large)))
    if small * small * large > 12 * 1024 * 1024 * 2816:
        rows, cols = rows // 2, cols // 2
    return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=dtype,
                out=rng.choice(["bf16", "bf16", "f16"]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda", dtype=torch.float32)

    s = dict(case)
    if case["op"] == "embed":
        N, V, D, dt = case["N"], case["V"], case["D"], _DTYPES[case["dtype"]]
        # Token frequencies fall as 1 / rank, as natural text's do.
        ids = torch.exp(uniform(N).double() * math.log(V + 1)).long() - 1
        ids = ids.clamp_(0, V - 1)
        if case["pad"] >= 0:
            ids[uniform(N) < 0.1] = case["pad"]
        s["ids"] = ids
        s["weight"] = (normal(V, D) * 0.02).to(dt)
        s["d_out"] = normal(N, D).to(dt) if case["train"] else None
        return s
    if case["op"] in ("scan", "step"):
        dt, gdt = _DTYPES[case["dtype"]], _DTYPES[case["gdtype"]]
        B, T, D = case["B"], case.get("T", 1), case["D"]
        x = normal(B, T, D).to(dt)
        # Log-decays of gates with horizons from a few tokens to hundreds, channel by channel.
        g = torch.nn.functional.logsigmoid(normal(B, T, D) + 5.0 * uniform(D))
        if case.get("packed"):
            g[:, uniform(T) < 1.0 / 200] = -math.inf  # a new sequence starts here
        g = g.to(gdt)
        state = normal(B, D)
        if case["op"] == "step":
            s.update(x=x[:, 0].contiguous(), g=g[:, 0].contiguous(), state=state)
            return s
        s.update(x=x, g=g, state=state if case["init"] else None)
        if case["train"]:
            s.update(d_h=normal(B, T, D).to(dt), d_final=normal(B, D))
        return s
    b, m, n = case["batch"], case["rows"], case["cols"]
    # Momenta of gradients: a few strong directions over a full-rank remainder.
    r = max(1, min(8, m, n))
    u = normal(b, m, r) * torch.logspace(0, -1, r, device="cuda")
    s["update"] = ((u @ normal(b, r, n)) / math.sqrt(r) + 0.1 * normal(b, m, n)).to(
        _DTYPES[case["dtype"]])
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _scan_plain(a, x):
    """h_t = a_t h_{t-1} + x_t along dimension 1 from a zero state: pairs of
    steps joined, the half-length recurrence, then the steps in between."""
    T = x.shape[1]
    if T == 1:
        return x
    if T % 2:
        h = _scan_plain(a[:, :-1], x[:, :-1])
        return torch.cat([h, a[:, -1:] * h[:, -1:] + x[:, -1:]], 1)
    a0, a1, x0, x1 = a[:, 0::2], a[:, 1::2], x[:, 0::2], x[:, 1::2]
    h1 = _scan_plain(a0 * a1, a1 * x0 + x1)
    h0 = torch.cat([x0[:, :1], a0[:, 1:] * h1[:, :-1] + x0[:, 1:]], 1)
    return torch.stack([h0, h1], 2).flatten(1, 2)


def _newton_schulz_plain(X, steps):
    if steps == 0:
        return X
    a, b, c = _COEFFICIENTS
    A = X @ X.transpose(-1, -2)
    return _newton_schulz_plain(a * X + (b * A + c * (A @ A)) @ X, steps - 1)


def _run_plain(s):
    if s["op"] == "embed":
        w, ids = s["weight"], s["ids"]
        y = (w[ids].float() * s["scale"]).to(w.dtype)
        if not s["train"]:
            return y
        d = s["d_out"].float()
        if s["pad"] >= 0:
            d = torch.where((ids == s["pad"])[:, None], torch.zeros_like(d), d)
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, ids, d)
        return {"y": y, "dweight": (dw * s["scale"]).to(w.dtype)}
    if s["op"] == "step":
        h = torch.exp(s["g"].float()) * s["state"] + s["x"].float()
        return {"h": h.to(s["x"].dtype), "state": h}
    if s["op"] == "scan":
        x, a = s["x"].float(), torch.exp(s["g"].float())
        if s["state"] is not None:
            x = torch.cat([x[:, :1] + a[:, :1] * s["state"][:, None], x[:, 1:]], 1)
        h = _scan_plain(a, x)
        out = {"h": h.to(s["x"].dtype), "state": h[:, -1].contiguous()}
        if not s["train"]:
            return out
        d = s["d_h"].float()
        d = torch.cat([d[:, :-1], d[:, -1:] + s["d_final"][:, None]], 1)
        later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        u = _scan_plain(later.flip(1), d.flip(1)).flip(1)
        start = torch.zeros_like(h[:, 0]) if s["state"] is None else s["state"]
        dg = u * a * torch.cat([start[:, None], h[:, :-1]], 1)
        out.update(dx=u.to(s["x"].dtype), dg=dg.to(s["g"].dtype))
        if s["state"] is not None:
            out["dstate"] = a[:, 0] * u[:, 0]
        return out
    X = s["update"].float()
    tall = X.shape[-2] > X.shape[-1]
    X = X.transpose(-1, -2) if tall else X
    X = X / (X.square().sum((-1, -2), keepdim=True).sqrt() + _EPS)
    X = _newton_schulz_plain(X, _STEPS)
    return (X.transpose(-1, -2) if tall else X).to(_DTYPES[s["out"]]).contiguous()


# ---------------------------------------------------------------------------
# The package's operators
# ---------------------------------------------------------------------------


def _run_own(s):
    import nested_recurrent_memory_b200 as nrm

    if s["op"] == "embed":
        pad = s["pad"] if s["pad"] >= 0 else None
        y = nrm.embed_tokens(s["ids"], s["weight"], scale=s["scale"], padding_idx=pad)
        if not s["train"]:
            return y
        return {"y": y, "dweight": nrm.embed_tokens_bwd(s["ids"], s["d_out"], s["V"],
                                                        scale=s["scale"], padding_idx=pad)}
    if s["op"] == "step":
        h, state = nrm.step_gated_scan(s["x"], s["g"], s["state"])
        return {"h": h, "state": state}
    if s["op"] == "scan":
        if not s["train"]:
            h, state = nrm.gated_scan_fwd(s["x"], s["g"], initial_state=s["state"],
                                          output_final_state=True)
            return {"h": h, "state": state}
        h, state, aux = nrm.gated_scan_fwd(s["x"], s["g"], initial_state=s["state"],
                                           output_final_state=True, return_aux=True)
        dx, dg, dinit = nrm.gated_scan_bwd(s["x"], s["g"], s["d_h"], d_final=s["d_final"],
                                           initial_state=s["state"], aux=aux)
        out = {"h": h, "state": state, "dx": dx, "dg": dg}
        if dinit is not None:
            out["dstate"] = dinit
        return out
    return nrm.orthogonalize(s["update"], steps=_STEPS, coefficients=_COEFFICIENTS, eps=_EPS,
                             dtype=_DTYPES[s["out"]])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "embed":
        N, V, D = case["N"], case["V"], case["D"]
        # Distinct rows that N tokens of these frequencies touch, as expected.
        v = np.arange(V, dtype=np.float64)
        p = np.log((v + 2.0) / (v + 1.0)) / math.log(V + 1)
        rows = float(np.sum(-np.expm1(N * np.log1p(-np.minimum(p, 1 - 1e-12)))))
        nbytes = rows * D * e + N * 8 + N * D * e
        flops = N * D
        if case["train"]:
            nbytes += N * D * e + V * D * e + N * 8
            flops += N * D
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "step":
        n = case["B"] * case["D"]
        return {"bytes": n * (2 * e + _BYTES[case["gdtype"]] + 8), "flops": 3 * n}
    if case["op"] == "scan":
        n, eg = case["B"] * case["T"] * case["D"], _BYTES[case["gdtype"]]
        edge = case["B"] * case["D"] * 4
        nbytes, flops = n * (2 * e + eg) + edge * (2 if case["init"] else 1), 3 * n
        if case["train"]:
            nbytes += n * (3 * e + 2 * eg) + edge * (3 if case["init"] else 1)
            flops += 7 * n
        return {"bytes": nbytes, "flops": flops}
    b, m, n = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # A and A A are symmetric: half of each product is enough.
    flops = b * _STEPS * (m * m * n + m * m * m + 2.0 * m * m * n)
    return {"bytes": b * m * n * (e + _BYTES[case["out"]]), "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "embed":
        ids, w = s["ids"], s["weight"].double()
        y = w.index_select(0, ids).mul_(s["scale"])
        if not s["train"]:
            return y
        d = s["d_out"].double()
        if s["pad"] >= 0:
            d[ids == s["pad"]] = 0.0
        # Sorted by token: the gradient is the difference of running sums at the rows' ends.
        # The order of the sum within a row does not matter in 64 bits.
        dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        dw.index_put_((ids,), d, accumulate=True)
        return {"y": y, "dweight": dw.mul_(s["scale"])}
    if s["op"] == "step":
        h = s["state"].double() * s["g"].double().exp() + s["x"].double()
        return {"h": h, "state": h}
    if s["op"] == "scan":
        # Token by token, as the definition has it.
        x, a = s["x"].double(), s["g"].double().exp()
        T = x.shape[1]
        h = torch.empty_like(x)
        prev = torch.zeros_like(x[:, 0]) if s["state"] is None else s["state"].double()
        start = prev
        for t in range(T):
            prev = torch.addcmul(x[:, t], a[:, t], prev)
            h[:, t] = prev
        out = {"h": h, "state": h[:, -1].contiguous()}
        if not s["train"]:
            return out
        d, dx, dg = s["d_h"].double(), torch.empty_like(x), torch.empty_like(x)
        carry = s["d_final"].double()
        for t in range(T - 1, -1, -1):
            u = d[:, t] + carry
            dx[:, t] = u
            carry = a[:, t] * u
            dg[:, t] = carry * (h[:, t - 1] if t else start)
        out.update(dx=dx, dg=dg)
        if s["state"] is not None:
            out["dstate"] = carry
        return out
    # The iteration is a polynomial of the singular values: X = U p(sigma) V^T = U f(lambda) U^T G
    # with lambda, U the eigenvalues and vectors of G G^T.
    G = s["update"].double()
    tall = G.shape[-2] > G.shape[-1]
    G = G.transpose(-1, -2) if tall else G
    G = G / (torch.linalg.matrix_norm(G, keepdim=True) + _EPS)
    lam, U = torch.linalg.eigh(G @ G.transpose(-1, -2))
    a, b, c = _COEFFICIENTS
    f = torch.ones_like(lam)
    for _ in range(_STEPS):
        q = a + b * lam + c * lam * lam
        f, lam = f * q, lam * q * q
    X = (U * f[..., None, :]) @ (U.transpose(-1, -2) @ G)
    return X.transpose(-1, -2).contiguous() if tall else X
