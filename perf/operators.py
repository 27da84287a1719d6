"""Workloads of the linear recurrence and of the matrix orthogonalisation, each in a plain form
(elementary tensor operations) and through the library's own entry points.

  scan   u = sigmoid(-f), p_t = h_{t-1} (zero where a new document starts), h_t = p_t + u_t (c_t - p_t),
         y_t = h_t silu(z_t); the training cases take all gradients as well
  orth   five Newton-Schulz steps X <- a X + (b A + c A A) X, A = X X^T, from X = G / (|G| + eps)
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    scan = lambda name, T, B, d, dtype, train=False, packed=True, document=0: {  # noqa: E731
        "name": name, "op": "scan", "T": T, "B": B, "d": d, "dtype": dtype, "train": train, "packed": packed,
        "document": document}
    orth = lambda name, count, m, n, dtype, kind="noise": {  # noqa: E731
        "name": name, "op": "orth", "count": count, "m": m, "n": n, "dtype": dtype, "kind": kind}
    return [
        scan("token_one_stream", 1, 1, 1280, "bf16"),                 # interactive generation: latency
        scan("token_many_streams", 1, 128, 2048, "bf16"),             # a serving batch, one token each
        scan("prompt_odd_fp32", 777, 5, 1001, "fp32", packed=False, document=200),   # odd width, packed texts
        scan("prompt_large", 4096, 64, 1536, "bf16"),                 # reading long prompts
        scan("train_layer", 512, 32, 1280, "bf16", train=True),       # one layer of the byte-level model's step
        scan("train_documents_fp32", 2048, 8, 512, "fp32", train=True, document=300),
        scan("train_long", 65536, 1, 1280, "bf16", train=True, document=20000),      # one very long sequence
        orth("one_small", 1, 256, 256, "bf16"),                       # smallest update: latency
        orth("model_square", 18, 1280, 1280, "bf16", kind="lowrank"),  # W_x, W_h, out_proj of six layers
        orth("model_in_proj", 6, 2560, 1280, "bf16"),                 # the tall input projections of six layers
        orth("lowrank_factors", 12, 270, 1536, "bf16", kind="lowrank"),  # U, V of low-rank layers: wide and ragged
        orth("odd_fp32", 4, 1000, 257, "fp32"),                       # fp32 training, ragged both ways
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if rng.random() < 0.6:
        T = 1 if rng.random() < 0.2 else _log(rng, 2, 65536)
        train = T > 1 and rng.random() < 0.6
        most = (1 << 25 if dtype == "fp32" else 1 << 26) if train else 1 << 27
        d = _log(rng, 16, 4096)
        B = _log(rng, 1, max(1, min(256, most // (T * d))))
        T = max(1, min(T, most // (B * d)))
        return {"op": "scan", "T": T, "B": B, "d": d, "dtype": dtype, "train": train, "packed": rng.random() < 0.5,
                "document": rng.choice([0, 0, _log(rng, 1, max(2, T))])}
    m, n = _log(rng, 16, 2560), _log(rng, 16, 2560)
    count = max(1, min(_log(rng, 1, 24), (18 * 1280 ** 3) // max(1, min(m, n) ** 2 * max(m, n))))
    return {"op": "orth", "count": count, "m": m, "n": n, "dtype": dtype, "kind": rng.choice(["noise", "lowrank"])}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "orth":
        count, m, n = case["count"], case["m"], case["n"]
        G = randn(count, m, n)
        if case["kind"] == "lowrank":     # a few strong directions above noise, as gradients of trained layers have
            G = 0.01 * G + 0.1 * randn(count, m, 16) @ randn(count, 16, n)
        return {"op": "orth", "G": (1e-3 * G).to(dtype)}
    T, B, d = case["T"], case["B"], case["d"]
    x = torch.empty(T, B, 3 * d, device="cuda", dtype=dtype) if case["packed"] else None
    parts = x.chunk(3, dim=-1) if case["packed"] else [torch.empty(T, B, d, device="cuda", dtype=dtype) for _ in range(3)]
    for i, p in enumerate(parts):
        p.normal_(generator=g)
        if i == 0:   # forget gates: every channel with a memory of its own, from two steps to some hundred
            p.add_((5 * torch.rand(d, generator=g, device="cuda")).to(dtype))
    s = {"op": "scan", "f": parts[0], "c": parts[1], "z": parts[2], "h0": 0.3 * randn(B, d), "train": case["train"],
         "reset": None}
    if case["document"]:
        s["reset"] = torch.rand(T, B, generator=g, device="cuda") < 1.0 / case["document"]
    if case["train"]:
        s["dy"] = torch.empty(T, B, d, device="cuda", dtype=dtype).normal_(generator=g)
        s["dh"] = randn(B, d)
    return s


# ------------------------------------------------------------------ plain forms

def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t over the first axis by doubling (a and x are overwritten)."""
    k = 1
    while k < a.shape[0]:
        x[k:] = x[k:] + a[k:] * x[:-k]
        a[k:] = a[k:] * a[:-k]
        k *= 2
    return x


def _plain_scan(s):
    f, c, z, h0, reset = s["f"].float(), s["c"].float(), s["z"].float(), s["h0"], s["reset"]
    u, sz = torch.sigmoid(-f), torch.sigmoid(z)
    a = torch.sigmoid(f)
    keep = a if reset is None else a.masked_fill(reset.unsqueeze(-1), 0.0)     # a_t, 0 where h_{t-1} is dropped
    x = u * c
    x[0] += keep[0] * h0
    h = _scan(keep.clone(), x)
    out = s["f"].dtype
    y = h * z * sz
    if not s["train"]:
        return [y.to(out), h[-1].clone()]
    dy = s["dy"].float()
    x = dy * z * sz
    x[-1] += s["dh"]
    after = torch.cat([keep[1:], torch.zeros_like(keep[:1])])
    gh = _scan(after.flip(0), x.flip(0)).flip(0)
    p = torch.cat([h0.unsqueeze(0), h[:-1]])
    if reset is not None:
        p = p.masked_fill(reset.unsqueeze(-1), 0.0)
    df = gh * (p - c) * u * a
    dz = dy * h * sz * (1.0 + z * (1.0 - sz))
    return [y.to(out), h[-1].clone(), df.to(out), (gh * u).to(out), dz.to(out), keep[0] * gh[0]]


def _plain_orth(G):
    a, b, c = COEFFICIENTS
    norm = G.double().square().sum(dim=(-2, -1), keepdim=True).sqrt()
    X = (G.double() / (norm + EPS)).float()
    tall = X.shape[-2] > X.shape[-1]
    if tall:
        X = X.transpose(-2, -1)
    left = STEPS
    while left:
        A = X @ X.transpose(-2, -1)
        X = a * X + (b * A + c * (A @ A)) @ X
        left -= 1
    return (X.transpose(-2, -1) if tall else X).to(G.dtype)


# ------------------------------------------------------------------ one pass

def run(s):
    if own:
        from elman_b200 import hasty_pytorch_lib as lib
        if s["op"] == "orth":
            return [lib.newton_schulz(s["G"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)]
        y, h, saved = lib.gated_linear_forward(s["train"], s["f"], s["c"], s["z"], s["h0"], s["reset"])
        if not s["train"]:
            return [y, h]
        df, dc, dz, dh0 = lib.gated_linear_backward(s["f"], s["c"], s["z"], saved, s["dy"], s["dh"], s["reset"])
        return [y, h, df, dc, dz, dh0]
    return [_plain_orth(s["G"])] if s["op"] == "orth" else _plain_scan(s)


def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "orth":
        # the Gram matrix and its square are symmetric: half of their products are the other half's
        r, q = sorted((case["m"], case["n"]))
        return {"bytes": 2 * size * case["count"] * r * q, "flops": STEPS * case["count"] * (3 * r * r * q + r ** 3)}
    n, rows, chan = case["T"] * case["B"] * case["d"], case["T"] * case["B"], case["B"] * case["d"]
    marks = rows if case["document"] else 0
    # training is two operators with the rest of the model between them: f, c, z are read by each
    values, states = (11, 4) if case["train"] else (4, 2)
    return {"bytes": values * size * n + 4 * states * chan + marks * (2 if case["train"] else 1),
            "flops": (30 if case["train"] else 10) * n}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    if case["op"] == "scan" and case["T"] * case["B"] * case["d"] > (1 << 27):
        return None
    s = prepare(case, seed)
    if case["op"] == "orth":
        a, b, c = COEFFICIENTS
        X = s["G"].double()
        X = X / (torch.linalg.matrix_norm(X, keepdim=True) + EPS)
        for _ in range(STEPS):
            if case["m"] <= case["n"]:
                A = X @ X.mT
                X = a * X + b * (A @ X) + c * (A @ (A @ X))
            else:
                A = X.mT @ X
                X = a * X + b * (X @ A) + c * ((X @ A) @ A)
        return [X]
    T, train, reset = case["T"], case["train"], s["reset"]
    f, c, z = (s[k].double() for k in "fcz")
    u = 1.0 / (1.0 + torch.exp(f))
    h, prev = torch.empty_like(f), torch.empty_like(f) if train else None
    p = s["h0"].double()
    for t in range(T):
        if reset is not None:
            p = torch.where(reset[t].unsqueeze(-1), 0.0, p)
        if train:
            prev[t] = p
        p = torch.lerp(p, c[t], u[t])
        h[t] = p
    e = torch.exp(-z)
    y = h * z / (1.0 + e)
    if not train:
        return [y, h[-1].clone()]
    dy = s["dy"].double()
    dz = dy * h * (1.0 + e + z * e) / (1.0 + e) ** 2
    last = h[-1].clone()
    del h
    gh, q = s["dh"].double(), dy * z / (1.0 + e)
    G = torch.empty_like(f)
    for t in reversed(range(T)):
        gh = gh + q[t]
        G[t] = gh
        gh = gh * (1.0 - u[t])
        if reset is not None:
            gh = torch.where(reset[t].unsqueeze(-1), 0.0, gh)
    return [y, last, G * (prev - c) * u * (1.0 - u), G * u, dz, gh]
