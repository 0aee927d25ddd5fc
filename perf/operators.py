"""Measured cases of two operators of the generation path: the 8-bit integer matrix product with a scale per row and per
channel (`dvq_hip.ops.linear_int8`, `linear_int8_batched`) and the verification of drafted codes against the prior's
distribution (`dvq_hip.ops.prior_verify`).

`run` computes them in elementary torch operations, or through the framework's entry points where `own` is true; `exact`
says in 64 bits what the outputs are.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "d-vqvae_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from dvq_hip import ops
    return ops


def listed():
    return [
        # one grasp through the decoder's first layer: the weights' bytes and the launch are all there is
        dict(name="linear one row", op="linear", M=1, K=2560, N=1024, type="fp32", relu=True),
        # a small serving batch through the position decoder's first layer
        dict(name="linear 16 rows bf16", op="linear", M=16, K=2048, N=1024, type="bf16", relu=True),
        # odd and ragged everywhere: no dimension is a multiple of a tile or of a load
        dict(name="linear odd", op="linear", M=333, K=1037, N=501, type="fp32", relu=False),
        # the timed generation batch through the decoder's first layer
        dict(name="linear 4096 rows", op="linear", M=4096, K=2560, N=1024, type="fp32", relu=True),
        # rows quantised once and read by several layers: the product alone, at a generic large size
        dict(name="product 8192 rows bf16", op="product", M=8192, K=4096, N=4096, type="bf16", relu=False),
        # the six part heads of the hand encoder, first layer, one launch for all
        dict(name="six heads", op="batched", M=512, K=1024, N=512, type="fp32", relu=True, heads=6),
        # one grid of the prior, drafted cell by cell, no cell behind the last one
        dict(name="verify one grid", op="verify", B=1, G=9, P=9, V=512, type="fp32", draft="probs", layout="cells", sigma=0.3,
             ragged=False, masked=0.0),
        # the timed batch: the prior's forward hands its logits over as [B, V, cells]
        dict(name="verify 4096 grids", op="verify", B=4096, G=9, P=9, V=512, type="fp32", draft="probs", layout="cells", sigma=0.3,
             ragged=False, masked=0.0),
        # rows that drafted different numbers of codes, from the largest codebook of the search benchmark, unused codes masked
        dict(name="verify ragged bf16", op="verify", B=1000, G=5, P=6, V=8192, type="bf16", draft="logits", layout="rows", sigma=0.5,
             ragged=True, masked=0.1),
        # few rows over the longest codebook the search takes: the codes of one position are the long axis
        dict(name="verify few long rows", op="verify", B=8, G=4, P=5, V=65536, type="fp32", draft="logits", layout="rows", sigma=0.5,
             ragged=False, masked=0.0),
        # a full serving batch over a large odd codebook
        dict(name="verify many long rows", op="verify", B=1024, G=4, P=5, V=16381, type="bf16", draft="logits", layout="rows",
             sigma=0.5, ragged=False, masked=0.0),
    ]


def _between(rng, low, high):
    """A whole number whose logarithm is spread evenly."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["linear", "product", "batched", "verify", "verify", "verify"])
    if kind == "verify":
        V = _between(rng, 2, 65536)
        G = rng.randint(1, 12)
        B = _between(rng, 1, max(1, min(4096, (512 * 4 * 16381) // (G * V))))
        layout = rng.choice(["rows", "cells"])
        return dict(op="verify", B=B, G=G, P=G + rng.randint(0, 1), V=V, type=rng.choice(["fp32", "bf16"]),
                    draft=rng.choice(["logits", "probs"]), layout=layout, sigma=round(rng.uniform(0.05, 1.0), 3),
                    ragged=rng.random() < 0.5, masked=round(rng.uniform(0.0, 0.5), 3) if V >= 16 and rng.random() < 0.5 else 0.0)
    M, K, N = _between(rng, 1, 4096), _between(rng, 16, 4096), _between(rng, 1, 4096)
    if rng.random() < 0.5:
        K = max(16, K // 16 * 16)
    case = dict(op=kind, M=M, K=K, N=N, type=rng.choice(["fp32", "bf16"]), relu=rng.random() < 0.5)
    if kind == "batched":
        case["heads"] = rng.randint(2, 8)
        case["M"], case["N"] = max(1, M // case["heads"]), max(1, N // 2)
    return case


# ------------------------------------------------------------------------------------------------------------- inputs
def _weights(g, N, K):
    """A layer as a quantised checkpoint holds it: int8 codes, one fp32 scale per output channel, an fp32 bias."""
    W = torch.randn(N, K, generator=g, device=DEV) / math.sqrt(K)
    a = W.abs().amax(1)
    codes = torch.round(W.double() * 127.0 / a.double()[:, None]).to(torch.int8)
    return codes, (a.double() / 127.0).float(), 0.1 * torch.randn(N, generator=g, device=DEV)


def _features(g, M, K, type_):
    """Activations behind a ReLU and un-quantised features mixed: row norms vary over two orders of magnitude."""
    x = torch.randn(M, K, generator=g, device=DEV)
    x = torch.where(torch.rand(M, 1, generator=g, device=DEV) < 0.5, x.clamp_min(0.0), x)
    return (x * torch.exp(1.5 * torch.randn(M, 1, generator=g, device=DEV))).to(TYPES[type_])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] != "verify":
        n = case.get("heads", 1)
        layers = [_weights(g, case["N"], case["K"]) for _ in range(n)]
        xs = [_features(g, case["M"], case["K"], case["type"]) for _ in range(n)]
        if case["op"] == "product":         # the rows come quantised already
            c, s = _quantized(xs[0])
            xs = [(c.to(torch.int8), s)]
        return dict(case=case, xs=xs, layers=layers)
    B, G, P, V, dt = case["B"], case["G"], case["P"], case["V"], TYPES[case["type"]]
    t = 2.0 * torch.randn(B, P, V, generator=g, device=DEV)
    if case["masked"]:                      # codes ruled out for everyone; code 0 stays
        out = torch.rand(V, generator=g, device=DEV) < case["masked"]
        out[0] = False
        t.masked_fill_(out, -math.inf)
    t = t.to(dt)
    d = t[:, :G].float() + case["sigma"] * torch.randn(B, G, V, generator=g, device=DEV)
    d = d.to(dt)
    gumbel = -torch.log(-torch.log(torch.rand(B, G, V, generator=g, device=DEV).clamp_(1e-7, 1.0 - 1e-7)))
    tokens = (d.float() + gumbel).argmax(2)
    del gumbel
    if case["draft"] == "probs":            # a drafting prior's generate() returns probabilities in fp32
        d = torch.softmax(d.float(), 2)
    if case["layout"] == "cells":           # the prior's forward returns [B, V, cells]
        t = t.transpose(1, 2).contiguous().transpose(1, 2)
    lengths = torch.randint(0, G + 1, (B,), generator=g, device=DEV) if case["ragged"] else None
    u = torch.rand(B, G, generator=g, device=DEV, dtype=torch.float64)
    r = torch.rand(B, generator=g, device=DEV, dtype=torch.float64)
    return dict(case=case, logits=t, draft=d, tokens=tokens, u=u, r=r, lengths=lengths)


# -------------------------------------------------------------------------------------------------------- plain forms
def _quantized(x):
    """Codes (whole numbers, as float64) and scales of the rows of x.  The quotient 127 x / max|x| next to a half decides
    a code, so it is taken in 64 bits."""
    a = x.abs().amax(1).double()
    q = x.double() * 127.0 / torch.where(a > 0, a, torch.ones_like(a))[:, None]
    return torch.round(q), (a / 127.0).float()


def _product(codes, s, layer, relu, dtype):
    w, t, b = layer
    acc = codes.double() @ w.double().T     # beyond 2^24 a sum of 8-bit products does not fit 32-bit floats
    y = acc.float() * s[:, None] * t + b
    return (y.clamp_min(0.0) if relu else y).to(dtype)


def _mass(logits):
    """softmax in 64 bits: a draw next to the border of two codes is decided by the last bits."""
    z = logits.double()
    e = torch.exp(z - z.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _verify(st):
    c, x, r = st["case"], st["tokens"], st["r"]
    B, G, P = c["B"], c["G"], c["P"]
    p = _mass(st["logits"])
    q = st["draft"].double() if c["draft"] == "probs" else _mass(st["draft"])
    px = p[:, :G].gather(2, x[..., None])[..., 0]
    qx = q.gather(2, x[..., None])[..., 0]
    n = st["lengths"] if st["lengths"] is not None else torch.full((B,), G, device=x.device)
    ok = (st["u"] * qx < px) & (torch.arange(G, device=x.device) < n[:, None])
    accepted = ok.long().cumprod(1).sum(1)
    rows = torch.arange(B, device=x.device)
    pa = p[rows, accepted.clamp_max(P - 1)]
    left = (pa - q[rows, accepted.clamp_max(G - 1)]).clamp_min(0.0)
    bonus = accepted >= n
    left = torch.where((bonus | (left.sum(1) <= 2.0 ** -40))[:, None], pa, left)
    cdf = left.cumsum(1)
    at = (cdf <= r[:, None] * cdf[:, -1:]).sum(1)
    last = (left > 0).long().mul(torch.arange(1, c["V"] + 1, device=x.device)).amax(1) - 1
    return accepted, torch.where(bonus & (n >= P), torch.full_like(at, -1), torch.minimum(at, last))


def run(state):
    c = state["case"]
    if c["op"] == "verify":
        if own:
            return _ops().prior_verify(state["logits"], state["draft"], state["tokens"], state["u"], state["r"],
                                       lengths=state["lengths"], draft_probs=c["draft"] == "probs")
        return _verify(state)
    dt = TYPES[c["type"]]
    if own:
        ops = _ops()
        if c["op"] == "batched":
            ws, ts, bs = zip(*state["layers"])
            return ops.linear_int8_batched(state["xs"], ws, ts, bs, relu=c["relu"], out_dtype=dt)
        w, t, b = state["layers"][0]
        return ops.linear_int8(state["xs"][0], w, t, b, relu=c["relu"], out_dtype=dt)
    ys = []
    for x, layer in zip(state["xs"], state["layers"]):
        codes, s = x if c["op"] == "product" else _quantized(x)
        ys.append(_product(codes, s, layer, c["relu"], dt))
    return ys if c["op"] == "batched" else ys[0]


# --------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] != "verify":
        M, K, N, n = case["M"], case["K"], case["N"], case.get("heads", 1)
        x = M * K + 4 * M if case["op"] == "product" else M * K * size
        return {"bytes": n * (x + N * K + 8 * N + M * N * size), "flops": n * 2 * M * N * K}
    B, G, P, V = case["B"], case["G"], case["P"], case["V"]
    # A position is needed only if every draft before it was accepted.  The drafts' logits are the target's plus normal
    # noise of deviation sigma: a draft is accepted with probability erfc(sigma / sqrt 8).
    a = math.erfc(case["sigma"] / math.sqrt(8.0))
    tests = [sum(a ** g for g in range(n)) for n in (range(G + 1) if case["ragged"] else [G])]
    ends = [a ** n if n < P else 0.0 for n in (range(G + 1) if case["ragged"] else [G])]
    tests, ends = sum(tests) / len(tests), sum(ends) / len(ends)
    dsize = 4 if case["draft"] == "probs" else size
    read = tests * V * (size + dsize) + ends * V * size + tests * 16 + 8
    return {"bytes": int(B * (read + 16)), "flops": int(B * V * (tests * 2 + ends) * 4)}


# ---------------------------------------------------------------------------------------------------- in 64 bits alone
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "verify":
        return None                         # whole numbers: compared as they are
    out = []
    for x, (w, t, b) in zip(st["xs"], st["layers"]):
        if case["op"] == "product":
            codes, s = x[0].double(), x[1].double()
        else:
            v = x.double()
            top = v.abs().max(dim=1, keepdim=True).values
            s = (top / 127.0)[:, 0]
            # 127 x and the quotient's neighbour halves are exact in 64 bits: nearest whole number, ties to even
            f = torch.nan_to_num(127.0 * v / top)
            low = torch.floor(f)
            up = (f - low > 0.5) | ((f - low == 0.5) & (torch.remainder(low, 2.0) == 1.0))
            codes = low + up.double()
        y = torch.matmul(codes, w.double().t()) * torch.outer(s, t.double()) + b.double()
        out.append(torch.relu(y) if case["relu"] else y)
    return out if case["op"] == "batched" else out[0]
