"""64-bit CPU restatements of the 8-bit integer product and of the verification of drafted codes (test infrastructure)."""
import numpy as np
import torch


def int8_codes(x):
    """(codes int64 [M,K], scale float32 [M]) of x [M,K]: the exact quotient 127 x / max|x| to the nearest whole number,
    ties to even.  Numerator and comparison are exact in 64 bits: 127 x needs 31 bits, (2 q + 1) a at most 33."""
    v = x.detach().cpu().to(torch.float32).numpy().astype(np.float64)
    M, K = v.shape
    a = np.abs(v).max(axis=1)
    fine = np.isfinite(a)
    codes = np.zeros((M, K), dtype=np.int64)
    for m in range(M):
        if not fine[m] or a[m] == 0:
            continue
        t = 127.0 * np.abs(v[m])
        q = np.floor(t / a[m])
        # t / a against q + 1/2 without dividing: 2 t against (2 q + 1) a; the floor above may be one off next to a whole number
        q = np.where(q * a[m] > t, q - 1, np.where((q + 1) * a[m] <= t, q + 1, q))
        up = (2 * t > (2 * q + 1) * a[m]) | ((2 * t == (2 * q + 1) * a[m]) & (q % 2 == 1))
        codes[m] = (np.sign(v[m]) * (q + up)).astype(np.int64)
    with np.errstate(over="ignore", invalid="ignore"):
        scale = np.where(fine, (a / 127.0).astype(np.float32), np.float32(np.nan))
    return codes, scale.astype(np.float32)


def linear_int8(codes, scale, W, w_scale, b=None, relu=False):
    """float64 [M,N] from whole-number codes and fp32 scales."""
    acc = codes.astype(np.int64) @ W.astype(np.int64).T
    y = acc.astype(np.float64) * (scale.astype(np.float64)[:, None] * w_scale.astype(np.float64)[None, :])
    if b is not None:
        y = y + b.astype(np.float64)[None, :]
    return np.where(y < 0, 0.0, y) if relu else y


def distribution(row):
    """softmax of a row of logits in 64 bits, None where it has no mass or holds a NaN or +inf."""
    row = row.astype(np.float64)
    if np.isnan(row).any() or (row == np.inf).any() or not np.isfinite(row.max()):
        return None
    e = np.exp(row - row.max())
    return e / e.sum()


def verify(logits, draft, tokens, u, r, lengths=None, draft_probs=False):
    """(accepted, next) row by row, position by position.  A given probability counts where it is read: that of the drafted
    code in the test, the whole row at a rejection."""
    logits, draft = (t.detach().cpu().to(torch.float32).numpy() for t in (logits, draft))
    tokens, u, r = tokens.cpu().numpy(), u.cpu().numpy(), r.cpu().numpy()
    B, P, V = logits.shape
    G = draft.shape[1]
    accepted, nxt = np.zeros(B, np.int64), np.full(B, -1, np.int64)

    def pick(w, total, at):
        cdf = np.cumsum(w)
        hit = np.nonzero((cdf > at * total) & (w > 0))[0]
        return hit[0] if len(hit) else np.nonzero(w > 0)[0][-1]

    for b in range(B):
        n = G if lengths is None else min(max(int(lengths[b]), 0), G)
        g = 0
        while g < n:
            p = distribution(logits[b, g])
            q = draft[b, g].astype(np.float64) if draft_probs else distribution(draft[b, g])
            if p is None or q is None:
                break
            x = tokens[b, g]
            inside = 0 <= x < V
            px, qx = (p[x], q[x]) if inside else (0.0, 0.0)
            if not (qx >= 0 and np.isfinite(qx)):
                break
            if not u[b, g] * qx < px:
                if not ((q >= 0) & np.isfinite(q)).all():
                    break
                w = np.maximum(p - q, 0.0)
                if w.sum() <= 2.0 ** -40:
                    w = p
                nxt[b] = pick(w, w.sum(), r[b])
                break
            g += 1
        accepted[b] = g
        if g == n and n < P:
            p = distribution(logits[b, n])
            if p is not None:
                nxt[b] = pick(p, p.sum(), r[b])
    return accepted, nxt
