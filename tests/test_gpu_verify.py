"""Verification of drafted codes (prior_verify) against the row-by-row 64-bit oracle.  Every output is a whole number and has
to be equal: inputs are random, so none lies within 64-bit rounding of a border unless a test puts it there, and those put it
1e-12 away, far outside the 1e-14 that a sum of exponentials in another order can move."""
import numpy as np
import pytest
import torch

from dvq_hip import ops
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


def make(B, G, P, V, tdt=torch.float32, ddt=torch.float32, probs=False, sigma=0.5, seed=0, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    t = 2.0 * torch.randn(B, P, V, generator=g)
    if masked:
        out = torch.rand(V, generator=g) < masked
        out[0] = False
        t[..., out] = -INF
    t = t.to(tdt)
    d = t[:, :G].float() + sigma * torch.randn(B, G, V, generator=g)
    x = torch.multinomial(torch.softmax(d.double(), 2).reshape(-1, V), 1, generator=g).reshape(B, G) if G else torch.zeros(B, 0, dtype=torch.int64)
    d = (torch.softmax(d, 2) if probs else d).to(ddt)
    return dict(logits=t, draft=d, tokens=x, u_accept=torch.rand(B, G, generator=g, dtype=torch.float64),
                u_draw=torch.rand(B, generator=g, dtype=torch.float64))


def check(c, lengths=None, probs=False, place=lambda k, v: v):
    dev = {k: place(k, v.to(DEV)) for k, v in c.items()}
    acc, nxt = ops.prior_verify(**dev, lengths=None if lengths is None else lengths.to(DEV), draft_probs=probs)
    assert acc.dtype == torch.int64 and nxt.dtype == torch.int64
    ra, rn = S.verify(c["logits"], c["draft"], c["tokens"], c["u_accept"], c["u_draw"], lengths, probs)
    assert np.array_equal(acc.cpu().numpy(), ra)
    assert np.array_equal(nxt.cpu().numpy(), rn)
    return ra, rn


SIZES = [(1, 1, 1, 1), (1, 1, 2, 2), (3, 2, 3, 3), (1, 9, 9, 512), (70, 9, 9, 512), (5, 4, 5, 63), (5, 4, 5, 64), (5, 4, 4, 65), (4, 3, 4, 1000),
         (4, 3, 4, 1025), (3, 2, 3, 4096), (3, 2, 3, 4097), (2, 3, 4, 8192), (300, 2, 3, 8193), (2, 2, 3, 65536), (1, 2, 2, 70001), (600, 3, 4, 300),
         (5, 0, 1, 500), (2, 0, 1, 20000), (2100, 3, 3, 130)]


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,G,P,V", SIZES)
def test_equals_the_oracle(B, G, P, V, dtype, probs):
    # (a draft's probabilities stay in 32 bits beside 16-bit logits, as a drafting prior returns them)
    check(make(B, G, P, V, dtype, torch.float32 if probs else dtype, probs, seed=B + V), probs=probs)


@pytest.mark.parametrize("tdt,ddt", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("probs", [False, True])
def test_mixed_types(tdt, ddt, probs):
    check(make(40, 4, 5, 700, tdt, ddt, probs, seed=4), probs=probs)


@pytest.mark.parametrize("V", [30, 600, 5000, 40000])
@pytest.mark.parametrize("sigma", [0.0, 0.02, 3.0])
def test_drafts_from_nearly_the_same_to_far_off(V, sigma):
    a, _ = check(make(24, 5, 6, V, sigma=sigma, seed=V))
    if sigma == 0.0:
        assert (a == 5).all()


@pytest.mark.parametrize("V", [40, 700, 9000])
def test_lengths_from_none_to_all(V):
    B, G = 50, 6
    lengths = torch.arange(B) % (G + 3) - 1                  # -1 .. G + 1: clamped to 0 .. G
    for P in (G, G + 1):
        check(make(B, G, P, V, seed=V + P), lengths=lengths)
        check(make(B, G, P, V, probs=True, seed=V + P), lengths=lengths, probs=True)


@pytest.mark.parametrize("V", [50, 513, 6000, 50000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_codes(V, dtype):
    check(make(16, 4, 5, V, dtype, dtype, masked=0.6, seed=V))
    c = make(8, 3, 4, V, dtype, dtype, seed=V)
    c["logits"][:, :, 1:] = -INF                             # one code left
    check(c)
    c["logits"][:, :, 1:] = torch.finfo(dtype).min           # the type's lowest value masks as well
    check(c)
    c["draft"][:, :, : V - 1] = torch.finfo(dtype).min
    check(c)
    c["draft"][:, :, : V - 1] = -INF
    c["tokens"][:] = V - 1
    a, _ = check(c)
    assert (a == 0).all()


@pytest.mark.parametrize("V", [50, 513, 6000, 50000])
@pytest.mark.parametrize("probs", [False, True])
def test_distributions_without_mass(V, probs):
    """All -inf, a NaN, a +inf -- in the target, in the draft, at the first, a middle and the bonus position."""
    bad = [("all", -INF), ("one", float("nan")), ("one", INF)]
    base = make(18, 4, 5, V, probs=probs, sigma=0.1, seed=V)
    for which in ("logits", "draft"):
        for kind, v in bad:
            c = {k: t.clone() for k, t in base.items()}
            for b in range(18):
                g = b % c[which].shape[1]
                if kind == "all":
                    c[which][b, g] = v
                else:
                    c[which][b, g, (b * 37) % V] = v
            check(c, probs=probs)
    if probs:
        c = {k: t.clone() for k, t in base.items()}
        c["draft"][:9, 1] = 0.0                              # a draft without any mass keeps what the prior allows
        c["draft"][9:, 2, V // 2] = -0.25
        check(c, probs=True)


@pytest.mark.parametrize("V", [12, 800, 9000])
def test_codes_outside_the_table_are_rejected(V):
    c = make(12, 3, 4, V, seed=V)
    for b, x in enumerate((-1, V, V + 5, -(1 << 62), (1 << 62), -V)):
        c["tokens"][b, b % 3] = x
        c["tokens"][b + 6, :] = x
    a, n = check(c)
    assert (a[6:] == 0).all() and (n >= 0).all()


@pytest.mark.parametrize("V", [16, 512, 5000, 30000])
@pytest.mark.parametrize("probs", [False, True])
def test_equal_distributions_with_a_code_that_neither_has(V, probs):
    """p = q and a drafted code of no mass: rejected, nothing is left over, the draw is from p."""
    c = make(20, 2, 3, V, sigma=0.0, seed=V)
    c["logits"][:, :, 3] = -INF
    c["draft"] = c["logits"][:, :2].clone()
    if probs:
        c["draft"] = torch.softmax(c["draft"].double(), 2).float()
    c["tokens"][:] = 3
    a, n = check(c, probs=probs)             # (probabilities rounded to 32 bits leave their rounding over: a draw from that)
    assert (a == 0).all() and (n != 3).all()


@pytest.mark.parametrize("V", [20, 512, 4500, 20000])
def test_acceptance_next_to_the_border(V):
    """u a 1e-12th below and above p / q: kept and rejected, whatever 32 bits would say."""
    B = 64
    c = make(B, 1, 2, V, seed=V + 1)
    c["draft"] = c["draft"] + 0.0
    want = []
    for b in range(B):
        p, q = S.distribution(c["logits"][b, 0].numpy()), S.distribution(c["draft"][b, 0].numpy())
        x = int(np.argmin(p / q))                            # a code the draft gives too much: p / q < 1
        c["tokens"][b, 0] = x
        keep = b % 2 == 0
        c["u_accept"][b, 0] = p[x] / q[x] * (1 - 1e-12 if keep else 1 + 1e-12)
        want.append(int(keep))
    a, _ = check(c)
    assert a.tolist() == want


@pytest.mark.parametrize("V", [20, 512, 4500, 20000])
def test_draws_next_to_the_border_of_two_codes(V):
    """The last draw behind all kept codes: r a 1e-11th of the mass below and above the border of two codes."""
    B = 40
    c = make(B, 0, 1, V, seed=V + 2)
    want = []
    for b in range(B):
        cdf = np.cumsum(S.distribution(c["logits"][b, 0].numpy()))
        k = (b * 31) % (V - 1)
        # a border between two codes with mass enough on both sides
        while min(cdf[k] - (cdf[k - 1] if k else 0.0), cdf[k + 1] - cdf[k]) < 1e-9:
            k = (k + 1) % (V - 1)
        c["u_draw"][b] = cdf[k] + (1e-11 if b % 2 else -1e-11)
        want.append(k + 1 if b % 2 else k)
    _, n = check(c)
    assert n.tolist() == want


@pytest.mark.parametrize("V", [5, 512, 5000, 20000])
def test_first_and_last_uniforms(V):
    c = make(8, 2, 3, V, masked=0.3, seed=V)
    c["u_draw"][:4] = 0.0
    c["u_draw"][4:] = 1.0 - 2.0 ** -53
    c["u_accept"][::2] = 0.0
    c["u_accept"][1::2] = 1.0 - 2.0 ** -53
    check(c)


@pytest.mark.parametrize("V", [70, 512, 900, 5000, 20000])
def test_strides(V):
    """The prior's [B, V, cells] layout, slices, every second row, broadcast uniforms and drafts, columns of wider buffers."""
    c = make(14, 4, 5, V, seed=3)

    def cells(k, v):
        return v.transpose(1, 2).contiguous().transpose(1, 2) if k in ("logits", "draft") else v

    def inside(k, v):
        pad = torch.full((*v.shape[:-1], v.shape[-1] + 5), 7, dtype=v.dtype, device=DEV)
        pad[..., 3:3 + v.shape[-1]] = v
        return pad[..., 3:3 + v.shape[-1]]

    def spread(k, v):
        wide = torch.full((2 * v.shape[0], *v.shape[1:]), 1, dtype=v.dtype, device=DEV)
        wide[::2] = v
        return wide[::2]
    def target_cells(k, v):
        return cells(k, v) if k == "logits" else v

    def draft_cells(k, v):
        return cells(k, v) if k == "draft" else v
    for place in (cells, inside, spread, target_cells, draft_cells):
        check(c, place=place)
        check(c, lengths=torch.arange(14) % 5, place=place)
    one = make(1, 4, 5, V, seed=8)
    same = {k: v.expand(14, *v.shape[1:]) for k, v in one.items()}
    check({k: v.contiguous() for k, v in same.items()}, place=lambda k, v: one[k].to(DEV).expand(14, *v.shape[1:]))


def test_first_emitted_code_is_distributed_as_the_priors():
    """20000 rows of one pair of distributions: counts within five binomial deviations of B p."""
    g = torch.Generator().manual_seed(5)
    V, B = 40, 20000
    t, d = torch.randn(V, generator=g), torch.randn(V, generator=g)
    x = torch.multinomial(torch.softmax(d.double(), 0).expand(B, V), 1, generator=g)
    acc, nxt = ops.prior_verify(t.to(DEV).expand(B, 1, V), d.to(DEV).expand(B, 1, V), x.to(DEV),
                                torch.rand(B, 1, generator=g, dtype=torch.float64).to(DEV), torch.rand(B, generator=g, dtype=torch.float64).to(DEV))
    first = torch.where(acc.cpu() == 1, x[:, 0], nxt.cpu()).numpy()
    p = torch.softmax(t.double(), 0).numpy()
    assert np.all(np.abs(np.bincount(first, minlength=V) - B * p) <= 5 * np.sqrt(B * p * (1 - p)))


def test_offsets_beyond_32_bits():
    B, G, V = 3, 2, 600
    c = make(B, G, G + 1, V, torch.bfloat16, torch.bfloat16, seed=6)

    def far(k, v):
        if k not in ("logits", "draft"):
            return v
        wide = torch.empty(v.shape[0], v.shape[1], 1 << 30, dtype=v.dtype, device=DEV)
        wide[..., :V] = v
        return wide[..., :V]
    check(c, place=far)


def test_empty_batch_and_refusals():
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=DEV)
    f64, i64 = torch.float64, torch.int64
    a, n = ops.prior_verify(z(0, 3, 8), z(0, 2, 8), z(0, 2, dt=i64), z(0, 2, dt=f64), z(0, dt=f64))
    assert a.shape == (0,) and n.shape == (0,)
    good = dict(logits=z(4, 3, 8), draft=z(4, 2, 8), tokens=z(4, 2, dt=i64), u_accept=z(4, 2, dt=f64), u_draw=z(4, dt=f64))
    ops.prior_verify(**good)
    for bad in (dict(logits=z(4, 4, 8)), dict(logits=z(4, 1, 8)), dict(logits=z(3, 3, 8)), dict(logits=z(4, 3, 9)), dict(logits=z(4, 3, 8, dt=f64)),
                dict(logits=z(4, 24)), dict(draft=z(4, 2, 7)), dict(draft=z(4, 3, 8)), dict(draft=z(4, 2, 8, dt=torch.float16)), dict(tokens=z(4, 2)),
                dict(tokens=z(4, 3, dt=i64)), dict(tokens=z(4, 2, dt=torch.int32)), dict(u_accept=z(4, 2)), dict(u_accept=z(4, 1, dt=f64)),
                dict(u_draw=z(4)), dict(u_draw=z(4, 1, dt=f64)), dict(lengths=z(3, dt=i64)), dict(lengths=z(4, dt=torch.int32)),
                dict(tokens=torch.zeros(4, 2, dtype=i64)), dict(draft=torch.zeros(4, 2, 8)), dict(logits=z(4, 3, 0), draft=z(4, 2, 0))):
        with pytest.raises(RuntimeError):
            ops.prior_verify(**{**good, **bad})


@pytest.mark.parametrize("B,V", [(3, 512), (40, 512), (2, 30000)])
def test_recorded_in_graphs_and_replayed(B, V):
    """Two recordings of one shape (they share no workspace), replayed in turns between eager calls."""
    cs = [{k: v.to(DEV) for k, v in make(B, 4, 5, V, seed=s).items()} for s in (1, 2)]
    for c in cs:
        ops.prior_verify(**c)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.prior_verify(**c))
        graphs.append(g)
    for i in range(4):
        for c, s in zip(cs, (1, 2)):
            for k, v in make(B, 4, 5, V, seed=10 * i + s).items():
                c[k].copy_(v.to(DEV))
        for j in ((0, 1), (1, 0))[i % 2]:
            graphs[j].replay()
        for c, (a, n) in zip(cs, outs):
            ea, en = ops.prior_verify(**c)
            assert torch.equal(a, ea) and torch.equal(n, en)
        torch.cuda.synchronize()


def test_two_streams_at_once():
    cs = [{k: v.to(DEV) for k, v in make(*shape, seed=9).items()} for shape in ((6, 4, 5, 40000), (500, 4, 5, 512))]
    want = [ops.prior_verify(**c) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.prior_verify(**cs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for a, n in got[i]:
            assert torch.equal(a, want[i][0]) and torch.equal(n, want[i][1])


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("B,G,P,V", [(1500, 70, 71, 20), (2, 130, 130, 40), (1, 70, 71, 600), (3, 65, 66, 520), (200, 66, 67, 1100), (800, 65, 65, 1030),
                                     (2, 66, 67, 2000)])
def test_more_drafted_codes_than_a_wave_has_lanes(B, G, P, V, probs):
    """Drafts next to the target: rows of every length up to all G codes kept."""
    c = make(B, G, P, V, probs=probs, sigma=0.01, seed=G + V)
    a, _ = check(c, probs=probs)
    assert (a > 64).any()
    if not probs and B < 10:
        c["draft"] = c["logits"][:, :G].clone()
        a, _ = check(c)
        assert (a == G).all()


@pytest.mark.parametrize("G,P", [(65, 65), (65, 66), (66, 67), (68, 69)])
@pytest.mark.parametrize("B,V", [(3, 40), (3, 1500), (200, 1500)])
def test_a_border_behind_the_64th_code(B, V, G, P):
    """The last drafted code's u a 1e-12th below and above p / q: an unsure test in the second set of drafted codes."""
    c = make(B, G, P, V, seed=G + V)
    c["draft"] = c["logits"][:, :G].clone()
    c["draft"][:, G - 1] += torch.randn(B, V, generator=torch.Generator().manual_seed(V))
    want = []
    for b in range(B):
        p, q = S.distribution(c["logits"][b, G - 1].numpy()), S.distribution(c["draft"][b, G - 1].numpy())
        x = int(np.argmin(p / q))
        c["tokens"][b, G - 1] = x
        c["u_accept"][b, G - 1] = p[x] / q[x] * (1 - 1e-12 if b % 2 else 1 + 1e-12)
        want.append(G if b % 2 else G - 1)
    a, _ = check(c)
    assert a.tolist() == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("B,G,P,V", [(192, 3, 3, 1025), (200, 3, 4, 1537), (768, 2, 3, 1025), (800, 3, 3, 2047), (200, 0, 1, 1300), (770, 0, 1, 1300),
                                     (191, 3, 4, 1025), (193, 2, 3, 9000)])
def test_a_workgroup_per_row(B, G, P, V, probs, dtype):
    check(make(B, G, P, V, dtype, torch.float32 if probs else dtype, probs, sigma=0.3, seed=B), probs=probs)
    check(make(B, G, P, V, dtype, torch.bfloat16, probs, sigma=0.3, seed=B, masked=0.4), lengths=torch.arange(B) % (G + 2), probs=probs)


@pytest.mark.parametrize("B", [200, 800])
def test_a_workgroup_per_row_with_odd_rows_of_its_own_types(B):
    """Rows of odd lengths inside wider buffers (no row starts at a multiple of 16 bytes), target and draft of different types."""
    def odd(k, v):
        if k not in ("logits", "draft"):
            return v
        wide = torch.full((*v.shape[:-1], v.shape[-1] + 6), 9, dtype=v.dtype, device=DEV)
        wide[..., 5:5 + v.shape[-1]] = v
        return wide[..., 5:5 + v.shape[-1]]
    for t, d in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)):
        for probs in (False, True):
            check(make(B, 3, 4, 1803, t, d, probs, sigma=0.3, seed=B), probs=probs, place=odd)


@pytest.mark.parametrize("B", [200, 800])
@pytest.mark.parametrize("sigma", [0.0, 1e-3, 3.0])
@pytest.mark.parametrize("probs", [False, True])
def test_a_workgroup_per_row_and_drafts_near_and_far(B, sigma, probs):
    """Next to equal distributions leave residual weights next to zero in every tile, and next to no mass."""
    c = make(B, 2, 3, 1600, probs=probs, sigma=sigma, seed=B)
    check(c, probs=probs)
    c["u_accept"][:, 1] = 1.0 - 2.0 ** -53                   # rejections even there
    c["tokens"][::3] = 0
    check(c, probs=probs)


@pytest.mark.parametrize("B", [200, 800])
@pytest.mark.parametrize("probs", [False, True])
def test_a_workgroup_per_row_and_distributions_without_mass(B, probs):
    c = make(B, 2, 3, 1100, probs=probs, sigma=0.1, seed=B)
    for b in range(0, B, 2):
        which = "logits" if b % 4 else "draft"
        g, v = b // 4 % c[which].shape[1], (-INF, float("nan"), INF)[b // 2 % 3]
        if v == -INF and not (probs and which == "draft"):
            c[which][b, g] = v
        else:
            c[which][b, g, (b * 37) % 1100] = v
    check(c, probs=probs)


@pytest.mark.parametrize("B", [200, 800])
def test_a_workgroup_per_row_next_to_the_borders(B):
    """Acceptance and draws a 1e-12th and a 1e-11th next to a border."""
    V = 1700
    c = make(B, 1, 2, V, seed=V + B)
    want = []
    for b in range(B):
        p, q = S.distribution(c["logits"][b, 0].numpy()), S.distribution(c["draft"][b, 0].numpy())
        x = int(np.argmin(p / q))
        c["tokens"][b, 0] = x
        c["u_accept"][b, 0] = p[x] / q[x] * (1 - 1e-12 if b % 2 else 1 + 1e-12)
        cdf = np.cumsum(S.distribution(c["logits"][b, 1].numpy()))
        k = (b * 31) % (V - 1)
        while min(cdf[k] - (cdf[k - 1] if k else 0.0), cdf[k + 1] - cdf[k]) < 1e-9:
            k = (k + 1) % (V - 1)
        c["u_draw"][b] = cdf[k] + (1e-11 if b % 4 == 3 else -1e-11)
        want.append((b % 2, k + 1 if b % 4 == 3 else k))
    a, n = check(c)
    assert a.tolist() == [w[0] for w in want]
    assert all(n[b] == w[1] for b, w in enumerate(want) if w[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,P", [(1, 2), (2, 3), (63, 5), (511, 3), (513, 9), (900, 9), (1000, 9), (1024, 16), (77, 16)])
def test_logits_with_all_positions_of_a_code_side_by_side(V, P, dtype):
    """The prior's layout in short rows: copied whole up to 32 KiB, read in place above."""
    place = lambda k, v: v.transpose(1, 2).contiguous().transpose(1, 2) if k == "logits" else v
    for B in (1, 40, 5000 if V * P < 400 else 60):
        check(make(B, P - 1, P, V, dtype, sigma=0.3, seed=V), place=place)
        check(make(B, P, P, V, dtype, probs=True, sigma=0.3, seed=V), probs=True, place=place)


@pytest.mark.parametrize("tdt,ddt", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("G,P,V", [(1, 1, 1100), (1, 2, 1300), (2, 2, 1025), (9, 10, 1537), (10, 10, 2600), (17, 18, 1111), (31, 32, 1500), (40, 41, 1200),
                                   (3, 4, 40000)])
def test_long_rows_with_all_positions_of_a_code_side_by_side(G, P, V, tdt, ddt):
    """Tiles of all positions in LDS as far as it reaches: target and draft, the target alone, neither; every second code of a wider
    buffer, and positions padded to more than there are, which are read in place."""
    B = 5
    cells = lambda k, v: v.transpose(1, 2).contiguous().transpose(1, 2) if k in ("logits", "draft") else v

    def padded(k, v):
        if k not in ("logits", "draft"):
            return v
        wide = torch.full((v.shape[0], 2 * v.shape[2], v.shape[1] + 3), 9, dtype=v.dtype, device=DEV)
        wide[:, ::2, 1:1 + v.shape[1]] = v.transpose(1, 2)
        return wide[:, ::2, 1:1 + v.shape[1]].transpose(1, 2)
    for place in (cells, padded):
        check(make(B, G, P, V, tdt, ddt, sigma=0.05, seed=V), place=place)
        check(make(B, G, P, V, tdt, ddt, probs=True, sigma=0.05, seed=V), lengths=torch.arange(B) * G // 4, probs=True, place=place)
    c = make(B, G, P, V, sigma=0.05, seed=V)
    c["draft"] = c["logits"][:, :G].clone()
    c["draft"][:, G - 1] += torch.randn(B, V, generator=torch.Generator().manual_seed(V))
    p, q = (np.stack([S.distribution(c[k][b, G - 1].numpy()) for b in range(B)]) for k in ("logits", "draft"))
    for b in range(B):                                           # an unsure test at the last draft
        x = int(np.argmin(p[b] / q[b]))
        c["tokens"][b, G - 1] = x
        c["u_accept"][b, G - 1] = p[b, x] / q[b, x] * (1 - 1e-12 if b % 2 else 1 + 1e-12)
    a, _ = check(c, place=cells)
    assert a.tolist() == [G if b % 2 else G - 1 for b in range(B)]


@pytest.mark.parametrize("V", [600, 1500, 3000, 20000])
@pytest.mark.parametrize("layout", ["rows", "cells"])
@pytest.mark.parametrize("B", [4, 600])
def test_a_nan_among_masked_codes(B, V, layout):
    """Whole tiles of -inf with one NaN in them, in target and draft: a distribution that is none, wherever the NaN lies."""
    if B * V > 2000000:
        B = 64
    c = make(B, 2, 3, V, sigma=0.1, seed=V)
    lo, hi = (0, 512) if V < 1024 else (512, min(V, 1536))
    for b in range(0, B, 2):
        which = "logits" if b % 4 else "draft"
        g = b // 4 % c[which].shape[1]
        c[which][b, g, lo:hi] = -INF
        c[which][b, g, lo + (b * 37) % (hi - lo)] = float("nan")
    place = (lambda k, v: v) if layout == "rows" else lambda k, v: v.transpose(1, 2).contiguous().transpose(1, 2) if k in ("logits", "draft") else v
    _, n = check(c, place=place)
    assert (n == -1).any() and (n >= 0).any()


def rising(V, kind, g):
    """Logits whose running reference point has to move: levels just below and above the slack of 8, slow and fast ascents."""
    at = torch.arange(V).float() / V
    tile = torch.arange(V) // 512
    if kind == "below":                                          # 7.9 above the first level for most of the row
        x = torch.where(at < 0.1, 0.0, 7.9)
    elif kind == "steps":                                        # most of the mass lies 7.9 above, then one tile 8.1 above moves it
        x = torch.where(at < 0.1, 0.0, 7.9)
        x[-600:] = 8.1
    elif kind == "stairs":                                       # every tile 8.1 above the one in front of it, up to the last six
        x = 8.1 * (tile - tile.max()).clamp_min(-6).float()
    elif kind == "gentle":                                       # moves in most tiles, each of them with mass
        x = 40.0 * at
    else:
        x = torch.sort(12.0 * torch.randn(V, generator=g)).values
    return x + 0.01 * torch.randn(V, generator=g)


@pytest.mark.parametrize("kind", ["below", "steps", "stairs", "gentle", "sorted"])
@pytest.mark.parametrize("B,V", [(8, 6000), (24, 20000), (130, 9000)])
def test_ascending_logits_and_uniforms_next_to_the_border(B, V, kind):
    """Rows whose reference point moves while its lane holds most of the mass: the test sums are joined over moves, and tests from
    1e-12 to 1e-4 next to the border have to come out as in 64 bits."""
    g = torch.Generator().manual_seed(V + B)
    c = make(B, 1, 2, V, seed=V)
    want = []
    for b in range(B):
        up = rising(V, kind, g)
        c["logits"][b, 0] = up
        c["draft"][b, 0] = up.flip(0) if b % 3 == 0 else up + 0.3 * torch.randn(V, generator=g)
        p, q = S.distribution(c["logits"][b, 0].numpy()), S.distribution(c["draft"][b, 0].numpy())
        x = int(np.argmin(np.where(q > 1e-9, p / np.maximum(q, 1e-300), np.inf)))
        if not p[x] > 1e-12:
            x = int(np.argmax(np.where(p < q, p, 0.0)))          # (flipped: a code that both have)
        assert 0 < p[x] < q[x]
        c["tokens"][b, 0] = x
        off = (1e-12, 1e-9, 1e-7, 1e-6, 5e-6, 1.5e-5, 3e-5, 1e-4)[b // 2 % 8]
        c["u_accept"][b, 0] = p[x] / q[x] * (1 - off if b % 2 else 1 + off)
        want.append(b % 2)
    for place in (lambda k, v: v, lambda k, v: v.transpose(1, 2).contiguous().transpose(1, 2) if k in ("logits", "draft") else v):
        a, _ = check(c, place=place)
        assert a.tolist() == want
