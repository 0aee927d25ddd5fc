"""The 8-bit heads and the verification of drafted grids where the models call them, and both together: a drafting head in
8 bits, its codes drawn from given uniforms, the prior's verification of them."""
import copy
import pickle

import numpy as np
import pytest
import torch

from dvq_hip import ops, rng, set_compute_dtype, set_head_dtype, synth
from network.DVQVAE import Decoder, DVQVAE, Encoder
from network.pixelcnn.models import GatedPixelCNN
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def head(cls, sizes, latent, seed):
    torch.manual_seed(seed)
    return cls(sizes, latent).to(DEV).eval()


def oracle_mlp(linears, x, relu_last):
    """The layers one after the other on the oracle's codes, each output rounded to fp32 as the kernel hands it on; the last
    layer's float64 output."""
    for i, l in enumerate(linears):
        W, t = S.int8_codes(l.weight.detach().cpu())
        c, s = S.int8_codes(x)
        y = S.linear_int8(c, s, W, t, l.bias.detach().cpu().numpy(), relu_last or i + 1 < len(linears))
        x = torch.from_numpy(y).float()
    return y


@pytest.mark.parametrize("B", [1, 7, 100, 600])
def test_heads_in_8_bits_equal_the_layers_one_by_one(B):
    """The same fp32 hand-over between layers: the oracle's rounding of a 64-bit value and the kernel's are the same one,
    so codes agree and the last output is off by its own rounding (2^-24) at most."""
    x = torch.randn(B, 1024, generator=torch.Generator().manual_seed(B))
    e = set_head_dtype(head(Encoder, [1024, 512], 256, 0), torch.int8)
    y = e(x.to(DEV)).cpu().double().numpy()
    ref = oracle_mlp([m for m in e.MLP if isinstance(m, torch.nn.Linear)] + [e.linear_means], x, False)
    assert np.all(np.abs(y - ref) <= 2.0 ** -24 * np.abs(ref) * (1 + 1e-6) + 2.0 ** -50)
    d = set_head_dtype(head(Decoder, [1024, 128, 6], 1024, 1), torch.int8)
    ref = oracle_mlp([m for m in d.MLP if isinstance(m, torch.nn.Linear)], x, False)
    assert np.all(np.abs(d(x.to(DEV)).cpu().double().numpy() - ref) <= 2.0 ** -24 * np.abs(ref) * (1 + 1e-6) + 2.0 ** -50)


def test_decoder_takes_its_input_in_pieces():
    d = set_head_dtype(head(Decoder, [1024, 128, 6], 2048, 2), torch.int8)
    g = torch.Generator().manual_seed(0)
    table, idx, f = torch.randn(128, 1024, generator=g).to(DEV), torch.randint(0, 128, (40,), generator=g).to(DEV), torch.randn(40, 1024, generator=g).to(DEV)
    assert torch.equal(d.forward_pieces([(idx, table), f]), d(torch.cat([table[idx], f], 1)))


def test_8_bit_heads_follow_their_weights_and_stay_out_of_copies():
    e = set_head_dtype(head(Encoder, [64, 32], 16, 3), torch.int8)
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    a = e(x)
    twin, loaded = copy.deepcopy(e), pickle.loads(pickle.dumps(e))
    assert torch.equal(twin(x), a) and torch.equal(loaded.to(DEV)(x), a)
    with torch.no_grad():
        e.linear_means.weight.mul_(2.0)
        e.linear_means.bias.mul_(2.0)
    assert torch.allclose(e(x), 2 * a, rtol=1e-6) and torch.equal(twin(x), a)
    set_compute_dtype(e, torch.float32)
    assert not torch.equal(e(x), 2 * a)


def test_error_of_8_bit_heads_is_that_of_their_rounding():
    """Against fp32: every layer's operands are off by at most half a code, |x| and |w| by max/254.  For the first layer that
    bounds an output by sum |w| a/254 + |x| a_w/254 + a a_w/254^2; here on the layer itself."""
    torch.manual_seed(4)
    l = torch.nn.Linear(1024, 512).to(DEV)
    x = torch.randn(300, 1024, device=DEV)
    y = ops.linear_int8(x, *ops.quantize_rows(l.weight.detach()), l.bias.detach()).double()
    ref = x.double() @ l.weight.detach().double().T + l.bias.detach().double()
    a, aw = x.abs().amax(1).double()[:, None], l.weight.detach().abs().amax(1).double()[None, :]
    lim = l.weight.detach().abs().double().sum(1)[None, :] * a / 254 + x.abs().double().sum(1)[:, None] * aw / 254 + 1024 * a * aw / 254 ** 2
    assert ((y - ref).abs() <= lim * (1 + 1e-6)).all()


def test_hand_encoder_with_8_bit_heads_equals_its_parts_one_by_one():
    torch.manual_seed(5)
    m = DVQVAE(obj_inchannel=4).to(DEV).eval()
    obj, hand = synth.object_clouds(3, 200, seed=1).to(DEV), torch.randn(3, 3, 778, generator=torch.Generator().manual_seed(2)).to(DEV)
    set_head_dtype(m, torch.int8)
    idx, emb = m(obj, hand)
    idx1, emb1 = m.forward_per_part(obj, hand)
    assert torch.equal(idx, idx1) and torch.equal(emb, emb1)


def test_generation_with_8_bit_heads_runs_and_stays_near_fp32():
    from dvq_hip.pipeline import GraspGenerator
    gen = GraspGenerator.synthetic(torch.device(DEV), seed=0, with_prior=True)
    objs = synth.object_clouds(3, 300, seed=4).to(DEV)
    xt = torch.randint(0, 128, (3, 3, 3), generator=torch.Generator().manual_seed(0)).to(DEV)
    ref = gen.generate(objs, x_tilde=xt)["vertices"]
    set_head_dtype(gen.model, torch.int8)
    out = gen.generate(objs, x_tilde=xt)["vertices"]
    assert torch.isfinite(out).all() and out.shape == ref.shape and not torch.equal(out, ref)


def prior(seed, layers=3, codes=128, dim=128):
    torch.manual_seed(seed)
    p = GatedPixelCNN(codes, dim, layers, n_classes=16).to(DEV).eval()
    with torch.no_grad():
        p.output_conv[2].weight.mul_(4.0)
    return p


@pytest.mark.parametrize("B", [1, 30])
def test_a_drafting_prior_is_verified_by_another(B):
    target, draft = prior(0), prior(1)
    g = torch.Generator().manual_seed(2)
    label = torch.randint(0, 16, (B,), generator=g).to(DEV)
    u = lambda *s: torch.rand(*s, generator=g, dtype=torch.float64).to(DEV)
    x, q = draft.generate(None, label, batch_size=B, uniforms=u(B, 9), return_probs=True)
    ua, ud = u(B, 9), u(B)
    lengths = torch.randint(0, 10, (B,), generator=g).to(DEV)
    for n in (None, lengths):
        acc, nxt = target.verify(x, label, q, ua, ud, lengths=n, draft_probs=True)
        with torch.no_grad():
            cells = target(x, label).flatten(2).transpose(1, 2)
        ra, rn = S.verify(cells, q, x.reshape(B, 9), ua, ud, n, True)
        assert np.array_equal(acc.cpu().numpy(), ra) and np.array_equal(nxt.cpu().numpy(), rn)
    acc, nxt = target.verify(x, label, cells, ua, ud)                 # drafted by itself: all kept, no cell behind the last
    assert (acc == 9).all() and (nxt == -1).all()
    with pytest.raises(RuntimeError):
        target.verify(x, label, q[:, :8], ua, ud, draft_probs=True)
    with pytest.raises(RuntimeError):
        target.verify(x.reshape(B, 9), label, q, ua, ud, draft_probs=True)
    empty = target.verify(x[:0], label[:0], q[:0], ua[:0], ud[:0], draft_probs=True)
    assert empty[0].shape == (0,) and empty[1].shape == (0,)


def test_8_bit_drafting_head_and_verification_together():
    """Object feature -> 9 x 128 draft logits in 8 bits (two products), codes drawn at given uniforms, one forward of the prior
    with them as the history, verification; against the same steps on the oracle from the feature and the prior's logits on."""
    B, V = 50, 128
    target = prior(3)
    h = set_head_dtype(head(Encoder, [1024, 256], 9 * V, 6), torch.int8)
    g = torch.Generator().manual_seed(7)
    feat = torch.randn(B, 1024, generator=g)
    label = torch.randint(0, 16, (B,), generator=g).to(DEV)
    u = rng.uniforms(torch.arange(B, device=DEV), 9, seed=1)
    ua, ud = rng.uniforms(torch.arange(B, device=DEV), 9, seed=2), rng.uniforms(torch.arange(B, device=DEV), 1, seed=3)[:, 0]

    d = h(feat.to(DEV)).view(B, 9, V)
    x = torch.empty(B, 9, dtype=torch.int64, device=DEV)
    ops.prior_sample(d.view(B * 9, V), u.reshape(-1), x.view(-1))
    acc, nxt = target.verify(x.view(B, 3, 3), label, d, ua, ud)

    lin = [m for m in h.MLP if isinstance(m, torch.nn.Linear)] + [h.linear_means]
    ref = oracle_mlp(lin, feat, False)
    assert np.all(np.abs(d.view(B, -1).cpu().double().numpy() - ref) <= 2.0 ** -24 * np.abs(ref) * (1 + 1e-6) + 2.0 ** -50)
    with torch.no_grad():
        cells = target(x.view(B, 3, 3), label).flatten(2).transpose(1, 2)
    ra, rn = S.verify(cells, d, x, ua, ud)
    assert np.array_equal(acc.cpu().numpy(), ra) and np.array_equal(nxt.cpu().numpy(), rn)
    assert 0 < acc.sum() < 9 * B


def test_cells_behind_the_drafts_and_codes_outside_the_table():
    """What lies behind a grid's drafts is not looked up; a drafted code outside the table is rejected, cells behind it are not
    reached.  Every position's history is unchanged by either."""
    B = 40
    target = prior(4)
    V = target.embedding.num_embeddings
    g = torch.Generator().manual_seed(8)
    label = torch.randint(0, 16, (B,), generator=g).to(DEV)
    x = torch.randint(0, V, (B, 9), generator=g).to(DEV)
    with torch.no_grad():
        q = target(x.view(B, 3, 3), label).flatten(2).transpose(1, 2).contiguous()
    u = lambda *s: torch.rand(*s, generator=g, dtype=torch.float64).to(DEV)
    ua, ud, lengths = u(B, 9), u(B), torch.arange(B, device=DEV) % 10
    acc, nxt = target.verify(x.view(B, 3, 3), label, q, ua, ud, lengths=lengths)
    assert torch.equal(acc, lengths)                                  # drafted by the prior itself
    behind = torch.arange(9, device=DEV)[None, :] >= lengths[:, None]
    for fill in (-1, V, 1 << 40, -(1 << 62)):
        y = torch.where(behind, fill, x)
        a, n = target.verify(y.view(B, 3, 3), label, q, ua, ud, lengths=lengths)
        assert torch.equal(a, acc) and torch.equal(n, nxt)
        a, n = target.verify(y.view(B, 3, 3), label, q, ua, ud)       # now they are drafts
        assert torch.equal(a, lengths) and (n[lengths < 9] >= 0).all() and (n[lengths == 9] == -1).all()


def test_8_bit_heads_in_recorded_graphs():
    """The first call recorded (the copy of the weights is not kept then), eager calls before its replay, a graph over a kept copy
    that a changed weight refreshes in place, and a graph and eager calls in turns."""
    e = set_head_dtype(head(Encoder, [64, 32], 16, 9), torch.int8)
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    spare = set_head_dtype(head(Encoder, [64, 32], 16, 9), torch.int8)
    want = spare(x)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            spare(x)                                                  # (the kernels are loaded)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(first):
            a = e(x)
        assert torch.equal(e(x), want)
        with torch.cuda.graph(second):
            b = e(x)
        for scale in (1.0, 2.0, 0.5):
            e.linear_means.weight.mul_(scale)
            spare.linear_means.weight.mul_(scale)
            want = spare(x)
            first.replay()                                            # quantises for itself
            assert torch.equal(a, want)
            assert torch.equal(e(x), want)
            second.replay()                                           # reads the copy that the call above refreshed
            assert torch.equal(b, want)
            torch.cuda.synchronize()


def test_recorded_graphs_follow_edited_weights_without_an_eager_call():
    """A graph recorded after an eager call quantises for itself as well: weights and biases that are edited in place or loaded
    count at the next replay, as they do for heads in fp32."""
    e = set_head_dtype(head(Encoder, [64, 32], 16, 10), torch.int8)
    d = set_head_dtype(head(Decoder, [48, 6], 64, 11), torch.int8)
    twins = [copy.deepcopy(m) for m in (e, d)]
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(2)).to(DEV)
    for m in (e, d, *twins):
        m(x)                                                          # eager calls first: copies of the weights are kept
    torch.cuda.synchronize()
    graphs, outs = [], []
    with torch.no_grad():
        for m in (e, d):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(m(x))
        for step in range(4):
            for m, t in zip((e, d), twins):
                if step == 1:
                    for p, q in zip(m.parameters(), t.parameters()):
                        p.mul_(1.5)
                        q.mul_(1.5)
                if step == 2:
                    state = {k: v + 0.25 for k, v in t.state_dict().items()}
                    m.load_state_dict(state)
                    t.load_state_dict(state)
                if step == 3:
                    m(x)                                              # an eager call in between
            for g in graphs:
                g.replay()
            got = [o.clone() for o in outs]
            for m, t, y in zip((e, d), twins, got):
                assert torch.equal(y, t(x))
            torch.cuda.synchronize()


def test_a_replaced_weight_at_an_earlier_address_is_quantised_anew():
    """Replaced twice between two calls, a weight can lie where the first one lay, at the same version."""
    e = set_head_dtype(head(Encoder, [64, 32], 16, 12), torch.int8)
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(3)).to(DEV)
    for seed in range(12):
        g = torch.Generator().manual_seed(seed)
        e.linear_means.weight = torch.nn.Parameter(torch.randn(16, 32, generator=g).to(DEV))
        if seed % 2:                                                  # (the call comes after every second replacement)
            fresh = copy.deepcopy(e)
            assert torch.equal(e(x), fresh(x))
            del fresh


def test_verify_is_recorded_once_its_tables_are_made(monkeypatch):
    """Packed weights and class tables that a first call makes would hold nothing until the graph's first replay, and eager calls
    would read them: refused.  A recorded graph has buffers of its own: calls of other batch sizes, which drop the kept ones,
    other graphs and changed weights leave it what it is."""
    target = prior(5)
    g = torch.Generator().manual_seed(9)
    u = lambda *s: torch.rand(*s, generator=g, dtype=torch.float64).to(DEV)

    def inputs(B):
        return [torch.randint(0, 128, (B, 3, 3), generator=g).to(DEV), torch.randint(0, 16, (B,), generator=g).to(DEV),
                torch.randn(B, 9, 128, generator=g).to(DEV), u(B, 9), u(B)]
    a, b, other = inputs(6), inputs(6), inputs(11)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="once before"):
            target.verify(*a)
    assert not target._bufs and target._packed_key is None
    target.verify(*a)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for args in (a, b):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(target.verify(*args))
    for i in range(4):
        for args in (a, b):
            for t, v in zip(args, inputs(6)):
                t.copy_(v)
        want = [[t.clone() for t in target.verify(*args)] for args in (a, b)]
        target.generate(None, other[1], batch_size=11, uniforms=other[3])         # (drops the buffers of other batch sizes)
        spoil = [torch.full((1 << 18,), float("nan"), device=DEV) for _ in range(64)]
        for j in ((0, 1), (1, 0))[i % 2]:
            graphs[j].replay()
        for got, w in zip(outs, want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
        assert all(t.isnan().all() for t in spoil)
        del spoil
        torch.cuda.synchronize()
    with torch.no_grad():
        target.embedding.weight.add_(0.0)                                         # (another version of the same weights)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="once before"):
            target.verify(*a)
    target.verify(*other)                                                         # packs them anew
    spoil = [torch.full((1 << 18,), float("nan"), device=DEV) for _ in range(64)]
    graphs[0].replay()
    assert torch.equal(outs[0][0], want[0][0]) and torch.equal(outs[0][1], want[0][1]) and all(t.isnan().all() for t in spoil)
    twin = copy.deepcopy(target)
    assert not twin._recorded and target._recorded


def test_generated_parameters_are_those_of_the_8_bit_layers_one_by_one():
    """Generation with 8-bit heads: what both decoders make of the pieces they are given equals their layers on the 64-bit oracle,
    and the parameter vector is made of that."""
    from dvq_hip.pipeline import GraspGenerator, assemble_param
    gen = GraspGenerator.synthetic(torch.device(DEV), seed=0, with_prior=True)
    objs = synth.object_clouds(5, 300, seed=4).to(DEV)
    xt = torch.randint(0, 128, (5, 3, 3), generator=torch.Generator().manual_seed(0)).to(DEV)
    set_head_dtype(gen.model, torch.int8)
    seen = {}
    for name in ("decoder", "pos_decoder"):
        def record(pieces, name=name, run=getattr(gen.model, name).forward_pieces):
            y = run(pieces)
            seen[name] = (torch.cat([p[1][p[0]] if isinstance(p, tuple) else p for p in pieces], 1).cpu(), y.clone())
            return y
        getattr(gen.model, name).forward_pieces = record
    param = gen.generate(objs, x_tilde=xt)["recon_param"]
    for name in ("decoder", "pos_decoder"):
        x, y = seen[name]
        ref = oracle_mlp([m for m in getattr(gen.model, name).MLP if isinstance(m, torch.nn.Linear)], x, False)
        assert np.all(np.abs(y.cpu().double().numpy() - ref) <= 2.0 ** -24 * np.abs(ref) * (1 + 1e-6) + 2.0 ** -50)
    assert torch.equal(param, assemble_param(seen["decoder"][1], seen["pos_decoder"][1]))
