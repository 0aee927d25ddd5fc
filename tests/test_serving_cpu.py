"""The oracles of the 8-bit product and of the verification against independent arithmetic, and what the entry points refuse.
Nothing here needs a GPU: the C entries refuse before they launch."""
import ctypes
from fractions import Fraction

import numpy as np
import pytest
import torch

from dvq_hip import _lib, ops, set_head_dtype
from oracle import serving_oracle as S

VP = ctypes.c_void_p


def test_codes_of_the_oracle_are_the_nearest_whole_numbers_of_exact_quotients():
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(40, 24, generator=g), torch.randn(40, 24, generator=g).to(torch.bfloat16).float(),
                   torch.randint(-254, 255, (40, 24), generator=g).float() * 0.5])
    x[80:, 0] = 127.0                          # halves: 127 x / a = x, ties throughout
    codes, scale = S.int8_codes(x)
    for m in range(x.shape[0]):
        a = max(Fraction(float(v)) for v in x[m].abs())
        for k in range(x.shape[1]):
            assert codes[m, k] == round(127 * Fraction(float(x[m, k])) / a)          # Fraction rounds halves to even
    assert codes.max() == 127 and codes.min() >= -127
    assert np.array_equal(scale, (x.abs().amax(1).double() / 127).float().numpy())


def test_codes_of_the_oracle_in_special_rows():
    x = torch.zeros(5, 4)
    x[1, 2] = float("inf")
    x[2, 0] = float("nan")
    x[3] = torch.tensor([1e-45, -1e-45, 0.0, 0.0])
    x[4] = torch.tensor([3.4e38, -1.7e38, 1.0, 0.0])
    codes, scale = S.int8_codes(x)
    assert not codes[:3].any() and scale[0] == 0 and np.isnan(scale[1:3]).all()
    assert codes[3].tolist() == [127, -127, 0, 0] and codes[4, 0] == 127 and np.isfinite(scale[4])


def test_verification_oracle_keeps_the_target_distribution():
    """Summed over drafted code and accept/reject, the first emitted code has probability p exactly: over all codes x,
    q(x) min(1, p(x)/q(x)) + P(reject) (p - q)+ / mass = p(x).  Here by counting: 20000 rows."""
    g = torch.Generator().manual_seed(1)
    V, B = 6, 20000
    t, d = torch.randn(V, generator=g), torch.randn(V, generator=g)
    q = torch.softmax(d.double(), 0)
    x = torch.multinomial(q.expand(B, V), 1, generator=g)
    acc, nxt = S.verify(t.expand(B, 1, V), d.expand(B, 1, V), x, torch.rand(B, 1, generator=g, dtype=torch.float64),
                        torch.rand(B, generator=g, dtype=torch.float64))
    first = np.where(acc == 1, x[:, 0].numpy(), nxt)
    p = torch.softmax(t.double(), 0).numpy()
    # binomial deviation of a count of 20000: five of them
    assert np.all(np.abs(np.bincount(first, minlength=V) / B - p) <= 5 * np.sqrt(p * (1 - p) / B))


def _quantize(lib, M=4, K=16, ldc=16, dtype=0, ldx=16, ptr=16, codes=16):
    return lib.dvq_int8_quantize_rows(ptr, dtype, ldx, M, K, codes, ldc, ptr, None)


def _product(lib, n=1, M=4, K=16, N=4, ldx=16, ldw=16, ldy=4, x_dtype=0, y_dtype=0, ptr=16, xs=True, ws=16, nbytes=1 << 40):
    arr = (VP * 8)(*[ptr] * 8)
    return lib.dvq_linear_int8_batched(n, arr, x_dtype, arr if xs else None, ldx, arr, arr, ldw, None, M, K, N, 0, arr, y_dtype, ldy, ws, nbytes, None)


@pytest.mark.parametrize("bad", [dict(K=0), dict(K=1 << 17, ldc=1 << 17), dict(ldc=24), dict(K=17), dict(M=-1), dict(dtype=2), dict(ptr=None),
                                 dict(codes=8), dict(ldx=-1)])
def test_quantize_refusals(bad):
    lib = _lib.load()
    assert _quantize(lib, **bad) == -1 and lib.dvq_last_error()


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=9), dict(K=0), dict(K=1 << 17), dict(M=-1), dict(N=0), dict(x_dtype=3), dict(y_dtype=2), dict(ldy=3),
                                 dict(ldx=-1), dict(ldw=-1), dict(ptr=None), dict(x_dtype=2, xs=False), dict(M=0x7FFFFFFF),
                                 dict(M=20000, ws=None), dict(M=20000, ws=8), dict(M=20000, nbytes=20000 * 64 + 80000 + 4 * 64 - 1), dict(K=4097, ws=None),
                                 dict(n=2, M=20000, nbytes=20000 * 64 + 80000 + 4 * 64)])
def test_product_refusals(bad):
    lib = _lib.load()
    assert _product(lib, **bad) == -1 and lib.dvq_last_error()


def test_single_product_refusals():
    lib = _lib.load()
    call = lambda x=16, W=16, y=16, x_dtype=0, xs=16, N=4, ws=16, M=4: lib.dvq_linear_int8(x, x_dtype, xs, 16, W, 16, 16, None, M, 16, N, 0, y, 0, 4,
                                                                                        ws, 1 << 40, None)
    assert call(M=0) == 0
    for bad in (dict(x=None), dict(W=None), dict(y=None), dict(x_dtype=2, xs=None), dict(N=0), dict(M=20000, ws=None)):
        assert call(**bad) == -1 and lib.dvq_last_error()


def test_workspace_of_the_product():
    size = _lib.load().dvq_linear_int8_workspace_bytes
    assert size(1, 20, 16, 4) == 20 * 64 + 80 + 4 * 64 and size(3, 20, 16, 4) == 3 * size(1, 20, 16, 4)
    assert size(1, 0, 16, 4) == 0 and size(0, 20, 16, 4) == 0
    assert size(8, 1 << 20, 1 << 16, 1 << 16) == 8 * ((1 << 36) + (1 << 22) + (1 << 32))


def _verify_args(**kw):
    a = _lib.DvqPriorVerify()
    for f in ("logits", "draft", "tokens", "u_accept", "u_draw", "accepted", "next"):
        setattr(a, f, 16)
    a.B, a.G, a.P, a.V = 2, 3, 4, 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(B=-1), dict(V=0), dict(V=(1 << 20) + 1), dict(B=1 << 30, V=1 << 20), dict(P=2), dict(P=5), dict(G=0, P=0), dict(G=-1), dict(logits_dtype=2),
                                 dict(draft_dtype=-1), dict(logits=None), dict(draft=None), dict(tokens=None), dict(u_accept=None),
                                 dict(u_draw=None), dict(accepted=None), dict(next=None)])
def test_verify_refusals(bad):
    lib = _lib.load()
    assert lib.dvq_prior_verify(ctypes.byref(_verify_args(**bad)), 16, 1 << 40, None) == -1 and lib.dvq_last_error()
    assert lib.dvq_prior_verify(None, 16, 1 << 40, None) == -1


def test_verify_refuses_a_workspace_too_small():
    """Long rows whose codes lie apart, and few long rows, need one."""
    lib = _lib.load()
    for kw in (dict(V=5000, logits_v=9, draft_v=1), dict(V=50000, logits_v=1, draft_v=1)):
        a = _verify_args(**kw)
        need = lib.dvq_prior_verify_workspace_bytes(ctypes.byref(a))
        assert need > 0
        for ws, size in ((None, need), (16, need - 1), (24, need)):
            assert lib.dvq_prior_verify(ctypes.byref(a), ws, size, None) == -1
    assert lib.dvq_prior_verify_workspace_bytes(ctypes.byref(_verify_args(V=1000, logits_v=1, draft_v=1))) == 0
    assert lib.dvq_prior_verify_workspace_bytes(ctypes.byref(_verify_args(V=5000, logits_v=1, draft_v=1))) == 0
    assert lib.dvq_prior_verify_workspace_bytes(ctypes.byref(_verify_args(V=50000, logits_v=1, draft_v=1, B=5000))) == 0


def test_empty_calls_return_without_a_launch():
    lib = _lib.load()
    assert _quantize(lib, M=0) == 0 and _product(lib, M=0) == 0
    assert lib.dvq_prior_verify(ctypes.byref(_verify_args(B=0)), None, 0, None) == 0


def test_cpu_tensors_and_wrong_types_are_refused():
    x, W, s = torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.linear_int8(x, W, s), lambda: ops.linear_int8((W, s), W, s),
                 lambda: ops.linear_int8(x.double(), W, s), lambda: ops.linear_int8(x, W, s, out_dtype=torch.float16),
                 lambda: ops.linear_int8_batched([], [], [], []), lambda: ops.linear_int8_batched([x, (W, s)], [W, W], [s, s], [None, None])):
        with pytest.raises(RuntimeError):
            call()
    lg, tok, u = torch.zeros(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.prior_verify(lg, lg, tok, u, u[:, 0])


def test_head_dtype_is_set_on_the_heads_alone():
    from network.gen_net import GenNet
    m = set_head_dtype(GenNet(), torch.int8)
    assert m.decoder.compute_dtype == torch.int8 and m.pos_decoder.compute_dtype == torch.int8
    assert m.obj_encoder_type.compute_dtype == torch.float32 and m.GatedPixelCNN.compute_dtype == torch.float32
    with pytest.raises(ValueError):
        set_head_dtype(m, torch.float16)


def test_sizes_that_no_launch_holds_are_refused():
    lib = _lib.load()
    assert _quantize(lib, M=1 << 26) == -1 and b"2^26" in lib.dvq_last_error()
    for bad in (dict(M=1 << 26, N=1 << 10, ldy=1 << 10), dict(M=(1 << 30) + 1), dict(N=(1 << 30) + 1, ldy=1 << 31), dict(N=1 << 28, ldy=1 << 28),
                dict(M=100, N=1 << 26, ldy=1 << 26, ldw=17)):
        assert _product(lib, **bad) == -1 and lib.dvq_last_error()
    for bad in (dict(B=1 << 26, V=8), dict(B=1 << 24, V=5000, logits_v=1, draft_v=1), dict(B=1 << 24, V=5000, logits_v=4, draft_v=4), dict(B=1 << 20, V=1 << 20, logits_v=9, draft_v=9)):
        assert lib.dvq_prior_verify(ctypes.byref(_verify_args(**bad)), 16, 1 << 60, None) == -1 and b"too large" in lib.dvq_last_error()


@pytest.mark.parametrize("logits_dtype,V,P,waves", [(0, 1000, 8, 5), (1, 1000, 16, 5), (0, 500, 7, 2), (0, 900, 9, 5)])
def test_short_rows_of_several_waves_that_no_launch_holds_are_refused(logits_dtype, V, P, waves):
    """Staged rows have up to five waves whatever their number: counted as launched, not as one."""
    lib = _lib.load()
    for B in (((1 << 32) - 1) // (64 * waves) + 1, 1 << 26):
        a = _verify_args(B=B, V=V, P=P, G=P - 1, logits_dtype=logits_dtype, logits_p=1, logits_v=P, draft_v=1)
        assert lib.dvq_prior_verify(ctypes.byref(a), 16, 1 << 60, None) == -1 and b"too large" in lib.dvq_last_error()


def test_8_bit_heads_on_the_cpu_are_refused():
    from network.DVQVAE import Decoder, Encoder
    for head in (Encoder([8, 6], 4), Decoder([6, 4], 8)):
        with pytest.raises(RuntimeError, match="HIP device"):
            set_head_dtype(head, torch.int8)(torch.zeros(2, 8))
