"""8-bit integer product (quantize_rows, linear_int8, linear_int8_batched) against whole-number arithmetic.

Codes and sums are whole numbers and have to be equal.  An output is (sum) * (s t) + b, taken in 64 bits and rounded once:
off by half a step of its type, eps/2 relative (eps of float32 2^-23, of bfloat16 2^-7), plus 2^-52 relative to the larger
of the two summands for the 64-bit operations before it, plus half the smallest subnormal."""
import numpy as np
import pytest
import torch

from dvq_hip import ops
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows(M, K, dtype, seed, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(spread * torch.randn(M, 1, generator=g))
    return x.to(dtype)


def layer(N, K, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    codes, scale = S.int8_codes(torch.randn(N, K, generator=g) / K ** 0.5)
    return torch.from_numpy(codes.astype(np.int8)), torch.from_numpy(scale), 0.1 * torch.randn(N, generator=g)


def check_output(y, codes, scale, W, t, b, relu):
    ref = S.linear_int8(codes, scale, W.numpy(), t.numpy(), None if b is None else b.numpy(), relu)
    prod = np.abs(S.linear_int8(codes, scale, W.numpy(), t.numpy()))
    size = np.maximum(prod, 0 if b is None else np.abs(b.numpy().astype(np.float64))[None, :])
    got = y.float().cpu().numpy().astype(np.float64)
    tol = torch.finfo(y.dtype).eps / 2 * np.abs(ref) * (1 + 1e-6) + 2.0 ** -51 * size + 2.0 ** -134
    over = np.abs(ref) > float(torch.finfo(y.dtype).max) * (1 + torch.finfo(y.dtype).eps / 4)      # beyond the type: infinite
    assert np.array_equal(got[over], np.sign(ref[over]) * np.inf)
    got, ref, tol = np.where(over, 0.0, got), np.where(over, 0.0, ref), np.where(over, 0.0, tol)
    assert got.shape == ref.shape and np.array_equal(np.isnan(got), np.isnan(ref))
    off = np.abs(got - ref) - tol
    assert np.nanmax(off, initial=-1.0) <= 0, f"worst excess {np.nanmax(off)}"


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 15), (1, 2560), (2, 16), (3, 17), (5, 1037), (16, 64), (17, 2048), (67, 4100), (2, 131071), (1000, 33)])
def test_codes_and_scales_are_the_exact_ones(M, K, dtype):
    x = rows(M, K, dtype, M * 7 + K)
    if K > 8:
        x[0, : K // 2] = (torch.randint(-254, 255, (K // 2,), generator=torch.Generator().manual_seed(K)).float() * 0.5).to(dtype)
        x[0, K // 2:] = 0
        x[0, 0] = 127.0                        # quotients that are halves: ties
    codes, scale = ops.quantize_rows(x.to(DEV))
    ref, ref_scale = S.int8_codes(x)
    assert codes.shape == (M, K) and codes.dtype == torch.int8 and scale.dtype == torch.float32
    assert np.array_equal(codes.cpu().numpy(), ref)
    assert np.array_equal(scale.cpu().numpy(), ref_scale)


def test_quotients_next_to_a_half_round_to_their_own_side():
    """x one 32-bit step below, at and above (k + 1/2) a / 127 for odd and even k and many a."""
    g = torch.Generator().manual_seed(3)
    a = (1 + torch.rand(400, generator=g)).double() * 2.0 ** torch.randint(-60, 60, (400,), generator=g).double()
    a = a.float()
    k = torch.randint(0, 127, (400, 40), generator=g).double()
    mid = ((k + 0.5) * a.double()[:, None] / 127.0).float()
    inf = torch.tensor(float("inf"))
    x = torch.cat([a[:, None], torch.nextafter(mid, -inf), mid, torch.nextafter(mid, inf)], 1)
    codes, _ = ops.quantize_rows(x.to(DEV))
    assert np.array_equal(codes.cpu().numpy(), S.int8_codes(x)[0])


@pytest.mark.parametrize("K", [7, 64, 300, 2560])
@pytest.mark.parametrize("M", [1, 9, 40])
def test_special_rows(M, K):
    """Zeros, infinities, NaN (first, middle and last element), subnormals and the largest values; a bad row spoils itself only."""
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(K))
    specials = [("zero", 0.0), ("inf", float("inf")), ("-inf", float("-inf")), ("nan", float("nan")), ("tiny", 1e-42), ("huge", 3.2e38)]
    W, t, b = layer(70, K, K)
    for i, (_, v) in enumerate(specials):
        y = x.clone()
        m = i % M
        y[m] = v if v == 0.0 else y[m]
        if v == 0.0:
            pass
        elif v == v and abs(v) < 1e-30:
            y[m] = y[m] * v
        elif v == v and abs(v) < float("inf"):
            y[m] = y[m] / y[m].abs().max() * v
        else:
            y[m, (0, K // 2, K - 1)[i % 3]] = v
        codes, scale = ops.quantize_rows(y.to(DEV))
        ref, ref_scale = S.int8_codes(y)
        assert np.array_equal(codes.cpu().numpy(), ref)
        assert np.array_equal(scale.cpu().numpy(), ref_scale, equal_nan=True)
        out = ops.linear_int8(y.to(DEV), W.to(DEV), t.to(DEV), b.to(DEV), relu=True)
        check_output(out, ref, ref_scale, W, t, b, True)
        assert torch.isnan(out[m]).all() == (not np.isfinite(ref_scale[m]))


# ---------------------------------------------------------------------- product
SHAPES = [(1, 1, 1), (1, 16, 1), (1, 2560, 1024), (1, 2048, 6), (2, 15, 55), (3, 100, 64), (4, 64, 65), (8, 1024, 512), (15, 2050, 17),
          (16, 2048, 1024), (17, 31, 33), (31, 1040, 129), (33, 512, 2048), (64, 64, 64), (65, 1037, 501), (100, 48, 200), (128, 128, 128),
          (130, 272, 260), (257, 2560, 300), (300, 1, 300), (513, 144, 55), (700, 1024, 640), (1030, 80, 1030)]


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product_equals_whole_number_arithmetic(M, K, N, dtype, out_dtype):
    x = rows(M, K, dtype, M + K + N)
    W, t, b = layer(N, K, N)
    relu, bias = (M + N) % 2 == 0, (K + N) % 3 != 0
    y = ops.linear_int8(x.to(DEV), W.to(DEV), t.to(DEV), b.to(DEV) if bias else None, relu=relu, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    codes, scale = S.int8_codes(x)
    check_output(y, codes, scale, W, t, b if bias else None, relu)
    # quantised before: the same bits
    pair = ops.quantize_rows(x.to(DEV))
    again = ops.linear_int8(pair, W.to(DEV), t.to(DEV), b.to(DEV) if bias else None, relu=relu, out_dtype=out_dtype)
    assert torch.equal(y, again)


def test_longest_sums_with_the_largest_codes_are_exact():
    """127 * 127 * 131071 and -128 * -128 * 131071 fit 32 bits."""
    K = ops.INT8_MAX_K
    for code in (127, -128):
        c = torch.full((3, K), code, dtype=torch.int8, device=DEV)
        one = torch.ones(3, device=DEV)
        y = ops.linear_int8((c, one), c, one)
        assert (y.double() == float(np.float32(code * code * K))).all()
        y = ops.linear_int8((c[:, :-2], one), c[:, :-2], one)
        assert (y.double() == float(np.float32(code * code * (K - 2)))).all()


@pytest.mark.parametrize("M,K,N", [(5, 37, 70), (70, 96, 130), (300, 512, 256)])
def test_strides_offsets_and_slices(M, K, N):
    """Rows inside wider buffers at any byte offset (x, codes, weights, outputs); what lies beside an output stays."""
    x = rows(M, K, torch.float32, 5)
    W, t, b = layer(N, K, 6)
    codes, scale = S.int8_codes(x)
    wide_x = torch.full((M, K + 13), 1e30, device=DEV)
    wide_x[:, 7:7 + K] = x.to(DEV)
    for off in (0, 1, 3, 16):
        wide_w = torch.full((N, K + 32), 127, dtype=torch.int8, device=DEV)
        wide_w[:, off:off + K] = W.to(DEV)
        wide_c = torch.full((M, K + 21), -127, dtype=torch.int8, device=DEV)
        wide_c[:, off:off + K] = torch.from_numpy(codes.astype(np.int8)).to(DEV)
        out = torch.full((M, N + 9), 5.0, device=DEV)
        y = ops.linear_int8(wide_x[:, 7:7 + K], wide_w[:, off:off + K], t.to(DEV), b.to(DEV), out=out[:, 4:4 + N])
        assert y.data_ptr() == out[:, 4:].data_ptr()
        check_output(y, codes, scale, W, t, b, False)
        assert (out[:, :4] == 5).all() and (out[:, 4 + N:] == 5).all()
        y = ops.linear_int8((wide_c[:, off:off + K], torch.from_numpy(scale).to(DEV)), wide_w[:, off:off + K], t.to(DEV), b.to(DEV))
        check_output(y, codes, scale, W, t, b, False)


def test_broadcast_rows():
    x = rows(1, 100, torch.float32, 9)
    W, t, b = layer(40, 100, 9)
    y = ops.linear_int8(x.to(DEV).expand(50, 100), W.to(DEV)[:1].expand(40, 100), t.to(DEV), b.to(DEV))
    codes, scale = S.int8_codes(x.expand(50, 100))
    check_output(y, codes, scale, W[:1].expand(40, 100), t, b, False)


def test_offsets_beyond_32_bits():
    """Rows of x, codes and out further than 2^31 elements apart."""
    M, K, N, far = 600, 64, 40, 1 << 22
    x = rows(M, K, torch.bfloat16, 11)
    W, t, b = layer(N, K, 11)
    codes, scale = S.int8_codes(x)
    wide = torch.empty(M, far, dtype=torch.bfloat16, device=DEV)
    wide[:, :K] = x.to(DEV)
    out = torch.empty(M, far, dtype=torch.bfloat16, device=DEV)
    out[:, N] = 3.0
    check_output(ops.linear_int8(wide[:, :K], W.to(DEV), t.to(DEV), b.to(DEV), out=out[:, :N]), codes, scale, W, t, b, False)
    assert (out[:, N] == 3.0).all()
    del wide, out
    wide = torch.empty(M, far, dtype=torch.int8, device=DEV)
    wide[:, :K] = torch.from_numpy(codes.astype(np.int8)).to(DEV)
    check_output(ops.linear_int8((wide[:, :K], torch.from_numpy(scale).to(DEV)), W.to(DEV), t.to(DEV), b.to(DEV)), codes, scale, W, t, b, False)


@pytest.mark.parametrize("n,M,K,N,dtype", [(1, 3, 70, 5, torch.float32), (6, 1, 1024, 512, torch.float32), (6, 70, 512, 256, torch.bfloat16),
                                           (8, 300, 129, 77, torch.float32), (6, 512, 1024, 512, torch.float32)])
def test_batched_equals_one_at_a_time(n, M, K, N, dtype):
    xs = [rows(M, K, dtype, i).to(DEV) for i in range(n)]
    layers = [layer(N, K, i) for i in range(n)]
    Ws, ts = [l[0].to(DEV) for l in layers], [l[1].to(DEV) for l in layers]
    bs = [l[2].to(DEV) if i % 3 else None for i, l in enumerate(layers)]
    ys = ops.linear_int8_batched(xs, Ws, ts, bs, relu=True)
    pairs = ops.linear_int8_batched([ops.quantize_rows(x) for x in xs], Ws, ts, bs, relu=True)
    for i in range(n):
        one = ops.linear_int8(xs[i], Ws[i], ts[i], bs[i], relu=True)
        assert torch.equal(ys[i], one) and torch.equal(pairs[i], one)


def test_empty_batches_and_layers():
    W, t, b = (v.to(DEV) for v in layer(7, 20, 1))
    assert ops.linear_int8(torch.empty(0, 20, device=DEV), W, t, b).shape == (0, 7)
    assert ops.linear_int8(torch.ones(3, 20, device=DEV), W[:0], t[:0], b[:0]).shape == (3, 0)
    c, s = ops.quantize_rows(torch.empty(0, 20, device=DEV))
    assert c.shape == (0, 20) and s.shape == (0,)
    assert ops.linear_int8((c, s), W, t, b).shape == (0, 7)


def test_refusals():
    W, t, b = (v.to(DEV) for v in layer(7, 20, 1))
    x = torch.ones(3, 20, device=DEV)
    for call in (lambda: ops.linear_int8(x[:, :19], W, t, b), lambda: ops.linear_int8(x.double(), W, t, b), lambda: ops.linear_int8(x, W.float(), t, b),
                 lambda: ops.linear_int8(x, W, t[:6], b), lambda: ops.linear_int8(x, W, t, b[:6]), lambda: ops.linear_int8(x, W, t.double(), b),
                 lambda: ops.linear_int8(x.T.contiguous().T, W, t, b), lambda: ops.linear_int8(x, W, t, b, out=torch.empty(3, 8, device=DEV)),
                 lambda: ops.linear_int8(x, W, t, b, out=torch.empty(1, 7, device=DEV).expand(3, 7)),
                 lambda: ops.linear_int8(x, W, t, b, out=torch.empty(3, 7, device=DEV, dtype=torch.float16)),
                 lambda: ops.linear_int8(x, W.cpu(), t, b), lambda: ops.linear_int8(x, W, t.cpu(), b), lambda: ops.linear_int8(x[0], W, t, b),
                 lambda: ops.linear_int8((W[:3], t[:2]), W, t, b), lambda: ops.quantize_rows(x[0]), lambda: ops.quantize_rows(x[:, :0]),
                 lambda: ops.quantize_rows(torch.empty(1, 1 << 17, device=DEV)), lambda: ops.quantize_rows(W),
                 lambda: ops.linear_int8_batched([x] * 9, [W] * 9, [t] * 9, [b] * 9),
                 lambda: ops.linear_int8_batched([x, x[:2]], [W, W], [t, t], [b, b]),
                 lambda: ops.linear_int8(x, W, t, b, out=x[:, :7])):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("M", [1, 12, 90, 600])
def test_recorded_in_a_graph_and_replayed(M):
    K, N = 520, 130
    W, t, b = (v.to(DEV) for v in layer(N, K, M))
    x = rows(M, K, torch.float32, 0).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear_int8(x, W, t, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_int8(x, W, t, b)
    for i in range(4):
        x.copy_(rows(M, K, torch.float32, i).to(DEV))
        graph.replay()
        got = y.clone()
        assert torch.equal(got, ops.linear_int8(x, W, t, b))
        torch.cuda.synchronize()


def test_two_streams_at_once():
    K, N = 1024, 512
    W, t, b = (v.to(DEV) for v in layer(N, K, 2))
    xs = [rows(M, K, torch.float32, M).to(DEV) for M in (8, 200)]
    want = [ops.linear_int8(x, W, t, b) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.linear_int8(xs[i], W, t, b))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


# ------------------------------------------------------------------- every tile
# 64 x 64, 128 x 128 and 256 x 256 tiles: tails in rows and channels, k of one stage and less, of an odd number of stages, of
# no whole pieces
TILES = [(700, 64, 650), (450, 1037, 640), (1500, 200, 1400), (1411, 528, 1345), (2048, 16, 1536), (4000, 130, 2100), (8193, 64, 1000), (4099, 304, 2049),
         (2048, 1040, 4096)]


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", TILES)
def test_product_of_many_rows_equals_whole_number_arithmetic(M, K, N, out_dtype):
    x = rows(M, K, torch.float32, M + K + N)
    W, t, b = layer(N, K, N)
    codes, scale = S.int8_codes(x)
    relu = N % 2 == 0
    y = ops.linear_int8(x.to(DEV), W.to(DEV), t.to(DEV), b.to(DEV), relu=relu, out_dtype=out_dtype)
    check_output(y, codes, scale, W, t, b, relu)
    # a row is the same bits alone, among few and among all
    for n in (1, 16, 40, 300):
        assert torch.equal(y[:n], ops.linear_int8(x[:n].to(DEV), W.to(DEV), t.to(DEV), b.to(DEV), relu=relu, out_dtype=out_dtype))
    # columns of a wider buffer, at offsets that 16-byte stores reach and at others; what lies beside them stays
    for left, right in ((8, 8), (3, 4)):
        out = torch.full((M + 2, left + N + right), 5.0, dtype=out_dtype, device=DEV)
        ops.linear_int8(x.to(DEV), W.to(DEV), t.to(DEV), b.to(DEV), relu=relu, out=out[1:-1, left:left + N])
        assert torch.equal(out[1:-1, left:left + N], y)
        assert (out[0] == 5).all() and (out[-1] == 5).all() and (out[:, :left] == 5).all() and (out[:, left + N:] == 5).all()


@pytest.mark.parametrize("M,K,N", [(700, 80, 650), (1500, 200, 1400), (2100, 48, 1100)])
def test_batches_of_many_rows_equal_one_at_a_time(M, K, N):
    xs = [rows(M, K, torch.bfloat16, i).to(DEV) for i in range(8)]
    layers = [layer(N, K, i) for i in range(8)]
    Ws, ts = [l[0].to(DEV) for l in layers], [l[1].to(DEV) for l in layers]
    bs = [l[2].to(DEV) if i % 3 else None for i, l in enumerate(layers)]
    for y, x, W, t, b in zip(ops.linear_int8_batched(xs, Ws, ts, bs, relu=True), xs, Ws, ts, bs):
        assert torch.equal(y, ops.linear_int8(x, W, t, b, relu=True))


def test_rows_and_channels_of_no_finite_scale_in_every_tile():
    for M, K, N in ((450, 96, 640), (1500, 96, 1400), (2048, 96, 4096)):
        x = rows(M, K, torch.float32, M)
        x[5, 3], x[M - 1, K - 1], x[M // 2] = float("nan"), float("inf"), 0.0
        W, t, b = layer(N, K, N)
        t[7], t[N - 1], b[9] = float("nan"), float("inf"), -float("inf")
        codes, scale = S.int8_codes(x)
        check_output(ops.linear_int8(x.to(DEV), W.to(DEV), t.to(DEV), b.to(DEV)), codes, scale, W, t, b, False)


def test_single_rows_and_features_of_any_stride_together():
    """One row's stride and one feature's are nobody's business."""
    W, t, b = layer(40, 70, 2)
    args = [W.to(DEV)] * 3, [t.to(DEV)] * 3, [b.to(DEV)] * 3
    wide = torch.randn(9, 200, generator=torch.Generator().manual_seed(3)).to(DEV)
    xs = [wide[1:2, :70], wide[3:4, 80:150].contiguous(), wide[::4][1:2, 10:80]]
    for y, x in zip(ops.linear_int8_batched(xs, *args), xs):
        assert torch.equal(y, ops.linear_int8(x, W.to(DEV), t.to(DEV), b.to(DEV)))
    with pytest.raises(RuntimeError):
        ops.linear_int8_batched([wide[:2, :70], wide[:2, 70:140].contiguous(), wide[:2, :70]], *args)
    one = layer(40, 1, 4)
    cols = [wide[:, 3:4], wide[:, 5:6].contiguous().t().contiguous().t(), wide[:, 9:10]]
    layers = [one[0].to(DEV)] * 2, [one[1].to(DEV)] * 2, [one[2].to(DEV)] * 2
    for y, x in zip(ops.linear_int8_batched([cols[0], cols[2]], *layers), (cols[0], cols[2])):
        assert torch.equal(y, ops.linear_int8(x.contiguous(), one[0].to(DEV), one[1].to(DEV), one[2].to(DEV)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(17, 4096, 33), (250, 4096, 250), (255, 2571, 241), (257, 2560, 240), (512, 1024, 512), (511, 1009, 497), (528, 1024, 512),
                                   (1000, 70, 256), (4000, 300, 16), (100, 4097, 40)])
def test_rows_quantised_by_every_workgroup_and_once_before(M, K, N, dtype):
    """At, below and above the sizes where a layer of floats is one launch."""
    x = rows(M, K, dtype, M + N)
    x[M // 2] = 0
    x[M - 1, 0] = float("inf")
    W, t, b = layer(N, K, N)
    y = ops.linear_int8(x.to(DEV), W.to(DEV), t.to(DEV), b.to(DEV), relu=True)
    codes, scale = S.int8_codes(x)
    check_output(y, codes, scale, W, t, b, True)
    xs = [x.to(DEV), x.to(DEV).flip(0)]
    for z, want in zip(ops.linear_int8_batched(xs, [W.to(DEV)] * 2, [t.to(DEV)] * 2, [b.to(DEV)] * 2, relu=True), (y, y.flip(0))):
        assert torch.equal(z.nan_to_num(7.0), want.nan_to_num(7.0)) and torch.equal(z.isnan(), want.isnan())


# ------------------------------------------------------------- rounded once
def to_bf16_exactly(v):
    """float64 -> the nearest bfloat16 (ties to even) as float64, in one rounding."""
    m, e = np.frexp(v)
    q = np.exp2(np.maximum(e - 8, -133).astype(np.float64))        # 8 significant bits, no finer than the smallest subnormal
    return np.rint(v / q) * q


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("M,N", [(3, 70), (30, 100), (70, 200), (700, 650), (1500, 1400), (2048, 4096)])
def test_bf16_outputs_are_rounded_once(M, N, relu):
    """Biases on the border of two bfloat16 values, sums that move them off it by less than 32 bits hold: rounded to 32 bits in
    between they would lie on the border again.  Everything up to the rounding is exact in 64 bits."""
    K = 64
    W = torch.zeros(N, K, dtype=torch.int8)
    W[:, 5] = 1
    b = (1 + (2 * (torch.arange(N) % 128) + 1) * 2.0 ** -8) * torch.exp2((torch.arange(N) % 7 - 3).float())
    b[::3] *= -1
    b[1::11] = 5 * 2.0 ** -134                                      # (a border of subnormals)
    t = torch.where(b.abs() < 1e-30, 2.0 ** -120, 1.0)              # (there the sums are a part of the subnormals' step as well)
    codes = torch.zeros(M, K, dtype=torch.int8)
    codes[:, 5] = torch.tensor([1, -1, 0, 1, 1, -1])[torch.arange(M) % 6].to(torch.int8) * 127
    s = torch.full((M,), 2.0 ** -40)
    x = codes.float() * 2.0 ** -40                                  # quantised in the call: the same codes and scales
    want = to_bf16_exactly(codes[:, 5].double().numpy()[:, None] * (s.double().numpy()[:, None] * t.double().numpy()[None, :]) + b.double().numpy()[None, :])
    want = np.where(want < 0, 0.0, want) if relu else want
    dev = [v.to(DEV) for v in (W, t, b)]
    for xs in (x.to(DEV), x.to(torch.bfloat16).to(DEV), (codes.to(DEV), s.to(DEV))):
        y = ops.linear_int8(xs, *dev, relu=relu, out_dtype=torch.bfloat16)
        assert np.array_equal(y.float().cpu().numpy().astype(np.float64), want)
        wide = torch.zeros(M, N + 7, dtype=torch.bfloat16, device=DEV)
        ops.linear_int8(xs, *dev, relu=relu, out=wide[:, 3:3 + N])
        assert torch.equal(wide[:, 3:3 + N], y)
    for y in ops.linear_int8_batched([x.to(DEV)] * 2, [dev[0]] * 2, [dev[1]] * 2, [dev[2]] * 2, relu=relu, out_dtype=torch.bfloat16):
        assert np.array_equal(y.float().cpu().numpy().astype(np.float64), want)
