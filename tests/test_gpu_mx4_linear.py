"""The product with one matrix of 4-bit weights against its value in 64 bits.

Tolerance per element: a sum of K products in f32 is off by at most K 2^-24 sum |x| |w|
(8-bit rows: plus what the matrix instruction cuts, 8 * 2^-13 max |x| max |w| for each
eight columns, see test_gpu_mx4.py); bias and add are two more f32 sums, each off by
2^-24 of the sum so far; the store by half a step of its type (2^-8 in bf16)."""

import numpy as np
import pytest
import torch

from tests.test_gpu_mx4 import sum_error

pytestmark = pytest.mark.gpu

ROWS = ("bf16", "mx8", "mx4")
SHAPES = [
    # T, K, N
    (1, 32, 16), (2, 96, 48), (1, 2048, 5120), (16, 1024, 64), (5, 544, 20000), (17, 160, 112), (31, 2048, 768),
    (33, 672, 144), (64, 512, 256), (65, 7168, 80), (129, 1408, 528), (300, 480, 1040), (257, 2080, 768),
    (700, 224, 2064),
]


def _mods():
    from vllm_moe_offload_amd import mxfp4, native

    return mxfp4, native


def make_rows(x, kind):
    """(operand, its values in 64 bits) of rows x in f32."""
    _, native = _mods()
    b = x.to(torch.bfloat16).cuda()
    if kind == "bf16":
        return b, b.double().cpu().numpy()
    rows = native.rows_to_mx8(b) if kind == "mx8" else native.rows_to_mx4(b)
    return rows, rows.float().double().cpu().numpy()


def make_weights(N, K, seed):
    mxfp4, _ = _mods()
    w = torch.randn((N, K), generator=torch.Generator().manual_seed(seed)) * 0.05
    codes, scales = mxfp4.quantize(w)
    return mxfp4.pack_w2(codes, scales).cuda(), mxfp4.dequantize(codes, scales).double().numpy()


def check(got, x, w, kind, bias=None, add=None):
    y = x @ w.T
    tol = sum_error(x, w, kind == "mx8")
    for extra in (bias, add):
        if extra is not None:
            y = y + extra.double().cpu().numpy()
            tol = tol + 2.0**-24 * (np.abs(y) + tol)
    half = 2.0**-8 if got.dtype is torch.bfloat16 else 2.0**-24
    tol = tol + half * (np.abs(y) + tol)
    off = np.abs(got.double().cpu().numpy() - y)
    assert np.all(off <= tol), float((off / tol).max())


@pytest.mark.parametrize("kind", ROWS)
@pytest.mark.parametrize("T,K,N", SHAPES)
def test_product(T, K, N, kind):
    _, native = _mods()
    g = torch.Generator().manual_seed(T * K + N)
    x, xv = make_rows(torch.randn((T, K), generator=g), kind)
    w, wv = make_weights(N, K, K)
    check(native.mx4_linear(x, w), xv, wv, kind)
    bias = torch.randn(N, generator=g).cuda()
    add = torch.randn((T, N), generator=g).to(torch.bfloat16).cuda()
    room = torch.full((T * N + 32,), 7.0, device="cuda")
    out = room[16:-16].view(T, N)
    assert native.mx4_linear(x, w, out, bias=bias, add=add) is out
    check(out, xv, wv, kind, bias, add)
    assert bool((room[:16] == 7).all()) and bool((room[-16:] == 7).all())
    half = bias.to(torch.bfloat16)
    check(native.mx4_linear(x, w, bias=half), xv, wv, kind, half)
    room = torch.full((T * N + 32,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = room[16:-16].view(T, N).copy_(add)
    native.mx4_linear(x, w, out, add=out)  # in place
    check(out, xv, wv, kind, None, add)
    assert bool((room[:16] == 7).all()) and bool((room[-16:] == 7).all())


@pytest.mark.parametrize("kind", ROWS)
@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_a_bad_row_stays_its_own(T, kind):
    """NaN and infinities of one row reach that row alone, and bad columns of the weights
    their own columns; rows of zeros are zeros."""
    mxfp4, native = _mods()
    K, N = 672, 144
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(T))
    w = torch.randn((N, K), generator=torch.Generator().manual_seed(3)) * 0.05
    w[7, 40] = float("nan")
    codes, scales = mxfp4.quantize(w)
    bank = mxfp4.pack_w2(codes, scales).cuda()
    clean = native.mx4_linear(make_rows(x, kind)[0], bank)
    x[-1, 3] = float("nan")
    got = native.mx4_linear(make_rows(x, kind)[0], bank)
    assert bool(torch.isnan(got[:, 7]).all()) and bool(torch.isnan(got[-1]).all())
    keep = torch.arange(N) != 7
    assert torch.equal(got[:-1, keep], clean[:-1, keep]) and not bool(torch.isnan(clean[:, keep]).any())
    x[-1] = 0.0
    got = native.mx4_linear(make_rows(x, kind)[0], bank)
    assert not bool(got[-1, keep].any())


@pytest.mark.parametrize("kind", ["mx8", "mx4"])
@pytest.mark.parametrize("T,K,N", [(1, 160, 32), (9, 544, 64), (50, 1056, 80), (300, 672, 272)])
def test_scales_at_any_address(T, K, N, kind):
    _, native = _mods()
    x, xv = make_rows(torch.randn((T, K), generator=torch.Generator().manual_seed(K)), kind)
    w, wv = make_weights(N, K, N)
    want = native.mx4_linear(x, w)
    check(want, xv, wv, kind)
    for shift in (1, 2, 5, 8):
        room = torch.full((x.scale.numel() + 32,), 255, dtype=torch.uint8, device="cuda")
        sc = room[shift:shift + x.scale.numel()].view(x.scale.shape).copy_(x.scale)
        assert torch.equal(native.mx4_linear(type(x)(x.q, sc), w), want)


@pytest.mark.parametrize("kind", ["mx8", "mx4"])
def test_extreme_scales(kind):
    """Sums stay f32's: largest rows by smallest weights, and the other way round."""
    mxfp4, native = _mods()
    T, K, N = 20, 256, 32
    g = torch.Generator().manual_seed(4)
    for ex, ew in ((100, -110), (-110, 100), (-60, -60), (60, 60)):
        x, xv = make_rows(torch.randn((T, K), generator=g) * 2.0**ex, kind)
        codes, scales = mxfp4.quantize(torch.randn((N, K), generator=g) * 2.0**ew)
        wv = mxfp4.dequantize(codes, scales).double().numpy()
        out = torch.empty((T, N), device="cuda")
        native.mx4_linear(x, mxfp4.pack_w2(codes, scales).cuda(), out)
        check(out, xv, wv, kind)


@pytest.mark.parametrize("kind", ROWS)
def test_outputs_past_32_bits(kind):
    """More than 2^31 outputs: the last rows are those of a small call."""
    _, native = _mods()
    T, K, N = 70_016, 32, 32_768
    g = torch.Generator().manual_seed(5)
    last = torch.randn((40, K), generator=g)
    x = torch.zeros((T, K))
    x[-40:] = last
    w, wv = make_weights(N, K, 1)
    rows, _ = make_rows(x, kind)
    out = native.mx4_linear(rows, w)
    _, lv = make_rows(last, kind)
    check(out[-40:], lv, wv, kind)
    assert not bool(out[:100].any())


def test_many_rows():
    """More row blocks than a grid's second dimension has."""
    _, native = _mods()
    T = 65_536 * 32 + 5
    x = torch.zeros((T, 32), dtype=torch.bfloat16, device="cuda")
    x[-7:] = 1.0
    w, wv = make_weights(16, 32, 1)
    for rows in (x, native.rows_to_mx4(x)):
        out = native.mx4_linear(rows, w)
        check(out[-7:], np.ones((7, 32)), wv, "bf16")
        assert not bool(out[:-7].any())


def test_empty_and_refused():
    mxfp4, native = _mods()
    w, _ = make_weights(48, 64, 1)
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    assert native.mx4_linear(x[:0], w).shape == (0, 48)
    assert native.mx4_linear(native.Mx4Rows.allocate(0, 64, "cuda"), w).shape == (0, 48)
    for bad in (x.float(), x.cpu(), x[0], torch.zeros((4, 128), dtype=torch.bfloat16, device="cuda")[:, ::2], None,
                torch.zeros((4, 192), dtype=torch.bfloat16, device="cuda"), native.Mx4Rows.allocate(4, 192, "cuda"),
                native.Mx4Rows(x, x), native.Mx4Rows(native.rows_to_mx4(x).q, native.rows_to_mx4(x).scale[:2])):
        with pytest.raises((ValueError, TypeError)):
            native.mx4_linear(bad, w)
    for bad in (w.unsqueeze(0), w[:24], w.float(), w.cpu(), None):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            native.mx4_linear(x, bad)
    for kw in (dict(out=torch.empty((4, 48), dtype=torch.float16, device="cuda")), dict(out=torch.empty((4, 32), device="cuda")),
               dict(bias=torch.zeros(32, device="cuda")), dict(bias=torch.zeros((1, 48), device="cuda")),
               dict(bias=torch.zeros(48, dtype=torch.float64, device="cuda")), dict(add=torch.zeros((4, 48), device="cuda")),
               dict(add=torch.zeros((48, 4), dtype=torch.bfloat16, device="cuda").t())):
        with pytest.raises(ValueError):
            native.mx4_linear(x, w, **kw)
    square, _ = make_weights(64, 64, 1)
    with pytest.raises(ValueError, match="overlap"):
        native.mx4_linear(x, square, x)
    buf = torch.zeros((5, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        native.mx4_linear(x, square, buf[1:], add=buf[:4])


@pytest.mark.parametrize("T", [1, 16, 40, 300])
def test_a_run_of_them_captured_and_replayed(T):
    """Norm to 4 bits, projection, the residual's addition, rows to 4 bits again and a
    head: one graph, replayed on new rows, gives the eager bits; calls on two streams at
    once too."""
    _, native = _mods()
    H, N, V = 544, 320, 1040
    g = torch.Generator().manual_seed(T)
    w1, _ = make_weights(H, H, 1)
    w2, _ = make_weights(V, H, 2)
    weight = torch.rand(H, generator=g).to(torch.bfloat16).cuda()
    bias = torch.randn(H, generator=g).cuda()

    def step(x, mx4, mid, logits):
        native.add_rms_norm(x, weight, mx4=mx4)
        native.mx4_linear(mx4, w1, mid, bias=bias, add=x)
        native.rows_to_mx4(mid, mx4)
        return native.mx4_linear(mx4, w2, logits)

    def bufs():
        return (native.Mx4Rows.allocate(T, H, "cuda"), torch.empty((T, H), dtype=torch.bfloat16, device="cuda"),
                torch.empty((T, V), device="cuda"))

    x, b = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda"), bufs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(x, *b)
    side, sx, sb = torch.cuda.Stream(), torch.empty_like(x), bufs()
    for _ in range(3):
        x.copy_(torch.randn((T, H), generator=g).to(torch.bfloat16))
        sx.copy_(torch.randn((T, H), generator=g).to(torch.bfloat16))
        want, swant = step(x, *bufs()).clone(), step(sx, *bufs()).clone()
        assert bool(want.any())
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(sx, *sb)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b[2], want) and torch.equal(sb[2], swant)


@pytest.mark.parametrize("kind", ROWS)
def test_rows_do_not_depend_on_their_neighbours(kind):
    """A row's bits are the same whatever lies beside it in a call of as many rows."""
    _, native = _mods()
    w, _ = make_weights(272, 672, 3)
    for T in (3, 16, 33, 130, 300):
        g = torch.Generator().manual_seed(T)
        a = torch.randn((T, 672), generator=g)
        b = torch.randn((T, 672), generator=g)
        b[T // 2] = a[T // 2]
        ya, yb = (native.mx4_linear(make_rows(t, kind)[0], w) for t in (a, b))
        assert torch.equal(ya[T // 2], yb[T // 2])


@pytest.mark.parametrize("kind", ["mx8", "mx4"])
@pytest.mark.parametrize("T,K,N", [(4090, 672, 4112), (1000, 2080, 7184), (500, 2080, 7184), (2050, 544, 2064)])
def test_tall_products(T, K, N, kind):
    """Enough of both for the tiles of 128 and 256, with ends inside a tile and a chunk."""
    _, native = _mods()
    x, xv = make_rows(torch.randn((T, K), generator=torch.Generator().manual_seed(T)), kind)
    w, wv = make_weights(N, K, N)
    check(native.mx4_linear(x, w), xv, wv, kind)
