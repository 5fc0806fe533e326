"""The kernel forms of the product with one 4-bit matrix, row tiles and split K, each by name.

Sizes end inside a tile, a chunk of 128 columns and a block of 32 outputs, K takes each
number of chunks past the last four (what is loaded ahead goes round several times).
Values in 64 bits are the GPU's.  Tolerance as test_gpu_mx4_linear.py has it: K 2^-24 of the
magnitudes (8-bit rows into bf16: and 8 * 2^-13 max |x| max |w| for each eight columns),
the store half a step."""

import pytest
import torch

from tests.test_gpu_mx4_linear import make_rows, make_weights

pytestmark = pytest.mark.gpu

#: kind of rows ("-f32": into f32), a workgroup's rows and columns, T, K, N
CASES = [
    ("bf16", 32, 256, 333, 672, 2064), ("bf16", 32, 256, 1030, 2080, 3088),
    ("bf16", 64, 256, 1000, 672, 4112), ("bf16", 64, 256, 1030, 1376, 6640),
    ("bf16", 128, 256, 2050, 2080, 5136), ("bf16", 128, 256, 4090, 2080, 3088),
    ("mx8", 64, 64, 301, 672, 2064), ("mx8", 64, 64, 600, 1184, 2064),
    ("mx8", 64, 128, 333, 2080, 3088), ("mx8", 64, 128, 600, 672, 5136),
    ("mx8", 128, 128, 1030, 672, 6640), ("mx8", 128, 128, 1030, 1376, 6640),
    ("mx8", 128, 256, 1000, 2080, 4112), ("mx8", 128, 256, 2050, 2080, 2064),
    ("mx8", 256, 256, 2050, 1376, 4112), ("mx8", 256, 256, 4090, 2080, 2064),
    ("mx8-f32", 64, 64, 301, 672, 2064), ("mx8-f32", 64, 64, 333, 1184, 2064),
    ("mx8-f32", 64, 128, 700, 672, 4112), ("mx8-f32", 64, 128, 1000, 2080, 5136),
    ("mx8-f32", 128, 128, 1030, 672, 5136), ("mx8-f32", 128, 128, 1500, 1440, 4112),
    ("mx4", 64, 64, 301, 672, 2064), ("mx4", 64, 64, 700, 1184, 1040),
    ("mx4", 64, 128, 700, 672, 4112), ("mx4", 64, 128, 1000, 1376, 4112),
    ("mx4", 128, 128, 1030, 672, 5136), ("mx4", 128, 128, 1500, 1376, 4112),
    ("mx4", 256, 256, 3001, 1376, 4112), ("mx4", 256, 256, 4090, 2080, 7184),
    ("bf16", 32, 256, 2050, 1440, 7184),  # more than two workgroups a unit
]
#: few rows: a workgroup's waves split K
SPLIT = [(kind, *size) for kind in ("bf16", "mx8", "mx8-f32", "mx4") for size in (
    (16, 32, 13, 1184, 2064), (16, 32, 40, 672, 1040), (16, 64, 40, 672, 4112), (32, 64, 61, 1440, 7184),
    (16, 128, 13, 672, 20016))]
ONE_EACH = CASES[::2] + SPLIT
SCALED = [c for c in ONE_EACH if c[0] != "bf16"]


def _mods():
    from vllm_moe_offload_amd import mxfp4, native

    return mxfp4, native


def _reaches(kind, rows, columns, T, K, N):
    _, native = _mods()
    form = native.mx4_linear_form(kind.removesuffix("-f32"), T, K, N, out_f32=kind.endswith("-f32"))
    assert form == (rows, columns, (kind, rows, columns, T, K, N) in SPLIT)


def _rows(kind, x):
    rows, v = make_rows(x, kind.removesuffix("-f32"))
    return rows, torch.from_numpy(v).cuda()


def _out(kind, T, N):
    return torch.empty((T, N), dtype=torch.float32 if kind.endswith("-f32") else torch.bfloat16, device="cuda")


def check(got, x, w, kind, bias=None, add=None):
    """got against the product of values x and w in 64 bits."""
    y = x @ w.T
    tol = x.abs() @ w.abs().T * (x.shape[1] * 2.0**-24)
    if kind == "mx8":
        eight = lambda v: v.abs().unflatten(1, (-1, 8)).amax(2)
        tol += 8 * 2.0**-13 * (eight(x) @ eight(w).T)
    for extra in (bias, add):
        if extra is not None:
            y = y + extra.double()
            tol = tol + 2.0**-24 * (y.abs() + tol)
    half = 2.0**-8 if got.dtype is torch.bfloat16 else 2.0**-24
    tol = tol + half * (y.abs() + tol)
    off = (got.double() - y).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("kind,rows,columns,T,K,N", CASES + SPLIT)
def test_product(kind, rows, columns, T, K, N):
    _, native = _mods()
    _reaches(kind, rows, columns, T, K, N)
    g = torch.Generator().manual_seed(T + K)
    x, xv = _rows(kind, torch.randn((T, K), generator=g))
    w, wv = make_weights(N, K, N)
    wv = torch.from_numpy(wv).cuda()
    bias = torch.randn(N, generator=g).cuda()
    add = torch.randn((T, N), generator=g).to(torch.bfloat16).cuda()
    room = torch.full((T * N + 64,), 7.0, dtype=_out(kind, 1, 1).dtype, device="cuda")
    out = room[32:-32].view(T, N)
    native.mx4_linear(x, w, out)
    check(out, xv, wv, kind)
    native.mx4_linear(x, w, out, bias=bias, add=add)
    check(out, xv, wv, kind, bias, add)
    assert bool((room[:32] == 7).all()) and bool((room[-32:] == 7).all())


@pytest.mark.parametrize("kind,rows,columns,T,K,N", ONE_EACH)
def test_a_bad_row_stays_its_own(kind, rows, columns, T, K, N):
    """NaN and infinities of one row reach that row alone, wherever in the row they are;
    bad columns of the weights their own columns; rows of zeros are zeros."""
    mxfp4, native = _mods()
    _reaches(kind, rows, columns, T, K, N)
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(T))
    w = torch.randn((N, K), generator=torch.Generator().manual_seed(3)) * 0.05
    w[7, 40], w[N - 2, K - 1] = float("nan"), float("inf")
    bank = mxfp4.pack_w2(*mxfp4.quantize(w)).cuda()
    call = lambda: native.mx4_linear(_rows(kind, x)[0], bank, _out(kind, T, N))
    clean = call()
    keep = torch.tensor([n for n in range(N) if n not in (7, N - 2)], device="cuda")
    assert bool(torch.isnan(clean[:, [7, N - 2]]).all()) and bool(torch.isfinite(clean[:, keep]).all())
    last = (K - 1) // 128 * 128  # the first column of the last chunk, K is no multiple of it
    bad = {T // 3: (3, "nan"), T // 2: (last, "nan"), T // 2 + 1: (K - 1, "nan"), T - 2: (last + 17, "inf"), T - 1: (K - 16, "-inf")}
    for r, (c, v) in bad.items():
        x[r, c] = float(v)
    x[1] = 0.0
    got = call()
    rest = torch.tensor([r for r in range(T) if r not in bad and r != 1], device="cuda")
    assert not bool(torch.isfinite(got[list(bad)][:, keep]).any())
    assert torch.equal(got[rest][:, keep], clean[rest][:, keep])
    assert not bool(got[1, keep].any())


@pytest.mark.parametrize("T,K,N", [(700, 672, 2064), (1000, 2080, 4112), (2050, 1376, 4112)])
def test_a_bad_8_bit_value_stays_in_its_row(T, K, N):
    """A value that is not a number in a group whose scale is one (rows made elsewhere)."""
    _, native = _mods()
    x, _ = _rows("mx8", torch.randn((T, K), generator=torch.Generator().manual_seed(T)))
    w, _ = make_weights(N, K, 3)
    for dtype in (torch.bfloat16, torch.float32):
        call = lambda: native.mx4_linear(x, w, torch.empty((T, N), dtype=dtype, device="cuda"))
        clean = call()
        saved = x.q.clone()
        last = (K - 1) // 128 * 128
        bad = [T // 2, T // 2 + 1, T - 1]
        for r, c in zip(bad, (last, last + 15, K - 1)):
            x.q.view(torch.uint8)[r, c] = 0xFF
        got = call()
        rest = torch.tensor([r for r in range(T) if r not in bad], device="cuda")
        assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[rest], clean[rest])
        x.q.copy_(saved)


@pytest.mark.parametrize("kind,rows,columns,T,K,N", SCALED)
def test_scales_at_any_address(kind, rows, columns, T, K, N):
    _, native = _mods()
    _reaches(kind, rows, columns, T, K, N)
    x, _ = _rows(kind, torch.randn((T, K), generator=torch.Generator().manual_seed(K)))
    w, _ = make_weights(N, K, N)
    want = native.mx4_linear(x, w, _out(kind, T, N))
    for shift in (1, 2, 5, 8):
        room = torch.full((x.scale.numel() + 32,), 255, dtype=torch.uint8, device="cuda")
        sc = room[shift:shift + x.scale.numel()].view(x.scale.shape).copy_(x.scale)
        assert torch.equal(native.mx4_linear(type(x)(x.q, sc), w, _out(kind, T, N)), want)


@pytest.mark.parametrize("kind,rows,columns,T,K,N", SCALED)
def test_extreme_scales(kind, rows, columns, T, K, N):
    """Rows and weights far from one, and groups far from each other: sums stay f32's."""
    mxfp4, native = _mods()
    _reaches(kind, rows, columns, T, K, N)
    g = torch.Generator().manual_seed(4)
    for ex, ew, spread in ((100, -110, 0), (-110, 100, 0), (-60, -60, 0), (0, 0, 6)):
        each = lambda n: torch.randint(-spread, spread + 1, (n, K // 32), generator=g).repeat_interleave(32, dim=1)
        x, xv = _rows(kind, torch.randn((T, K), generator=g) * 2.0**(ex + each(T)))
        codes, scales = mxfp4.quantize(torch.randn((N, K), generator=g) * 2.0**(ew + each(N)))
        wv = mxfp4.dequantize(codes, scales).double().cuda()
        check(native.mx4_linear(x, mxfp4.pack_w2(codes, scales).cuda(), _out(kind, T, N)), xv, wv, kind)


@pytest.mark.parametrize("kind,rows,columns,T,K,N", ONE_EACH)
def test_rows_do_not_depend_on_their_neighbours(kind, rows, columns, T, K, N):
    """A row's bits are the same whatever lies beside it, and wherever in the call it is."""
    _, native = _mods()
    _reaches(kind, rows, columns, T, K, N)
    w, _ = make_weights(N, K, 3)
    g = torch.Generator().manual_seed(T)
    a, b = torch.randn((T, K), generator=g), torch.randn((T, K), generator=g)
    b[T // 2], b[T - 1], b[0] = a[T // 2], a[T // 2], a[T // 2]
    ya, yb = (native.mx4_linear(_rows(kind, t)[0], w, _out(kind, T, N)) for t in (a, b))
    for r in (T // 2, T - 1, 0):
        assert torch.equal(ya[T // 2], yb[r])


def test_shapes_give_the_same_bits():
    """Row tiles add a row's chunks in order, whatever the call's size makes the shape."""
    _, native = _mods()
    K, N = 1376, 4112
    w, _ = make_weights(N, K, 3)
    x = torch.randn((4090, K), generator=torch.Generator().manual_seed(1))
    for kind in ("bf16", "mx8", "mx4", "mx8-f32"):
        forms, first = set(), None
        for T in (300, 600, 1000, 2050, 4090):
            form = native.mx4_linear_form(kind.removesuffix("-f32"), T, K, N, out_f32=kind.endswith("-f32"))
            if form[2]:
                continue
            forms.add(form)
            y = native.mx4_linear(_rows(kind, x[:T])[0], w, _out(kind, T, N))[:300]
            first = y if first is None else first
            assert torch.equal(y, first), (kind, T, form)
        assert len(forms) > 1, (kind, forms)


@pytest.mark.parametrize("kind,rows,columns,T,K,N", ONE_EACH)
def test_captured_and_on_two_streams(kind, rows, columns, T, K, N):
    """One graph replayed on new rows beside a call on another stream: the eager bits."""
    _, native = _mods()
    _reaches(kind, rows, columns, T, K, N)
    w, _ = make_weights(N, K, 5)
    g = torch.Generator(device="cuda").manual_seed(T)
    fresh = lambda: torch.empty((T, K), device="cuda").normal_(generator=g).to(torch.bfloat16)
    name = kind.removesuffix("-f32")
    make = {"bf16": lambda b: b.clone(), "mx8": native.rows_to_mx8, "mx4": native.rows_to_mx4}[name]
    parts = lambda r: (r,) if isinstance(r, torch.Tensor) else (r.q.view(torch.uint8), r.scale)
    x, sx, out, sout = make(fresh()), make(fresh()), _out(kind, T, N), _out(kind, T, N)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        native.mx4_linear(x, w, out)
    for _ in range(3):
        for rows_of in (x, sx):
            for to, new in zip(parts(rows_of), parts(make(fresh()))):
                to.copy_(new)
        want, swant = native.mx4_linear(x, w, _out(kind, T, N)), native.mx4_linear(sx, w, _out(kind, T, N))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            native.mx4_linear(sx, w, sout)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(sout, swant) and bool(want.any())


@pytest.mark.parametrize("kind,rows,columns,T,K,N", [c for c in ONE_EACH if not c[0].endswith("-f32")])
def test_added_in_place(kind, rows, columns, T, K, N):
    """out over add has the bits of out beside it: each value is read before its sum is
    written, by whichever lanes."""
    _, native = _mods()
    _reaches(kind, rows, columns, T, K, N)
    g = torch.Generator().manual_seed(T + N)
    x, _ = _rows(kind, torch.randn((T, K), generator=g))
    w, _ = make_weights(N, K, N)
    add = torch.randn((T, N), generator=g).to(torch.bfloat16).cuda()
    bias = torch.randn(N, generator=g).to(torch.bfloat16).cuda()
    want = native.mx4_linear(x, w, bias=bias, add=add)
    for _ in range(3):
        out = add.clone()
        native.mx4_linear(x, w, out, bias=bias, add=out)
        assert torch.equal(out, want)
