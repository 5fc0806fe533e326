"""Rows and weights to 4 bits and back.

Quantisation is exact: from the definition (scales are powers of two, so v / 2^e is
exact, and the nearest value is a comparison), codes, scales and the bank's bytes are
those of mxfp4.quantize and pack_w13 / pack_w2 on the CPU, which tests/test_mx_formats.py
holds against the 64-bit oracle.  Only the norm has a tolerance."""

import numpy as np
import pytest
import torch

from oracle import mx

pytestmark = pytest.mark.gpu


def _mods():
    from vllm_moe_offload_amd import mxfp4, native

    return mxfp4, native


def _bits(n, seed, dtype):
    """Random bit patterns: every exponent, subnormals, NaN and infinities."""
    g = torch.Generator().manual_seed(seed)
    if dtype is torch.bfloat16:
        return torch.randint(-2**15, 2**15, (n,), generator=g, dtype=torch.int16).view(torch.bfloat16)
    return torch.randint(-2**31, 2**31 - 1, (n,), generator=g, dtype=torch.int32).view(torch.float32)


def _borders(dtype):
    """Groups around every border between two codes, at every scale that dtype has: the
    border and its neighbours on either side, with 6 or 5 as the group's largest."""
    one = []
    for b in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
        t = torch.tensor([b, b], dtype=dtype)
        up = torch.nextafter(t, torch.full_like(t, 9.0)) if dtype is torch.float32 else t + t * 2.0**-7
        dn = torch.nextafter(t, torch.zeros_like(t)) if dtype is torch.float32 else t - t * 2.0**-8
        one += [b, -b, float(up[0]), float(dn[0])]
    one = torch.tensor(one + [6.0, 3.0, -0.0, 0.0], dtype=torch.float64)
    rows = [one * 2.0**e for e in range(-150, 126)]
    rows.append(torch.tensor([4.5] * 16 + [-5.75, 3.25] * 8, dtype=torch.float64))
    return torch.stack(rows).to(dtype)


def _equal(got, codes, scales):
    assert torch.equal(got.scale.cpu(), scales)
    assert torch.equal(got.q.cpu(), codes)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 32), (3, 96), (1, 2048), (257, 160), (64, 7168), (5, 40000)])
def test_rows_are_the_definitions(T, H, dtype):
    mxfp4, native = _mods()
    x = (torch.randn((T, H), generator=torch.Generator().manual_seed(T + H)) * 3).to(dtype)
    x[0, :32] = 0
    _equal(native.rows_to_mx4(x.cuda()), *mxfp4.quantize(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_any_bits(dtype):
    mxfp4, native = _mods()
    if dtype is torch.bfloat16:  # every value, beside 31 others
        x = torch.arange(-2**15, 2**15, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
        x = torch.cat([x[torch.randperm(2**16, generator=torch.Generator().manual_seed(s))] for s in range(8)]).view(-1, 256)
    else:
        x = _bits(1 << 20, 5, dtype).view(-1, 256)
    # patterns of one binade, so that all codes come up
    y = _bits(1 << 18, 6, dtype).float()
    m, _ = torch.frexp(torch.where(torch.isfinite(y), y, torch.ones_like(y)))
    y = (m * 2.0 ** torch.randint(-4, 4, m.shape, generator=torch.Generator().manual_seed(1))).to(dtype).view(-1, 256)
    z = _bits(1 << 14, 7, dtype) * 0.0  # zeros of either sign, NaN
    tiny = torch.ldexp(y[:16].float(), torch.tensor(-127)).to(dtype)  # subnormal numbers
    x = torch.cat([x, y, z.view(-1, 256), tiny])
    codes, scales = mxfp4.quantize(x)
    assert (scales == 255).any() and (scales == 0).any() and len(torch.unique(codes & 15)) == 16
    _equal(native.rows_to_mx4(x.cuda()), codes, scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_borders_between_codes(dtype):
    mxfp4, native = _mods()
    x = _borders(dtype)
    got = native.rows_to_mx4(x.cuda())
    _equal(got, *mxfp4.quantize(x))
    codes, scales = mx.quantize_mx4(x.double().numpy())  # the definition in 64 bits
    assert np.array_equal(got.scale.cpu().numpy(), scales)
    assert np.array_equal(got.q.cpu().numpy(), codes)


SHAPES = [(1, 16, 32), (3, 16, 96), (2, 64, 128), (1, 64, 160), (5, 192, 480), (2, 128, 512), (3, 64, 544),
          (1, 320, 1056), (4, 1536, 2048), (2, 112, 7168)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gate_up", [False, True])
@pytest.mark.parametrize("E,N,K", SHAPES)
def test_banks_are_the_definitions(E, N, K, gate_up, dtype):
    mxfp4, native = _mods()
    if gate_up and N % 64:
        N = 64
    w = (torch.randn((E, N, K), generator=torch.Generator().manual_seed(N + K)) * 0.05).to(dtype)
    w[0, 0, :32] = 0
    w[-1, -1, -32:] = _bits(32, 3, dtype)
    w[0, 1, 5] = float("nan")
    want = (mxfp4.pack_w13 if gate_up else mxfp4.pack_w2)(*mxfp4.quantize(w))
    room = torch.full((want.numel() + 512,), 77, dtype=torch.uint8, device="cuda")
    bank = room[256:-256].view(want.shape)
    got = native.quantize_mx4(w.cuda(), bank, gate_up=gate_up)
    assert got is bank and torch.equal(bank.cpu(), want)
    assert bool((room[:256] == 77).all()) and bool((room[-256:] == 77).all())
    assert torch.equal(native.quantize_mx4(w.cuda(), gate_up=gate_up).cpu(), want)
    # one matrix without an expert's dimension
    assert torch.equal(native.quantize_mx4(w[0].cuda(), gate_up=gate_up).cpu(), want[0])


def _same_values(got, want):
    """Bit for bit, NaN as NaN."""
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], want[~nan])
    assert torch.equal(torch.signbit(got[~nan]), torch.signbit(want[~nan]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_of_every_code_and_scale(dtype):
    mxfp4, native = _mods()
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)  # [256, 512 columns]
    scales = torch.arange(256, dtype=torch.uint8).unsqueeze(1).repeat(1, 16)
    rows = native.Mx4Rows(codes.cuda(), scales.cuda())
    out = torch.empty((256, 512), dtype=dtype, device="cuda")
    # in 64 bits: 2^128 and past it becomes an infinity of either type
    v = mx.values_mx4(codes.numpy(), scales.numpy())
    v[255] = np.nan
    with np.errstate(over="ignore"):
        want = torch.from_numpy(v.astype(np.float32)).to(dtype)
    _same_values(native.mx4_values(rows, out).cpu(), want)
    bank = mxfp4.pack_w2(codes, scales).cuda()
    _same_values(native.mx4_values(bank, out).cpu(), want)
    bank = mxfp4.pack_w13(codes, scales).cuda()
    _same_values(native.mx4_values(bank, out, gate_up=True).cpu(), want)


@pytest.mark.parametrize("gate_up", [False, True])
@pytest.mark.parametrize("E,N,K", SHAPES)
def test_values_of_banks(E, N, K, gate_up):
    mxfp4, native = _mods()
    if gate_up and N % 64:
        N = 64
    w = torch.randn((E, N, K), generator=torch.Generator().manual_seed(N + K)) * 0.05
    codes, scales = mxfp4.quantize(w)
    bank = (mxfp4.pack_w13 if gate_up else mxfp4.pack_w2)(codes, scales).cuda()
    want = mxfp4.dequantize(codes, scales)
    _same_values(native.mx4_values(bank, columns=K, gate_up=gate_up).float().cpu(), want)
    room = torch.full((want.numel() + 32,), 7.0, device="cuda")
    out = room[16:-16].view(want.shape)
    _same_values(native.mx4_values(bank, out, gate_up=gate_up).cpu(), want)
    assert bool((room[:16] == 7).all()) and bool((room[-16:] == 7).all())


def test_pack_experts_on_the_gpu_is_that_of_the_cpu():
    mxfp4, _ = _mods()
    g = torch.Generator().manual_seed(2)
    for dtype in (torch.bfloat16, torch.float32, torch.float16):
        w13 = (torch.randn((3, 128, 160), generator=g) * 0.1).to(dtype)
        w2 = (torch.randn((3, 160, 64), generator=g) * 0.1).to(dtype)
        want = mxfp4.pack_experts(w13, w2)
        got = mxfp4.pack_experts(w13.cuda(), w2.cuda())
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)), dtype
        # weights whose strides the kernel does not take
        got = mxfp4.pack_experts(w13.cuda().transpose(1, 2).contiguous().transpose(1, 2), w2.cuda())
        assert torch.equal(got[0].cpu(), want[0])


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H", [(1, 32), (3, 160), (17, 2048), (5, 7168), (2, 32768)])
def test_norm_to_4_bits(T, H, residual):
    """y in f32 is off by at most d = (H + 8) 2^-24 |y| (the sum of squares, halved by the
    root, then a root, a division and two products), so a group's scale is that of a
    largest magnitude within d, and a code's value is within half a step of some y within
    d: the codes' steps are 0.5 up to 2, then 1 up to 4, then 2, times the scale."""
    mxfp4, native = _mods()
    g = torch.Generator().manual_seed(T * H)
    x = torch.randn((T, H), generator=g).to(torch.bfloat16)
    w = torch.rand(H, generator=g).to(torch.bfloat16) + 0.5
    r = None if residual is None else (torch.randn((T, H), generator=g) * 4).to(residual)
    mx4 = native.Mx4Rows.allocate(T, H, "cuda")
    out = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
    res = None if r is None else r.cuda()
    res_out = None if r is None else torch.empty_like(res)
    ret = native.add_rms_norm(x.cuda(), w.cuda(), residual=res, residual_out=res_out, out=out, mx4=mx4)
    assert ret[0] is out and ret[1] is mx4 and ret[2] is res_out
    # the other outputs are those of the norm without 4-bit rows
    plain = native.add_rms_norm(x.cuda(), w.cuda(), residual=None if r is None else r.cuda(),
                                residual_out=None if r is None else torch.empty_like(res))
    assert torch.equal(plain[0].view(torch.int16), out.view(torch.int16))
    s = x.double().numpy() + (0.0 if r is None else r.double().numpy())
    y = mx.rms_norm(s.astype(np.float32).astype(np.float64), w.double().numpy(), 1e-6)
    d = (H + 8) * 2.0**-24 * np.abs(y)
    e = mx4.scale.cpu().numpy().astype(np.int64) - 127
    lo, hi = (mx.group_exponents(np.abs(y) + k * d, 6.0) for k in (-1, 1))
    assert np.all((e >= lo) & (e <= hi))
    scale = np.ldexp(1.0, np.repeat(e, 32, axis=1))
    got = mx4.float().cpu().double().numpy()
    a = np.abs(y) / scale + d / scale
    half = np.where(a <= 2, 0.25, np.where(a <= 4, 0.5, 1.0)) * scale
    assert np.all(np.abs(got - y) <= half * (1 + 2.0**-40) + d)


def test_norm_refuses():
    _, native = _mods()
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    mx4, mx8 = native.Mx4Rows.allocate(4, 64, "cuda"), native.Mx8Rows.allocate(4, 64, "cuda")
    with pytest.raises(ValueError, match="not both"):
        native.add_rms_norm(x, w, mx4=mx4, mx8=mx8)
    with pytest.raises(TypeError):
        native.add_rms_norm(x, w, mx4=mx8)
    with pytest.raises(TypeError):
        native.add_rms_norm(x, w, mx8=mx4)
    with pytest.raises(ValueError):
        native.add_rms_norm(x, w, mx4=native.Mx4Rows.allocate(4, 96, "cuda"))
    over = native.Mx4Rows(x.view(torch.uint8).view(-1)[: 4 * 32].view(4, 32), mx4.scale)
    with pytest.raises(ValueError, match="overlap"):
        native.add_rms_norm(x, w, mx4=over)
    with pytest.raises(ValueError, match="overlap"):
        native.add_rms_norm(x, w, out=x, mx4=native.Mx4Rows(mx4.q, mx4.q.view(-1)[4:12].view(4, 2)))
    x40 = torch.zeros((4, 40), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        native.add_rms_norm(x40, torch.ones(40, dtype=torch.bfloat16, device="cuda"), mx4=mx4)


def test_empty_and_refused():
    mxfp4, native = _mods()
    assert native.rows_to_mx4(torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")).shape == (0, 64)
    assert native.mx4_values(native.Mx4Rows.allocate(0, 64, "cuda")).shape == (0, 64)
    assert native.quantize_mx4(torch.empty((0, 64, 64), device="cuda")).shape == (0, 64, mxfp4.row_bytes(64))
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    for bad in (x[:, :32], x.half(), x.cpu(), x[0], torch.zeros((4, 48), dtype=torch.bfloat16, device="cuda"), None):
        with pytest.raises((ValueError, TypeError)):
            native.rows_to_mx4(bad)
    with pytest.raises(TypeError):
        native.rows_to_mx4(x, native.Mx8Rows.allocate(4, 64, "cuda"))
    with pytest.raises(ValueError):
        native.rows_to_mx4(x, native.Mx4Rows.allocate(5, 64, "cuda"))
    with pytest.raises(ValueError, match="overlap"):
        native.rows_to_mx4(x, native.Mx4Rows(x.view(torch.uint8).view(-1)[:128].view(4, 32),
                                             torch.empty((4, 2), dtype=torch.uint8, device="cuda")))
    w = torch.zeros((2, 64, 64), dtype=torch.bfloat16, device="cuda")
    for bad in (w.transpose(1, 2), w.half(), w.cpu(), w[0, 0], w[..., :48].contiguous(), None):
        with pytest.raises((ValueError, RuntimeError)):
            native.quantize_mx4(bad)
    with pytest.raises(RuntimeError):
        native.quantize_mx4(w[:, :24].contiguous())
    with pytest.raises(RuntimeError):
        native.quantize_mx4(w[:, :32].contiguous(), gate_up=True)
    bank = native.quantize_mx4(w)
    with pytest.raises(ValueError):
        native.quantize_mx4(w, bank[:1])
    with pytest.raises(ValueError):
        native.mx4_values(bank)
    with pytest.raises(ValueError):
        native.mx4_values(bank, columns=640)
    with pytest.raises(ValueError):
        native.mx4_values(bank, torch.empty((2, 64, 64), dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError):
        native.mx4_values(bank, torch.empty((2, 32, 64), device="cuda"))
    with pytest.raises(ValueError):
        native.mx4_values(native.rows_to_mx4(x), columns=32)


def test_rows_past_32_bits():
    """Offsets past 2^31 values, and past 2^32 bytes of the f32 values."""
    mxfp4, native = _mods()
    T, H = 300_100, 7168  # 2.15e9 values
    x = torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn((3, H), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    got = native.rows_to_mx4(x)
    codes, scales = mxfp4.quantize(x[-4:].cpu())
    assert torch.equal(got.q[-4:].cpu(), codes) and torch.equal(got.scale[-4:].cpu(), scales)
    del x
    out = native.mx4_values(got, torch.empty((T, H), device="cuda"))
    assert torch.equal(out[-4:].cpu(), mxfp4.dequantize(codes, scales))


def test_a_bank_past_32_bits():
    mxfp4, native = _mods()
    E, N, K = 90, 4096, 7168  # 2.6e9 weights
    w = torch.zeros((E, N, K), dtype=torch.bfloat16, device="cuda")
    w[-1, -64:] = (torch.randn((64, K), generator=torch.Generator().manual_seed(1)) * 0.02).to(torch.bfloat16).cuda()
    bank = native.quantize_mx4(w)
    want = mxfp4.pack_w2(*mxfp4.quantize(w[-1, -64:].cpu()))
    assert torch.equal(bank[-1, -64:].cpu(), want)
    values = native.mx4_values(bank, w)
    assert torch.equal(values[-1, -64:].float().cpu(), mxfp4.dequantize(*mxfp4.unpack_w2(want, K)))
    assert not bool(values[0].any()) and not bool(values[-1, :-64].any())


def test_captured_and_replayed_on_another_stream():
    mxfp4, native = _mods()
    g = torch.Generator().manual_seed(9)
    x = torch.empty((33, 544), dtype=torch.bfloat16, device="cuda")
    w = torch.empty((2, 64, 544), device="cuda")
    mx4, bank = native.Mx4Rows.allocate(33, 544, "cuda"), native.quantize_mx4(w.zero_())
    back, wback = torch.empty_like(x), torch.empty_like(w)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        native.mx4_values(native.rows_to_mx4(x, mx4), back)
        native.mx4_values(native.quantize_mx4(w, bank, gate_up=True), wback, gate_up=True)
    for _ in range(3):
        hx, hw = torch.randn((33, 544), generator=g).to(torch.bfloat16), torch.randn((2, 64, 544), generator=g)
        x.copy_(hx)
        w.copy_(hw)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(back.float().cpu(), mxfp4.dequantize(*mxfp4.quantize(hx)))
        assert torch.equal(wback.cpu(), mxfp4.dequantize(*mxfp4.quantize(hw)))
    # outputs that a call makes under stream= come from that stream's pool
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    rows = native.rows_to_mx4(x, stream=side)
    vals = native.mx4_values(rows, stream=side)
    side.synchronize()
    assert torch.equal(vals.float().cpu(), mxfp4.dequantize(*mxfp4.quantize(hx)))
