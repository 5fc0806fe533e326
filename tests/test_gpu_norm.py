"""The residual's addition and root-mean-square norm, and rows in 8 bits,
against the formula in 64 bits.

Tolerances.  r = x + residual is one f32 addition: 2^-24 |r|.  The sum of
squares adds at most 32 terms per thread, then 6 and 16 steps: under 64
roundings, so the root's reciprocal is off by at most 32 * 2^-24 and its own
few; y takes two more products: 2^-18 |y| in all.  bf16 adds half a step, 2^-8
relative; e4m3 2^-4 relative or half its smallest step, 2^-10 of the scale."""

import numpy as np
import pytest
import torch

from oracle import mx

F32 = 2.0**-18


def _native():
    from vllm_moe_offload_amd import native

    return native


def _f64(t):
    return t.detach().cpu().double().numpy()


def check_mx8(rows, y):
    """MX8 rows against their unrounded values y (64 bits, off by F32)."""
    q, s = rows.q.float().cpu().double().numpy(), rows.scale.cpu().numpy().astype(np.int64) - 127
    want = mx.group_exponents(y, 448.0)
    amax = np.abs(y).reshape(y.shape[0], -1, 32).max(axis=2)
    border = np.abs(amax / (448.0 * np.ldexp(1.0, s)) - 1.0) < F32
    border |= np.abs(amax / (224.0 * np.ldexp(1.0, s)) - 1.0) < F32
    assert np.all((s == want) | border)
    assert np.max(np.abs(q), initial=0.0) <= 448.0
    scale = np.repeat(np.ldexp(1.0, s), 32, axis=1)
    err = np.abs(q * scale - y)
    assert np.all(err <= np.maximum(2.0**-4 * np.abs(y), 2.0**-10 * scale) + F32 * np.abs(y))


def _case(T, H, res, wdt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty((T, H), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    r = None
    if res is not None:
        r = (torch.empty((T, H), device="cuda").normal_(0, 3, generator=g)).to(res)
        r[:, :: max(1, H // 3)] *= 40
    w = torch.empty(H, device="cuda").uniform_(0.5, 1.5, generator=g).to(wdt)
    return x, r, w


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,res,wdt,out,mx8", [
    (1, 2048, torch.bfloat16, torch.bfloat16, True, False),
    (1, 32, None, torch.bfloat16, True, True),
    (3, 8, torch.float32, torch.float32, True, False),
    (7, 40, torch.bfloat16, torch.float32, True, False),       # a row of five threads
    (5, 512, torch.bfloat16, torch.bfloat16, False, True),
    (17, 544, torch.float32, torch.bfloat16, True, True),
    (33, 2880, torch.bfloat16, torch.bfloat16, True, True),
    (300, 2048, torch.bfloat16, torch.bfloat16, True, True),
    (65, 7168, torch.float32, torch.bfloat16, True, True),
    (2, 8192, None, torch.float32, True, True),                # a full workgroup
    (2, 8224, torch.bfloat16, torch.bfloat16, True, True),     # two steps per thread, the second short
    (3, 16416, torch.float32, torch.bfloat16, True, True),     # three steps
    (2, 32768, torch.bfloat16, torch.bfloat16, True, True),    # the longest row
])
def test_norm_is_the_formula(T, H, res, wdt, out, mx8):
    native = _native()
    print(f"case norm T={T} H={H} {res} {wdt}", flush=True)
    x, r, w = _case(T, H, res, wdt, T * 31 + H)
    ro = torch.full_like(r, 7.0) if r is not None else None
    o = torch.full_like(x, 7.0) if out else None
    m = native.Mx8Rows.allocate(T, H, "cuda") if mx8 else None
    got = native.add_rms_norm(x, w, residual=r, residual_out=ro, out=o, mx8=m, eps=1e-5)
    assert got[0] is o and got[1] is m and got[2] is ro
    rr = _f64(x) + (_f64(r) if r is not None else 0.0)
    y = mx.rms_norm(rr, _f64(w), 1e-5)
    if r is not None:
        tol = 2.0**-24 if res == torch.float32 else 2.0**-8 + 2.0**-24
        assert np.all(np.abs(_f64(ro) - rr) <= tol * np.abs(rr))
    if out:
        assert np.all(np.abs(_f64(o) - y) <= (2.0**-8 + F32) * np.abs(y))
    if mx8:
        check_mx8(m, y)
        assert torch.equal(m.float(), m.q.float() * torch.repeat_interleave(
            torch.exp2(m.scale.float() - 127), 32, dim=1))


@pytest.mark.gpu
def test_norm_in_place_and_defaults():
    native = _native()
    x, r, w = _case(9, 1056, torch.bfloat16, torch.bfloat16, 3)
    want, _, ro = native.add_rms_norm(x, w, residual=r, residual_out=torch.empty_like(r))
    x2, r2 = x.clone(), r.clone()
    out, m, r3 = native.add_rms_norm(x2, w, residual=r2, out=x2)
    assert out is x2 and m is None and r3 is r2
    assert torch.equal(x2, want) and torch.equal(r2, ro)
    y, _, none = native.add_rms_norm(x, w)
    assert none is None and y.dtype == torch.bfloat16


@pytest.mark.gpu
def test_rows_of_zeros_tiny_and_not_a_number():
    """A row of zeros is zeros; a NaN or an infinity reaches its own row (its
    own group, where rows are only rounded) and no other."""
    native = _native()
    x, r, w = _case(6, 256, torch.bfloat16, torch.bfloat16, 5)
    x[1], r[1] = 0, 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    x[4] = 1e-30
    r[4] = 0
    m = native.Mx8Rows.allocate(6, 256, "cuda")
    o, _, _ = native.add_rms_norm(x, w, residual=r, residual_out=torch.empty_like(r), out=torch.empty_like(x), mx8=m)
    v = m.float()
    assert not o[1].any() and not v[1].any()
    assert o[2].isnan().all() and v[2].isnan().all()
    assert o[3, 9].isnan() and v[3, :32].isnan().all()
    y = mx.rms_norm(_f64(x[4:5]), _f64(w), 1e-6)  # 1e-30 / 1e-3
    assert np.all(np.abs(_f64(o[4:5]) - y) <= (2.0**-8 + F32) * np.abs(y))
    for t in (0, 5):
        assert o[t].isfinite().all() and v[t].isfinite().all()
    z = torch.zeros((3, 96), dtype=torch.bfloat16, device="cuda")
    z[0, 40], z[1, 70], z[2, 3] = float("nan"), float("-inf"), 2.0**-133  # the smallest bf16
    f = native.rows_to_mx8(z).float()
    assert f[0, 32:64].isnan().all() and not f[0, :32].any() and not f[0, 64:].any()
    assert f[1, 64:].isnan().all() and not f[1, :64].any()
    # 2^-133 is an eighth of 2^-127 * 2^-3: a value of the smallest scale
    assert f[2, 3] == 2.0**-133 and f[2].count_nonzero() == 1


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(1, 32), (5, 96), (40, 2048), (3, 8224), (2, 32768)])
def test_rows_to_mx8(T, H):
    native = _native()
    g = torch.Generator(device="cuda").manual_seed(H)
    x = torch.empty((T, H), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    x[0, :32] = torch.tensor([448.0, -448.0, 0.0, 2.0**-9, 2.0**-10, 3 * 2.0**-10] + [1.0] * 26)
    m = native.rows_to_mx8(x)
    # every step is exact but the rounding: bit for bit
    assert np.array_equal(m.float().cpu().double().numpy(), mx.round_mx8(_f64(x)))
    assert np.array_equal(m.scale.cpu().numpy().astype(np.int64) - 127, mx.group_exponents(_f64(x), 448.0))


@pytest.mark.gpu
def test_norm_on_a_stream_and_in_a_graph():
    native = _native()
    x, r, w = _case(50, 2048, torch.bfloat16, torch.bfloat16, 11)
    ro, o, m = torch.empty_like(r), torch.empty_like(x), native.Mx8Rows.allocate(50, 2048, "cuda")
    want = native.add_rms_norm(x, w, residual=r, residual_out=torch.empty_like(r))[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        native.add_rms_norm(x, w, residual=r, residual_out=ro, out=o, mx8=m)
        native.add_rms_norm(x, w, residual=r, residual_out=ro, out=o, mx8=m, stream=side)
    side.synchronize()
    assert torch.equal(o, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        native.add_rms_norm(x, w, residual=r, residual_out=ro, out=o, mx8=m)
    for seed in range(3):
        x.normal_(generator=torch.Generator(device="cuda").manual_seed(seed))
        graph.replay()
        torch.cuda.synchronize()
        e = native.Mx8Rows.allocate(50, 2048, "cuda")
        want = native.add_rms_norm(x, w, residual=r, residual_out=torch.empty_like(r), out=torch.empty_like(x), mx8=e)
        assert torch.equal(o, want[0]) and torch.equal(ro, want[2])
        assert torch.equal(m.q.view(torch.uint8), e.q.view(torch.uint8)) and torch.equal(m.scale, e.scale)


@pytest.mark.gpu
def test_norm_empty_and_refusals():
    native = _native()
    x, r, w = _case(4, 64, torch.bfloat16, torch.bfloat16, 1)
    assert native.add_rms_norm(x[:0], w, residual=r[:0])[0].shape == (0, 64)
    assert native.rows_to_mx8(x[:0]).shape == (0, 64)
    bad = [
        lambda: native.add_rms_norm(x.float(), w),
        lambda: native.add_rms_norm(x, w.half()),
        lambda: native.add_rms_norm(x, w[:32]),
        lambda: native.add_rms_norm(x, w, residual=r[:2]),
        lambda: native.add_rms_norm(x, w, residual=r.half()),
        lambda: native.add_rms_norm(x, w, residual_out=r),
        lambda: native.add_rms_norm(x, w, residual=r, residual_out=r.float()),
        lambda: native.add_rms_norm(x.t(), w),
        lambda: native.add_rms_norm(x[:, :32], w[:32]),                      # not contiguous
        lambda: native.add_rms_norm(x, w, eps=-1.0),
        lambda: native.add_rms_norm(x, w, eps=float("nan")),
        lambda: native.add_rms_norm(x, w, mx8=native.Mx8Rows.allocate(4, 32, "cuda")),
        lambda: native.add_rms_norm(x.cpu(), w),
        lambda: native.Mx8Rows.allocate(4, 40, "cuda"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    odd = torch.zeros((4, 36), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="unsupported shape"):
        native.add_rms_norm(odd, torch.ones(36, dtype=torch.bfloat16, device="cuda"))
    buf = torch.zeros(4 * 64 + 4, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="unsupported shape"):
        native.add_rms_norm(buf[4:].view(4, 64), w)                          # 8 bytes off


@pytest.mark.gpu
def test_norm_keeps_outputs_apart():
    """Outputs in one buffer, or over rows that other workgroups still read."""
    native = _native()
    x, r, w = _case(4, 64, torch.bfloat16, torch.bfloat16, 2)
    _, rf, _ = _case(4, 64, torch.float32, torch.bfloat16, 2)
    wide = torch.zeros((8, 64), dtype=torch.bfloat16, device="cuda")
    over = native.Mx8Rows(wide.view(torch.float8_e4m3fn)[:2].reshape(4, 64), torch.zeros((4, 2), dtype=torch.uint8, device="cuda"))
    bad = [
        lambda: native.add_rms_norm(x, w, residual=r, out=r),                    # residual_out is residual
        lambda: native.add_rms_norm(x, w, residual=r, residual_out=x, out=x),
        lambda: native.add_rms_norm(x, w, residual=rf, residual_out=torch.empty_like(rf),
                                    out=rf.view(torch.bfloat16).view(-1)[:256].view(4, 64)),
        lambda: native.add_rms_norm(wide[:4], w, mx8=over),
        lambda: native.rows_to_mx8(wide[:4], over),
    ]
    before = [t.clone() for t in (x, r, rf, wide)]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail(f"call {i} was taken")
    assert all(torch.equal(a, b) for a, b in zip((x, r, rf, wide), before))
    want = native.add_rms_norm(x, w, residual=r, residual_out=torch.empty_like(r))
    a, b = x.clone(), r.clone()
    native.add_rms_norm(a, w, residual=b, out=b, residual_out=a)                 # each over the other's input
    assert torch.equal(b, want[0]) and torch.equal(a, want[2])


@pytest.mark.gpu
def test_norm_past_32_bits():
    """More than 2^32 bytes of rows: the last rows and those around 2^31 elements."""
    native = _native()
    T, H = 300_100, 7168
    x = torch.empty((T, H), dtype=torch.bfloat16, device="cuda").normal_()
    w = torch.empty(H, device="cuda").uniform_(0.5, 1.5)
    m = native.Mx8Rows.allocate(T, H, "cuda")
    out = native.add_rms_norm(x, w, out=torch.empty_like(x), mx8=m)[0]
    q = native.rows_to_mx8(x)
    for a, b in ((0, 64), (299_560, 299_660), (T - 64, T)):
        e, f = native.Mx8Rows.allocate(b - a, H, "cuda"), native.rows_to_mx8(x[a:b].clone())
        assert torch.equal(native.add_rms_norm(x[a:b].clone(), w, out=torch.empty_like(x[a:b]), mx8=e)[0], out[a:b])
        for got, want in ((m[a:b], e), (q[a:b], f)):
            assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.scale, want.scale)


@pytest.mark.gpu
def test_norm_refuses_rows_that_others_still_read():
    """Outputs that start inside an input, or scales over one: refused, nothing
    written; next to it, and row for row, the call is taken."""
    native = _native()
    buf = torch.empty((9, 64), dtype=torch.bfloat16, device="cuda").normal_()
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    keep, x = buf.clone(), buf[:4]
    m = native.Mx8Rows.allocate(4, 64, "cuda")
    over_q = native.Mx8Rows(buf.view(torch.float8_e4m3fn).view(-1)[64:320].view(4, 64), m.scale)
    over_s = native.Mx8Rows(m.q, buf.view(torch.uint8).view(-1)[3:11].view(4, 2))
    other = torch.zeros_like(x)
    bad = [
        lambda: native.add_rms_norm(x, w, out=buf[1:5]),
        lambda: native.add_rms_norm(buf[1:5], w, out=x),
        lambda: native.add_rms_norm(other, w, residual=x, residual_out=buf[3:7]),
        lambda: native.add_rms_norm(other, w, residual=buf[3:7], out=x),
        lambda: native.add_rms_norm(x, w, mx8=over_q),
        lambda: native.add_rms_norm(x, w, mx8=over_s),
        lambda: native.add_rms_norm(x, buf[4], out=buf[4:8]),
        lambda: native.rows_to_mx8(x, over_q),
        lambda: native.rows_to_mx8(x, over_s),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError, match="overlap"):
            call()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()
    assert torch.equal(buf, keep) and not other.any()
    want = native.add_rms_norm(keep[:4], w)[0]
    native.add_rms_norm(x, w, out=buf[4:8])
    assert torch.equal(buf[4:8], want) and torch.equal(buf[:4], keep[:4])
    native.add_rms_norm(x, w, out=x)
    assert torch.equal(buf[:4], want) and torch.equal(buf[8], keep[8])


@pytest.mark.gpu
def test_outputs_made_for_a_stream_are_its_own():
    """With stream= an output that the call makes is memory of that stream's pool:
    what the current stream still has queued on a freed block does not reach it."""
    native = _native()
    side = torch.cuda.Stream()
    x, _, w = _case(64, 2048, torch.bfloat16, torch.bfloat16, 4)
    gate = torch.empty((64, 2048), device="cuda").normal_(0, 0.05).to(torch.bfloat16)
    logits = native.router_gate(x, gate, torch.empty((64, 64), dtype=torch.bfloat16, device="cuda"))
    ids = native.router_topk(logits, 4)[1]
    perm = native.permute(ids, native.Permutation.allocate(256, 64, "cuda"))
    flat = lambda r: [t.view(torch.uint8) for t in (  # noqa: E731
        (r.q, r.scale) if isinstance(r, native.Mx8Rows) else (r,) if isinstance(r, torch.Tensor) else
        [v for v in r if v is not None])]
    calls = [lambda **s: native.add_rms_norm(x, w, **s), lambda **s: native.rows_to_mx8(x, **s),
             lambda **s: native.router_topk(logits, 4, **s)[:2], lambda **s: native.gather_rows(x, 4, perm, **s)]
    for i, call in enumerate(calls):
        print(f"case own stream {i}", flush=True)
        want = [t.clone() for t in flat(call())]
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        old = [torch.empty_like(t) for t in want]
        torch.cuda._sleep(20_000_000)          # the current stream is behind
        for t in old:
            t.fill_(0x55)
        del old, t                             # their blocks are free for this stream, the fills still queued
        got = call(stream=side)
        side.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(got), want)), i
