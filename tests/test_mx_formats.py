"""Microscaling formats on the host: the quantizer against the definition in
64 bits, the bank's byte order, what is refused."""

import numpy as np
import pytest
import torch

from oracle import mx


def _m():
    from vllm_moe_offload_amd import mxfp4

    return mxfp4


def _special_rows(K, rng):
    """Rows whose groups sit on the format's borders."""
    w = rng.standard_normal((32, K)).astype(np.float32) * 0.02
    w[0] = 0.0
    w[1, :8] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]         # ties of scale 1
    w[1, 8:16] = -w[1, :8]
    w[2] = np.float32(1e-40)                                         # subnormal f32
    w[3] = np.nextafter(np.float32(6.0), np.float32(7.0))            # just past a scale's reach
    w[4] = 6.0 * 2.0 ** rng.integers(-20, 20)
    w[5] = np.float32(2.0**120) * rng.standard_normal(K)
    w[6] = np.float32(2.0**-125) * rng.standard_normal(K)
    w[7, ::2] = -0.0
    return w


@pytest.mark.parametrize("K", [32, 96, 160, 512, 1056])
def test_quantize_is_the_definition(K):
    w = _special_rows(K, np.random.default_rng(K))
    codes, scales = _m().quantize(torch.from_numpy(w))
    want_c, want_s = mx.quantize_mx4(w)
    assert np.array_equal(scales.numpy(), want_s)
    assert np.array_equal(codes.numpy(), want_c)
    got = _m().dequantize(codes, scales).numpy()
    assert np.array_equal(got.astype(np.float64), mx.values_mx4(want_c, want_s))


def test_quantize_bf16_and_not_a_number():
    w = torch.randn(32, 64).to(torch.bfloat16)
    c, s = _m().quantize(w)
    c32, s32 = _m().quantize(w.float())
    assert torch.equal(c, c32) and torch.equal(s, s32)
    w[3, 5], w[4, 40] = float("nan"), float("inf")
    c, s = _m().quantize(w)
    assert s[3, 0] == 255 and s[4, 1] == 255 and s[3, 1] != 255 and s[4, 0] != 255
    v = _m().dequantize(c, s)
    assert v[3, :32].isnan().all() and v[4, 32:].isnan().all() and not v[3, 32:].isnan().any()


@pytest.mark.parametrize("K", [32, 128, 160, 480, 512, 768, 1056])
def test_bank_bytes_are_where_the_kernels_read_them(K):
    m = _m()
    N = 64
    rng = np.random.default_rng(K)
    codes = torch.from_numpy(rng.integers(0, 256, (2, N, K // 2), dtype=np.uint8))
    scales = torch.from_numpy(rng.integers(0, 255, (2, N, K // 32), dtype=np.uint8))
    bank = m.pack_w2(codes, scales)
    assert bank.shape == (2, N, m.row_bytes(K)) and bank.is_contiguous()
    flat = bank.reshape(2, -1)
    block = 16 * m.row_bytes(K)
    c, s = codes.numpy(), scales.numpy()
    for e, n, k in [(0, 0, 0), (1, 63, K - 1), (1, 17, K // 2), (0, 33, K - 32), (1, 40, 31)]:
        quad, chunk, group = k // 512, k // 128, k % 128 // 32
        lane = n % 16 + 16 * group
        base = (n // 16) * block + quad * 4352
        byte = int(flat[e, base + 256 + (chunk % 4) * 1024 + lane * 16 + k % 32 // 2])
        assert byte == c[e, n, k // 2]
        assert int(flat[e, base + lane * 4 + chunk % 4]) == s[e, n, k // 32]
    c2, s2 = m.unpack_w2(bank, K)
    assert torch.equal(c2, codes) and torch.equal(s2, scales)
    # gate and up rows in alternating blocks of 16
    b13 = m.pack_w13(codes, scales)
    order = torch.cat([torch.arange(h + 16 * b, h + 16 * b + 16) for b in range(2) for h in (0, 32)])
    assert torch.equal(b13, m.pack_w2(codes[:, order], scales[:, order]))
    c3, s3 = m.unpack_w13(b13, K)
    assert torch.equal(c3, codes) and torch.equal(s3, scales)


def test_library_and_host_agree_on_bytes():
    from vllm_moe_offload_amd import native

    lib = native.load_library()
    for N, K in ((16, 32), (64, 160), (1536, 2048), (4096, 7168), (2048, 768)):
        assert lib.lmoe_mx4_bytes(N, K) == N * _m().row_bytes(K)
    for N, K in ((15, 32), (16, 48), (0, 32), (16, 0), (-16, 32)):
        assert lib.lmoe_mx4_bytes(N, K) == -1


def test_pack_experts_is_quantize_then_pack():
    m = _m()
    w13, w2 = torch.randn(3, 128, 96).to(torch.bfloat16), torch.randn(3, 96, 64).to(torch.bfloat16)
    b13, b2 = m.pack_experts(w13, w2)
    assert torch.equal(b13, m.pack_w13(*m.quantize(w13))) and torch.equal(b2, m.pack_w2(*m.quantize(w2)))


def test_refusals():
    m = _m()
    with pytest.raises(ValueError):
        m.row_bytes(48)
    with pytest.raises(ValueError):
        m.quantize(torch.zeros(16, 40))
    with pytest.raises(ValueError):
        m.quantize(torch.zeros(16, 64, dtype=torch.int8))
    c, s = torch.zeros(32, 32, dtype=torch.uint8), torch.zeros(32, 2, dtype=torch.uint8)
    with pytest.raises(ValueError):
        m.pack_w2(c[:20], s[:20])           # no whole blocks of 16 rows
    with pytest.raises(ValueError):
        m.pack_w13(c, s)                    # gate and up of 16 rows each
    with pytest.raises(ValueError):
        m.pack_w2(c, s[:, :1])
    with pytest.raises(ValueError):
        m.pack_w2(c.int(), s)
    with pytest.raises(ValueError):
        m.unpack_w2(m.pack_w2(c, s), 128 + 32)
    with pytest.raises(ValueError):
        m.pack_experts(c, c)


P16, N = 4096, None  # a placeholder address, never read: these calls fail on the host


def test_c_entries_check_their_arguments():
    from vllm_moe_offload_amd import native

    lib = native.load_library()
    norm = lambda x=P16, T=1, H=64, r=P16, w=P16, eps=1e-6, ro=P16, out=P16, q=P16, s=P16: \
        lib.lmoe_add_rms_norm(x, T, H, r, 0, w, 0, eps, ro, out, q, s, N)
    assert norm(T=0, x=N, r=N, w=N, ro=N, out=N, q=N, s=N) == 0
    assert norm(T=-1) == 1000 and norm(H=0) == 1000 and norm(eps=-1.0) == 1000 and norm(eps=float("nan")) == 1000
    assert norm(x=N) == 1000 and norm(w=N) == 1000 and norm(out=N, q=N, s=N) == 1000
    assert norm(r=N) == 1000 and norm(ro=N) == 1000 and norm(q=N) == 1000 and norm(s=N) == 1000
    assert norm(H=36) == 1001 and norm(H=40) == 1001 and norm(H=32800) == 1001
    for k in ("x", "r", "w", "ro", "out", "q"):
        assert norm(**{k: P16 + 8}) == 1001, k
    rows = lambda x=P16, T=1, H=64, q=P16, s=P16: lib.lmoe_rows_to_mx8(x, T, H, q, s, N)
    assert rows(T=0, x=N, q=N, s=N) == 0 and rows(T=-1) == 1000 and rows(x=N) == 1000 and rows(q=N) == 1000
    assert rows(s=N) == 1000 and rows(H=40) == 1001 and rows(x=P16 + 2) == 1001 and rows(H=65536) == 1001
    gu = lambda x=P16, xs=P16, T=2, H=64, I=32, k=2, w=P16, P=4, n=4, path=0, act=P16, as_=P16, bm=128, split=0: \
        lib.lmoe_mx4_gateup_silu(x, xs, T, H, I, k, w, P, P16, P16, P16, P16, P16, n, bm, path, act, as_, split, N)
    assert gu(T=0, n=0, x=N, act=N) == 0
    assert gu(T=-1) == 1000 and gu(k=0) == 1000 and gu(n=5) == 1000 and gu(P=0) == 1000 and gu(x=N) == 1000
    assert gu(xs=N) == 1000 and gu(as_=N) == 1000 and gu(act=N) == 1000 and gu(w=N) == 1000
    assert gu(H=48) == 1001 and gu(I=48) == 1001 and gu(x=P16 + 8) == 1001 and gu(w=P16 + 4) == 1001
    assert gu(path=9) == 1003 and gu(path=3) == 1003
    assert gu(split=1) == 1000 and gu(split=1, xs=N, as_=N, path=2) == 1003  # two parts: bf16 rows, no row tiles
    dn = lambda act=P16, as_=P16, H=64, I=32, w=P16, P=4, n=4, path=0, y=P16, bm=128, split=0: \
        lib.lmoe_mx4_down(act, as_, split, H, I, w, P, P16, P16, P16, P16, P16, n, bm, path, y, 0, N)
    assert dn(n=0, act=N, y=N) == 0 and dn(n=-1) == 1000 and dn(act=N) == 1000 and dn(y=N) == 1000
    assert dn(H=48) == 1001 and dn(I=16) == 1001 and dn(y=P16 + 8) == 1001 and dn(path=9) == 1003
    assert dn(split=1) == 1000 and dn(split=1, as_=N, path=2) == 1003
    from vllm_moe_offload_amd.native import _Mx4Workspace
    import ctypes

    def ws(**kw):
        v = {n: P16 for n, _ in _Mx4Workspace._fields_}
        return _Mx4Workspace(**{**v, "y_f32": 1, "act_split": 0, **kw})

    def fused(x=P16, xs=P16, T=2, H=64, I=32, k=2, w13=P16, w2=P16, P=4, w=P16, ids=P16, path=0, bm=32, wsp=None,
              add=N, out=P16):
        s = ws() if wsp is None else wsp
        return lib.lmoe_mx4_fused_moe(x, xs, T, H, I, k, w13, w2, P, w, ids, N, 0, path, bm, ctypes.addressof(s), add,
                                      out, N)

    assert lib.lmoe_mx4_fused_moe(P16, P16, 2, 64, 32, 2, P16, P16, 4, P16, P16, N, 0, 0, 32, N, N, P16, N) == 1000
    assert fused(T=-1) == 1000 and fused(k=0) == 1000 and fused(P=0) == 1000 and fused(x=N) == 1000 and fused(ids=N) == 1000
    assert fused(w=N) == 1000 and fused(out=N) == 1000 and fused(xs=N) == 1000 and fused(w13=N) == 1000 and fused(w2=N) == 1000
    assert fused(wsp=ws(act=None)) == 1000 and fused(wsp=ws(y=None)) == 1000 and fused(wsp=ws(act_scale=None)) == 1000
    assert fused(wsp=ws(act_split=1)) == 1000
    assert fused(H=48) == 1001 and fused(I=40) == 1001 and fused(P=70000) == 1001 and fused(T=1 << 30, k=4) == 1001
    assert fused(x=P16 + 8) == 1001 and fused(add=P16 + 8) == 1001 and fused(out=P16 + 8) == 1001
    assert fused(path=2, bm=256) == 1001 and fused(path=2, bm=128, H=32 * 4096) == 1001 and fused(path=3) == 1003
    one = lambda x=P16, xs=P16, H=64, I=32, k=2, w13=P16, w2=P16, P=4, w=P16, ids=P16, n=0, add=N, act=P16, as_=P16, out=P16, tab=N, b13=N, b2=N, pb=0, tb=N, nb=0: \
        lib.lmoe_mx4_decode_one(x, xs, H, I, k, w13, w2, P, w, ids, tab, n, b13, b2, pb, tb, nb, add, act, as_, out, N)
    assert one(b13=P16, tb=P16, tab=P16) == 1000 and one(b13=P16, b2=P16, tb=P16) == 1000
    assert one(b13=P16, b2=P16, tb=P16, tab=P16, pb=-1) == 1000 and one(b13=P16 + 8, b2=P16, tb=P16, tab=P16) == 1001
    assert one(x=N) == 1000 and one(xs=N) == 1000 and one(as_=N) == 1000 and one(w=N) == 1000 and one(ids=N) == 1000
    assert one(act=N) == 1000 and one(out=N) == 1000 and one(k=0) == 1000 and one(n=-1) == 1000 and one(w2=N) == 1000
    assert one(H=40) == 1001 and one(I=40) == 1001 and one(k=70000) == 1001 and one(add=P16 + 2) == 1001
    comb = lambda y=P16, w=P16, T=1, k=2, H=64, out=P16, add=N: \
        lib.lmoe_combine_f32(y, N, w, T, k, H, add, out, N)
    assert comb(T=0, y=N, out=N) == 0 and comb(y=N) == 1000 and comb(H=60) == 1001 and comb(out=P16 + 2) == 1001


def test_norm_entries_refuse_shared_buffers():
    from vllm_moe_offload_amd import native

    lib = native.load_library()
    a, b, c, d, e = (P16 * i for i in range(1, 6))
    norm = lambda x=a, r=b, rf=0, ro=c, out=d, q=e: lib.lmoe_add_rms_norm(x, 1, 64, r, rf, a, 0, 1e-6, ro, out, q, P16, N)
    assert norm(out=c) == 1000 and norm(ro=b, out=b) == 1000 and norm(ro=a, out=a) == 1000
    assert norm(rf=1, out=b) == 1000 and norm(rf=1, ro=a) == 1000
    for t in (a, b, c, d):
        assert norm(q=t) == 1000, t
    assert lib.lmoe_rows_to_mx8(a, 1, 64, a, P16, N) == 1000


def test_few_tokens_entry_checks_its_arguments():
    from vllm_moe_offload_amd import native

    lib = native.load_library()
    few = lambda x=P16, xs=P16, T=2, H=64, I=32, k=2, w13=P16, w2=P16, P=4, w=P16, ids=P16, n=0, add=N, act=P16, as_=P16, \
        y=P16, out=P16: lib.lmoe_mx4_decode_few(x, xs, T, H, I, k, w13, w2, P, w, ids, N, n, add, act, as_, y, out, N)
    assert few(T=0, x=N, y=N, out=N) == 0
    assert few(T=-1) == 1000 and few(k=0) == 1000 and few(P=0) == 1000 and few(n=-1) == 1000 and few(H=0) == 1000
    for t in ("x", "xs", "w13", "w2", "w", "ids", "act", "as_", "y", "out"):
        assert few(**{t: N}) == 1000, t
    assert few(H=48) == 1001 and few(I=40) == 1001 and few(P=70000) == 1001 and few(T=33) == 1001
    assert few(T=1 << 30, k=1 << 30) == 1001
    for t in ("x", "w13", "w2", "act", "y", "out", "add"):
        assert few(**{t: P16 + 8}) == 1001, t


def test_norm_entries_refuse_any_overlap_but_row_for_row():
    """Every output against every input and the other outputs, from either side,
    by one byte or one row: refused before any device work."""
    from vllm_moe_offload_amd import native

    lib = native.load_library()
    T, H = 3, 64
    size = {"x": 2 * T * H, "r": 2 * T * H, "w": 2 * H, "ro": 2 * T * H, "out": 2 * T * H, "q": T * H, "s": T * H // 32}
    at = {n: 65536 * (i + 1) for i, n in enumerate(size)}

    def norm(f32=0, **kw):
        a = {**at, **kw}
        return lib.lmoe_add_rms_norm(a["x"], T, H, a["r"], f32, a["w"], 0, 1e-6, a["ro"], a["out"], a["q"], a["s"], N)

    for o in ("ro", "out", "q", "s"):
        step = 1 if o == "s" else 16
        for other in size:
            if other == o:
                continue
            ends = [at[other] + size[other] - step, at[other] + 2 * H, at[other] + step]
            ends += [at[other] + step - size[o]] if size[o] % 16 == 0 or o == "s" else []
            for p in ends:
                if p < at[other] + size[other] and p % step == 0:  # else refused for its address
                    assert norm(**{o: p}) == 1000, (o, other, p - at[other])
            # row for row: a bf16 output over x, or over a residual that is no output's as well
            if (o, other) not in (("ro", "x"), ("ro", "r"), ("out", "x"), ("out", "r")):
                assert norm(**{o: at[other]}) == 1000, (o, other)
    f32 = 4 * T * H
    for kw in (dict(ro=at["r"] + 16), dict(ro=at["r"] + f32 - 16), dict(out=at["r"] + f32 - 16), dict(out=at["r"]),
               dict(ro=at["x"]), dict(x=at["ro"] + f32 - 16), dict(s=at["r"] + f32 - 1), dict(s=at["ro"] + f32 - 1)):
        assert norm(f32=1, **kw) == 1000, kw
    rows = lambda x=at["x"], q=at["q"], s=at["s"]: lib.lmoe_rows_to_mx8(x, T, H, q, s, N)
    x, q = at["x"], at["q"]
    for kw in (dict(q=x + 16), dict(q=x + size["x"] - 16), dict(q=x + 16 - size["q"]), dict(s=x), dict(s=x + size["x"] - 1),
               dict(s=x + 1 - size["s"]), dict(s=q), dict(s=q + size["q"] - 1)):
        assert rows(**kw) == 1000, kw


def test_row_tiles_take_8_bit_rows_up_to_their_limits():
    """The heights that the rules choose hold the rows, and the library draws the
    same lines."""
    from vllm_moe_offload_amd import native

    lib = native.load_library()
    limits = native.MX4_MAX_COLUMNS_MX8
    assert tuple(limits) == native.MX4_BLOCK_M
    gu = lambda bm, H, I: lib.lmoe_mx4_gateup_silu(P16, P16, 2, H, I, 1, P16, 4, P16, P16, P16, P16, P16, 2, bm, 2, P16, P16, 0, N)
    dn = lambda bm, H, I: lib.lmoe_mx4_down(P16, P16, 0, H, I, P16, 4, P16, P16, P16, P16, P16, 2, bm, 2, P16, 0, N)
    for bm, top in limits.items():
        # LDS: two stages of rows (32-row tiles: of two chunks), a pair id and all scales a row
        room = 160 * 1024 - bm * 128 * (4 if bm == 32 else 2) - 4 * bm
        chunks = room // (4 * bm)
        assert top == 128 * (chunks - chunks % 2 if bm == 32 else chunks)
        assert gu(bm, top + 32, 32) == 1001 and dn(bm, 32, top + 32) == 1001
    for columns in (32, 2048, 32640, 32672, 73600, 73632, 147200):
        for pairs, experts in ((1 << 20, 1), (1 << 20, 128), (5000, 16), (100, 8)):
            assert native.mx4_path(pairs, experts, True, columns) == native.LMOE_PATH_MFMA
            bm = native.mx4_block_m(pairs, experts, 4096, columns)
            assert columns <= limits[bm] and bm <= native.mx4_block_m(pairs, experts, 4096)
            if columns <= limits[128]:
                assert bm == native.mx4_block_m(pairs, experts, 4096)
    assert native.mx4_path(1 << 20, 1, True, 147232) == native.LMOE_PATH_GEMV
    assert native.mx4_path(1 << 20, 1, False, 147232) == native.LMOE_PATH_MFMA  # bf16 rows need no room for scales


def test_auto_refuses_tiles_of_another_kernel():
    """A permutation built for other row tiles, where row tiles are due: refused by
    AUTO as by an explicit path; with few pairs per slot no height is needed."""
    import ctypes

    from vllm_moe_offload_amd import native

    lib = native.load_library()
    P = 4
    v = {n: P16 for n, _ in native._Mx4Workspace._fields_}
    for a8, few in ((P16, 6), (N, 4)):
        n = few * P + 1
        ws = native._Mx4Workspace(**{**v, "y_f32": 1, "act_split": 0, "act_scale": a8})
        for bm in (96, 256, 320, 0):
            assert lib.lmoe_mx4_gateup_silu(P16, a8, n, 64, 32, 1, P16, P, P16, P16, P16, P16, P16, n, bm, 0, P16, a8, 0, N) == 1001
            assert lib.lmoe_mx4_down(P16, a8, 0, 64, 32, P16, P, P16, P16, P16, P16, P16, n, bm, 0, P16, 1, N) == 1001
            assert lib.lmoe_mx4_fused_moe(P16, a8, n, 64, 32, 1, P16, P16, P, P16, P16, N, 0, 0, bm, ctypes.addressof(ws), N,
                                          P16, N) == 1001


@pytest.mark.parametrize("fmt", ["mxfp4", "bf16"])
def test_a_checkpoint_in_4_bits_page_locks_no_bf16_copy(fmt, tmp_path, monkeypatch):
    """What from_checkpoint asks to page-lock: the blocks that the host store keeps."""
    from safetensors.torch import save_file

    from vllm_moe_offload_amd import layer as layer_mod
    from vllm_moe_offload_amd.moe_offload.config import MoeOffloadConfig
    from vllm_moe_offload_amd.moe_offload.runtime import MoeOffloadRuntime

    E, H, I = 2, 64, 32
    w13, w2 = torch.randn(E, 2 * I, H).to(torch.bfloat16), torch.randn(E, H, I).to(torch.bfloat16)
    save_file({f"m.experts.{e}.{n}.weight": t.contiguous() for e in range(E)
               for n, t in (("gate_proj", w13[e, :I]), ("up_proj", w13[e, I:]), ("down_proj", w2[e]))},
              str(tmp_path / "e.safetensors"))
    asked = {}
    make, pack = layer_mod.create_cpu_first_expert_weights, layer_mod.mxfp4.pack_experts

    def make_spy(*a, pin_memory, **kw):
        asked["bf16"] = pin_memory
        return make(*a, pin_memory=pin_memory, **kw)

    def pack_spy(*a, pin_memory=False):
        asked["4 bits"] = pin_memory
        return pack(*a, pin_memory=pin_memory)

    monkeypatch.setattr(layer_mod, "create_cpu_first_expert_weights", make_spy)
    monkeypatch.setattr(layer_mod.mxfp4, "pack_experts", pack_spy)
    rt = MoeOffloadRuntime(MoeOffloadConfig(enabled=True, num_slots=2, async_load=True, pin_host_memory=True, cpu_first_load=True))
    assert rt.config.should_pin_host_memory
    layer = layer_mod.SlotMoELayer.from_checkpoint(
        tmp_path / "e.safetensors", prefix="m", layer_id=3, runtime=rt, num_experts=E, hidden_size=H, intermediate_size=I,
        gate_weight=torch.zeros(E, H, dtype=torch.bfloat16), top_k=1, weight_format=fmt, device="cpu")
    if fmt == "mxfp4":
        assert asked == {"bf16": False, "4 bits": True}
        b13, b2 = pack(w13, w2)
        assert torch.equal(layer.w13_weight, b13) and torch.equal(layer.w2_weight, b2)
    else:
        assert asked == {"bf16": True} and torch.equal(layer.w13_weight, w13)


@pytest.mark.gpu
def test_every_scale_is_exact_on_the_gpu():
    """Values of every scale byte, and quantizing rows of every size, as on the host:
    powers of two are built from their bits (a device's pow is off by a bit for some)."""
    from vllm_moe_offload_amd import native

    m = _m()
    byte = torch.arange(256, dtype=torch.uint8)
    codes = torch.arange(16, dtype=torch.uint8).repeat(256, 1)
    codes = (codes | (codes.flip(1) << 4)).contiguous()                       # [256, 16]: 32 columns
    want = torch.from_numpy(mx.values_mx4(codes.numpy(), byte.view(256, 1).numpy())).float()
    want[255] = float("nan")
    q = torch.arange(32, dtype=torch.uint8).repeat(256, 1) * 4                # e4m3 codes, no NaN
    rows = native.Mx8Rows(q.view(torch.float8_e4m3fn), byte.view(256, 1))
    v8 = torch.from_numpy(q.view(torch.float8_e4m3fn).float().numpy().astype(np.float64) *
                          np.ldexp(1.0, byte.numpy().astype(np.int64) - 127)[:, None]).float()
    v8[255] = float("nan")
    for dev in ("cpu", "cuda"):
        got = m.dequantize(codes.to(dev), byte.view(256, 1).to(dev)).cpu()
        assert torch.equal(got[:255], want[:255]) and got[255].isnan().all(), dev
        got = native.Mx8Rows(rows.q.to(dev), rows.scale.to(dev)).float().cpu()
        assert torch.equal(got[:255], v8[:255]) and got[255].isnan().all(), dev
    rng = np.random.default_rng(3)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4, dtype=np.float32) * rng.choice([-1.0, 1.0], 32)
    w = np.stack([np.ldexp(ties, e) for e in range(-126, 126)]).astype(np.float32)
    w = np.concatenate([w, np.nextafter(w, np.float32(0)), rng.standard_normal(w.shape).astype(np.float32) *
                        np.ldexp(np.float32(1), rng.integers(-120, 120, (w.shape[0], 1)))])
    c, s = mx.quantize_mx4(w)
    for dev in ("cpu", "cuda"):
        got_c, got_s = m.quantize(torch.from_numpy(w).to(dev))
        assert np.array_equal(got_s.cpu().numpy(), s) and np.array_equal(got_c.cpu().numpy(), c), dev
