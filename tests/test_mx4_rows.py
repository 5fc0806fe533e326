"""4-bit rows, quantisation and products of 4-bit weights: what is refused (no GPU needed)."""

import ctypes

import pytest
import torch

P16 = 4096  # placeholders: no call here gets as far as a launch


def _lib():
    from vllm_moe_offload_amd import native

    return native.load_library()


def test_rows_entries_check_their_arguments():
    lib = _lib()
    q, sc, x = 1 << 20, 2 << 20, 3 << 20
    for fn, args in ((lib.lmoe_rows_to_mx4, lambda v, T, H, q, s: (v, 0, T, H, q, s, None)),
                     (lib.lmoe_mx4_rows_values, lambda v, T, H, q, s: (q, s, T, H, v, 0, None))):
        assert fn(*args(None, 0, 64, None, None)) == 0       # no rows: null operands
        assert fn(*args(x, -1, 64, q, sc)) == 1000
        assert fn(*args(x, 4, 0, q, sc)) == 1000
        assert fn(*args(x, 4, 48, q, sc)) == 1001            # a row of one group and a half
        assert fn(*args(None, 4, 64, q, sc)) == 1000
        assert fn(*args(x, 4, 64, None, sc)) == 1000
        assert fn(*args(x, 4, 64, q, None)) == 1000
        assert fn(*args(x + 8, 4, 64, q, sc)) == 1001
        assert fn(*args(x, 4, 64, q + 4, sc)) == 1001
        assert fn(*args(x, 4, 64, x + 496, sc)) == 1000      # the last 16 of x's 512 bytes
        assert fn(*args(x, 4, 64, q, q + 127)) == 1000       # the last of q's 128
        assert fn(*args(x, 4, 64, q, x)) == 1000


def test_bank_entries_check_their_arguments():
    lib = _lib()
    w, bank = 1 << 20, 64 << 20
    for fn, args in ((lib.lmoe_mx4_quantize, lambda w, E, N, K, g, b: (w, 0, E, N, K, g, b, None)),
                     (lib.lmoe_mx4_bank_values, lambda w, E, N, K, g, b: (b, E, N, K, g, w, 0, None))):
        assert fn(*args(None, 0, 64, 64, 1, None)) == 0
        assert fn(*args(w, -1, 64, 64, 0, bank)) == 1000
        assert fn(*args(w, 2, 0, 64, 0, bank)) == 1000
        assert fn(*args(w, 2, 64, 0, 0, bank)) == 1000
        assert fn(*args(w, 2, 24, 64, 0, bank)) == 1001
        assert fn(*args(w, 2, 64, 40, 0, bank)) == 1001
        assert fn(*args(w, 2, 32, 64, 1, bank)) == 1001      # halves of 16 rows: no whole group of act
        assert fn(*args(None, 2, 64, 64, 0, bank)) == 1000
        assert fn(*args(w, 2, 64, 64, 0, None)) == 1000
        assert fn(*args(w + 2, 2, 64, 64, 0, bank)) == 1001
        assert fn(*args(w, 2, 64, 64, 0, bank + 8)) == 1001
        assert fn(*args(w, 2, 64, 64, 0, w + 2 * 64 * 64 * 2 - 16)) == 1000
        assert fn(*args(w, 1 << 30, 1 << 20, 1 << 20, 0, bank)) == 1001  # more than a grid


def test_linear_checks_its_arguments():
    lib = _lib()
    mb = 1 << 20
    x, xs, w, bias, add, out = (i * mb for i in range(1, 7))

    def call(x=x, xs=None, rows=0, T=4, K=64, N=32, w=w, bias=bias, bias_f32=1, add=add, out=out, f32=0):
        return lib.lmoe_mx4_linear(x, xs, rows, T, K, N, w, bias, bias_f32, add, out, f32, None)

    assert call(T=0, x=None, w=None, bias=None, add=None, out=None) == 0
    assert call(T=-1) == 1000 and call(K=0) == 1000 and call(N=0) == 1000
    assert call(rows=3) == 1003 and call(rows=-1) == 1003
    assert call(K=48) == 1001 and call(N=24) == 1001
    for name in ("x", "w", "out"):
        assert call(**{name: None}) == 1000, name
    assert call(xs=xs) == 1000                      # bf16 rows have no scales
    assert call(rows=1) == 1000 and call(rows=2) == 1000
    for name, v in (("x", x), ("w", w), ("bias", bias), ("add", add), ("out", out)):
        assert call(**{name: v + 8}) == 1001, name
    assert call(out=x) == 1000 and call(out=w) == 1000 and call(out=bias) == 1000
    assert call(rows=2, xs=xs, out=xs & ~15) == 1000
    assert call(add=out + 16) == 1000               # over add, but not in place
    assert call(add=out, f32=1) == 1000             # rows of two types


def test_experts_of_4_bit_rows_check_their_arguments():
    lib = _lib()
    p, N = ctypes.c_void_p(P16), None
    i = [p] * 5  # offsets, sorted_pairs, active, tile_off, meta
    assert lib.lmoe_mx44_gateup_silu(N, N, 0, 64, 64, 2, N, 4, N, N, N, N, N, 0, 32, 0, N, N, 0, N) == 0
    assert lib.lmoe_mx44_gateup_silu(p, N, 2, 64, 64, 2, p, 4, *i, 4, 32, 0, p, p, 0, N) == 1000  # no scales
    assert lib.lmoe_mx44_gateup_silu(p, p, 2, 64, 64, 2, p, 4, *i, 4, 32, 0, p, N, 0, N) == 1000
    assert lib.lmoe_mx44_gateup_silu(p, p, 2, 64, 64, 2, p, 4, *i, 4, 32, 0, p, p, 1, N) == 1000  # no two parts
    assert lib.lmoe_mx44_gateup_silu(p, p, 2, 48, 64, 2, p, 4, *i, 4, 32, 0, p, p, 0, N) == 1001
    assert lib.lmoe_mx44_gateup_silu(p, p, 2, 64, 64, 2, p, 4, *i, 4, 32, 3, p, p, 0, N) == 1003
    assert lib.lmoe_mx44_down(p, N, 0, 64, 64, p, 4, *i, 4, 32, 0, p, 0, N) == 1000
    assert lib.lmoe_mx44_down(p, p, 1, 64, 64, p, 4, *i, 4, 32, 0, p, 0, N) == 1000
    assert lib.lmoe_mx44_decode_few(p, N, 2, 64, 64, 2, p, p, 4, p, p, N, 0, N, p, p, p, p, N) == 1000
    assert lib.lmoe_mx44_decode_one(p, N, 64, 64, 2, p, p, 4, p, p, N, 0, N, N, 0, N, 0, N, p, p, p, N) == 1000


def test_rows_are_what_they_say():
    from vllm_moe_offload_amd import mxfp4, native

    rows = native.Mx4Rows.allocate(5, 96, "cpu")
    assert rows.shape == (5, 96) and rows.q.shape == (5, 48) and rows.scale.shape == (5, 3)
    assert rows[1:3].shape == (2, 96)
    with pytest.raises(TypeError):
        rows[0]
    for columns in (0, 48, -32):
        with pytest.raises(ValueError):
            native.Mx4Rows.allocate(5, columns, "cpu")
    x = torch.randn(5, 96)
    q = native.Mx4Rows(*mxfp4.quantize(x))
    assert torch.equal(q.float(), mxfp4.dequantize(q.q, q.scale)) and q.float().shape == x.shape


def test_kinds_of_rows():
    from vllm_moe_offload_amd import fused_moe, native

    bank = torch.empty((2, 64, 32), dtype=torch.uint8)
    x = torch.empty((3, 32), dtype=torch.bfloat16)
    assert fused_moe.rows_kind(x, bank) == "bf16"
    assert fused_moe.rows_kind(native.Mx8Rows.allocate(3, 32, "cpu"), bank) == "mx8"
    assert fused_moe.rows_kind(native.Mx4Rows.allocate(3, 32, "cpu"), bank) == "mx4"
    with pytest.raises(ValueError, match="4-bit rows"):
        fused_moe.rows_kind(native.Mx4Rows.allocate(3, 32, "cpu"), x)


def test_sizes_past_the_tiles_offsets_are_refused():
    lib = _lib()
    mb = 1 << 20
    long = (1 << 23) + 32
    x, xs, w, out = mb, 1 << 40, 1 << 41, 1 << 42
    for rows in (0, 1, 2):
        scale = xs if rows else None
        assert lib.lmoe_mx4_linear(x, scale, rows, 1, long, 16, w, None, 0, None, out, 0, None) == 1001
    assert lib.lmoe_mx4_quantize(x, 0, 1, 16, long, 0, w, None) == 1001
    assert lib.lmoe_mx4_bank_values(w, 1, 16, long, 0, x, 0, None) == 1001
    assert lib.lmoe_mx4_quantize(x, 0, 1 << 30, 1 << 30, 1 << 22, 0, w, None) == 1001  # 2^68 quads
    p, N = ctypes.c_void_p(P16), None
    i = [p] * 5
    tiles = 2  # LMOE_PATH_MFMA

    def gateup(T, H, I, block_m, path=tiles):
        return lib.lmoe_mx44_gateup_silu(p, p, T, H, I, 1, p, 4, *i, T, block_m, path, p, p, 0, N)

    assert gateup(1 << 19, 1 << 14, 64, 64) == 1001          # 2^33 values of x
    assert gateup(64, long, 64, 64) == 1001
    assert lib.lmoe_mx44_down(p, p, 0, 64, long, p, 4, *i, 64, 64, tiles, p, 0, N) == 1001
    for block_m in (0, 16, 32, 96, 320, 512):                # no tile of 4-bit rows is so high
        assert gateup(64, 64, 64, block_m) == 1001, block_m
        assert gateup(64, 64, 64, block_m, 0) == 1001, block_m  # AUTO, where tiles are due
        assert lib.lmoe_mx44_down(p, p, 0, 64, 64, p, 4, *i, 64, block_m, tiles, p, 0, N) == 1001, block_m
    assert lib.lmoe_mx4_gateup_silu(p, p, 64, 64, 64, 1, p, 4, *i, 64, 256, tiles, p, p, 0, N) == 1001  # nor of 8-bit ones


def test_path_and_height_of_4_bit_rows():
    from vllm_moe_offload_amd import native

    few, tiles = native.LMOE_PATH_GEMV, native.LMOE_PATH_MFMA
    per = native.MX4_FEW_PAIRS_PER_EXPERT_MX4
    assert native.mx4_path(per * 8, 8, mx4=True) == few and native.mx4_path(per * 8 + 1, 8, mx4=True) == tiles
    assert native.mx4_path(1 << 20, 8, columns=native.MX4_MAX_COLUMNS_MX4, mx4=True) == tiles
    assert native.mx4_path(1 << 20, 8, columns=native.MX4_MAX_COLUMNS_MX4 + 32, mx4=True) == few
    assert native.mx4_path(1 << 20, 8, mx4=True, row_values=(1 << 33) - 2) == tiles
    assert native.mx4_path(1 << 20, 8, mx4=True, row_values=1 << 33) == few
    for pairs in (1, 63, 64, 500, 5_000, 33_000, 100_000, 1_000_000):
        for experts in (1, 8, 60, 128):
            for wide in (32, 768, 2048):
                for columns in (64, 2048, 7168):
                    assert native.mx4_block_m(pairs, experts, wide, mx4_columns=columns) in native.MX4_ROWS_BLOCK_M
    # low while the card is not full, then 128, 256 where rows are long
    assert [native.mx4_block_m(n * 128, 128, 768, mx4_columns=2048) for n in (1, 50, 51, 300)] == [64, 64, 128, 128]
    assert [native.mx4_block_m(n * 32, 32, 2048, mx4_columns=7168) for n in (1, 50, 51, 300)] == [64, 64, 256, 256]
    assert native.mx4_block_m(201 * 128, 128, 768, mx4_columns=4096) == 256
    assert native.mx4_block_m(201, 1, 768, mx4_columns=4096) == 64


def test_python_refusals_before_any_launch():
    """What the wrappers refuse by looking: nothing here needs a device."""
    from vllm_moe_offload_amd import native

    rows = native.Mx4Rows.allocate(2, 64, "cpu")
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        native._need_mx4_rows(x, "x")
    with pytest.raises(ValueError):
        native._need_mx4_rows(native.Mx4Rows(rows.q[:, :24], rows.scale), "x", (2, 48))
    with pytest.raises(ValueError):
        native._need_alike(rows, x)
    with pytest.raises(ValueError):
        native._need_alike(rows, native.Mx8Rows.allocate(2, 64, "cpu"))
    native._need_alike(rows, rows)
    native._need_alike(x, x)
