"""The plain product of 8-bit rows with f32 outputs: its sums are f32's.

Tolerance: a sum of K products in f32 is off by at most K 2^-24 sum |x| |w|, the store by
2^-24 of the result.  Rows and weights are such that less than f32 shows: in every eight
columns one product is 448 * 6 (of alternating sign, so that these cancel) and the others
are up to 7 * 2^-9 * 6, below 2^-15 of it, all positive; over 512 columns they sum to 10 and
more where the tolerance is 6."""

import numpy as np
import pytest
import torch

from tests.test_gpu_mx4_linear import check, make_rows, make_weights

pytestmark = pytest.mark.gpu

# the split-K forms, then row tiles of each shape that 8-bit rows have
SHAPES = [(1, 32, 16), (16, 512, 64), (5, 160, 20000), (40, 512, 4096), (64, 480, 7168), (301, 96, 2048),
          (700, 480, 2064), (1024, 512, 2048), (500, 480, 7184), (2050, 416, 7184), (4090, 480, 7184)]


def _mods():
    from vllm_moe_offload_amd import mxfp4, native

    return mxfp4, native


def cancelling(T, K, N, seed):
    """(rows, their values, weights, theirs): codes as the docstring has them, groups'
    scales from 2^-3 to 2^3, the same for two eights that cancel."""
    mxfp4, native = _mods()
    rng = np.random.default_rng(seed)
    q = rng.integers(1, 8, (T, K)).astype(np.uint8)            # m 2^-9
    q[:, ::16], q[:, 8::16] = 0x7E, 0xFE                        # 448, -448
    sc = rng.integers(124, 131, (T, K // 32)).astype(np.uint8)
    code = rng.integers(1, 8, (N, K)).astype(np.uint8)          # .5 to 6
    code[:, ::8] = 7
    ws = rng.integers(124, 131, (N, K // 32)).astype(np.uint8)
    rows = native.Mx8Rows(torch.from_numpy(q).cuda().view(torch.float8_e4m3fn), torch.from_numpy(sc).cuda())
    codes, scales = torch.from_numpy(code[:, 0::2] | code[:, 1::2] << 4), torch.from_numpy(ws)
    return (rows, rows.float().double().cpu().numpy(), mxfp4.pack_w2(codes, scales).cuda(),
            mxfp4.dequantize(codes, scales).double().numpy())


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_small_products_beside_large_ones_count(T, K, N):
    _, native = _mods()
    x, xv, w, wv = cancelling(T, K, N, T + K)
    out = torch.empty((T, N), device="cuda")
    native.mx4_linear(x, w, out)
    check(out, xv, wv, "mx4")  # f32's sums alone


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_bias_and_add(T, K, N):
    _, native = _mods()
    g = torch.Generator().manual_seed(T * K + N)
    x, xv = make_rows(torch.randn((T, K), generator=g), "mx8")
    w, wv = make_weights(N, K, K)
    bias = torch.randn(N, generator=g).cuda()
    add = torch.randn((T, N), generator=g).to(torch.bfloat16).cuda()
    room = torch.full((T * N + 32,), 7.0, device="cuda")
    out = room[16:-16].view(T, N)
    native.mx4_linear(x, w, out, bias=bias, add=add)
    check(out, xv, wv, "mx4", bias, add)
    assert bool((room[:16] == 7).all()) and bool((room[-16:] == 7).all())


@pytest.mark.parametrize("T,K,N", [(20, 256, 32), (700, 224, 2064)])
def test_every_value_and_scale(T, K, N):
    """All e4m3 values; rows and weights whose scales are far from one."""
    mxfp4, native = _mods()
    rng = np.random.default_rng(T)
    for ex, ew in ((0, 0), (100, -110), (-120, 110), (-60, -60)):
        q = rng.integers(0, 255, (T, K)).astype(np.uint8)
        q[(q & 127) == 127] = 0
        x = native.Mx8Rows(torch.from_numpy(q).cuda().view(torch.float8_e4m3fn),
                           torch.full((T, K // 32), 127 + ex, dtype=torch.uint8, device="cuda"))
        codes, scales = mxfp4.quantize(torch.randn((N, K), generator=torch.Generator().manual_seed(N)) * 2.0**ew)
        out = torch.empty((T, N), device="cuda")
        native.mx4_linear(x, mxfp4.pack_w2(codes, scales).cuda(), out)
        check(out, x.float().double().cpu().numpy(), mxfp4.dequantize(codes, scales).double().numpy(), "mx4")


@pytest.mark.parametrize("T,K,N", [(40, 672, 144), (700, 672, 2064)])
def test_a_bad_value_stays_in_its_row(T, K, N):
    mxfp4, native = _mods()
    x, _ = make_rows(torch.randn((T, K), generator=torch.Generator().manual_seed(T)), "mx8")
    w, _ = make_weights(N, K, N)
    call = lambda: native.mx4_linear(x, w, torch.empty((T, N), device="cuda"))
    clean = call()
    x.q.view(torch.uint8)[-1, 3] = 0x7F   # NaN as a value
    x.scale[1, 2] = 255                   # and as a scale
    got = call()
    assert bool(torch.isnan(got[[1, -1]]).all())
    keep = [r for r in range(T) if r not in (1, T - 1)]
    assert torch.equal(got[keep], clean[keep]) and not bool(torch.isnan(clean).any())
