"""Which rows of 4-bit experts' second product stay f32 up to the weighted sum.

Where they do, out is that sum of the f32 rows (the products' call gives them) rounded
once: off by 2^-8 of itself and k + 2 f32 roundings of the magnitudes.  Rows in bf16 are off
by 2^-8 each, which past a few tokens shows in some output at least."""

import numpy as np
import pytest
import torch

from tests._util import to_dev_i32
from tests.test_gpu_mx4 import Layer, _f64
from tests.test_gpu_mx44 import Layer4

pytestmark = pytest.mark.gpu

H, I, E, K = 256, 160, 8, 4


def _layer(rows, T):
    rng = np.random.default_rng(T)
    ids = to_dev_i32(np.stack([rng.choice(E, K, replace=False) for _ in range(T)]))
    layer = Layer4(H, I, E, T, T) if rows == "mx4" else Layer(H, I, E, T, rows, T)
    g = torch.Generator(device="cuda").manual_seed(T)
    w = torch.empty((T, K), device="cuda").uniform_(0.05, 1, generator=g).to(torch.bfloat16)
    add = torch.empty((T, H), device="cuda").normal_(generator=g).to(torch.bfloat16)
    return layer, ids, w, add


def _sum_is_of_f32_rows(layer, ids, w, add, out):
    """Whether out is the rounded sum of f32 rows."""
    from vllm_moe_offload_amd import fused_moe, native

    T = ids.shape[0]
    mx4 = isinstance(layer.x, native.Mx4Rows)
    perm = native.Permutation.allocate(T * K, E, "cuda")
    bm = native.mx4_block_m(T * K, E, I, max(H, I) if layer.rows == "mx8" else 0, mx4_columns=max(H, I) if mx4 else 0)
    native.permute(ids, perm, block_m=bm)
    y = torch.empty((T * K, H), device="cuda")
    native.grouped_mlp(layer.x, K, layer.w13, layer.w2, perm, layer.act_buffer(T * K), y, path=native.LMOE_PATH_MFMA)
    y, wv, av = _f64(y).reshape(T, K, H), _f64(w)[:, :, None], _f64(add)
    want, mag = (wv * y).sum(1) + av, (np.abs(wv * y)).sum(1) + np.abs(av)
    return bool(np.all(np.abs(_f64(out) - want) <= 2.0**-8 * np.abs(want) + (K + 2) * 2.0**-24 * mag))


@pytest.mark.parametrize("T", [257, 333, 700, 1024])
def test_rows_of_4_bit_experts_and_rows(T):
    """Up to 4096 pairs without being asked."""
    from vllm_moe_offload_amd import fused_moe

    layer, ids, w, add = _layer("mx4", T)
    out = fused_moe.fused_experts(layer.x, w, ids, layer.w13, layer.w2, None, add=add)
    assert _sum_is_of_f32_rows(layer, ids, w, add, out)


@pytest.mark.parametrize("rows", ["bf16", "mx8", "mx4"])
@pytest.mark.parametrize("T", [300, 1025])
def test_a_workspace_that_keeps_them(rows, T):
    from vllm_moe_offload_amd import fused_moe

    layer, ids, w, add = _layer(rows, T)
    get = lambda **kw: fused_moe.get_workspace(T, K, E, H, I, "cuda", rows=rows, **kw)
    ws = get(y_f32=True)
    assert ws.y.dtype is torch.float32 and get(y_f32=True) is ws and (get() is ws) == (rows == "mx4" and T * K <= 4096)
    out = fused_moe.fused_experts(layer.x, w, ids, layer.w13, layer.w2, None, add=add, workspace=ws)
    assert _sum_is_of_f32_rows(layer, ids, w, add, out)
    plain = fused_moe.fused_experts(layer.x, w, ids, layer.w13, layer.w2, None, add=add, workspace=get())
    assert torch.equal(plain, fused_moe.fused_experts(layer.x, w, ids, layer.w13, layer.w2, None, add=add))
    if get() is not ws:  # bf16 rows do show: the check above is no empty one
        assert not _sum_is_of_f32_rows(layer, ids, w, add, plain)


def test_bf16_experts_have_none():
    from vllm_moe_offload_amd import fused_moe

    with pytest.raises(ValueError, match="4-bit experts"):
        fused_moe.get_workspace(4, 2, 4, 64, 32, "cuda", y_f32=True)
