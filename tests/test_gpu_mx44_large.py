"""Rows of 4-bit experts whose offsets pass 31 and 32 bits: the last tokens' act and y are
those of a call of these tokens alone, on every path and tile height that reaches them."""

import numpy as np
import pytest
import torch

from tests.test_gpu_mx44 import Layer4, _bits, _native, _paths, check_layer, run_layer

pytestmark = pytest.mark.gpu

LAST, H, I, P = 40, 7168, 32, 2


@pytest.mark.parametrize("T", [
    300_100,    # columns past 2^31
    1_198_300,  # bytes up to 2^32, the last that row tiles reach
    1_300_000,  # and past it: the split-K kernel
])
def test_the_last_tokens_are_those_of_a_small_call(T):
    native = _native()
    reached = T * (H // 2) <= 0xFFFFFFFF
    layer = Layer4(H, I, P, LAST, 6)
    ids = np.arange(LAST).reshape(-1, 1).astype(np.int32) % P
    q = torch.zeros((T, H // 2), dtype=torch.uint8, device="cuda")
    sc = torch.full((T, H // 32), 127, dtype=torch.uint8, device="cuda")
    q[-LAST:], sc[-LAST:] = layer.x.q, layer.x.scale
    big = Layer4.__new__(Layer4)
    big.__dict__.update(layer.__dict__, x=native.Mx4Rows(q, sc))
    many = np.concatenate([np.zeros((T - LAST, 1), np.int32), ids])  # the others' slot is 0
    for path, bm in _paths() if reached else _paths()[:1]:
        perm, *small = run_layer(layer, ids, 1, path, block_m=bm)
        check_layer(layer, perm, 1, small[0], small[1], ids[:, 0])
        at = {s: perm.offsets[s].item() for s in range(P + 1)}
        perm, act, y = run_layer(big, many, 1, path, block_m=bm)
        offsets = perm.offsets.cpu().numpy()
        assert offsets.tolist() == [0, T - LAST // P, T]
        assert torch.equal(y[-LAST:].view(torch.int16), small[1].view(torch.int16)), (path, bm)
        for s in range(P):  # a slot's last rows
            n = at[s + 1] - at[s]
            for got, want in zip(_bits(act, y)[:2], _bits(*small)[:2]):
                assert torch.equal(got[offsets[s + 1] - n:offsets[s + 1]], want[at[s]:at[s + 1]]), (path, bm, s)
        assert bool(small[0].q.any()) and not bool(y[:-LAST].any())
        del act, y
