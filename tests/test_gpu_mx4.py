"""Expert products over 4-bit slot banks against the experts in 64 bits.

Tolerances, per element and by stage.  A product of K terms in f32 is off by at
most K 2^-24 sum |x| |w| (dg, du for gate and up).  act = silu(gate) up then
moves by 1.1 |up| dg + |silu(gate)| du (|silu'| <= 1.1); its own exp, reciprocal
and products by 2^-20; the store by half a step, 2^-8 in bf16, 2^-4 (or 2^-10 of
the scale) in 8 bits.  y is checked against the act that the kernel stored, so
only its own sum and store (2^-8 in bf16) count.

8-bit rows: the matrix instruction adds each 8 neighbouring columns in fixed
point.  With 2^m the largest product of the operands' powers of two among them,
every product loses what lies below 2^(m - 13) (towards zero); blocks of 8 are
then added in f32.  (One product of 2^8 beside one of 2^(8 - d): whole for d <=
13, gone from 14 on, at columns 1 to 7; whole at any d <= 23 from column 8 on.)
So a block of 8 is off by at most 8 * 2^-13 * max |x| max |w|, as 2^m <= max |x|
max |w|, and that is added to K 2^-24 sum |x| |w|."""

import numpy as np
import pytest
import torch

from oracle import mx
from tests._util import to_dev_i32

ROWS = ("bf16", "mx8")
SHAPES = [
    # H, I, rows of each slot
    (32, 32, [1, 0, 2]),                        # one group of K either way
    (64, 96, [3, 17, 1]),
    (160, 64, [15, 16, 0, 31]),                 # K tails of one and two groups
    (544, 288, [1, 32, 33, 2]),                 # a quad and one group; two chunks and one group
    (1024, 480, [5, 65, 100, 1]),               # several passes of 32 rows
    (2048, 768, [1, 9, 40]),
    (7168, 64, [2, 33]),
    (96, 1056, [7, 129, 257]),
]


def _native():
    from vllm_moe_offload_amd import native

    return native


def _paths():
    """(path, row-tile height): the split-K kernel, then row tiles."""
    native = _native()
    return [(native.LMOE_PATH_GEMV, 32)] + [(native.LMOE_PATH_MFMA, bm) for bm in native.MX4_BLOCK_M]


def _f64(t):
    return t.detach().cpu().double().numpy()


class Layer:
    """Random 4-bit experts and rows, on the device and as 64-bit values."""

    def __init__(self, H, I, P, T, rows, seed):
        from vllm_moe_offload_amd import mxfp4, native

        rng = np.random.default_rng(seed)
        self.H, self.I, self.P, self.rows = H, I, P, rows
        w13 = torch.from_numpy(rng.standard_normal((P, 2 * I, H)).astype(np.float32) * 0.05)
        w2 = torch.from_numpy(rng.standard_normal((P, H, I)).astype(np.float32) * 0.05)
        c13, s13 = mxfp4.quantize(w13)
        c2, s2 = mxfp4.quantize(w2)
        self.w13 = mxfp4.pack_w13(c13, s13).cuda()
        self.w2 = mxfp4.pack_w2(c2, s2).cuda()
        self.v13 = [mx.values_mx4(c13[p].numpy(), s13[p].numpy()) for p in range(P)]
        self.v2 = [mx.values_mx4(c2[p].numpy(), s2[p].numpy()) for p in range(P)]
        x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(torch.bfloat16).cuda()
        self.x = x if rows == "bf16" else native.rows_to_mx8(x)
        self.xv = _f64(self.x if rows == "bf16" else self.x.float())

    def act_buffer(self, n, split=False):
        native = _native()
        if self.rows == "mx8":
            a = native.Mx8Rows.allocate(n, self.I, "cuda")
            a.q.view(torch.uint8).fill_(0x31)
            a.scale.fill_(99)
            return a
        return torch.full((n, 2, self.I) if split else (n, self.I), 7.0, dtype=torch.bfloat16, device="cuda")


def sum_error(x, w, mx8):
    """How far f32 sums over the columns of rows x and weight rows w may be off."""
    e = np.abs(x) @ np.abs(w).T * (x.shape[1] * 2.0**-24)
    if mx8:
        eight = lambda v: np.abs(v).reshape(v.shape[0], -1, 8).max(axis=2)
        e = e + 8 * 2.0**-13 * (eight(x) @ eight(w).T)
    return e


def act_values(act):
    """act rows in 64 bits: bf16, MX8, or bf16 in two parts."""
    if not isinstance(act, torch.Tensor):
        return _f64(act.float())
    return _f64(act) if act.dim() == 2 else _f64(act).sum(1)


def check_act(got, gate, up, dg, du, mx8_scale=None, step=2.0**-8):
    sg = gate / (1.0 + np.exp(-gate))
    act = sg * up
    tol = 1.1 * np.abs(up) * dg + np.abs(sg) * du + dg * du + 2.0**-20 * np.abs(act)
    if mx8_scale is None:
        tol = tol * (1 + step) + step * np.abs(act)
    else:
        tol = tol * (1 + 2.0**-4) + np.maximum(2.0**-4 * np.abs(act), 2.0**-10 * np.repeat(mx8_scale, 32, axis=1))
    assert np.all(np.abs(got - act) <= tol), float(np.max(np.abs(got - act) / np.maximum(tol, 1e-300)))


def check_layer(layer, perm, k, act, y, ids_slot):
    """Every placed pair's act and y; ids_slot[p]: the slot of pair p or -1."""
    offs = perm.offsets.cpu().numpy()
    pairs = perm.sorted_pairs.cpu().numpy()
    mx8 = layer.rows == "mx8"
    a = act_values(act)
    # two parts: the high one is off by 2^-8 of the value at most and the low one by
    # 2^-8 of that; their products are twice as many terms of 1 + 2^-8 the size
    split = not mx8 and act.dim() == 3
    step, terms = (2.0**-16, 2.01) if split else (2.0**-8, 1.0)
    sc = np.ldexp(1.0, act.scale.cpu().numpy().astype(np.int64) - 127) if mx8 else None
    yv = _f64(y)
    ystep = 2.0**-8 if y.dtype == torch.bfloat16 else 2.0**-24
    for s in range(layer.P):
        pos = np.arange(offs[s], offs[s + 1])
        if not len(pos):
            continue
        assert np.all(ids_slot[pairs[pos]] == s)
        x, w = layer.xv[pairs[pos] // k], layer.v13[s]
        g, ab = x @ w.T, sum_error(x, w, mx8)
        I = layer.I
        check_act(a[pos], g[:, :I], g[:, I:], ab[:, :I], ab[:, I:], sc[pos] if mx8 else None, step)
        want = a[pos] @ layer.v2[s].T
        tol = terms * sum_error(a[pos], layer.v2[s], mx8) * (1 + ystep) + ystep * np.abs(want)
        got = yv[pairs[pos]]
        assert np.all(np.abs(got - want) <= tol + 1e-30), float(np.max(np.abs(got - want) / (tol + 1e-30)))


def _ids(counts, extra, rng):
    ids = np.concatenate([np.repeat(np.arange(len(counts)), counts), np.full(extra, -1)]).astype(np.int32)
    return rng.permutation(ids).reshape(-1, 1)


def run_layer(layer, ids, k, path, *, block_m=None, log2phy=None, y_dtype=torch.bfloat16, split=False):
    native = _native()
    n = ids.size
    perm = native.Permutation.allocate(n, layer.P, "cuda")
    bm = native.mx4_block_m(n, layer.P) if block_m is None else block_m
    native.permute(to_dev_i32(ids), perm, log2phy=log2phy, skip_unmapped=True, block_m=bm)
    act = layer.act_buffer(n, split)
    y = torch.full((n, layer.H), -7.0, dtype=y_dtype, device="cuda")
    native.grouped_mlp(layer.x, k, layer.w13, layer.w2, perm, act, y, path=path)
    return perm, act, y


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("H,I,counts", SHAPES)
def test_products_are_the_experts(H, I, counts, rows):
    native = _native()
    rng = np.random.default_rng(H * 7 + I)
    P, T = len(counts), sum(counts) + 3
    ids = _ids(counts, 3, rng)
    l2p = rng.permutation(P).astype(np.int32)
    layer = Layer(H, I, P, T, rows, H + I)
    slot_of = np.where(ids[:, 0] >= 0, l2p[np.maximum(ids[:, 0], 0)], -1)
    for path, bm in _paths():
        for y_dtype in (torch.bfloat16, torch.float32):
            print(f"case mx4 H={H} I={I} {rows} path={path} block_m={bm} {y_dtype}", flush=True)
            perm, act, y = run_layer(layer, ids, 1, path, block_m=bm, log2phy=to_dev_i32(l2p), y_dtype=y_dtype)
            torch.cuda.synchronize()
            check_layer(layer, perm, 1, act, y, slot_of)
            placed = int(perm.meta[native.META_PAIRS])
            assert placed == sum(counts)
            # what no pair owns is left as it was
            assert torch.all(y[torch.from_numpy(ids[:, 0] < 0).cuda()] == -7.0)
            if rows == "mx8":
                assert torch.all(act.q.view(torch.uint8)[placed:] == 0x31) and torch.all(act.scale[placed:] == 99)
            else:
                assert torch.all(act[placed:] == 7.0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("H,I,counts", [(160, 96, [1, 31, 32, 33, 63, 64, 65]), (1024, 416, [127, 128, 129, 5, 300])])
def test_tile_heights_give_the_same_bits(H, I, counts, rows):
    native = _native()
    layer = Layer(H, I, len(counts), sum(counts), rows, 9)
    ids = _ids(counts, 0, np.random.default_rng(9))
    bits = lambda a, y: (y.view(torch.int16), a.q.view(torch.uint8) if rows == "mx8" else a.view(torch.int16))
    _, *want = run_layer(layer, ids, 1, native.LMOE_PATH_MFMA, block_m=32)
    for bm in native.MX4_BLOCK_M[1:]:
        _, *got = run_layer(layer, ids, 1, native.LMOE_PATH_MFMA, block_m=bm)
        for a, b in zip(bits(*got), bits(*want)):
            assert torch.equal(a, b)
    # a row alone, in whichever kernel form its tile then takes
    for t in (0, sum(counts) - 1):
        one = Layer.__new__(Layer)
        one.__dict__.update(layer.__dict__, x=layer.x[t:t + 1])
        _, _, y1 = run_layer(one, ids[t:t + 1], 1, native.LMOE_PATH_MFMA, block_m=64)
        assert torch.equal(y1[0].view(torch.int16), want[1][t].view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [
    [0] * 63 + [40, 3],                             # the last of the first 64 slots, then the next
    [0] * 64 + [33],
    [5] * 64,
    [1] * 130 + [0] * 70 + [65],                    # past 128 slots, empty ones between
    [0] * 300 + [2, 0, 0, 31],
    [200] + [0] * 400,
])
def test_tiles_find_their_slot(counts):
    native = _native()
    P = len(counts)
    layer = Layer(32, 32, P, sum(counts), "bf16", P)
    ids = _ids(counts, 0, np.random.default_rng(P))
    for bm in native.MX4_BLOCK_M:
        print(f"case mx4 slots P={P} block_m={bm}", flush=True)
        perm, act, y = run_layer(layer, ids, 1, native.LMOE_PATH_MFMA, block_m=bm)
        torch.cuda.synchronize()
        check_layer(layer, perm, 1, act, y, ids[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_several_experts_per_token_and_the_same_twice(rows):
    """top_k 3; a token may name one expert twice: both pairs get their row."""
    rng = np.random.default_rng(5)
    T, k, P = 21, 3, 5
    ids = rng.integers(0, P, (T, k)).astype(np.int32)
    ids[4] = [2, 2, 2]
    layer = Layer(96, 64, P, T, rows, 17)
    for path, bm in _paths():
        perm, act, y = run_layer(layer, ids, k, path, block_m=bm)
        torch.cuda.synchronize()
        check_layer(layer, perm, k, act, y, ids.flatten())
        assert torch.equal(y[12], y[13]) and torch.equal(y[12], y[14])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_a_bad_row_stays_its_own(rows):
    """A token that is not a number spoils its own pairs and nothing else, also
    where K ends inside a fragment."""
    from vllm_moe_offload_amd import native

    rng = np.random.default_rng(8)
    ids = _ids([6, 20], 0, rng)
    layer = Layer(160, 96, 2, 26, rows, 3)
    for path, bm in _paths():
        _, _, clean = run_layer(layer, ids, 1, path, block_m=bm)
        for value in (float("nan"), float("inf")):
            bad = layer.x.clone() if rows == "bf16" else layer.x.float().to(torch.bfloat16)
            bad[5, 159] = value
            keep, layer.x = layer.x, bad if rows == "bf16" else native.rows_to_mx8(bad)
            _, _, y = run_layer(layer, ids, 1, path, block_m=bm)
            layer.x = keep
            assert not y[5].isfinite().any()
            other = torch.arange(26, device="cuda") != 5
            assert torch.equal(y[other], clean[other])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_extreme_scales(rows):
    """Weights near both ends of the scales' range: exact powers of two pass through."""
    from vllm_moe_offload_amd import mxfp4

    layer = Layer(64, 32, 1, 2, rows, 1)
    w13 = torch.zeros(1, 64, 64)
    w13[0, :32] = torch.eye(32, 64) * 6.0
    w13[0, 32:] = torch.eye(32, 64) * 2.0**100
    w2 = torch.zeros(1, 64, 32)
    w2[0, :32] = torch.eye(32) * 2.0**-100
    layer.w13, layer.w2 = mxfp4.pack_w13(*mxfp4.quantize(w13)).cuda(), mxfp4.pack_w2(*mxfp4.quantize(w2)).cuda()
    c, s = mxfp4.quantize(w13[0]); layer.v13 = [mx.values_mx4(c.numpy(), s.numpy())]
    c, s = mxfp4.quantize(w2[0]); layer.v2 = [mx.values_mx4(c.numpy(), s.numpy())]
    ids = np.zeros((2, 1), dtype=np.int32)
    for path, bm in _paths():
        perm, act, y = run_layer(layer, ids, 1, path, block_m=bm)
        check_layer(layer, perm, 1, act, y, ids.flatten())
        assert y[:, :32].abs().max() > 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("T,k,E", [(1, 4, 8), (1, 8, 8), (3, 2, 8), (40, 4, 16), (300, 4, 8)])
def test_fused_experts_over_a_4_bit_bank(T, k, E, rows):
    """Permutation, products and combine through the layer's own call: out
    against the sum of the pairs' rows, each taken from the products' call."""
    from vllm_moe_offload_amd import fused_moe, native

    H, I = 256, 160
    rng = np.random.default_rng(T + k)
    ids = np.stack([rng.choice(E, k, replace=False) for _ in range(T)]).astype(np.int32)
    layer = Layer(H, I, E, T, rows, T)
    g = torch.Generator(device="cuda").manual_seed(T)
    w = torch.empty((T, k), device="cuda").uniform_(0.05, 1, generator=g).to(torch.bfloat16)
    add = torch.empty((T, H), device="cuda").normal_(generator=g).to(torch.bfloat16)
    l2p = to_dev_i32(rng.permutation(E))
    out = fused_moe.fused_experts(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, l2p, add=add).clone()
    ws = fused_moe.get_workspace(T, k, E, H, I, "cuda", rows=fused_moe.rows_kind(layer.x, layer.w13))
    assert ws.y.dtype == (torch.float32 if T * k <= native.FUSED_DECODE_MAX_PAIRS else torch.bfloat16)
    assert isinstance(ws.act, native.Mx8Rows) == (rows == "mx8")
    path = native.mx4_path(T * k, E)
    split = rows == "bf16" and path == native.LMOE_PATH_GEMV  # as the workspace of so few pairs has it
    _, act, y = run_layer(layer, ids, k, path, log2phy=l2p, y_dtype=torch.float32, split=split)
    yv = _f64(y).reshape(T, k, H)
    want = (_f64(w)[:, :, None] * yv).sum(1) + _f64(add)
    mag = (np.abs(_f64(w))[:, :, None] * np.abs(yv)).sum(1) + np.abs(_f64(add))
    tol = 2.0**-8 * np.abs(want) + (k + 2) * 2.0**-24 * mag
    # the rows themselves: bf16 past FUSED_DECODE_MAX_PAIRS pairs; a fused form
    # may add the same products of act in another order
    rowtol = 2.0**-8 if ws.y.dtype == torch.bfloat16 else 0.0
    av = act_values(act)
    worst = max(sum_error(av, v, rows == "mx8").max() for v in layer.v2) * (2.01 if split else 1.0)
    tol = tol + rowtol * mag + 2 * k * worst
    assert np.all(np.abs(_f64(out) - want) <= tol)
    again = fused_moe.fused_experts(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, l2p, add=add)
    assert torch.equal(again, out)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("H,I,k,E", [(32, 32, 1, 2), (160, 96, 3, 5), (1024, 416, 5, 8), (2048, 768, 8, 16),
                                     (544, 1056, 9, 12), (64, 64, 20, 4)])
def test_one_token_straight_from_its_ids(H, I, k, E, rows):
    """act is the formula's (its sums over K are cut otherwise than the split-K
    kernel's, so its last bits may be others), out the pairs' weighted sum; a pair
    without a slot adds nothing and is counted; a slot may serve several pairs."""
    from vllm_moe_offload_amd import fused_moe, native

    rng = np.random.default_rng(H + k)
    ids = rng.integers(0, E, (1, k)).astype(np.int32)  # k > E, or by chance: the same twice
    if k > 2:
        ids[0, 1] = E + 3                              # outside the table
    l2p = rng.permutation(E).astype(np.int32)
    if k > 3:
        l2p[ids[0, 3]] = -1
    layer = Layer(H, I, E, 1, rows, H)
    d_ids, d_l2p = to_dev_i32(ids), to_dev_i32(l2p)
    w = torch.empty((1, k), device="cuda").uniform_(0.05, 1).to(torch.bfloat16)
    add = torch.randn((1, H), device="cuda").to(torch.bfloat16)
    split = rows == "bf16"
    bufs = native.Mx4Buffers(native.Permutation.allocate(k, E, "cuda"), layer.act_buffer(k, split),
                             torch.empty((k, H), dtype=torch.float32, device="cuda"))
    native.device_flags(clear=True)
    out = native.mx4_decode_one(layer.x, w, d_ids, layer.w13, layer.w2, d_l2p, bufs,
                                torch.empty((1, H), dtype=torch.bfloat16, device="cuda"), add=add)
    slots = np.array([l2p[e] if e < E else -1 for e in ids[0]])
    assert native.device_flags(clear=True)[native.FLAG_UNPLACED] == int((slots < 0).sum())
    bits = lambda a: a.q.view(torch.uint8) if rows == "mx8" else a.view(torch.int16)
    mx8 = rows == "mx8"
    av, wv = act_values(bufs.act), _f64(w)[0]
    sc = np.ldexp(1.0, bufs.act.scale.cpu().numpy().astype(np.int64) - 127) if mx8 else None
    want, mag, sums = _f64(add)[0].copy(), np.abs(_f64(add))[0], np.zeros(H)
    for j in range(k):
        if slots[j] < 0:
            assert torch.equal(bits(bufs.act)[j], bits(layer.act_buffer(1, split))[0])
            continue
        gu, e = layer.xv @ layer.v13[slots[j]].T, sum_error(layer.xv, layer.v13[slots[j]], mx8)
        check_act(av[j:j + 1], gu[:, :I], gu[:, I:], e[:, :I], e[:, I:], sc[j:j + 1] if mx8 else None, 2.0**-16)
        y = wv[j] * (layer.v2[slots[j]] @ av[j])
        want, mag = want + y, mag + np.abs(y)
        # both parts' products: twice as many terms
        sums += wv[j] * sum_error(av[j:j + 1], layer.v2[slots[j]], mx8)[0] * (2.01 if split else 1.0)
    # a sum by up to eight waves, the addend and the bf16 rounding on top
    tol = 2.0**-8 * np.abs(want) + (1 + 2.0**-8) * (sums + (k + 10) * 2.0**-24 * (mag + sums))
    assert np.all(np.abs(_f64(out)[0] - want) <= tol)
    # the layer's calls take this form, with the same bits
    if (slots >= 0).all():
        again = fused_moe.fused_experts(layer.x, w, d_ids, layer.w13, layer.w2, d_l2p, add=add)
        assert torch.equal(again, out)
        inp = fused_moe.MoEFusedExpertsInput(
            hidden_states=layer.x, topk_weights=w, topk_ids=d_ids, weights=fused_moe.MoEWeights(layer.w13, layer.w2),
            routing=fused_moe.MoERoutingParams(log2phy=d_l2p), shared_output=add)
        res = fused_moe.run_fused_experts_contract(inp)
        assert torch.equal(res.routed_out, out)
        assert np.array_equal(res.expert_tokens.cpu().numpy(), np.bincount(slots, minlength=E))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("T", [1, 2, 33])
def test_decode_layer_over_a_4_bit_bank(T, rows):
    """Router, permutation and experts of a decode step: the norm's two outputs
    in, the same bits as the separate calls, captured as well as eager."""
    from vllm_moe_offload_amd import fused_moe, native

    E, H, I, k = 16, 256, 96, 4
    layer = Layer(H, I, E, T, rows, 6)
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.empty((T, H), device="cuda").normal_(generator=g).to(torch.bfloat16)
    res = torch.empty((T, H), device="cuda").normal_(generator=g).to(torch.bfloat16)
    nw = torch.empty(H, device="cuda").uniform_(0.5, 1.5, generator=g).to(torch.bfloat16)
    gate = torch.empty((E, H), device="cuda").normal_(0, 0.2, generator=g).to(torch.bfloat16)
    hidden, ro = torch.empty_like(x), torch.empty_like(res)
    mx8 = native.Mx8Rows.allocate(T, H, "cuda") if rows == "mx8" else None
    spec = fused_moe.RouterSpec(top_k=k)
    ws = fused_moe.get_workspace(T, k, E, H, I, "cuda", tag="dl", rows=rows)
    logits = torch.empty((T, E), dtype=torch.bfloat16, device="cuda")
    w, ids = torch.empty((T, k), dtype=torch.bfloat16, device="cuda"), torch.empty((T, k), dtype=torch.int32, device="cuda")
    l2p = to_dev_i32(np.random.default_rng(1).permutation(E))
    out = torch.empty_like(x)

    def step():
        native.add_rms_norm(x, nw, residual=res, residual_out=ro, out=hidden, mx8=mx8)
        fused_moe.decode_layer(hidden, gate, spec, layer.w13, layer.w2, l2p, workspace=ws, out=out, logits_out=logits,
                               w_out=w, ids_out=ids, expert_rows=mx8)

    step()
    torch.cuda.synchronize()
    want = fused_moe.fused_experts(hidden if mx8 is None else mx8, w, ids, layer.w13, layer.w2, l2p).clone()
    assert torch.equal(out, want)
    rw, rids, _ = fused_moe.route(hidden, gate, spec)
    assert torch.equal(rw, w) and torch.equal(rids, ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        x.normal_(generator=torch.Generator(device="cuda").manual_seed(seed + 50))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
        want = fused_moe.fused_experts(hidden if mx8 is None else mx8, w, ids, layer.w13, layer.w2, l2p)
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_masked_pairs_and_a_token_without_any(rows):
    """Pairs whose expert has no slot add nothing; a token without a pair is its
    addend; the status words count what was dropped."""
    from vllm_moe_offload_amd import fused_moe, native

    T, k, E, H, I = 5, 2, 6, 64, 32
    layer = Layer(H, I, 4, T, rows, 2)
    ids = np.array([[0, 1], [4, 5], [2, 4], [3, 0], [5, 1]], dtype=np.int32)
    l2p = to_dev_i32(np.array([0, 1, 2, 3, -1, -1]))
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")
    add = torch.randn((T, H), device="cuda").to(torch.bfloat16)
    native.device_flags(clear=True)
    out = fused_moe.fused_experts(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, l2p, add=add).clone()
    assert native.device_flags(clear=True)[native.FLAG_UNPLACED] == 4
    assert torch.equal(out[1], add[1])
    full = fused_moe.fused_experts(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2,
                                   to_dev_i32(np.array([0, 1, 2, 3, 0, 0])), add=add).clone()
    native.device_flags(clear=True)
    assert torch.equal(out[0], full[0]) and torch.equal(out[3], full[3]) and not torch.equal(out[2], full[2])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_a_captured_step_replays(rows):
    from vllm_moe_offload_amd import fused_moe, native

    T, k, E, H, I = 6, 2, 8, 256, 96
    rng = np.random.default_rng(1)
    layer = Layer(H, I, E, T, rows, 4)
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")
    d_ids = to_dev_i32(rng.integers(0, E, (T, k)))
    ws = fused_moe.get_workspace(T, k, E, H, I, "cuda", tag="graph", rows=fused_moe.rows_kind(layer.x, layer.w13))
    out = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
    call = lambda o, s: fused_moe.fused_experts(layer.x, w, d_ids, layer.w13, layer.w2, None, out=o, workspace=s)
    call(out, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, ws)
    for _ in range(3):
        d_ids.copy_(to_dev_i32(rng.integers(0, E, (T, k))))
        graph.replay()
        torch.cuda.synchronize()
        want = call(torch.empty_like(out), None)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    native.device_flags(clear=True)


@pytest.mark.gpu
def test_empty_batches_and_refusals():
    from vllm_moe_offload_amd import fused_moe, native

    layer = Layer(64, 32, 2, 4, "bf16", 0)
    ids = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    w = torch.ones((4, 1), dtype=torch.bfloat16, device="cuda")
    for x in (layer.x[:0], native.rows_to_mx8(layer.x)[:0]):
        assert fused_moe.fused_experts(x, w[:0], ids[:0], layer.w13, layer.w2, None).shape == (0, 64)
    perm = native.Permutation.allocate(4, 2, "cuda")
    native.permute(ids, perm)
    act, y = layer.act_buffer(4), torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    x8, a8 = native.rows_to_mx8(layer.x), native.Mx8Rows.allocate(4, 32, "cuda")
    wrong = [
        lambda: native.gateup_silu(layer.x, 1, layer.w13, perm, a8),            # rows of two kinds
        lambda: native.gateup_silu(x8, 1, layer.w13, perm, act),
        lambda: native.gateup_silu(layer.x.float(), 1, layer.w13, perm, act),
        lambda: native.gateup_silu(layer.x, 1, layer.w13[:, :, :-1].contiguous(), perm, act),
        lambda: native.gateup_silu(layer.x, 1, layer.w13[:1], perm, act),       # fewer slots
        lambda: native.gateup_silu(layer.x, 2, layer.w13, perm, act),
        lambda: native.gateup_silu(torch.zeros((4, 160), dtype=torch.bfloat16, device="cuda"), 1, layer.w13, perm, act),
        # a row of 32 columns takes as many bytes as one of 64: the down bank tells them apart
        lambda: native.grouped_mlp(layer.x[:, :32].contiguous(), 1, layer.w13, layer.w2, perm, act, y),
        lambda: fused_moe.fused_experts(layer.x[:, :32].contiguous(), w, ids, layer.w13, layer.w2, None),
        lambda: native.down(act, layer.w2, perm, y.half()),
        lambda: native.down(act, layer.w2, perm, y[:2]),
        lambda: native.down(act[:2], layer.w2, perm, y),
        lambda: native.gateup_silu(x8, 1, torch.zeros((2, 64, 64), dtype=torch.bfloat16, device="cuda"), perm, act),
        lambda: native.fused_moe_decode(layer.x, w, layer.w13, layer.w2, perm, act, y),
        lambda: native.down_combine(act, w, layer.w2, perm, y),
    ]
    bf = [torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in ((2, 64, 64), (2, 64, 32))]
    bufs = native.Mx4Buffers(perm, act, y)
    one = native.Mx4Buffers(native.Permutation.allocate(1, 2, "cuda"), layer.act_buffer(1, True), y[:1])
    whole = native.Mx4Buffers(native.Permutation.allocate(1, 2, "cuda"), act[:1], y[:1])
    out = torch.empty((4, 64), dtype=torch.bfloat16, device="cuda")
    layer_call = lambda x=layer.x, w=w, ids=ids, b=bufs, w13=layer.w13, w2=layer.w2, l2p=None, o=out, **kw: \
        native.mx4_fused_moe(x, w, ids, w13, w2, l2p, b, o, block_m=32, **kw)
    wrong += [
        lambda: fused_moe.fused_experts(x8, w, ids, *bf, None),                 # 8-bit rows, bf16 experts
        lambda: fused_moe.fused_experts(layer.x, w, ids, layer.w13, layer.w2, None,
                                        workspace=fused_moe.get_workspace(4, 1, 2, 64, 32, "cuda")),
        lambda: fused_moe.get_workspace(4, 1, 2, 64, 32, "cuda", rows="int8"),
        lambda: layer_call(x=x8),
        lambda: layer_call(w=w.float()),
        lambda: layer_call(ids=ids.long()),
        lambda: layer_call(ids=ids[:2]),
        lambda: layer_call(w13=layer.w13[:1]),
        lambda: layer_call(o=out[:2]),
        lambda: layer_call(l2p=torch.zeros(2, device="cuda")),
        lambda: layer_call(add=out.float()),
        lambda: native.mx4_decode_one(layer.x, w, ids, layer.w13, layer.w2, None, bufs, out),
        lambda: native.mx4_decode_one(layer.x[:1], w[:1], ids[:1], layer.w13, layer.w2, None, whole, out[:1]),
        lambda: native.gateup_silu(layer.x, 1, layer.w13, perm, layer.act_buffer(3, True)),
        lambda: native.down(torch.zeros((4, 3, 32), dtype=torch.bfloat16, device="cuda"), layer.w2, perm, y),
        lambda: native.gateup_silu(x8, 1, layer.w13, perm, layer.act_buffer(4, True)),
        lambda: native.Mx4Buffers(perm, act[:2], y),
        lambda: native.Mx4Buffers(perm, act, y.half()),
        lambda: fused_moe.decode_layer(layer.x, bf[0][0, :16, :].contiguous(), fused_moe.RouterSpec(top_k=1), layer.w13,
                                       layer.w2, None, workspace=fused_moe.get_workspace(4, 1, 2, 64, 32, "cuda", rows="mx8"),
                                       expert_rows=native.Mx8Rows.allocate(3, 64, "cuda")),
    ]
    layer_call()
    native.mx4_decode_one(layer.x[:1], w[:1], ids[:1], layer.w13, layer.w2, None, one, out[:1])
    for i, call in enumerate(wrong):
        with pytest.raises((ValueError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(RuntimeError, match="unsupported shape"):
        native.mx4_fused_moe(layer.x, w, ids, layer.w13, layer.w2, None, bufs, out, block_m=96,
                             path=native.LMOE_PATH_MFMA)
    with pytest.raises(RuntimeError, match="unsupported option"):
        native.gateup_silu(layer.x, 1, layer.w13, perm, act, path=native.LMOE_PATH_STREAM)
    native.permute(ids, perm, block_m=32)
    with pytest.raises(RuntimeError, match="unsupported option"):            # two parts in row tiles
        native.grouped_mlp(layer.x, 1, layer.w13, layer.w2, perm, layer.act_buffer(4, True), y, path=native.LMOE_PATH_MFMA)


@pytest.mark.gpu
@pytest.mark.parametrize("H,I,counts", [(256, 128, [1, 40, 0, 129]), (1024, 640, [3, 70, 17]), (160, 96, [5, 33])])
def test_scales_at_any_address(H, I, counts):
    """MX8 scales that start off a four-byte boundary: the same bits."""
    native = _native()
    rng = np.random.default_rng(H)
    ids = _ids(counts, 2, rng)
    layer = Layer(H, I, len(counts), len(ids), "mx8", 3)
    n = len(ids)

    def off(rows, shift):
        buf = torch.zeros(rows.scale.numel() + 4, dtype=torch.uint8, device="cuda")
        s = buf[shift:shift + rows.scale.numel()].view(rows.scale.shape)
        s.copy_(rows.scale)
        return native.Mx8Rows(rows.q, s)

    for path, bm in _paths():
        perm, act, y = run_layer(layer, ids, 1, path, block_m=bm)
        for shift in (1, 2, 3):
            a2, y2 = off(layer.act_buffer(n), shift), torch.full_like(y, -7.0)
            native.grouped_mlp(off(layer.x, shift), 1, layer.w13, layer.w2, perm, a2, y2, path=path)
            assert torch.equal(a2.q.view(torch.uint8), act.q.view(torch.uint8)) and torch.equal(a2.scale, act.scale)
            assert torch.equal(y2, y)


@pytest.mark.gpu
def test_a_slot_past_32_bits():
    """The last slot of banks of more than 2^32 bytes, by every kernel."""
    from vllm_moe_offload_amd import mxfp4, native

    H, I, P = 7168, 2048, 600
    w13, w2 = mxfp4.pack_experts(torch.empty((1, 2 * I, H), device="cuda").normal_(0, 0.05),
                                 torch.empty((1, H, I), device="cuda").normal_(0, 0.05))
    b13 = torch.zeros((P, *w13.shape[1:]), dtype=torch.uint8, device="cuda")
    b2 = torch.zeros((P, *w2.shape[1:]), dtype=torch.uint8, device="cuda")
    b13[P - 1], b2[P - 1] = w13[0], w2[0]
    assert b2.numel() > 2**32
    x = torch.empty((40, H), device="cuda").normal_().to(torch.bfloat16)
    for rows in (x, native.rows_to_mx8(x)):
        for T, path, bm in ((3, native.LMOE_PATH_GEMV, 32), (40, native.LMOE_PATH_MFMA, 32),
                            (40, native.LMOE_PATH_MFMA, 128)):
            res = []
            for slots, a, b in ((P, b13, b2), (1, w13, w2)):
                ids = torch.full((T, 1), slots - 1, dtype=torch.int32, device="cuda")
                perm = native.permute(ids, native.Permutation.allocate(T, slots, "cuda"), block_m=bm)
                act = torch.empty((T, I), dtype=torch.bfloat16, device="cuda") if rows is x else \
                    native.Mx8Rows.allocate(T, I, "cuda")
                y = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
                res.append(native.grouped_mlp(rows[:T], 1, a, b, perm, act, y, path=path))
            assert torch.equal(*res)
        one = []
        for slots, a, b in ((P, b13, b2), (1, w13, w2)):
            act = torch.empty((1, 2, I), dtype=torch.bfloat16, device="cuda") if rows is x else \
                native.Mx8Rows.allocate(1, I, "cuda")
            bufs = native.Mx4Buffers(native.Permutation.allocate(1, slots, "cuda"), act,
                                     torch.empty((1, H), dtype=torch.float32, device="cuda"))
            one.append(native.mx4_decode_one(
                rows[:1], torch.ones((1, 1), dtype=torch.bfloat16, device="cuda"),
                torch.full((1, 1), slots - 1, dtype=torch.int32, device="cuda"), a, b, None, bufs,
                torch.empty((1, H), dtype=torch.bfloat16, device="cuda")))
        assert torch.equal(*one)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_rows_past_32_bits(rows):
    """More than 2^31 elements of x and y: rows around that border and the last."""
    native = _native()
    T, H, I, P = 300_100, 7168, 32, 2
    layer = Layer(H, I, P, 1, "bf16", 1)
    x = torch.empty((T, H), dtype=torch.bfloat16, device="cuda").normal_()
    x = native.rows_to_mx8(x) if rows == "mx8" else x
    ids = torch.randint(0, P, (T, 1), dtype=torch.int32, device="cuda")
    layer.rows = rows

    def run(a, b):
        n = b - a
        part = native.Mx8Rows(x.q[a:b].clone(), x.scale[a:b].clone()) if rows == "mx8" else x[a:b].clone()
        perm = native.permute(ids[a:b].clone(), native.Permutation.allocate(n, P, "cuda"), block_m=128)
        return native.grouped_mlp(x if n == T else part, 1, layer.w13, layer.w2, perm, layer.act_buffer(n),
                                  torch.empty((n, H), dtype=torch.bfloat16, device="cuda"), path=native.LMOE_PATH_MFMA)

    y = run(0, T)
    out = native.combine(y, torch.ones((T, 1), dtype=torch.bfloat16, device="cuda"), torch.empty_like(y))
    for a, b in ((0, 64), (299_560, 299_660), (T - 64, T)):
        want = run(a, b)
        assert torch.equal(y[a:b], want) and torch.equal(out[a:b], want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("T", [1, 9, 200])
def test_two_calls_at_once(T, rows):
    """Two streams, a workspace each."""
    from vllm_moe_offload_amd import fused_moe

    k, E, H, I = 2, 8, 512, 256
    layers = [Layer(H, I, E, T, rows, s) for s in (5, 6)]
    rng = np.random.default_rng(T)
    ids = [to_dev_i32(rng.integers(0, E, (T, k))) for _ in layers]
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")
    spaces = [fused_moe.get_workspace(T, k, E, H, I, "cuda", tag=f"call{i}", rows=fused_moe.rows_kind(v.x, v.w13))
              for i, v in enumerate(layers)]
    call = lambda i: fused_moe.fused_experts(layers[i].x, w, ids[i], layers[i].w13, layers[i].w2, None,
                                             out=torch.empty((T, H), dtype=torch.bfloat16, device="cuda"), workspace=spaces[i])
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in (0, 1) for o in got[i])


@pytest.mark.gpu
def test_buffers_and_workspaces_of_another_kind_are_refused():
    from vllm_moe_offload_amd import fused_moe, native

    layer = Layer(64, 32, 2, 1, "bf16", 0)
    perm, act = native.Permutation.allocate(1, 2, "cuda"), layer.act_buffer(1)
    y = torch.empty((1, 64), dtype=torch.float32, device="cuda")
    ids = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    w = torch.ones((1, 1), dtype=torch.bfloat16, device="cuda")
    ws = fused_moe.get_workspace(1, 1, 2, 64, 32, "cuda")
    for call in (lambda: native.Mx4Buffers(native.Permutation.allocate(1, 2, "cpu"), act, y),
                 lambda: native.Mx4Buffers(perm, act, y[0]),
                 lambda: fused_moe._fused_experts_ws(layer.x, w, ids, layer.w13, layer.w2, None, workspace=ws)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("H,I,counts", [
    (32, 32, [1]),
    (64, 96, [8, 9, 1, 0, 16]),                    # a fragment for both parts, one for each
    (160, 160, [17, 7, 33]),                       # several passes, K inside a fragment
    (1024, 416, [2, 40, 24]),
    (2048, 768, [3, 12]),
])
def test_act_in_two_parts(H, I, counts):
    """Twice the bits between the products; a row's bits do not depend on the
    rows beside it, and no path has other values than the formula's."""
    native = _native()
    rng = np.random.default_rng(H + I)
    ids = _ids(counts, 3, rng)
    layer = Layer(H, I, len(counts), len(ids), "bf16", 21)
    for y_dtype in (torch.float32, torch.bfloat16):
        perm, act, y = run_layer(layer, ids, 1, native.LMOE_PATH_GEMV, y_dtype=y_dtype, split=True)
        torch.cuda.synchronize()
        check_layer(layer, perm, 1, act, y, ids[:, 0])
        assert torch.all(y[torch.from_numpy(ids[:, 0] < 0).cuda()] == -7.0)
        assert torch.all(act[sum(counts):] == 7.0)
    whole = run_layer(layer, ids, 1, native.LMOE_PATH_GEMV)[1]
    assert torch.equal(act[:sum(counts), 0], whole[:sum(counts)])                # the high part is the rounded value
    for t in (int(np.argmax(ids[:, 0] == s)) for s in range(len(counts)) if counts[s]):
        one = Layer.__new__(Layer)
        one.__dict__.update(layer.__dict__, x=layer.x[t:t + 1])
        y1 = run_layer(one, ids[t:t + 1], 1, native.LMOE_PATH_GEMV, split=True)[2]
        assert torch.equal(y1[0], y[t])


@pytest.mark.gpu
def test_act_in_two_parts_past_the_numbers():
    """Values that overflow, or are none, keep the high part's."""
    native = _native()
    layer = Layer(64, 32, 1, 3, "bf16", 2)
    layer.x[0] *= 3e36
    layer.x[1, 5] = float("nan")
    ids = np.zeros((3, 1), np.int32)
    whole = run_layer(layer, ids, 1, native.LMOE_PATH_GEMV)[1]
    _, act, y = run_layer(layer, ids, 1, native.LMOE_PATH_GEMV, split=True)
    assert torch.equal(act[:, 0].view(torch.int16), whole.view(torch.int16))
    assert torch.all(act[:, 1][~whole.isfinite()] == 0) and act[:, 1].isfinite().all()
    assert not whole[0].isfinite().all() and y[1].isnan().all() and y[2].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,H,I", [(1, 1, 4, 256, 128), (1, 2, 8, 512, 128), (2, 1, 4, 256, 128), (3, 4, 24, 1024, 416)])
def test_few_tokens_lose_no_bits_between_the_products(T, k, E, H, I):
    """out of few tokens: its own rounding and the sums', nothing of act's."""
    from vllm_moe_offload_amd import fused_moe, native

    for seed in range(4):
        rng = np.random.default_rng(100 * seed + H)
        ids = np.stack([rng.choice(E, k, replace=False) for _ in range(T)]).astype(np.int32)
        layer = Layer(H, I, E, T, "bf16", seed)
        assert native.mx4_path(T * k, E) == native.LMOE_PATH_GEMV
        w = torch.empty((T, k), device="cuda").uniform_(0.05, 1).to(torch.bfloat16)
        out = _f64(fused_moe.fused_experts(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, None))
        for t in range(T):
            want, slack = np.zeros(H), np.zeros(H)
            for j in range(k):
                v13, v2 = layer.v13[ids[t, j]], layer.v2[ids[t, j]]
                gu, e = layer.xv[t] @ v13.T, sum_error(layer.xv[t:t + 1], v13, False)[0]
                sg = gu[:I] / (1.0 + np.exp(-gu[:I]))
                act = sg * gu[I:]
                da = 1.1 * np.abs(gu[I:]) * e[:I] + np.abs(sg) * e[I:] + e[:I] * e[I:] + 2.0**-20 * np.abs(act)
                da = da * (1 + 2.0**-16) + 2.0**-16 * np.abs(act)
                wj = _f64(w)[t, j]
                want += wj * (v2 @ act)
                slack += wj * (np.abs(v2) @ da + 2.01 * sum_error((np.abs(act) + da)[None], v2, False)[0])
                slack += 2 * k * 2.0**-24 * wj * (np.abs(v2) @ np.abs(act))
            assert np.all(np.abs(out[t] - want) <= slack * (1 + 2.0**-8) + 2.0**-8 * np.abs(want))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("T,k,E,H,I", [
    (2, 1, 3, 32, 32),
    (5, 3, 40, 160, 96),
    (21, 3, 5, 96, 64),             # more pairs than slots
    (3, 8, 200, 1024, 416),
    (8, 8, 400, 64, 32),            # the most pairs
    (64, 1, 2, 32, 32),             # several passes of rows
])
def test_few_tokens_straight_from_their_ids(T, k, E, H, I, rows):
    """The permuted form's bits, of every pair and token; pairs without a slot add
    nothing, are counted and leave their rows; one slot may serve several pairs."""
    native = _native()
    rng = np.random.default_rng(T * k)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    ids[T // 2] = ids[T // 2, 0]                        # the same expert every time
    if k > 1:
        ids[T - 1, 1], ids[0, 1] = -1, E + 7            # outside the table
    l2p = rng.permutation(E).astype(np.int32)
    l2p[rng.integers(0, E)] = -1
    layer = Layer(H, I, E, T, rows, T)
    d_ids, d_l2p, n = to_dev_i32(ids), to_dev_i32(l2p), T * k
    w = torch.empty((T, k), device="cuda").uniform_(0.05, 1).to(torch.bfloat16)
    add = torch.randn((T, H), device="cuda").to(torch.bfloat16)
    slots = np.where((ids >= 0) & (ids < E), l2p[np.clip(ids, 0, E - 1)], -1).flatten()
    bits = lambda a: a.q.view(torch.uint8) if rows == "mx8" else a.view(torch.int16)
    for addend, table in ((add, d_l2p), (None, d_l2p), (add, None)):
        s = slots if table is not None else np.where((ids >= 0) & (ids < E), ids, -1).flatten()
        res = []
        for call in (native.mx4_fused_moe, native.mx4_decode_few):
            bufs = native.Mx4Buffers(native.Permutation.allocate(n, E, "cuda"), layer.act_buffer(n, rows == "bf16"),
                                     torch.full((n, H), -7.0, dtype=torch.float32, device="cuda"))
            opt = dict(path=native.LMOE_PATH_GEMV, block_m=32) if call is native.mx4_fused_moe else {}
            native.device_flags(clear=True)
            out = call(layer.x, w, d_ids, layer.w13, layer.w2, table, bufs,
                       torch.empty((T, H), dtype=torch.bfloat16, device="cuda"), add=addend, **opt)
            flags = native.device_flags(clear=True)
            assert flags[native.FLAG_UNPLACED] == int((s < 0).sum())
            res.append((out, bufs))
        (want, a), (got, b) = res
        assert torch.equal(got, want) and torch.equal(b.y, a.y)
        assert torch.all(b.y[torch.from_numpy(s < 0).cuda()] == -7.0)
        pos = a.perm.row_idx.cpu().numpy()
        placed = np.flatnonzero(s >= 0)
        assert torch.equal(bits(b.act)[placed], bits(a.act)[pos[placed]])
        left = np.flatnonzero(s < 0)
        assert torch.equal(bits(b.act)[left], bits(layer.act_buffer(len(left), rows == "bf16")))


@pytest.mark.gpu
def test_few_tokens_refusals():
    from vllm_moe_offload_amd import fused_moe, native

    layer = Layer(64, 32, 400, 4, "bf16", 0)
    w, ids = torch.ones((4, 1), dtype=torch.bfloat16, device="cuda"), torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    out = torch.empty((4, 64), dtype=torch.bfloat16, device="cuda")
    perm = native.Permutation.allocate(4, 400, "cuda")
    y = torch.empty((4, 64), dtype=torch.float32, device="cuda")
    few = lambda b, i=ids: native.mx4_decode_few(layer.x, w, i, layer.w13, layer.w2, None, b, out)
    for bufs in (native.Mx4Buffers(perm, layer.act_buffer(4), y), native.Mx4Buffers(perm, layer.act_buffer(4, True), y.bfloat16())):
        with pytest.raises(ValueError):
            few(bufs)
    with pytest.raises(ValueError):
        few(native.Mx4Buffers(perm, layer.act_buffer(4, True), y), ids.long())
    # past the most pairs the layer's call takes the permuted form
    big = Layer(64, 32, 400, 9, "bf16", 1)
    ids8 = torch.randint(0, 400, (9, 8), dtype=torch.int32, device="cuda")
    w8 = torch.full((9, 8), 0.1, dtype=torch.bfloat16, device="cuda")
    bufs = native.Mx4Buffers(native.Permutation.allocate(72, 400, "cuda"), big.act_buffer(72, True),
                             torch.empty((72, 64), dtype=torch.float32, device="cuda"))
    o8 = torch.empty((9, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="unsupported shape"):
        native.mx4_decode_few(big.x, w8, ids8, big.w13, big.w2, None, bufs, o8)
    assert fused_moe.fused_experts(big.x, w8, ids8, big.w13, big.w2, None).isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("T,k,E,bm", [(1, 2, 8, 0), (9, 2, 8, 0), (40, 2, 40, 0), (50, 2, 8, 32), (200, 2, 700, 32),
                                      (200, 2, 8, 64), (600, 4, 8, 128)])
def test_every_form_captured_and_replayed(T, k, E, bm, rows):
    """Few tokens, the permuted split-K kernel (bm 0), row tiles of every height and
    grid: replays on new ids, with eager calls of the same shape between them."""
    from vllm_moe_offload_amd import fused_moe, native

    H, I = 256, 96
    rng = np.random.default_rng(T)
    layer = Layer(H, I, E, T, rows, 4)
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")
    d_ids = to_dev_i32(rng.integers(0, E, (T, k)))
    ws = [fused_moe.get_workspace(T, k, E, H, I, "cuda", tag=t, rows=rows) for t in ("forms", "forms eager")]
    out = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")

    def call(o, s):
        if bm:
            return native.mx4_fused_moe(layer.x, w, d_ids, layer.w13, layer.w2, None, s.mx4, o,
                                        path=native.LMOE_PATH_MFMA, block_m=bm)
        return fused_moe.fused_experts(layer.x, w, d_ids, layer.w13, layer.w2, None, out=o, workspace=s)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, ws[0])
    for _ in range(3):
        d_ids.copy_(to_dev_i32(rng.integers(0, E, (T, k))))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = call(torch.empty_like(out), ws[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    native.device_flags(clear=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("H,I", [(32, 32), (128, 160), (384, 128), (672, 416), (1120, 96)])
def test_one_and_two_chunks_a_stage_give_the_same_bits(H, I, rows):
    """32-row tiles on grids of few and of many workgroups (two chunks a stage, one),
    odd numbers of chunks, a row that is not a number among the others."""
    native = _native()
    layer = Layer(H, I, 3, 40, rows, H)
    ids = np.random.default_rng(I).integers(0, 3, (40, 1)).astype(np.int32)
    if rows == "mx8":
        layer.x.scale[7, -1] = 255
    else:
        layer.x[7, H - 1] = float("nan")
    few = run_layer(layer, ids, 1, native.LMOE_PATH_MFMA, block_m=32)
    wide = Layer.__new__(Layer)                    # the same experts before many that get no row
    extra = lambda b: torch.cat([b, torch.zeros((600, *b.shape[1:]), dtype=torch.uint8, device="cuda")])
    wide.__dict__.update(layer.__dict__, P=603, w13=extra(layer.w13), w2=extra(layer.w2))
    ids2 = np.concatenate([ids, np.full((600, 1), -1, np.int32)])
    keep = layer.x
    wide.x = torch.cat([keep, keep[:1].expand(600, H)]) if rows == "bf16" else native.Mx8Rows(
        torch.cat([keep.q.view(torch.uint8), keep.q.view(torch.uint8)[:1].expand(600, H)]).view(torch.float8_e4m3fn),
        torch.cat([keep.scale, keep.scale[:1].expand(600, H // 32)]))
    many = run_layer(wide, ids2, 1, native.LMOE_PATH_MFMA, block_m=32)
    bits = lambda a: a.q.view(torch.uint8) if rows == "mx8" else a.view(torch.int16)
    assert torch.equal(bits(few[1]), bits(many[1])[:40])
    assert torch.equal(few[2].view(torch.int16), many[2][:40].view(torch.int16))
    assert few[2][7].isnan().all() and few[2][torch.arange(40, device="cuda") != 7].isfinite().all()
