"""Expert products of 4-bit rows over 4-bit slot banks against the experts in 64 bits.

Tolerances, per element and by stage.  4-bit by 4-bit products are multiples of a quarter
of their scales, at most 36 of them: the matrix instruction's sums of eight lose nothing,
so a sum over K columns is off by at most K 2^-24 sum |x| |w| (dg, du for gate and up).
act = silu(gate) up then moves by da = 1.1 |up| dg + |silu(gate)| du + dg du + 2^-20 |act|
(see test_gpu_mx4.py).  Its rounding is the definition's of some value within da: a group's
scale is that of a largest magnitude within da, and a code's value lies within half a step
of a value within da (steps 0.5 up to 2, 1 up to 4, 2 up to 6, times the scale).  y is
checked against the act that the kernel stored, so only its own sum and store count."""

import numpy as np
import pytest
import torch

from oracle import mx
from tests._util import to_dev_i32
from tests.test_gpu_mx4 import SHAPES, Layer, _f64, _ids, run_layer, sum_error

pytestmark = pytest.mark.gpu


def _native():
    from vllm_moe_offload_amd import native

    return native


def _paths():
    """(path, row-tile height): the split-K kernel, then row tiles."""
    native = _native()
    return [(native.LMOE_PATH_GEMV, 32)] + [(native.LMOE_PATH_MFMA, bm) for bm in native.MX4_ROWS_BLOCK_M]


class Layer4(Layer):
    """Random 4-bit experts and 4-bit rows."""

    def __init__(self, H, I, P, T, seed):
        super().__init__(H, I, P, T, "bf16", seed)
        self.rows, self.dense = "mx4", self.x
        self.x = _native().rows_to_mx4(self.x)
        self.xv = _f64(self.x.float())

    def act_buffer(self, n, split=False):
        a = _native().Mx4Rows.allocate(n, self.I, "cuda")
        a.q.fill_(0x31)
        a.scale.fill_(99)
        return a


def act_error(gate, up, dg, du):
    sg = gate / (1.0 + np.exp(-np.clip(gate, -700, 700)))
    act = sg * up
    return act, 1.1 * np.abs(up) * dg + np.abs(sg) * du + dg * du + 2.0**-20 * np.abs(act)


def check_rounding(got, scale_bytes, v, d):
    """got and its scales are the 4-bit rounding of values within d of v."""
    e = scale_bytes.astype(np.int64) - 127
    big, small = np.abs(v) + d, np.maximum(np.abs(v) - d, 0.0)
    assert np.all(e <= mx.group_exponents(big, 6.0)) and np.all(e >= mx.group_exponents(small, 6.0))
    s = np.ldexp(1.0, np.repeat(e, 32, axis=1))
    half = np.where(big <= 2 * s, 0.25, np.where(big <= 4 * s, 0.5, 1.0)) * s
    off = np.abs(got - v)
    assert np.all(off <= half * (1 + 2.0**-40) + d), float(np.max(off / (half + d)))


def check_layer(layer, perm, k, act, y, ids_slot):
    offs, pairs = perm.offsets.cpu().numpy(), perm.sorted_pairs.cpu().numpy()
    a, sc, yv = _f64(act.float()), act.scale.cpu().numpy(), _f64(y)
    ystep = 2.0**-8 if y.dtype == torch.bfloat16 else 2.0**-24
    I = layer.I
    for s in range(layer.P):
        pos = np.arange(offs[s], offs[s + 1])
        if not len(pos):
            continue
        assert np.all(ids_slot[pairs[pos]] == s)
        x, w = layer.xv[pairs[pos] // k], layer.v13[s]
        g, e = x @ w.T, sum_error(x, w, False)
        v, d = act_error(g[:, :I], g[:, I:], e[:, :I], e[:, I:])
        check_rounding(a[pos], sc[pos], v, d)
        want = a[pos] @ layer.v2[s].T
        tol = sum_error(a[pos], layer.v2[s], False) * (1 + ystep) + ystep * np.abs(want)
        off = np.abs(yv[pairs[pos]] - want)
        assert np.all(off <= tol + 1e-30), float(np.max(off / (tol + 1e-30)))


def _bits(act, y):
    return act.q, act.scale, y.view(torch.int16) if y.dtype is torch.bfloat16 else y.view(torch.int32)


@pytest.mark.parametrize("H,I,counts", SHAPES + [(4096, 256, [300, 0, 1, 511])])
def test_products_are_the_experts(H, I, counts):
    native = _native()
    rng = np.random.default_rng(H * 7 + I)
    P, T = len(counts), sum(counts) + 3
    ids = _ids(counts, 3, rng)
    l2p = rng.permutation(P).astype(np.int32)
    layer = Layer4(H, I, P, T, H + I)
    slot_of = np.where(ids[:, 0] >= 0, l2p[np.maximum(ids[:, 0], 0)], -1)
    for path, bm in _paths():
        for y_dtype in (torch.bfloat16, torch.float32):
            print(f"case mx44 H={H} I={I} path={path} block_m={bm} {y_dtype}", flush=True)
            perm, act, y = run_layer(layer, ids, 1, path, block_m=bm, log2phy=to_dev_i32(l2p), y_dtype=y_dtype)
            torch.cuda.synchronize()
            check_layer(layer, perm, 1, act, y, slot_of)
            placed = int(perm.meta[native.META_PAIRS])
            assert placed == sum(counts)
            # what no pair owns is left as it was
            assert torch.all(y[torch.from_numpy(ids[:, 0] < 0).cuda()] == -7.0)
            assert torch.all(act.q[placed:] == 0x31) and torch.all(act.scale[placed:] == 99)


@pytest.mark.parametrize("H,I,counts", [(160, 96, [1, 31, 32, 33, 63, 64, 65]), (1024, 416, [127, 128, 129, 5, 300]),
                                        (544, 1056, [255, 256, 257, 1])])
def test_tile_heights_give_the_same_bits(H, I, counts):
    native = _native()
    if not native.MX4_ROWS_BLOCK_M:
        pytest.skip("one height")
    layer = Layer4(H, I, len(counts), sum(counts), 9)
    ids = _ids(counts, 0, np.random.default_rng(9))
    _, *want = run_layer(layer, ids, 1, native.LMOE_PATH_MFMA, block_m=native.MX4_ROWS_BLOCK_M[0])
    for bm in native.MX4_ROWS_BLOCK_M[1:]:
        _, *got = run_layer(layer, ids, 1, native.LMOE_PATH_MFMA, block_m=bm)
        for a, b in zip(_bits(*got), _bits(*want)):
            assert torch.equal(a, b)
    for t in (0, sum(counts) - 1):  # a row alone, in whichever kernel form its tile then takes
        one = Layer4.__new__(Layer4)
        one.__dict__.update(layer.__dict__, x=layer.x[t:t + 1])
        _, _, y1 = run_layer(one, ids[t:t + 1], 1, native.LMOE_PATH_MFMA, block_m=native.MX4_ROWS_BLOCK_M[-1])
        assert torch.equal(y1[0].view(torch.int16), want[1][t].view(torch.int16))


def test_several_experts_per_token_and_the_same_twice():
    rng = np.random.default_rng(5)
    T, k, P = 21, 3, 5
    ids = rng.integers(0, P, (T, k)).astype(np.int32)
    ids[4] = [2, 2, 2]
    layer = Layer4(96, 64, P, T, 17)
    for path, bm in _paths():
        perm, act, y = run_layer(layer, ids, k, path, block_m=bm)
        torch.cuda.synchronize()
        check_layer(layer, perm, k, act, y, ids.flatten())
        assert torch.equal(y[12], y[13]) and torch.equal(y[12], y[14])


def test_a_bad_row_stays_its_own():
    """A group that is not a number spoils its own token's pairs and nothing else, also
    where K ends inside a fragment; act's scales say so."""
    native = _native()
    ids = _ids([6, 20], 0, np.random.default_rng(8))
    layer = Layer4(160, 96, 2, 26, 3)
    for path, bm in _paths():
        _, _, clean = run_layer(layer, ids, 1, path, block_m=bm)
        for value in (float("nan"), float("inf")):
            bad = layer.dense.clone()
            bad[5, 159] = value
            keep, layer.x = layer.x, native.rows_to_mx4(bad)
            perm, act, y = run_layer(layer, ids, 1, path, block_m=bm)
            layer.x = keep
            rest = torch.arange(26, device="cuda") != 5
            assert y[5].isnan().all() and torch.equal(y[rest], clean[rest])
            at = int(perm.row_idx[5])
            assert bool((act.scale[at] == 255).all()) and not bool(act.q[at].any())


def test_extreme_scales():
    """Scales far from 1 on either side, that multiply to ordinary numbers."""
    from vllm_moe_offload_amd import mxfp4, native

    H, I, T = 256, 64, 40
    g = torch.Generator().manual_seed(3)
    ids = np.zeros((T, 1), np.int32)
    for ex in (-100, 60):
        layer = Layer4(H, I, 1, T, 5)
        layer.x = native.rows_to_mx4((torch.randn((T, H), generator=g) * 2.0**ex).cuda())
        layer.xv = _f64(layer.x.float())
        codes, scales = mxfp4.quantize(torch.randn((1, 2 * I, H), generator=g) * 2.0**-ex * 0.05)
        layer.w13 = mxfp4.pack_w13(codes, scales).cuda()
        layer.v13 = [mx.values_mx4(codes[0].numpy(), scales[0].numpy())]
        for path, bm in _paths():
            perm, act, y = run_layer(layer, ids, 1, path, block_m=bm)
            torch.cuda.synchronize()
            check_layer(layer, perm, 1, act, y, ids[:, 0])


@pytest.mark.parametrize("H,I,counts", [(256, 128, [1, 40, 0, 129]), (1024, 640, [3, 70, 17]), (160, 96, [5, 33])])
def test_scales_at_any_address(H, I, counts):
    native = _native()
    layer = Layer4(H, I, len(counts), sum(counts), 4)
    ids = _ids(counts, 0, np.random.default_rng(4))
    for path, bm in _paths():
        want = run_layer(layer, ids, 1, path, block_m=bm)
        keep = layer.x
        for shift in (1, 2, 7):
            room = torch.full((keep.scale.numel() + 32,), 255, dtype=torch.uint8, device="cuda")
            sc = room[shift:shift + keep.scale.numel()].view(keep.scale.shape).copy_(keep.scale)
            layer.x = native.Mx4Rows(keep.q, sc)
            got = run_layer(layer, ids, 1, path, block_m=bm)
            assert all(torch.equal(a, b) for a, b in zip(_bits(*got[1:]), _bits(*want[1:])))
        layer.x = keep


def layer_value(layer, ids, slots, w, add=None):
    """The layer in 64 bits from the kernel-independent definition, act rounded to 4 bits,
    and how far the combine of f32 rows may be off where act's codes are the definition's."""
    T, k = ids.shape
    out, mag = np.zeros((T, layer.H)), np.zeros((T, layer.H))
    for t in range(T):
        for j in range(k):
            s = slots[t, j]
            if s < 0:
                continue
            gu = layer.v13[s] @ layer.xv[t]
            gate, up = gu[:layer.I], gu[layer.I:]
            v = (gate / (1.0 + np.exp(-gate)) * up)[None]
            act = mx.values_mx4(*mx.quantize_mx4(v))
            out[t] += w[t, j] * (layer.v2[s] @ act[0])
            mag[t] += np.abs(w[t, j]) * (np.abs(layer.v2[s]) @ np.abs(act[0]))
    if add is not None:
        out, mag = out + add, mag + np.abs(add)
    return out, mag


@pytest.mark.parametrize("T,k,E,H,I", [(1, 4, 8, 256, 160), (1, 1, 3, 64, 32), (2, 2, 8, 512, 128), (9, 4, 8, 256, 96),
                                       (40, 4, 16, 256, 160), (300, 4, 8, 256, 160)])
def test_layer_end_to_end(T, k, E, H, I):
    """fused_experts against the definition in 64 bits.  A code of act at a border goes
    either way (its value moves by a step of its group), so outputs are compared in the
    2-norm: codes within d of a border, a part of about 7 d / 6 of them, d some 2^-20 of the
    group's scale, are too few to show beside the store's 2^-9 (y rows past 1024 pairs are
    stored in bf16 as well: twice that)."""
    from vllm_moe_offload_amd import fused_moe

    rng = np.random.default_rng(T + k)
    ids = np.stack([rng.choice(E, k, replace=False) for _ in range(T)]).astype(np.int32)
    layer = Layer4(H, I, E, T, T)
    l2p = rng.permutation(E).astype(np.int32)
    g = torch.Generator(device="cuda").manual_seed(T)
    w = torch.empty((T, k), device="cuda").uniform_(0.05, 1, generator=g).to(torch.bfloat16)
    add = torch.empty((T, H), device="cuda").normal_(0, 0.01, generator=g).to(torch.bfloat16)
    out = fused_moe.fused_experts(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, to_dev_i32(l2p), add=add)
    want, _ = layer_value(layer, ids, l2p[ids], _f64(w), _f64(add))
    rel = np.linalg.norm(_f64(out) - want) / np.linalg.norm(want)
    assert rel <= (2 if T * k > 1024 else 1) * 2.0**-8, rel
    again = fused_moe.fused_experts(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, to_dev_i32(l2p), add=add)
    assert torch.equal(again, out)


@pytest.mark.parametrize("H,I,k,E", [(32, 32, 1, 2), (160, 96, 3, 5), (1024, 416, 5, 8), (2048, 768, 8, 16),
                                     (544, 1056, 9, 12), (64, 64, 20, 4)])
def test_one_token_straight_from_its_ids(H, I, k, E):
    from vllm_moe_offload_amd import native

    rng = np.random.default_rng(H + k)
    ids = rng.integers(0, E, (1, k)).astype(np.int32)
    if k > 2:
        ids[0, 1] = E + 3                              # outside the table
    l2p = rng.permutation(E).astype(np.int32)
    if k > 3:
        l2p[ids[0, 3]] = -1
    layer = Layer4(H, I, E, 1, H)
    w = torch.empty((1, k), device="cuda").uniform_(0.05, 1).to(torch.bfloat16)
    add = torch.randn((1, H), device="cuda").to(torch.bfloat16)
    bufs = native.Mx4Buffers(native.Permutation.allocate(k, E, "cuda"), layer.act_buffer(k),
                             torch.empty((k, H), dtype=torch.float32, device="cuda"))
    native.device_flags(clear=True)
    out = native.mx4_decode_one(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, to_dev_i32(l2p), bufs,
                                torch.empty((1, H), dtype=torch.bfloat16, device="cuda"), add=add)
    slots = np.array([l2p[e] if e < E else -1 for e in ids[0]])
    assert native.device_flags(clear=True)[native.FLAG_UNPLACED] == int((slots < 0).sum())
    a, sc, wv = _f64(bufs.act.float()), bufs.act.scale.cpu().numpy(), _f64(w)[0]
    want, mag, sums = _f64(add)[0].copy(), np.abs(_f64(add))[0], np.zeros(H)
    for j in range(k):
        if slots[j] < 0:
            assert bool((bufs.act.q[j] == 0x31).all())
            continue
        gu, e = layer.xv @ layer.v13[slots[j]].T, sum_error(layer.xv, layer.v13[slots[j]], False)
        check_rounding(a[j:j + 1], sc[j:j + 1], *act_error(gu[:, :I], gu[:, I:], e[:, :I], e[:, I:]))
        y = wv[j] * (layer.v2[slots[j]] @ a[j])
        want, mag = want + y, mag + np.abs(y)
        sums += wv[j] * sum_error(a[j:j + 1], layer.v2[slots[j]], False)[0]
    tol = 2.0**-8 * np.abs(want) + (1 + 2.0**-8) * (sums + (k + 10) * 2.0**-24 * (mag + sums))
    assert np.all(np.abs(_f64(out)[0] - want) <= tol)


@pytest.mark.parametrize("T,k,E,H,I", [(2, 1, 4, 256, 128), (3, 4, 24, 1024, 416), (8, 4, 6, 160, 96), (16, 4, 3, 64, 32)])
def test_few_tokens_straight_from_their_ids(T, k, E, H, I):
    """The same bits as with a permutation."""
    from vllm_moe_offload_amd import native

    rng = np.random.default_rng(T)
    ids = rng.integers(-1, E + 1, (T, k)).astype(np.int32)
    layer = Layer4(H, I, E, T, T)
    w = torch.empty((T, k), device="cuda").uniform_(0.05, 1).to(torch.bfloat16)
    l2p = to_dev_i32(rng.permutation(E))

    def bufs():
        return native.Mx4Buffers(native.Permutation.allocate(T * k, E, "cuda"), layer.act_buffer(T * k),
                                 torch.empty((T * k, H), dtype=torch.float32, device="cuda"))

    out = lambda: torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
    args = (layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, l2p)
    few = native.mx4_decode_few(*args, bufs(), out())
    want = native.mx4_fused_moe(*args, bufs(), out(), path=native.LMOE_PATH_GEMV, block_m=32)
    assert torch.equal(few, want)
    native.device_flags(clear=True)


@pytest.mark.parametrize("T", [1, 2, 33, 200])
def test_decode_layer_with_4_bit_rows(T):
    """The norm's two outputs into the router and the experts: the bits of the separate
    calls, captured as well as eager."""
    from vllm_moe_offload_amd import fused_moe, native

    E, H, I, k = 16, 256, 96, 4
    layer = Layer4(H, I, E, T, 6)
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.empty((T, H), device="cuda").normal_(generator=g).to(torch.bfloat16)
    res = torch.empty((T, H), device="cuda").normal_(generator=g).to(torch.bfloat16)
    nw = torch.empty(H, device="cuda").uniform_(0.5, 1.5, generator=g).to(torch.bfloat16)
    gate = torch.empty((E, H), device="cuda").normal_(0, 0.2, generator=g).to(torch.bfloat16)
    hidden, ro = torch.empty_like(x), torch.empty_like(res)
    mx4 = native.Mx4Rows.allocate(T, H, "cuda")
    spec = fused_moe.RouterSpec(top_k=k)
    ws = fused_moe.get_workspace(T, k, E, H, I, "cuda", tag="dl", rows="mx4")
    logits = torch.empty((T, E), dtype=torch.bfloat16, device="cuda")
    w, ids = torch.empty((T, k), dtype=torch.bfloat16, device="cuda"), torch.empty((T, k), dtype=torch.int32, device="cuda")
    l2p = to_dev_i32(np.random.default_rng(1).permutation(E))
    out = torch.empty_like(x)

    def step():
        native.add_rms_norm(x, nw, residual=res, residual_out=ro, out=hidden, mx4=mx4)
        fused_moe.decode_layer(hidden, gate, spec, layer.w13, layer.w2, l2p, workspace=ws, out=out, logits_out=logits,
                               w_out=w, ids_out=ids, expert_rows=mx4)

    step()
    want = fused_moe.fused_experts(mx4, w, ids, layer.w13, layer.w2, l2p)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
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
        assert torch.equal(got, fused_moe.fused_experts(mx4, w, ids, layer.w13, layer.w2, l2p))


@pytest.mark.parametrize("T,k,E", [(1, 2, 8), (9, 2, 8), (40, 2, 40), (50, 2, 8), (200, 2, 300), (600, 4, 8)])
def test_calls_at_once_and_captured(T, k, E):
    """Default calls on two streams, and two graphs of them replayed at once: each has
    memory of its own."""
    from vllm_moe_offload_amd import fused_moe, native

    H, I = 256, 96
    rng = np.random.default_rng(T)
    parts = [Layer4(H, I, E, T, s) for s in (4, 5)]
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")
    ids = [to_dev_i32(rng.integers(0, E, (T, k))) for _ in parts]
    outs = [torch.empty((T, H), dtype=torch.bfloat16, device="cuda") for _ in parts]
    call = lambda i, **kw: fused_moe.fused_experts(parts[i].x, w, ids[i], parts[i].w13, parts[i].w2, None, **kw)
    graphs, streams = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], [torch.cuda.Stream(), torch.cuda.Stream()]
    call(0)
    torch.cuda.synchronize()
    for i in (0, 1):
        with torch.cuda.graph(graphs[i]):
            call(i, out=outs[i])
    for _ in range(3):
        for i in (0, 1):
            ids[i].copy_(to_dev_i32(rng.integers(0, E, (T, k))))
        want = [call(i) for i in (0, 1)]
        torch.cuda.synchronize()
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                got.append(call(i))
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(got[i], want[i]) and torch.equal(outs[i], want[i])
    native.device_flags(clear=True)


def test_rows_past_32_bits():
    """More than 2^31 columns of rows: the last tokens are those of a small call."""
    native = _native()
    T, H, I, P = 300_100, 7168, 32, 2
    layer = Layer4(H, I, P, 40, 6)
    small = run_layer(layer, np.zeros((40, 1), np.int32), 1, native.LMOE_PATH_GEMV)
    big = Layer4.__new__(Layer4)
    big.__dict__.update(layer.__dict__)
    q = torch.zeros((T, H // 2), dtype=torch.uint8, device="cuda")
    sc = torch.full((T, H // 32), 127, dtype=torch.uint8, device="cuda")
    q[-40:], sc[-40:] = layer.x.q, layer.x.scale
    big.x = native.Mx4Rows(q, sc)
    for path, bm in _paths()[1:] or _paths():
        perm, act, y = run_layer(big, np.zeros((T, 1), np.int32), 1, path, block_m=bm)
        torch.cuda.synchronize()
        if path == native.LMOE_PATH_GEMV:
            assert torch.equal(y[-40:], small[2])
        check_rows = Layer4.__new__(Layer4)
        check_rows.__dict__.update(layer.__dict__)
        want = _f64(act[T - 40:].float()) @ layer.v2[0].T
        tol = sum_error(_f64(act[T - 40:].float()), layer.v2[0], False) * 1.01 + 2.0**-8 * np.abs(want)
        assert np.all(np.abs(_f64(y[-40:]) - want) <= tol + 1e-30)
        assert not bool(y[:1000].any())
        del act, y


def test_buffers_and_rows_of_another_kind_are_refused():
    from vllm_moe_offload_amd import fused_moe, native

    layer = Layer4(64, 32, 2, 4, 1)
    ids = to_dev_i32(np.zeros((4, 1)))
    w = torch.ones((4, 1), dtype=torch.bfloat16, device="cuda")
    x8 = native.rows_to_mx8(layer.dense)
    for rows, x in (("bf16", layer.x), ("mx8", layer.x), ("mx4", layer.dense), ("mx4", x8)):
        ws = fused_moe.get_workspace(4, 1, 2, 64, 32, "cuda", rows=rows)
        with pytest.raises(ValueError, match="x and act"):
            fused_moe.fused_experts(x, w, ids, layer.w13, layer.w2, None, workspace=ws)
        with pytest.raises(ValueError, match="x and act"):
            native.gateup_silu(x, 1, layer.w13, ws.perm, ws.act_rows(4, native.LMOE_PATH_MFMA))
    with pytest.raises(ValueError, match="4-bit rows"):
        fused_moe.fused_experts(layer.x, w, ids, torch.zeros((2, 64, 64), dtype=torch.bfloat16, device="cuda"),
                                torch.zeros((2, 64, 32), dtype=torch.bfloat16, device="cuda"), None)
    with pytest.raises(ValueError):  # rows of another length
        fused_moe.fused_experts(native.Mx4Rows.allocate(4, 96, "cuda"), w, ids, layer.w13, layer.w2, None)
    with pytest.raises(ValueError):  # scales of too few rows
        fused_moe.fused_experts(native.Mx4Rows(layer.x.q, layer.x.scale[:3]), w, ids, layer.w13, layer.w2, None)


def test_empty_batches():
    from vllm_moe_offload_amd import fused_moe

    layer = Layer4(64, 32, 2, 4, 1)
    none = layer.x[:0]
    out = fused_moe.fused_experts(none, torch.empty((0, 2), dtype=torch.bfloat16, device="cuda"),
                                  torch.empty((0, 2), dtype=torch.int32, device="cuda"), layer.w13, layer.w2, None)
    assert out.shape == (0, 64)


@pytest.mark.parametrize("device_waves", [False, True])
@pytest.mark.parametrize("T", [5, 150, 600])
def test_capacity_waves_and_the_full_layer_equal_one_bank(T, device_waves):
    from tests.test_gpu_mx4_layer import E, _layer, _weights, _x
    from vllm_moe_offload_amd import fused_moe, mxfp4, native

    w13, w2, gate = _weights(2)
    layer, rt = _layer(260, w13, w2, gate, slots=8, b2_wave_prefill=True, device_wave_prefill=device_waves)
    x = _x(T, T)
    w, ids, _ = fused_moe.route(x, gate, layer.router_spec)
    rows = native.rows_to_mx4(x)
    args = dict(layer_id=260, hidden=rows, topk_weights=w, topk_ids=ids, num_logical_experts=E)
    b13, b2 = (t.cuda() for t in mxfp4.pack_experts(w13, w2))
    want = fused_moe.fused_experts(rows, w, ids, b13, b2, torch.arange(E, dtype=torch.int32, device="cuda"))
    out = fused_moe.run_device_waves(rt, **args) if device_waves else fused_moe.run_wave_prefill(rt, **args)[0]
    full = fused_moe.run_full_layer(rt, **args)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(full, want)


@pytest.mark.parametrize("T,top_k", [(10, 4), (1, 12)])
def test_decode_overflow_equals_one_bank(T, top_k):
    from tests.test_gpu_mx4_layer import E, H, I, _layer, _weights, _x
    from vllm_moe_offload_amd import fused_moe, mxfp4, native

    w13, w2, gate = _weights(3)
    slots = 16 if T > 1 else 8
    layer, rt = _layer(261, w13, w2, gate, slots=slots, top_k=top_k, decode_overflow=True, graph_compatible_offload=True)
    b13, b2 = (t.cuda() for t in mxfp4.pack_experts(w13, w2))
    spec = layer.router_spec
    ws = fused_moe.get_workspace(T, top_k, slots, H, I, torch.device("cuda"), tag="ovf4", rows="mx4")
    for step in range(3):
        x = _x(T, 70 + step)
        rows = native.rows_to_mx4(x)
        w, ids, _ = fused_moe.route(x, gate, spec)
        active = tuple(sorted(set(ids.cpu().flatten().tolist())))
        plan = rt.stage_fixed_slot_plan(layer_id=261, active_experts=active, num_logical_experts=E)
        bank = rt.slot_bank(261)
        out, _, _ = fused_moe.decode_layer(x, gate, spec, bank.w13_slots, bank.w2_slots, rt.log2phy_buffer(261), workspace=ws,
                                           overflow=rt.decode_overflow_slot_weights(layer_id=261, n_pairs=T * top_k),
                                           expert_rows=rows)
        rt.record_layer_compute(261)
        want = fused_moe.fused_experts(rows, w, ids, b13, b2, torch.arange(E, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert torch.equal(out, want), (step, plan.overflow is not None)


def test_rows_past_2_gib():
    """x of more than 2^31 bytes: the last tokens' act is that of a small call, bit for bit
    (row tiles add a row's chunks in order, whatever lies beside it)."""
    native = _native()
    T, H, I, P = 300_100, 16384, 32, 2
    layer = Layer4(H, I, P, 40, 11)
    ids = to_dev_i32(np.zeros((40, 1), np.int32))
    perm = native.Permutation.allocate(40, P, "cuda")
    want = layer.act_buffer(40)
    native.permute(ids, perm, block_m=64)
    native.gateup_silu(layer.x, 1, layer.w13, perm, want, path=native.LMOE_PATH_MFMA)
    q = torch.zeros((T, H // 2), dtype=torch.uint8, device="cuda")
    sc = torch.full((T, H // 32), 127, dtype=torch.uint8, device="cuda")
    q[-40:], sc[-40:] = layer.x.q, layer.x.scale
    act = layer.act_buffer(T)
    perm = native.Permutation.allocate(T, P, "cuda")
    for bm in native.MX4_ROWS_BLOCK_M:
        native.permute(to_dev_i32(np.zeros((T, 1), np.int32)), perm, block_m=bm)
        native.gateup_silu(native.Mx4Rows(q, sc), 1, layer.w13, perm, act, path=native.LMOE_PATH_MFMA)
        torch.cuda.synchronize()
        assert torch.equal(act.q[-40:], want.q) and torch.equal(act.scale[-40:], want.scale), bm
        assert not bool(act.q[:-40].bitwise_and(0x77).any()), bm


def test_two_threads_at_once():
    """A thread each with a stream of its own: rows, projection and experts, over and over."""
    import threading

    from vllm_moe_offload_amd import fused_moe, mxfp4

    native = _native()
    H, I, E, k, T = 512, 96, 8, 2, 33
    layers = [Layer4(H, I, E, T, s) for s in (21, 22)]
    proj = [native.quantize_mx4(torch.randn((H, H), generator=torch.Generator().manual_seed(s)).cuda() * 0.05)
            for s in (1, 2)]
    assert proj[0].shape == (H, mxfp4.row_bytes(H))
    ids = [to_dev_i32(np.random.default_rng(s).integers(0, E, (T, k))) for s in (1, 2)]
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")

    def once(i):
        mid = native.rows_to_mx4(native.mx4_linear(layers[i].x, proj[i]))
        return fused_moe.fused_experts(mid, w, ids[i], layers[i].w13, layers[i].w2, None)

    want = [once(i) for i in (0, 1)]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got[i].append(once(i))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # reported by the test's own thread
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for i in (0, 1):
        assert all(torch.equal(y, want[i]) for y in got[i])
