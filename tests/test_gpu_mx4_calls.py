"""Calls over 4-bit experts as programs make them: a decode step beside its
separate calls, the full layer's check, calls on several streams and threads,
results that are kept, events, very long rows.  (tests/test_gpu_mx4.py checks the
values, tests/test_gpu_mx4_layer.py the layer.)"""

import threading

import numpy as np
import pytest
import torch

from oracle import mx
from tests._util import to_dev_i32
from tests.test_gpu_mx4 import ROWS, Layer, check_act, check_layer, run_layer, sum_error

pytestmark = pytest.mark.gpu


def _bits(t):
    return t.view(torch.int16)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("T", [12, 18, 24, 28])
def test_a_decode_step_takes_the_path_of_its_separate_calls(T, rows, monkeypatch):
    """3, 4.5, 6 and 7 pairs per expert, around the borders of both kinds of rows:
    the router reads bf16 rows, the experts' rows choose the path."""
    from vllm_moe_offload_amd import fused_moe, native

    E, H, I, k = 16, 2048, 416, 4
    layer = Layer(H, I, E, T, rows, 6)
    g = torch.Generator(device="cuda").manual_seed(T)
    hidden = torch.empty((T, H), device="cuda").normal_(generator=g).to(torch.bfloat16)
    x = hidden if rows == "bf16" else native.rows_to_mx8(hidden)
    gate = torch.empty((E, H), device="cuda").normal_(0, 0.2, generator=g).to(torch.bfloat16)
    l2p = to_dev_i32(np.random.default_rng(1).permutation(E))
    ws = fused_moe.get_workspace(T, k, E, H, I, "cuda", tag="step", rows=rows)
    paths, mlp = [], native.grouped_mlp

    def spy(*a, **kw):
        paths.append(kw["path"])
        return mlp(*a, **kw)

    monkeypatch.setattr(native, "grouped_mlp", spy)
    out, w, ids = fused_moe.decode_layer(hidden, gate, fused_moe.RouterSpec(top_k=k), layer.w13, layer.w2, l2p,
                                         workspace=ws, out=torch.empty_like(hidden),
                                         expert_rows=x if rows == "mx8" else None)
    want = fused_moe.fused_experts(x, w, ids, layer.w13, layer.w2, l2p, out=torch.empty_like(hidden))
    torch.cuda.synchronize()
    assert paths == [native.mx4_path(T * k, E, rows == "mx8")]
    assert torch.equal(_bits(out), _bits(want))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("T", [1, 2, 8, 9, 60])
def test_the_full_layer_fails_closed_on_any_number_of_tokens(T, rows):
    """A pair without a slot is an error, with few pairs (no permutation in the
    call of fused_experts) as with many; good ids pass, whatever came before."""
    from tests.test_gpu_mx4_layer import E, H, _layer, _weights, _x
    from vllm_moe_offload_amd import fused_moe, mxfp4, native

    w13, w2, gate = _weights(11)
    layer, rt = _layer(210, w13, w2, gate, slots=8, b2_wave_prefill=True)
    b13, b2 = (t.cuda() for t in mxfp4.pack_experts(w13, w2))
    x = _x(T, T)
    w, ids, _ = fused_moe.route(x, gate, layer.router_spec)
    x = x if rows == "bf16" else native.rows_to_mx8(x)
    bad = ids.clone()
    bad[T - 1, 2] = E + 5
    run = lambda i, **kw: fused_moe.run_full_layer(rt, layer_id=210, hidden=x, topk_weights=w, topk_ids=i,  # noqa: E731
                                                   num_logical_experts=E, **kw)
    want = fused_moe.fused_experts(x, w, ids, b13, b2, torch.arange(E, dtype=torch.int32, device="cuda")).clone()
    for path in (native.LMOE_PATH_AUTO, native.LMOE_PATH_GEMV):
        with pytest.raises(RuntimeError, match="without ready slots: 1 pairs"):
            run(bad, path=path)
        assert torch.equal(_bits(run(ids)), _bits(want))
    native.device_flags(clear=True)


def _experts(kind, E, H, I, T, seed):
    """(rows, w13, w2) of bf16 experts, or of 4-bit ones with bf16 or 8-bit rows."""
    layer = Layer(H, I, E, T, "mx8" if kind == "mx8" else "bf16", seed)
    if kind != "bf16 experts":
        return layer.x, layer.w13, layer.w2
    g = torch.Generator(device="cuda").manual_seed(seed)
    w13, w2 = (torch.empty(s, device="cuda").normal_(0, 0.05, generator=g).to(torch.bfloat16)
               for s in ((E, 2 * I, H), (E, H, I)))
    return layer.x, w13, w2


KINDS = ("bf16 experts", "bf16", "mx8")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 3, 9, 200])
def test_default_calls_on_two_streams_and_from_two_threads(T, kind):
    """Calls of one shape without a workspace of the caller's, at once."""
    from vllm_moe_offload_amd import fused_moe

    k, E, H, I = 2, 8, 512, 256
    parts = [_experts(kind, E, H, I, T, s) for s in (5, 6)]
    rng = np.random.default_rng(T)
    ids = [to_dev_i32(np.stack([rng.permutation(E)[:k] for _ in range(T)])) for _ in parts]
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")

    def call(i):
        x, w13, w2 = parts[i]
        return fused_moe.fused_experts(x, w, ids[i], w13, w2, None,
                                       out=torch.empty((T, H), dtype=torch.bfloat16, device="cuda"))

    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(_bits(o), _bits(want[i])) for i in (0, 1) for o in got[i])

    got = [[], []]
    ready = threading.Barrier(2)

    def work(i):
        ready.wait()
        for _ in range(20):
            got[i].append(call(i))  # both on the default stream

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(len(g) == 20 for g in got)
    assert all(torch.equal(_bits(o), _bits(want[i])) for i in (0, 1) for o in got[i])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 3, 9, 200])
def test_graphs_of_default_calls_replayed_at_once(T, kind):
    """Two graphs of one shape on two streams, eager calls of the shape on a third; each
    graph holds the layer twice, the second over the first's result."""
    from vllm_moe_offload_amd import fused_moe, native

    k, E, H, I = 2, 8, 512, 256
    parts = [_experts(kind, E, H, I, T, s) for s in (5, 6, 7)]
    rng = np.random.default_rng(T)
    ids = [to_dev_i32(np.stack([rng.permutation(E)[:k] for _ in range(T)])) for _ in parts]
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")

    def layers(i):
        x, w13, w2 = parts[i]
        first = fused_moe.fused_experts(x, w, ids[i], w13, w2, None)
        again = native.rows_to_mx8(first) if kind == "mx8" else first
        return first, fused_moe.fused_experts(again, w, ids[i], w13, w2, None)

    want = [tuple(t.clone() for t in layers(i)) for i in range(3)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in (0, 1):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(layers(i))
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        eager = []
        for _ in range(4):
            for i in (0, 1):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
            with torch.cuda.stream(streams[2]):
                eager.append(layers(2))
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(outs[i], want[i]))
        assert all(torch.equal(_bits(a), _bits(b)) for e in eager for a, b in zip(e, want[2]))


def test_workspaces_of_streams_threads_and_captures():
    from vllm_moe_offload_amd import fused_moe

    get = lambda device="cuda", **kw: fused_moe.get_workspace(7, 2, 4, 64, 32, device, **kw)  # noqa: E731
    here = get()
    assert get("cuda:0") is here and get(torch.device("cuda", 0)) is here and get(tag="other") is not here
    side, other = torch.cuda.Stream(), []
    with torch.cuda.stream(side):
        there = get()
        assert there is not here and get() is there
    t = threading.Thread(target=lambda: other.append(get()))
    t.start()
    t.join()
    assert other[0] is not here and other[0] is not there
    assert get() is here
    # a capture's is its own, one that a caller asks for there starts as zeros
    warm = get(tag="warm")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = get(tag="warm")
        meta = inside.perm.meta.clone()
        inside.perm.meta.fill_(5)
        inside.out.fill_(1.0)
    assert inside is not warm and get(tag="warm") is warm
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert not meta.any() and (inside.perm.meta == 5).all() and not warm.perm.meta.any()
    fused_moe.clear_workspaces()
    assert get(tag="warm") is not warm


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 5, 60])
def test_results_are_the_callers(T, kind):
    """A result made by the call outlives the next call of its shape."""
    from vllm_moe_offload_amd import fused_moe

    E, H, I, k = 16, 256, 128, 4
    x, w13, w2 = _experts(kind, E, H, I, T, 6)
    rng = np.random.default_rng(T)
    w = torch.full((T, k), 0.25, dtype=torch.bfloat16, device="cuda")
    ids = [to_dev_i32(np.stack([rng.permutation(E)[:k] for _ in range(T)])) for _ in range(2)]
    ident = torch.arange(E, dtype=torch.int32, device="cuda")

    def contract(i):
        inp = fused_moe.MoEFusedExpertsInput(
            hidden_states=x, topk_weights=w, topk_ids=i, weights=fused_moe.MoEWeights(w13, w2),
            routing=fused_moe.MoERoutingParams(log2phy=ident))
        return fused_moe.run_fused_experts_contract(inp).routed_out

    for call in (contract, lambda i: fused_moe.fused_experts(x, w, i, w13, w2, ident)):
        first = call(ids[0])
        kept = first.clone()
        second = call(ids[1])
        assert torch.equal(_bits(first), _bits(kept)) and not torch.equal(first, second)


@pytest.mark.parametrize("device_waves", [False, True])
def test_results_of_waves_and_of_the_full_layer_are_the_callers(device_waves):
    from tests.test_gpu_mx4_layer import E, _layer, _weights, _x
    from vllm_moe_offload_amd import fused_moe

    w13, w2, gate = _weights(12)
    layer, rt = _layer(211, w13, w2, gate, slots=8, b2_wave_prefill=True, device_wave_prefill=device_waves)
    runs = [lambda **a: fused_moe.run_full_layer(rt, **a),
            lambda **a: fused_moe.run_device_waves(rt, **a) if device_waves else fused_moe.run_wave_prefill(rt, **a)[0]]
    for run in runs:
        res = []
        for seed in (1, 2):
            x = _x(150, seed)
            w, ids, _ = fused_moe.route(x, gate, layer.router_spec)
            out = run(layer_id=211, hidden=x, topk_weights=w, topk_ids=ids, num_logical_experts=E)
            res.append((out, out.clone()))
        assert torch.equal(*res[0]) and not torch.equal(res[0][0], res[1][0])


@pytest.mark.parametrize("T", [1, 3])
def test_events_come_where_the_contract_has_them(T, monkeypatch):
    """Before the permutation, before GMM2 and before the combine; one token, whose
    down product has the combine in it, records the last two after its permutation."""
    from vllm_moe_offload_amd import fused_moe, native

    E, H, I, k = 8, 256, 96, 2
    layer = Layer(H, I, E, T, "bf16", 3)
    w = torch.full((T, k), 0.5, dtype=torch.bfloat16, device="cuda")
    ids = to_dev_i32(np.stack([np.random.default_rng(t).permutation(E)[:k] for t in range(T)]))
    order = []

    def spy(name):
        call = getattr(native, name)

        def run(*a, **kw):
            order.append(name)
            return call(*a, **kw)

        monkeypatch.setattr(native, name, run)

    for name in ("permute", "gateup_silu", "down", "combine", "mx4_decode_one", "mx4_fused_moe"):
        spy(name)

    class Event(torch.cuda.Event):
        def record(self, stream=None):
            order.append("event")
            super().record(*([] if stream is None else [stream]))

    monkeypatch.setattr(torch.cuda, "Event", Event)
    inp = fused_moe.MoEFusedExpertsInput(hidden_states=layer.x, topk_weights=w, topk_ids=ids,
                                         weights=fused_moe.MoEWeights(layer.w13, layer.w2))
    res = fused_moe.run_fused_experts_contract(inp, record_events=True)
    torch.cuda.synchronize()
    assert all(e.query() for e in (res.before_dispatch_evt, res.before_gmm2_evt, res.before_combine_evt))
    if T == 1:
        assert order == ["event", "permute", "event", "event", "mx4_decode_one"]
    else:
        assert order == ["event", "permute", "gateup_silu", "event", "down", "event", "combine"]


def _long_rows(T, K, seed):
    """8-bit rows of more columns than one call of rows_to_mx8 takes."""
    from vllm_moe_offload_amd import native

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty((T * (K // 320), 320), device="cuda").normal_(generator=g).to(torch.bfloat16)
    r = native.rows_to_mx8(x)
    return native.Mx8Rows(r.q.view(T, K), r.scale.view(T, K // 32))


@pytest.mark.parametrize("bm", [32, 64, 128])
@pytest.mark.parametrize("side", ["gateup", "down"])
def test_the_longest_8_bit_rows_of_each_height(bm, side):
    """Rows whose scales just fit a tile's LDS, against the split-K kernel, which
    keeps none there: sums of the same products, cut otherwise."""
    from vllm_moe_offload_amd import mxfp4, native

    K, T, out = native.MX4_MAX_COLUMNS_MX8[bm], bm + 3, 64
    print(f"case longest rows K={K} block_m={bm} {side}", flush=True)
    x = _long_rows(T, K, bm)
    g = torch.Generator(device="cuda").manual_seed(1)
    codes, scales = mxfp4.quantize(torch.empty((1, out, K), device="cuda").normal_(0, 0.05, generator=g))
    ids = torch.zeros((T, 1), dtype=torch.int32, device="cuda")
    ids[T - 2] = -1
    perm = native.permute(ids, native.Permutation.allocate(T, 1, "cuda"), skip_unmapped=True, block_m=bm)
    xv = x.float().double().cpu().numpy()[perm.sorted_pairs.cpu().numpy()[:T - 1]] if side == "gateup" else \
        x.float().double().cpu().numpy()[:T - 1]
    wv = mxfp4.dequantize(codes, scales)[0].double().cpu().numpy()
    want, err = xv @ wv.T, sum_error(xv, wv, True)
    if side == "down":
        bank = mxfp4.pack_w2(codes, scales)
        for path in (native.LMOE_PATH_GEMV, native.LMOE_PATH_MFMA):
            y = torch.full((T, out), -7.0, dtype=torch.float32, device="cuda")
            native.down(x, bank, perm, y, path=path)
            got = y.cpu().double().numpy()[perm.sorted_pairs.cpu().numpy()[:T - 1]]
            assert np.all(np.abs(got - want) <= err * (1 + 2.0**-24) + 2.0**-24 * np.abs(want))
            assert torch.all(y[T - 2] == -7.0)
    else:
        bank = mxfp4.pack_w13(codes, scales)
        for path in (native.LMOE_PATH_GEMV, native.LMOE_PATH_MFMA):
            act = native.Mx8Rows.allocate(T, out // 2, "cuda")
            native.gateup_silu(x, 1, bank, perm, act, path=path)
            sc = np.ldexp(1.0, act.scale.cpu().numpy().astype(np.int64) - 127)[:T - 1]
            check_act(act.float().double().cpu().numpy()[:T - 1], want[:, :32], want[:, 32:], err[:, :32], err[:, 32:], sc)


def test_many_long_8_bit_rows_choose_a_height_that_holds_them():
    """The norm gives rows up to 32768 columns, more than the tallest tile holds."""
    from vllm_moe_offload_amd import fused_moe, mxfp4, native

    T, H, I = 8300, 32704, 1024
    assert native.mx4_block_m(T, 1, I) == 128 and H > native.MX4_MAX_COLUMNS_MX8[128]
    g = torch.Generator(device="cuda").manual_seed(1)
    w13, w2 = mxfp4.pack_experts(torch.empty((1, 2 * I, H), device="cuda").normal_(0, 0.05, generator=g),
                                 torch.empty((1, H, I), device="cuda").normal_(0, 0.05, generator=g))
    x = native.rows_to_mx8(torch.empty((T, H), dtype=torch.bfloat16, device="cuda").normal_(generator=g))
    ids, w = torch.zeros((T, 1), dtype=torch.int32, device="cuda"), torch.ones((T, 1), dtype=torch.bfloat16, device="cuda")
    out = fused_moe.fused_experts(x, w, ids, w13, w2, None)
    ws = fused_moe.get_workspace(T, 1, 1, H, I, "cuda", tag="long", rows="mx8")
    want = native.mx4_fused_moe(x, w, ids, w13, w2, None, ws.mx4, torch.empty_like(out), path=native.LMOE_PATH_MFMA,
                                block_m=32)
    torch.cuda.synchronize()
    assert torch.equal(_bits(out), _bits(want)) and out[::100].isfinite().all()
    fused_moe.clear_workspaces()


@pytest.mark.parametrize("rows", ROWS)
def test_auto_needs_a_permutation_of_its_own_tiles(rows):
    """One built at the default height, the bf16 kernels': taken with few pairs per
    slot, refused by name past them; the split-K kernel by name takes it."""
    from vllm_moe_offload_amd import native

    E, H, I = 4, 256, 96
    few = native.MX4_FEW_PAIRS_PER_EXPERT_MX8 if rows == "mx8" else native.MX4_FEW_PAIRS_PER_EXPERT
    for T in (few * E, few * E + 1):
        layer = Layer(H, I, E, T, rows, 6)
        ids = torch.arange(T, dtype=torch.int32, device="cuda").remainder_(E).view(T, 1)
        perm = native.permute(ids, native.Permutation.allocate(T, E, "cuda"))
        act, y = layer.act_buffer(T), torch.empty((T, H), dtype=torch.float32, device="cuda")
        want = native.grouped_mlp(layer.x, 1, layer.w13, layer.w2, perm, act, y, path=native.LMOE_PATH_GEMV).clone()
        if T == few * E:
            assert torch.equal(native.grouped_mlp(layer.x, 1, layer.w13, layer.w2, perm, act, y), want)
            continue
        for call in (lambda: native.gateup_silu(layer.x, 1, layer.w13, perm, act),
                     lambda: native.down(act, layer.w2, perm, y),
                     lambda: native.grouped_mlp(layer.x, 1, layer.w13, layer.w2, perm, act, y)):
            with pytest.raises(ValueError, match="block_m 256"):
                call()
        native.permute(ids, perm, block_m=native.mx4_block_m(T, E, I))
        native.grouped_mlp(layer.x, 1, layer.w13, layer.w2, perm, act, y)
        check_layer(layer, perm, 1, act, y, ids.cpu().numpy().flatten())


def _at(v, e):
    """v [R, K] rounded to e4m3 at the given group exponents."""
    s = np.ldexp(1.0, np.repeat(e, 32, axis=1))
    g = mx.e4m3_grid()
    return np.sign(v) * g[mx._nearest(v / s, g)] * s


def check_rounded_act(got, act, da):
    """MX8 act rows (values, exponents) against act in 64 bits, off by da at most: the
    exponent is the smallest that holds the group (the formula's, or where its largest
    value lies within da of a border the one beyond it), and the values are act's own
    rounding at that exponent, or where act lies within da of a tie its neighbour."""
    values, e = got
    amax = np.abs(act).reshape(act.shape[0], -1, 32)
    slack = da.reshape(amax.shape)
    low, high = (np.maximum(amax - slack, 0.0)).max(axis=2), (amax + slack).max(axis=2)
    top = lambda v: mx.group_exponents(np.repeat(v, 32, axis=1), 448.0)  # noqa: E731
    assert np.all((top(low) <= e) & (e <= top(high)))
    sign = np.where(act < 0, -1.0, 1.0)
    a, b = _at(sign * np.maximum(np.abs(act) - da, 0.0), e), _at(sign * (np.abs(act) + da), e)
    crossing = np.abs(act) <= da  # either sign
    lo, hi = np.minimum(a, b), np.maximum(a, b)
    lo, hi = np.where(crossing, np.minimum(lo, -hi), lo), np.where(crossing, np.maximum(hi, -lo), hi)
    assert np.all((lo <= values) & (values <= hi)), float(np.max(np.maximum(lo - values, values - hi)))


@pytest.mark.parametrize("H,I,counts", [(32, 32, [1, 0, 2]), (64, 96, [3, 17, 1]), (544, 288, [1, 32, 33, 2]),
                                        (1024, 416, [5, 65, 100, 1]), (2048, 768, [1, 9, 40])])
def test_act_in_8_bits_is_its_own_rounding(H, I, counts):
    """The scale that the gate-up product gives a group of act, from the formula and
    not from what it stored; groups of one row are far from those beside them."""
    from vllm_moe_offload_amd import native

    rng = np.random.default_rng(H + I)
    P, T = len(counts), sum(counts)
    layer = Layer(H, I, P, T, "mx8", 31)
    # rows of very different sizes: a scale taken from another row would show at once
    step = torch.from_numpy(rng.integers(-12, 13, (T, 1)).astype(np.int16)).cuda()
    layer.x = native.Mx8Rows(layer.x.q, (layer.x.scale.to(torch.int16) + step).to(torch.uint8))
    layer.xv = layer.x.float().double().cpu().numpy()
    ids = rng.permutation(np.repeat(np.arange(P), counts)).astype(np.int32).reshape(-1, 1)

    def check(values, exps, t, slot):
        x, w = layer.xv[t], layer.v13[slot]
        gu, err = x @ w.T, sum_error(x, w, True)
        gate, up, dg, du = gu[:, :I], gu[:, I:], err[:, :I], err[:, I:]
        sg = gate / (1.0 + np.exp(-gate))
        act = sg * up
        da = 1.1 * np.abs(up) * dg + np.abs(sg) * du + dg * du + 2.0**-20 * np.abs(act)
        check_rounded_act((values, exps), act, da)

    take = lambda rows: (rows.float().double().cpu().numpy(), rows.scale.cpu().numpy().astype(np.int64) - 127)  # noqa: E731
    for path, bm in [(native.LMOE_PATH_GEMV, 32)] + [(native.LMOE_PATH_MFMA, b) for b in native.MX4_BLOCK_M]:
        print(f"case act scales H={H} I={I} path={path} block_m={bm}", flush=True)
        perm, act, _ = run_layer(layer, ids, 1, path, block_m=bm)
        values, exps = take(act)
        pairs, offs = perm.sorted_pairs.cpu().numpy(), perm.offsets.cpu().numpy()
        for s in range(P):
            pos = np.arange(offs[s], offs[s + 1])
            if len(pos):
                check(values[pos], exps[pos], pairs[pos], s)
    # one token and few, straight from their ids: act rows lie by pair
    for t, call in ((1, native.mx4_decode_one), (min(T, 30), native.mx4_decode_few)):
        part = native.Mx8Rows(layer.x.q[:t].clone(), layer.x.scale[:t].clone())
        bufs = native.Mx4Buffers(native.Permutation.allocate(t, P, "cuda"), layer.act_buffer(t),
                                 torch.empty((t, H), dtype=torch.float32, device="cuda"))
        call(part, torch.ones((t, 1), dtype=torch.bfloat16, device="cuda"), to_dev_i32(ids[:t]), layer.w13, layer.w2, None,
             bufs, torch.empty((t, H), dtype=torch.bfloat16, device="cuda"))
        values, exps = take(bufs.act)
        for s in range(P):
            pos = np.flatnonzero(ids[:t, 0] == s)
            if len(pos):
                check(values[pos], exps[pos], pos, s)


@pytest.mark.parametrize("T,k,E,H,I", [(1, 2, 8, 512, 128), (3, 4, 24, 1024, 416), (12, 4, 8, 256, 160), (90, 3, 8, 512, 256)])
def test_8_bit_rows_end_to_end(T, k, E, H, I):
    """out of every form against the experts in 64 bits, act rounded to MX8 in between:
    where act lies near a tie its other neighbour is allowed, nothing more."""
    from vllm_moe_offload_amd import fused_moe, native

    rng = np.random.default_rng(T)
    layer = Layer(H, I, E, T, "mx8", 17)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    w = torch.empty((T, k), device="cuda").uniform_(0.05, 1, generator=torch.Generator(device="cuda").manual_seed(T)).to(torch.bfloat16)
    out = fused_moe.fused_experts(layer.x, w, to_dev_i32(ids), layer.w13, layer.w2, None).double().cpu().numpy()
    wv = w.double().cpu().numpy()
    want, slack = np.zeros((T, H)), np.zeros((T, H))
    for s in range(E):
        t, j = np.nonzero(ids == s)
        if not len(t):
            continue
        x, v13, v2 = layer.xv[t], layer.v13[s], layer.v2[s]
        gu, err = x @ v13.T, sum_error(x, v13, True)
        gate, up, dg, du = gu[:, :I], gu[:, I:], err[:, :I], err[:, I:]
        sg = gate / (1.0 + np.exp(-gate))
        exact = sg * up
        da = 1.1 * np.abs(up) * dg + np.abs(sg) * du + dg * du + 2.0**-20 * np.abs(exact)
        act, y = mx.expert(x, v13, v2, True)
        # how far the stored act may be from the rounded one: at the group's exponent and,
        # where its largest value is within da of a border, at the next one
        grp = np.abs(exact).reshape(len(t), -1, 32)
        top = lambda v: mx.group_exponents(np.repeat(v, 32, axis=1), 448.0)  # noqa: E731
        e0 = top(np.maximum(grp - da.reshape(grp.shape), 0.0).max(axis=2))
        e1 = top((grp + da.reshape(grp.shape)).max(axis=2))
        off = np.zeros_like(act)
        for e in (e0, e1):
            for v in (exact - da, exact, exact + da):
                off = np.maximum(off, np.abs(_at(v, e) - act))
        wj = wv[t, j][:, None]
        dy = off @ np.abs(v2).T + sum_error(np.abs(act) + off, v2, True)
        np.add.at(want, t, wj * y)
        np.add.at(slack, t, wj * (dy + 2 * k * 2.0**-24 * (np.abs(y) + dy)))
    assert np.all(np.abs(out - want) <= slack * (1 + 2.0**-8) + 2.0**-8 * np.abs(want))


def test_constants_are_there_for_every_stream():
    """The shared expert's ones and zeros, made on a stream that is behind and read on
    another; one made in a capture is not kept for eager calls."""
    from vllm_moe_offload_amd import layer as layer_mod

    dev, side = torch.device("cuda", 0), torch.cuda.Stream()
    layer_mod.clear_constants()
    torch.cuda._sleep(20_000_000)
    a, b = layer_mod._ones_bf16(4099, dev), layer_mod._zeros_i32(4099, dev)
    with torch.cuda.stream(side):
        got = layer_mod._ones_bf16(4099, dev).clone(), layer_mod._zeros_i32(4099, dev).clone()
    side.synchronize()
    assert (got[0] == 1).all() and not got[1].any()
    assert layer_mod._ones_bf16(4099, dev) is a and layer_mod._zeros_i32(4099, dev) is b
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = layer_mod._ones_bf16(4101, dev)
        out = inside + 1
    assert layer_mod._ones_bf16(4101, dev) is not inside and (layer_mod._ones_bf16(4101, dev) == 1).all()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert (out == 2).all()
