"""4-bit experts through the layer: host store, slot bank, staging, capacity
waves, decode overflow and shared experts move 4-bit experts as they move bf16
ones; the results are, bit for bit, those of one call over a bank that holds every
expert (whose values tests/test_gpu_mx4.py checks)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _mods():
    from vllm_moe_offload_amd import fused_moe, mxfp4, native
    from vllm_moe_offload_amd.layer import SlotMoELayer
    from vllm_moe_offload_amd.moe_offload.config import MoeOffloadConfig
    from vllm_moe_offload_amd.moe_offload.runtime import MoeOffloadRuntime

    return fused_moe, mxfp4, native, SlotMoELayer, MoeOffloadConfig, MoeOffloadRuntime


E, H, I = 32, 512, 160


def _weights(seed, experts=E):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.empty(s).normal_(0.0, 0.05, generator=g).to(torch.bfloat16)  # noqa: E731
    return mk(experts, 2 * I, H), mk(experts, H, I), mk(experts, H).cuda()


def _layer(layer_id, w13, w2, gate, *, slots, top_k=4, **kw):
    _, _, _, SlotMoELayer, Cfg, Runtime = _mods()
    cfg = {k: kw.pop(k) for k in list(kw) if k in ("decode_overflow", "b2_wave_prefill", "device_wave_prefill",
                                                   "graph_compatible_offload")}
    rt = Runtime(Cfg(enabled=True, num_slots=slots, async_load=True, pin_host_memory=True, **cfg))
    layer = SlotMoELayer(layer_id=layer_id, runtime=rt, gate_weight=gate, w13_weight=w13, w2_weight=w2, top_k=top_k,
                         weight_format="mxfp4", **kw)
    layer.register()
    return layer, rt


def _x(T, seed):
    return torch.empty((T, H), device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(seed)).to(
        torch.bfloat16)


@pytest.mark.parametrize("slots", [16, 32])
def test_decode_steps_with_staging_equal_one_bank(slots):
    fused_moe, mxfp4, native, *_ = _mods()
    w13, w2, gate = _weights(1)
    layer, rt = _layer(200, w13, w2, gate, slots=slots)
    buf = rt.host_store.get_layer_buffer(200)
    assert buf.w13.dtype == torch.uint8 and buf.w13.is_pinned()
    # 4 bits a column and a byte for 32 (rows of 160 columns are stored as 256)
    assert buf.total_bytes == E * (2 * I * (H // 2 + H // 32) + H * (256 // 2 + 512 // 32))
    b13, b2 = (t.cuda() for t in mxfp4.pack_experts(w13, w2))
    assert torch.equal(b13.cpu(), buf.w13) and layer.hidden_size == H and layer.intermediate_size == I
    for step, T in enumerate((1, 4, 1, 3, 2, 4)):
        print(f"case mx4 decode step {step} T={T}", flush=True)
        x = _x(T, step)
        out = layer.forward(x).clone()
        w, ids, _ = fused_moe.route(x, gate, layer.router_spec)
        want = fused_moe.fused_experts(x, w, ids, b13, b2, torch.arange(E, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
    assert rt.transfer_engine.bytes_issued > 0


@pytest.mark.parametrize("device_waves", [False, True])
@pytest.mark.parametrize("T", [150, 600])
def test_capacity_waves_equal_the_unsplit_layer(T, device_waves):
    fused_moe, mxfp4, native, *_ = _mods()
    w13, w2, gate = _weights(2)
    layer, rt = _layer(201, w13, w2, gate, slots=8, b2_wave_prefill=True, device_wave_prefill=device_waves)
    x = _x(T, T)
    w, ids, _ = fused_moe.route(x, gate, layer.router_spec)
    args = dict(layer_id=201, hidden=x, topk_weights=w, topk_ids=ids, num_logical_experts=E)
    b13, b2 = (t.cuda() for t in mxfp4.pack_experts(w13, w2))
    want = fused_moe.fused_experts(x, w, ids, b13, b2, torch.arange(E, dtype=torch.int32, device="cuda")).clone()
    if device_waves:
        out = fused_moe.run_device_waves(rt, **args).clone()
    else:
        out, report = fused_moe.run_wave_prefill(rt, **args)
        out = out.clone()
        assert len(report.waves) == 4
    full = fused_moe.run_full_layer(rt, **args).clone()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(full, want)
    # 8-bit rows through the same waves
    x8 = native.rows_to_mx8(x)
    args["hidden"] = x8
    want = fused_moe.fused_experts(x8, w, ids, b13, b2, torch.arange(E, dtype=torch.int32, device="cuda")).clone()
    out = fused_moe.run_device_waves(rt, **args) if device_waves else fused_moe.run_wave_prefill(rt, **args)[0]
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("T,top_k", [(10, 4), (1, 12)])
def test_decode_overflow_equals_one_bank_eager_and_replayed(T, top_k):
    fused_moe, mxfp4, native, *_ = _mods()
    w13, w2, gate = _weights(3)
    slots = 16 if T > 1 else 8
    layer, rt = _layer(202, w13, w2, gate, slots=slots, top_k=top_k, decode_overflow=True, graph_compatible_offload=True)
    b13, b2 = (t.cuda() for t in mxfp4.pack_experts(w13, w2))
    ident = torch.arange(E, dtype=torch.int32, device="cuda")
    spec = layer.router_spec
    ws = fused_moe.get_workspace(T, top_k, slots, H, I, torch.device("cuda"), tag="ovf", rows="bf16")
    static_x, out = torch.empty((T, H), dtype=torch.bfloat16, device="cuda"), torch.empty((T, H), dtype=torch.bfloat16,
                                                                                          device="cuda")

    def stage(x):
        _, ids, _ = fused_moe.route(x, gate, spec)
        active = tuple(sorted(set(ids.cpu().flatten().tolist())))
        return rt.stage_fixed_slot_plan(layer_id=202, active_experts=active, num_logical_experts=E)

    def run():
        ovf = rt.decode_overflow_slot_weights(layer_id=202, n_pairs=T * top_k)
        bank = rt.slot_bank(202)
        fused_moe.decode_layer(static_x, gate, spec, bank.w13_slots, bank.w2_slots, rt.log2phy_buffer(202), workspace=ws,
                               out=out, overflow=ovf)

    graph, over = None, []
    for step in range(5):
        x = _x(T, 70 + step) if step != 2 else torch.zeros((T, H), dtype=torch.bfloat16, device="cuda")
        static_x.copy_(x)
        plan = stage(x)
        over.append(plan.overflow is not None)
        print(f"case mx4 overflow step {step} {over[-1]}", flush=True)
        if graph is None:
            run()
        else:
            graph.replay()
        rt.record_layer_compute(202)
        w, ids, _ = fused_moe.route(x, gate, spec)
        want = fused_moe.fused_experts(x, w, ids, b13, b2, ident)
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
        if graph is None:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                run()
            torch.cuda.current_stream().wait_stream(s)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                run()
            rt.record_layer_compute(202)
    assert any(over)
    # the seam takes the same passes
    for step in range(2):
        x = _x(T, 90 + step)
        got = layer.forward(x).clone()
        w, ids, _ = fused_moe.route(x, gate, spec)
        want = fused_moe.fused_experts(x, w, ids, b13, b2, ident)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_shared_experts_in_4_bits():
    """A shared expert of the routed shape is a pinned slot; a wider one runs as a
    one-slot pass whose output the combine adds."""
    fused_moe, mxfp4, native, *_ = _mods()
    w13, w2, gate = _weights(4)
    s13, s2, _ = _weights(5, 1)
    layer, rt = _layer(203, w13, w2, gate, slots=E + 1, shared_w13=s13[0], shared_w2=s2[0])
    assert layer.mix_placement
    b13, b2 = (t.cuda() for t in mxfp4.pack_experts(torch.cat([w13, s13]), torch.cat([w2, s2])))
    ident = torch.arange(E + 1, dtype=torch.int32, device="cuda")
    for T in (1, 5, 90):
        x = _x(T, T)
        out = layer.forward(x).clone()
        w, ids, _ = fused_moe.route(x, gate, layer.router_spec)
        assert ids.shape[1] == 5 and int(ids[0, 4]) == E
        want = fused_moe.fused_experts(x, w, ids, b13, b2, ident)
        torch.cuda.synchronize()
        assert torch.equal(out, want), T
    g = torch.Generator().manual_seed(9)
    wide13 = torch.empty(2 * 3 * I, H).normal_(0, 0.05, generator=g).to(torch.bfloat16)
    wide2 = torch.empty(H, 3 * I).normal_(0, 0.05, generator=g).to(torch.bfloat16)
    layer, rt = _layer(204, w13, w2, gate, slots=E, shared_w13=wide13.cuda(), shared_w2=wide2.cuda())
    assert not layer.mix_placement and layer.shared_w13.dtype == torch.uint8
    d13, d2 = mxfp4.pack_experts(wide13[None].cuda(), wide2[None].cuda())
    for T in (1, 7):
        x = _x(T, 30 + T)
        ones, zeros = torch.ones((T, 1), dtype=torch.bfloat16, device="cuda"), torch.zeros((T, 1), dtype=torch.int32, device="cuda")
        shared = fused_moe.fused_experts(x, ones, zeros, d13, d2, None).clone()
        w, ids, _ = fused_moe.route(x, gate, layer.router_spec)
        want = fused_moe.fused_experts(x, w, ids, b13[:E].contiguous(), b2[:E].contiguous(), ident[:E], add=shared)
        out = layer.forward(x).clone()
        torch.cuda.synchronize()
        assert torch.equal(out, want), T


def test_layer_from_a_checkpoint_in_4_bits(tmp_path):
    from safetensors.torch import save_file

    fused_moe, mxfp4, native, SlotMoELayer, Cfg, Runtime = _mods()
    w13, w2, gate = _weights(6)
    save_file({f"model.layers.6.mlp.experts.{e}.{n}.weight": t.contiguous()
               for e in range(E)
               for n, t in (("gate_proj", w13[e, :I]), ("up_proj", w13[e, I:]), ("down_proj", w2[e]))},
              str(tmp_path / "experts.safetensors"))
    rt = Runtime(Cfg(enabled=True, num_slots=16, async_load=True, pin_host_memory=True, cpu_first_load=True,
                     release_original_expert_weights=True))
    layer = SlotMoELayer.from_checkpoint(tmp_path / "experts.safetensors", prefix="model.layers.6.mlp", layer_id=6,
                                         runtime=rt, num_experts=E, hidden_size=H, intermediate_size=I, gate_weight=gate,
                                         top_k=4, weight_format="mxfp4")
    block = layer.w13_weight.data_ptr()
    layer.register()
    buf = rt.host_store.get_layer_buffer(6)
    b13, b2 = mxfp4.pack_experts(w13, w2)
    assert buf.pinned and buf.w13.data_ptr() == block and torch.equal(buf.w13, b13) and torch.equal(buf.w2, b2)
    x = _x(3, 1)
    out = layer.forward(x).clone()
    w, ids, _ = fused_moe.route(x, gate, layer.router_spec)
    want = fused_moe.fused_experts(x, w, ids, b13.cuda(), b2.cuda(), torch.arange(E, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_layer_refuses_what_it_cannot_hold():
    _, mxfp4, _, SlotMoELayer, Cfg, Runtime = _mods()
    w13, w2, gate = _weights(7, 4)
    rt = Runtime(Cfg(enabled=True, num_slots=4))
    b13, b2 = mxfp4.pack_experts(w13, w2)
    mk = lambda a, b, **kw: SlotMoELayer(layer_id=1, runtime=rt, gate_weight=gate, w13_weight=a, w2_weight=b, top_k=2, **kw)  # noqa: E731
    mk(b13, b2, weight_format="mxfp4")
    for a, b, kw in ((b13, b2, {}), (w13, w2, dict(weight_format="int4")), (b13, w2, dict(weight_format="mxfp4")),
                     (b13[:, :64], b2, dict(weight_format="mxfp4")), (w13[:, :48], w2, dict(weight_format="mxfp4"))):
        with pytest.raises(ValueError):
            mk(a, b, **kw)
