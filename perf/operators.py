"""The operators around 4-bit experts: what is measured, their plain forms, and
their values in 64 bits.

norm     the residual's addition and the root-mean-square norm in front of a
         MoE layer: native.add_rms_norm.  r = x + residual, y = r / rms(r) * w;
         y in bf16 for the router gate, in 8 bits for the experts, or both.
decode   the experts of a few tokens over a 4-bit slot bank, permutation and
         weighted combine included: fused_moe.fused_experts.
experts  the experts' products of a prefill chunk over a 4-bit slot bank, one
         row for each (token, expert) pair: native.permute, native.grouped_mlp.

Formats (OCP microscaling): groups of 32 values along the row share a scale
2^e.  Weights are e2m1 (4 bits), two per byte, the even column in the low half.
8-bit rows are e4m3.  e is the smallest integer that keeps the group's largest
value within the format (6 and 448), so nothing saturates.

"rows" of a case: the experts' input is bf16 ("bf16") or 8 bits with scales
("mx8"); with "mx8" the SwiGLU output is rounded to the same 8-bit format
before the down projection: that format is part of the operator.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "vllm-ascend-hust-latchmoe_amd")
GROUP = 32
EPS = 1e-6


def listed():
    return [
        # one user's token in front of the gate: latency
        dict(name="norm-1", kind="norm", tokens=1, hidden=2048, residual="bf16", out=True, mx8=False),
        # a long prefill: bf16 for the gate and 8 bits for the experts
        dict(name="norm-4096", kind="norm", tokens=4096, hidden=2048, residual="bf16", out=True, mx8=True),
        # an odd chunk of long rows, the residual stream held in 32 bits
        dict(name="norm-1237-long", kind="norm", tokens=1237, hidden=7168, residual="f32", out=True, mx8=True),
        # one user's token: the smallest step
        dict(name="decode-1", kind="decode", rows="bf16", tokens=1, hidden=2048, width=768, experts=128, top_k=8, skew=1.0),
        # an ordinary serving batch
        dict(name="decode-16", kind="decode", rows="bf16", tokens=16, hidden=2048, width=768, experts=128, top_k=8, skew=1.0),
        # the large experts, a few users, 8-bit rows
        dict(name="decode-7-mx8", kind="decode", rows="mx8", tokens=7, hidden=7168, width=2048, experts=64, top_k=8, skew=0.0),
        # an odd batch over experts whose width is no multiple of 256 columns
        dict(name="decode-61-wide", kind="decode", rows="bf16", tokens=61, hidden=2048, width=1408, experts=60, top_k=4, skew=0.5),
        # a chunk of a chunked prefill, some experts hot, in both kinds of rows
        dict(name="chunk-300", kind="experts", rows="bf16", tokens=300, hidden=2048, width=768, experts=128, top_k=8, skew=0.5),
        dict(name="chunk-301-mx8", kind="experts", rows="mx8", tokens=301, hidden=2048, width=768, experts=128, top_k=8, skew=0.5),
        # a long prefill, in both kinds of rows
        dict(name="prefill-4096", kind="experts", rows="bf16", tokens=4096, hidden=2048, width=768, experts=128, top_k=8, skew=0.0),
        dict(name="prefill-4096-mx8", kind="experts", rows="mx8", tokens=4096, hidden=2048, width=768, experts=128, top_k=8, skew=0.0),
        # an odd prefill of the large experts
        dict(name="prefill-2049-large-mx8", kind="experts", rows="mx8", tokens=2049, hidden=7168, width=2048, experts=32, top_k=4, skew=0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


#: (hidden, width, experts, top_k) of the benchmark's layers
_LAYERS = ((2048, 768, 128, 8), (2048, 1408, 60, 4), (7168, 2048, 32, 8))


def draw(rng):
    kind = rng.choices(["norm", "decode", "experts"], [3, 4, 4])[0]
    if kind == "norm":
        out = rng.random() < 0.7
        return dict(kind=kind, tokens=_log_int(rng, 1, 4096), hidden=GROUP * _log_int(rng, 8, 256),
                    residual=rng.choice(["bf16", "f32", "none"]), out=out, mx8=not out or rng.random() < 0.6)
    if rng.random() < 0.5:
        hidden, width, experts, top_k = rng.choice(_LAYERS)
    else:
        hidden, width = GROUP * _log_int(rng, 8, 128), GROUP * _log_int(rng, 4, 48)
        experts = _log_int(rng, 4, 96)
        top_k = rng.randint(1, min(8, experts))
    most = 4096 * 8 * 2048 * 768 // (top_k * hidden * width)  # the largest listed case's products
    tokens = _log_int(rng, 1, 64) if kind == "decode" else _log_int(rng, 65, max(66, min(4096, most)))
    return dict(kind=kind, rows=rng.choice(["bf16", "mx8"]), tokens=tokens, hidden=hidden, width=width,
                experts=experts, top_k=top_k, skew=round(rng.uniform(0.0, 1.0), 3))


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------
def _gen(seed, part):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + part)


def _rank_bias(case, seed):
    """Zipf(1.1) over a random rank of the experts, mapped onto [-2, 2] and
    scaled by the case's skew."""
    E = case["experts"]
    ranks = np.random.RandomState(int(seed) % (1 << 31)).permutation(E) + 1
    return case["skew"] * (2.0 - 4.0 * np.log(ranks) / math.log(max(E, 2)))


def _exponent(amax, top):
    """The smallest e with amax <= top * 2^e (a whole tensor), -127 at least."""
    m, ex = torch.frexp(amax)
    tm, tex = math.frexp(top)
    e = ex - tex + (m > tm)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp_(min=-127)


def _codes4(w):
    """e2m1 codes (two per byte) and e8m0 scales of rows w, round to nearest even."""
    g = w.float().unflatten(-1, (-1, GROUP))
    e = _exponent(g.abs().amax(-1), 6.0)
    v = torch.ldexp(g, -e.unsqueeze(-1))
    a = v.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (v < 0)).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _rows8(y):
    """(e4m3 values, e) of rows y: y ~ value * 2^e."""
    g = y.unflatten(-1, (-1, GROUP))
    e = _exponent(g.abs().amax(-1), 448.0)
    q = torch.ldexp(g, -e.unsqueeze(-1)).float().to(torch.float8_e4m3fn)
    return q.flatten(-2), e


def _weights(g, experts, n, k):
    """Random experts of N(0, 0.02) rows in 4 bits, some experts at a time."""
    codes = torch.empty((experts, n, k // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((experts, n, k // GROUP), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (n * k))
    for e in range(0, experts, step):
        m = min(step, experts - e)
        w = torch.empty((m, n, k), dtype=torch.float32, device="cuda").normal_(0.0, 0.02, generator=g)
        codes[e:e + m], scales[e:e + m] = _codes4(w)
    return codes, scales


def prepare(case, seed):
    g = _gen(seed, 0)
    T, H = case["tokens"], case["hidden"]
    x = torch.empty((T, H), dtype=torch.bfloat16, device="cuda").normal_(0.0, 1.0, generator=g)
    s = dict(case=dict(case), x=x)
    if case["kind"] == "norm":
        if case["residual"] != "none":
            dt = torch.float32 if case["residual"] == "f32" else torch.bfloat16
            # the residual stream of a deep model: larger than one layer's output, a few channels far larger
            scale = torch.ones(H, device="cuda")
            scale[:: max(1, H // 4)] = 20.0
            s["residual"] = (torch.empty((T, H), device="cuda").normal_(0.0, 3.0, generator=g) * scale).to(dt)
            s["residual_out"] = torch.empty_like(s["residual"])
        s["weight"] = torch.empty(H, device="cuda").uniform_(0.5, 1.5, generator=g).to(torch.bfloat16)
        s["out"] = torch.empty_like(x) if case["out"] else None
        if case["mx8"]:
            s["q"] = torch.empty((T, H), dtype=torch.float8_e4m3fn, device="cuda")
            s["scale"] = torch.empty((T, H // GROUP), dtype=torch.uint8, device="cuda")
        return s
    E, I, k = case["experts"], case["width"], case["top_k"]
    bias = torch.from_numpy(_rank_bias(case, seed)).cuda()
    logits = torch.empty((T, E), dtype=torch.float64, device="cuda").normal_(0.0, 1.0, generator=g) + bias
    top, ids = torch.topk(logits, k, dim=1)
    s["ids"] = ids.to(torch.int32)
    s["weights"] = torch.softmax(top, dim=1).to(torch.bfloat16)
    s["capacity"] = int(torch.bincount(ids.flatten(), minlength=E).max())
    s["c13"], s["s13"] = _weights(g, E, 2 * I, H)
    s["c2"], s["s2"] = _weights(g, E, H, I)
    if case["rows"] == "mx8":
        s["q"], e = _rows8(x.float())
        s["scale"] = (e + 127).to(torch.uint8)
    if own:
        fw = _framework()
        s["w13"] = fw.mxfp4.pack_w13(s["c13"], s["s13"])
        s["w2"] = fw.mxfp4.pack_w2(s["c2"], s["s2"])
        s["perm"] = fw.native.Permutation.allocate(T * k, E, "cuda")
        if case["rows"] == "mx8":
            s["act"] = fw.native.Mx8Rows.allocate(T * k, I, "cuda")
        else:
            s["act"] = torch.empty((T * k, I), dtype=torch.bfloat16, device="cuda")
        s["y"] = torch.empty((T * k, H), dtype=torch.bfloat16, device="cuda")
    return s


# ---------------------------------------------------------------------------
# the calls a program makes
# ---------------------------------------------------------------------------
def _framework():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import vllm_moe_offload_amd.fused_moe
    import vllm_moe_offload_amd.mxfp4
    import vllm_moe_offload_amd.native

    return vllm_moe_offload_amd


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    return _plain_norm(state) if kind == "norm" else _plain_experts(state)


def _run_own(s):
    fw, case = _framework(), s["case"]
    if case["kind"] == "norm":
        mx8 = fw.native.Mx8Rows(s["q"], s["scale"]) if case["mx8"] else None
        fw.native.add_rms_norm(s["x"], s["weight"], residual=s.get("residual"), residual_out=s.get("residual_out"),
                               out=s["out"], mx8=mx8, eps=EPS)
        return dict(residual=s.get("residual_out"), out=s["out"], q=s.get("q"),
                    scale=s["scale"].view(torch.float8_e8m0fnu) if case["mx8"] else None)
    x = s["x"] if case["rows"] == "bf16" else fw.native.Mx8Rows(s["q"], s["scale"])
    if case["kind"] == "decode":
        return fw.fused_moe.fused_experts(x, s["weights"], s["ids"], s["w13"], s["w2"], None)
    block_m = fw.native.mx4_block_m(case["tokens"] * case["top_k"], case["experts"])
    fw.native.permute(s["ids"], s["perm"], block_m=block_m)
    return fw.native.grouped_mlp(x, case["top_k"], s["w13"], s["w2"], s["perm"], s["act"], s["y"])


# ---------------------------------------------------------------------------
# the plain forms: 32 bits, rounded once at the end
# ---------------------------------------------------------------------------
def _plain_norm(s):
    case = s["case"]
    r = s["x"].float()
    if "residual" in s:
        r = r + s["residual"].float()
    y = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    q = scale = None
    if case["mx8"]:
        q, e = _rows8(y)
        scale = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    return dict(residual=r.to(s["residual"].dtype) if "residual" in s else None,
                out=y.to(torch.bfloat16) if case["out"] else None, q=q, scale=scale)


def _values4(codes, scales):
    """The f32 weights that codes and scales stand for."""
    lut = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    lut = torch.cat([lut, -lut])
    v = torch.stack([lut[(codes & 15).int()], lut[(codes >> 4).int()]], dim=-1)
    v = v.flatten(-2).unflatten(-1, (-1, GROUP))
    return (v * torch.exp2(scales.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _plain_experts(s):
    case = s["case"]
    E, I, k, T, H = case["experts"], case["width"], case["top_k"], case["tokens"], case["hidden"]
    mx8 = case["rows"] == "mx8"
    x = s["x"].float()
    if mx8:
        x = (s["q"].float().unflatten(-1, (-1, GROUP)) * torch.exp2(s["scale"].float() - 127.0).unsqueeze(-1)).flatten(-2)
    ids = s["ids"].flatten().long()
    pair = torch.arange(T * k, device="cuda")
    if T * k <= E:  # few pairs: each pair's own expert
        rows, dest = x[pair // k].unsqueeze(1), pair
        c13, s13, c2, s2 = s["c13"][ids], s["s13"][ids], s["c2"][ids], s["s2"][ids]
    else:  # each expert's pairs, padded to the largest count
        C = s["capacity"]
        order = torch.argsort(ids, stable=True)
        first = torch.searchsorted(ids[order], torch.arange(E, device="cuda"))
        dest = torch.empty_like(ids)
        dest[order] = ids[order] * C + pair - first[ids[order]]
        rows = torch.zeros((E * C, H), device="cuda")
        rows[dest] = x[pair // k]
        rows = rows.view(E, C, H)
        c13, s13, c2, s2 = s["c13"], s["s13"], s["c2"], s["s2"]
    h = torch.bmm(rows, _values4(c13, s13).transpose(1, 2))
    gate, up = h[..., :I], h[..., I:]
    act = gate / (1.0 + torch.exp(-gate)) * up
    if mx8:
        q, e = _rows8(act)
        act = torch.ldexp(q.float().unflatten(-1, (-1, GROUP)), e.unsqueeze(-1)).flatten(-2)
    y = torch.bmm(act, _values4(c2, s2).transpose(1, 2)).reshape(-1, H)[dest]
    if case["kind"] == "decode":
        y = (y.view(T, k, H) * s["weights"].float().unsqueeze(-1)).sum(1)
    return y.to(torch.bfloat16)


# ---------------------------------------------------------------------------
# the operators in 64 bits
# ---------------------------------------------------------------------------
def _scale_of(v, top):
    """2^e, e the smallest with every |v| of a group (last axis) <= top * 2^e."""
    big = v.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(big / top)).clamp(min=-127)
    # log2 next to a whole number: settle by comparison
    e = torch.where(big <= top * torch.exp2(e - 1), e - 1, e)
    e = torch.where(big > top * torch.exp2(e), e + 1, e)
    return torch.exp2(torch.where(big > 0, e, torch.full_like(e, -127)).clamp(min=-127))


def _round_e4m3(v):
    """The nearest e4m3 value (ties to even) of |v| <= 448, in 64 bits: steps of
    an eighth of the binade, 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        r = s["x"].double() + (s["residual"].double() if "residual" in s else 0.0)
        y = r / torch.sqrt((r * r).sum(-1, keepdim=True) / r.shape[-1] + EPS) * s["weight"].double()
        q = None
        if case["mx8"]:  # the values on their group's scale, before their rounding to 8 bits
            g = y.view(y.shape[0], -1, GROUP)
            q = (g / _scale_of(g, 448.0)).view_as(y)
        # a scale is a choice between two powers of two, no computed number
        return dict(residual=r if "residual" in s else None, out=y if case["out"] else None, q=q, scale=None)
    E, I, k, T, H = case["experts"], case["width"], case["top_k"], case["tokens"], case["hidden"]
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
    grid = torch.tensor(grid, dtype=torch.float64, device="cuda")

    def values(codes, scales):
        v = torch.empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.float64, device="cuda")
        v[:, 0::2] = grid[(codes % 16).long()]
        v[:, 1::2] = grid[(codes // 16).long()]
        return v * (2.0 ** (scales.double() - 127.0)).repeat_interleave(GROUP, dim=1)

    x = s["x"].double()
    if case["rows"] == "mx8":
        x = s["q"].double() * (2.0 ** (s["scale"].double() - 127.0)).repeat_interleave(GROUP, dim=1)
    y = torch.zeros((T * k, H), dtype=torch.float64, device="cuda")
    flat = s["ids"].flatten()
    for e in range(E):
        at = (flat == e).nonzero().flatten()
        if not at.numel():
            continue
        w = values(s["c13"][e], s["s13"][e])
        rows = x[at // k]
        gate = rows @ w[:I].t()
        act = gate * torch.sigmoid(gate) * (rows @ w[I:].t())
        if case["rows"] == "mx8":
            g = act.view(act.shape[0], -1, GROUP)
            sc = _scale_of(g, 448.0)
            act = (_round_e4m3(g / sc) * sc).view_as(act)
        y[at] = act @ values(s["c2"][e], s["s2"][e]).t()
    if case["kind"] == "decode":
        return torch.einsum("tkh,tk->th", y.view(T, k, H), s["weights"].double())
    return y


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def _active(case):
    """Experts with a pair, of routing drawn like prepare's."""
    r = np.random.RandomState(1)
    z = r.standard_normal((case["tokens"], case["experts"])) + _rank_bias(case, 1)
    return int(np.unique(np.argpartition(-z, case["top_k"] - 1, axis=1)[:, :case["top_k"]]).size)


def work(case):
    T, H = case["tokens"], case["hidden"]
    if case["kind"] == "norm":
        res = {"none": 0, "bf16": 4, "f32": 8}[case["residual"]]  # read and written
        per = 2 + res + (2 if case["out"] else 0) + (1 + 1 / GROUP if case["mx8"] else 0)
        return dict(bytes=T * H * per + 2 * H, flops=T * H * 6)
    I, k = case["width"], case["top_k"]
    row = H * 2 if case["rows"] == "bf16" else H * (1 + 1 / GROUP)
    result = T * H * 2 if case["kind"] == "decode" else T * k * H * 2
    weights = _active(case) * 3 * I * H * (0.5 + 1 / GROUP)
    return dict(bytes=weights + T * row + T * k * 6 + result, flops=2 * T * k * 3 * I * H)
