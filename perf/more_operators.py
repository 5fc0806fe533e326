"""4-bit rows: what is measured of them, their plain forms, and their values in 64 bits.

rows     rows of activations to 4 bits and back: native.rows_to_mx4, native.mx4_values.
bank     weights to the 4-bit form that the slot bank holds, and back:
         native.quantize_mx4, native.mx4_values.
linear   y = x W^T (+ bias) (+ add) over one matrix of 4-bit weights, x in bf16, in
         8 bits or in 4 bits: native.mx4_linear.
experts  a MoE layer whose rows and weights are both in 4 bits, its SwiGLU output
         rounded to 4 bits between the two products: fused_moe.fused_experts.

Formats (OCP microscaling): groups of 32 values along the row share a scale 2^e.
4-bit values are e2m1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), two per byte,
the even column in the low half; 8-bit values are e4m3.  e is the smallest integer,
-127 at least, that keeps the group's largest magnitude within the format (6 and 448),
so nothing saturates.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "vllm-ascend-hust-latchmoe_amd")
GROUP = 32
HALF_BLOCK = 16  # weight rows come in blocks of 16


def listed():
    return [
        # one user's token on its way to 4 bits: latency
        dict(name="rows-1", kind="rows", dtype="bf16", tokens=1, hidden=2048),
        # a long prefill's rows
        dict(name="rows-4096", kind="rows", dtype="bf16", tokens=4096, hidden=7168),
        # gate and up weights of a layer of many experts, as a checkpoint has them
        dict(name="bank-128-gate-up", kind="bank", dtype="bf16", gate_up=True, experts=128, rows=1536, hidden=2048),
        # down weights of a few experts, an odd width, from f32 master weights
        dict(name="bank-5-f32", kind="bank", dtype="f32", gate_up=False, experts=5, rows=2048, hidden=1408),
        # one user's token through the attention's joint projection
        dict(name="linear-1", kind="linear", rows="mx4", tokens=1, hidden=2048, out=5120, f32=False, bias=True, add=False),
        # a serving batch through the head, logits in f32
        dict(name="linear-16-head", kind="linear", rows="bf16", tokens=16, hidden=2048, out=50000, f32=True, bias=False, add=False),
        # an odd chunk of 8-bit rows through an odd width, the residual stream added
        dict(name="linear-301-mx8", kind="linear", rows="mx8", tokens=301, hidden=1408, out=2048, f32=False, bias=False, add=True),
        # a long prefill of a wide model, rows in 4 bits
        dict(name="linear-4096", kind="linear", rows="mx4", tokens=4096, hidden=7168, out=7168, f32=False, bias=False, add=False),
        # one user's token through the experts: the smallest step
        dict(name="experts-1", kind="experts", tokens=1, hidden=2048, width=768, experts=128, top_k=8, skew=1.0),
        # an ordinary serving batch
        dict(name="experts-16", kind="experts", tokens=16, hidden=2048, width=768, experts=128, top_k=8, skew=1.0),
        # an odd chunk of a chunked prefill, some experts hot, a width that is no multiple of 256
        dict(name="experts-333", kind="experts", tokens=333, hidden=2048, width=1408, experts=60, top_k=4, skew=0.5),
        # a long prefill
        dict(name="experts-4096", kind="experts", tokens=4096, hidden=2048, width=768, experts=128, top_k=8, skew=0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


#: (hidden, width, experts, top_k) of the benchmark's layers
_LAYERS = ((2048, 768, 128, 8), (2048, 1408, 60, 4), (7168, 2048, 32, 8))


def draw(rng):
    kind = rng.choices(["rows", "bank", "linear", "experts"], [2, 2, 4, 4])[0]
    if kind == "rows":
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), tokens=_log_int(rng, 1, 4096), hidden=GROUP * _log_int(rng, 1, 224))
    if kind == "bank":
        hidden, gate_up = GROUP * _log_int(rng, 2, 224), rng.random() < 0.5
        rows = 2 * GROUP * _log_int(rng, 1, 64) if gate_up else HALF_BLOCK * _log_int(rng, 1, 256)
        most = 128 * 1536 * 2048 // (rows * hidden)  # the largest listed case's values
        return dict(kind=kind, dtype=rng.choice(["bf16", "f32"]), gate_up=gate_up,
                    experts=_log_int(rng, 1, max(1, min(128, most))), rows=rows, hidden=hidden)
    if kind == "linear":
        hidden, out = GROUP * _log_int(rng, 2, 224), HALF_BLOCK * _log_int(rng, 4, 2048)
        most = 4096 * 7168 * 7168 // (out * hidden)  # the largest listed case's products
        rows = rng.choice(["bf16", "mx8", "mx4", "mx4"])
        # 8-bit rows: products are summed in fixed point, 32-bit results are for the others
        return dict(kind=kind, rows=rows, tokens=_log_int(rng, 1, max(1, min(4096, most))), hidden=hidden, out=out,
                    f32=rows != "mx8" and rng.random() < 0.3, bias=rng.random() < 0.4, add=rng.random() < 0.4)
    if rng.random() < 0.5:
        hidden, width, experts, top_k = rng.choice(_LAYERS)
    else:
        hidden, width = GROUP * _log_int(rng, 8, 128), GROUP * _log_int(rng, 8, 48)
        experts = _log_int(rng, 4, 96)
        top_k = rng.randint(1, min(8, experts))
    most = 4096 * 8 * 2048 * 768 // (top_k * hidden * width)
    return dict(kind=kind, tokens=_log_int(rng, 1, max(1, min(4096, most))), hidden=hidden, width=width,
                experts=experts, top_k=top_k, skew=round(rng.uniform(0.0, 1.0), 3))


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1013 + 7)


def _rank_bias(case, seed):
    """Zipf over a random rank of the experts, mapped onto [-2, 2] and scaled by the
    case's skew."""
    E = case["experts"]
    ranks = np.random.RandomState(int(seed) % (1 << 31)).permutation(E) + 1
    return case["skew"] * (2.0 - 4.0 * np.log(ranks) / math.log(max(E, 2)))


def _exponent(amax, top):
    """The smallest e >= -127 with amax <= top * 2^e (a whole tensor)."""
    m, ex = torch.frexp(amax)
    tm, tex = math.frexp(top)
    e = ex - tex + (m > tm)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp_(min=-127)


def _nearest4(w):
    """(indices into the e2m1 values, sign in bit 3; e) of rows w in f32, ties to even."""
    g = w.unflatten(-1, (-1, GROUP))
    e = _exponent(g.abs().amax(-1), 6.0)
    v = torch.ldexp(g, -e.unsqueeze(-1))
    a = v.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return (code + 8 * (v < 0)).flatten(-2).to(torch.uint8), e


def _codes4(w):
    """e2m1 codes (two per byte) and e8m0 scales of rows w."""
    code, e = _nearest4(w.float())
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _rows8(y):
    """(e4m3 values, scale bytes) of rows y in f32."""
    g = y.unflatten(-1, (-1, GROUP))
    e = _exponent(g.abs().amax(-1), 448.0)
    return torch.ldexp(g, -e.unsqueeze(-1)).to(torch.float8_e4m3fn).flatten(-2), (e + 127).to(torch.uint8)


def _weights(g, n, k, experts=1):
    """Random matrices of N(0, 0.02) in 4 bits, some at a time."""
    codes = torch.empty((experts, n, k // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((experts, n, k // GROUP), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (n * k))
    for e in range(0, experts, step):
        m = min(step, experts - e)
        codes[e:e + m], scales[e:e + m] = _codes4(torch.empty((m, n, k), device="cuda").normal_(0.0, 0.02, generator=g))
    return codes, scales


def _activations(g, tokens, hidden):
    """Rows as a norm leaves them: a few channels far larger than the others."""
    channel = torch.ones(hidden, device="cuda")
    channel[:: max(1, hidden // 4)] = 8.0
    return torch.empty((tokens, hidden), device="cuda").normal_(0.0, 1.0, generator=g) * channel


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=dict(case))
    dtype = torch.float32 if case.get("dtype") == "f32" else torch.bfloat16
    kind, H = case["kind"], case["hidden"]
    if kind == "rows":
        s["x"] = _activations(g, case["tokens"], H).to(dtype)
        s["values"] = torch.empty((case["tokens"], H), dtype=torch.bfloat16, device="cuda")
        if own:
            s["mx4"] = _framework().native.Mx4Rows.allocate(case["tokens"], H, "cuda")
        return s
    if kind == "bank":
        shape = (case["experts"], case["rows"], H)
        s["w"] = torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 0.02, generator=g)
        s["values"] = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        if own:
            s["bank"] = torch.empty((*shape[:2], _framework().mxfp4.row_bytes(H)), dtype=torch.uint8, device="cuda")
        return s
    T = case["tokens"]
    x = _activations(g, T, H)
    rows = case["rows"] if kind == "linear" else "mx4"
    if rows == "bf16":
        s["x"] = x.to(torch.bfloat16)
    else:
        s["q"], s["scale"] = _rows8(x) if rows == "mx8" else _codes4(x)
    if kind == "linear":
        N = case["out"]
        c, sc = _weights(g, N, H)
        s["codes"], s["scales"] = c[0], sc[0]
        s["bias"] = torch.empty(N, device="cuda").normal_(0.0, 0.5, generator=g) if case["bias"] else None
        s["add"] = None
        if case["add"]:
            s["add"] = torch.empty((T, N), device="cuda").normal_(0.0, 1.0, generator=g).to(torch.bfloat16)
        s["y"] = torch.empty((T, N), dtype=torch.float32 if case["f32"] else torch.bfloat16, device="cuda")
        if own:
            s["w"] = _framework().mxfp4.pack_w2(s["codes"], s["scales"])
        return s
    E, I, k = case["experts"], case["width"], case["top_k"]
    logits = torch.empty((T, E), dtype=torch.float64, device="cuda").normal_(0.0, 1.0, generator=g)
    top, ids = torch.topk(logits + torch.from_numpy(_rank_bias(case, seed)).cuda(), k, dim=1)
    s["ids"] = ids.to(torch.int32)
    s["weights"] = torch.softmax(top, dim=1).to(torch.bfloat16)
    s["capacity"] = int(torch.bincount(ids.flatten(), minlength=E).max())
    s["c13"], s["s13"] = _weights(g, 2 * I, H, E)
    s["c2"], s["s2"] = _weights(g, H, I, E)
    if own:
        fw = _framework()
        s["w13"] = fw.mxfp4.pack_w13(s["c13"], s["s13"])
        s["w2"] = fw.mxfp4.pack_w2(s["c2"], s["s2"])
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
    return dict(rows=_plain_rows, bank=_plain_bank, linear=_plain_linear, experts=_plain_experts)[state["case"]["kind"]](state)


def _run_own(s):
    fw, case = _framework(), s["case"]
    if case["kind"] == "rows":
        return fw.native.mx4_values(fw.native.rows_to_mx4(s["x"], s["mx4"]), s["values"])
    if case["kind"] == "bank":
        fw.native.quantize_mx4(s["w"], s["bank"], gate_up=case["gate_up"])
        return fw.native.mx4_values(s["bank"], s["values"], gate_up=case["gate_up"])
    if case["kind"] == "linear":
        kinds = dict(mx8=fw.native.Mx8Rows, mx4=fw.native.Mx4Rows)
        x = s["x"] if case["rows"] == "bf16" else kinds[case["rows"]](s["q"], s["scale"])
        return fw.native.mx4_linear(x, s["w"], s["y"], bias=s["bias"], add=s["add"])
    x = fw.native.Mx4Rows(s["q"], s["scale"])
    return fw.fused_moe.fused_experts(x, s["weights"], s["ids"], s["w13"], s["w2"], None)


# ---------------------------------------------------------------------------
# the plain forms: 32 bits, rounded once at the end
# ---------------------------------------------------------------------------
def _e2m1(device):
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=device)
    return torch.cat([v, -v])


def _round4(w):
    """w in f32 rounded to 4 bits, as the values that they stand for."""
    code, e = _nearest4(w)
    v = _e2m1(w.device)[code.int()].unflatten(-1, (-1, GROUP))
    return torch.ldexp(v, e.unsqueeze(-1)).flatten(-2)


def _values4(codes, scales):
    """The f32 values that codes and scales stand for."""
    lut = _e2m1(codes.device)
    v = torch.stack([lut[(codes & 15).int()], lut[(codes >> 4).int()]], dim=-1)
    v = v.flatten(-2).unflatten(-1, (-1, GROUP))
    return (v * torch.exp2(scales.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _values8(q, scale):
    return (q.float().unflatten(-1, (-1, GROUP)) * torch.exp2(scale.float() - 127.0).unsqueeze(-1)).flatten(-2)


def _plain_rows(s):
    return _round4(s["x"].float()).to(torch.bfloat16)


def _plain_bank(s):
    return _round4(s["w"].float()).to(torch.bfloat16)


def _plain_linear(s):
    rows = s["case"]["rows"]
    x = s["x"].float() if rows == "bf16" else (_values8 if rows == "mx8" else _values4)(s["q"], s["scale"])
    y = x @ _values4(s["codes"], s["scales"]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["add"] is not None:
        y = y + s["add"].float()
    return y.to(s["y"].dtype)


def _plain_experts(s):
    case = s["case"]
    E, I, k, T, H = case["experts"], case["width"], case["top_k"], case["tokens"], case["hidden"]
    x = _values4(s["q"], s["scale"])
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
    act = _round4(gate / (1.0 + torch.exp(-gate)) * up)
    y = torch.bmm(act, _values4(c2, s2).transpose(1, 2)).reshape(-1, H)[dest]
    return (y.view(T, k, H) * s["weights"].float().unsqueeze(-1)).sum(1).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# the operators in 64 bits
# ---------------------------------------------------------------------------
def _scale_of(v, top):
    """2^e, e the smallest >= -127 with every |v| of a group (last axis) <= top * 2^e."""
    big = v.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(big / top)).clamp(min=-127)
    # log2 next to a whole number: settle by comparison
    e = torch.where(big <= top * torch.exp2(e - 1), e - 1, e)
    e = torch.where(big > top * torch.exp2(e), e + 1, e)
    return torch.exp2(torch.where(big > 0, e, torch.full_like(e, -127)).clamp(min=-127))


def _round_mx4(w):
    """w in 64 bits to the nearest values of its groups: steps of half the binade's
    power of two, 0.5 below 1; ties to even."""
    g = w.unflatten(-1, (-1, GROUP))
    scale = _scale_of(g, 6.0)
    v = g / scale
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=1.0))) - 1)
    return (torch.round(v / step) * step * scale).flatten(-2)


def _grid_values(codes, scales):
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
    grid = torch.tensor(grid, dtype=torch.float64, device="cuda")
    v = torch.empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.float64, device="cuda")
    v[:, 0::2] = grid[(codes % 16).long()]
    v[:, 1::2] = grid[(codes // 16).long()]
    return v * (2.0 ** (scales.double() - 127.0)).repeat_interleave(GROUP, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rows":
        return _round_mx4(s["x"].double())
    if case["kind"] == "bank":
        return torch.stack([_round_mx4(w.double()) for w in s["w"]])
    rows = case["rows"] if case["kind"] == "linear" else "mx4"
    if rows == "bf16":
        x = s["x"].double()
    elif rows == "mx8":
        x = s["q"].double() * (2.0 ** (s["scale"].double() - 127.0)).repeat_interleave(GROUP, dim=1)
    else:
        x = _grid_values(s["q"], s["scale"])
    if case["kind"] == "linear":
        y = x @ _grid_values(s["codes"], s["scales"]).t()
        if s["bias"] is not None:
            y += s["bias"].double()
        if s["add"] is not None:
            y += s["add"].double()
        return y
    E, I, k, T, H = case["experts"], case["width"], case["top_k"], case["tokens"], case["hidden"]
    y = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    for e in range(E):
        token, choice = (s["ids"] == e).nonzero(as_tuple=True)
        if not token.numel():
            continue
        w = _grid_values(s["c13"][e], s["s13"][e])
        gate = x[token] @ w[:I].t()
        act = _round_mx4(gate * torch.sigmoid(gate) * (x[token] @ w[I:].t()))
        part = act @ _grid_values(s["c2"][e], s["s2"][e]).t()
        y[token] += part * s["weights"][token, choice].double().unsqueeze(1)  # a token names an expert once
    return y


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
_MX4 = 0.5 + 1 / GROUP  # bytes of a 4-bit value and its share of the scale


def _active(case):
    """Experts with a pair, of routing drawn like prepare's."""
    r = np.random.RandomState(1)
    z = r.standard_normal((case["tokens"], case["experts"])) + _rank_bias(case, 1)
    return int(np.unique(np.argpartition(-z, case["top_k"] - 1, axis=1)[:, :case["top_k"]]).size)


def work(case):
    kind, H = case["kind"], case["hidden"]
    if kind in ("rows", "bank"):
        n = case["tokens"] * H if kind == "rows" else case["experts"] * case["rows"] * H
        # read, written in 4 bits, written as values
        return dict(bytes=n * ((4 if case["dtype"] == "f32" else 2) + _MX4 + 2), flops=n * 4)
    T = case["tokens"]
    if kind == "linear":
        N = case["out"]
        row = {"bf16": 2.0, "mx8": 1 + 1 / GROUP, "mx4": _MX4}[case["rows"]]
        y = (4 if case["f32"] else 2) + (2 if case["add"] else 0)
        return dict(bytes=N * H * _MX4 + T * H * row + T * N * y + (4 * N if case["bias"] else 0), flops=2 * T * N * H)
    I, k = case["width"], case["top_k"]
    return dict(bytes=_active(case) * 3 * I * H * _MX4 + T * H * (_MX4 + 2) + T * k * 6, flops=2 * T * k * 3 * I * H)
