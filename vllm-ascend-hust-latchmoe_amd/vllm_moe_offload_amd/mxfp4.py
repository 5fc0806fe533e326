"""Expert weights in 4 bits (OCP MXFP4) as the slot bank holds them.

A checkpoint's form of an [N, K] matrix is codes, uint8 [N, K / 2] (two e2m1
values per byte, the even column in the low half), and scales, uint8 [N, K / 32]
(2^(byte - 127) for 32 columns).  quantize() makes it from bf16 or f32 weights.

The bank's form is one uint8 tensor with the same leading dimensions,
[..., N, row_bytes(K)]: codes and scales of 16 rows x 128 columns in the order
that the matrix instructions read them, so that a wave's weights are one
contiguous run (include/latchmoe.h, lmoe_mx4_gateup_silu).  The rows of w13 are
the checkpoint's [gate; up] halves interleaved in blocks of 16, so that a wave
holds a gate and its up column together.  An expert is one contiguous run of
bytes either way: host store, slot bank and staging move it like any other
weight.

Everything here runs on the tensors' own device, once per weight; pack_experts takes
weights on the GPU through its kernel (native.quantize_mx4), which gives the same bytes.
"""

from __future__ import annotations

import torch

GROUP = 32    # values that share a scale
CHUNK = 128   # columns of one matrix-instruction fragment
QUAD = 512    # columns whose scales are stored together
ROWS = 16     # rows of one block

_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def row_bytes(K: int) -> int:
    """Bytes of one weight row of K columns in the bank's form."""
    if K <= 0 or K % GROUP:
        raise ValueError(f"rows of 4-bit weights are multiples of {GROUP} columns, got {K}")
    return -(-K // CHUNK) * (CHUNK // 2) + -(-K // QUAD) * (QUAD // GROUP)


def is_mx4(bank) -> bool:
    """Whether a slot bank holds 4-bit experts (its dtype says so)."""
    return isinstance(bank, torch.Tensor) and bank.dtype == torch.uint8


def exp2i(e: torch.Tensor) -> torch.Tensor:
    """2^e in f32 of integers e in [-149, 127], from its bits: torch.ldexp and pow are
    off by a bit for some of them on a GPU."""
    e = e.to(torch.int32)
    small = torch.ones_like(e) << (e + 149).clamp(0, 22)  # below the normal numbers
    return torch.where(e >= -126, (e + 127) << 23, small).view(torch.float32)


def scale_values(scales: torch.Tensor) -> torch.Tensor:
    """The f32 scales that scale bytes stand for (255: NaN)."""
    v = exp2i((scales.to(torch.int32) - 127).clamp(max=127))
    return torch.where(scales == 255, torch.full_like(v, float("nan")), v)


def quantize(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of weights w [..., N, K].  Round to nearest even; the
    scale is the smallest power of two that keeps the group within +-6 (nothing
    saturates).  A group with a NaN or an infinity becomes NaN (scale byte 255)."""
    K = int(w.shape[-1])
    if K % GROUP:
        raise ValueError(f"rows of 4-bit weights are multiples of {GROUP} columns, got {K}")
    if not w.is_floating_point():
        raise ValueError(f"weights must be floating point, got {w.dtype}")
    g = w.detach().float().unflatten(-1, (-1, GROUP))
    amax = g.abs().amax(-1)
    bad = ~torch.isfinite(amax)
    m, ex = torch.frexp(torch.where(bad, torch.ones_like(amax), amax))
    e = (ex - 3 + (m > 0.75)).clamp_(min=-127)          # 6 = 0.75 * 2^3
    e = torch.where(amax > 0, e, torch.full_like(e, -127))
    # two exact steps: 2^127 alone would not reach the smallest scales' inverses
    v = g * exp2i(-e // 2).unsqueeze(-1) * exp2i(-e - (-e // 2)).unsqueeze(-1)
    a = v.abs()
    code = torch.zeros(a.shape, dtype=torch.uint8, device=a.device)
    for border, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= border) if up else (a > border)
    code |= torch.signbit(v).to(torch.uint8) << 3
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).flatten(-2)
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The f32 weights that (codes, scales) stand for."""
    lut = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    v = torch.stack([lut[(codes & 15).long()], lut[(codes >> 4).long()]], dim=-1).flatten(-2)
    s = scale_values(scales)
    return (v.unflatten(-1, (-1, GROUP)) * s.unsqueeze(-1)).flatten(-2)


def _check(codes: torch.Tensor, scales: torch.Tensor) -> tuple[int, int]:
    for t, name in ((codes, "codes"), (scales, "scales")):
        if t.dtype != torch.uint8 or t.dim() < 2:
            raise ValueError(f"{name} must be uint8 [..., N, columns], got {t.dtype} {tuple(t.shape)}")
    N, K = int(codes.shape[-2]), 2 * int(codes.shape[-1])
    if tuple(scales.shape) != (*codes.shape[:-1], K // GROUP) or K % GROUP:
        raise ValueError(f"scales {tuple(scales.shape)} do not match codes {tuple(codes.shape)}")
    if N % ROWS:
        raise ValueError(f"4-bit weights come in blocks of {ROWS} rows, got {N}")
    return N, K


def _pad(t: torch.Tensor, columns: int, value: int) -> torch.Tensor:
    return torch.nn.functional.pad(t, (0, columns - int(t.shape[-1])), value=value)


def pack_w2(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The bank's form of [..., N, K] weights (the down projection: N = H, K = I)."""
    N, K = _check(codes, scales)
    chunks, quads = -(-K // CHUNK), -(-K // QUAD)
    lead = codes.shape[:-2]
    c = _pad(codes, chunks * CHUNK // 2, 0).reshape(-1, N // ROWS, ROWS, chunks, 4, 16)
    c = c.permute(0, 1, 3, 4, 2, 5).reshape(-1, N // ROWS, chunks, 1024)
    s = _pad(scales, quads * QUAD // GROUP, 127).reshape(-1, N // ROWS, ROWS, quads, 4, 4)
    s = s.permute(0, 1, 3, 5, 2, 4).reshape(-1, N // ROWS, quads, 256)  # [.., group, row, chunk]
    parts = []
    for q in range(quads):
        parts += [s[:, :, q], c[:, :, 4 * q:4 * q + 4].flatten(2)]
    return torch.cat(parts, dim=-1).reshape(*lead, N, row_bytes(K)).contiguous()


def pack_w13(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The bank's form of [..., 2I, H] gate and up weights (gate rows first)."""
    N, _ = _check(codes, scales)
    if N % (2 * GROUP):
        raise ValueError(f"the expert width must be a multiple of {GROUP}, got {N} / 2")

    def mix(t):
        t = t.unflatten(-2, (2, N // 2 // ROWS, ROWS))
        return t.transpose(-4, -3).flatten(-4, -2)

    return pack_w2(mix(codes), mix(scales))


def unpack_w2(bank: torch.Tensor, K: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of a bank of K columns: the inverse of pack_w2."""
    N = int(bank.shape[-2])
    if bank.dtype != torch.uint8 or int(bank.shape[-1]) != row_bytes(K) or N % ROWS:
        raise ValueError(f"no bank of {K} columns: {bank.dtype} {tuple(bank.shape)}")
    chunks, quads = -(-K // CHUNK), -(-K // QUAD)
    b = bank.reshape(-1, N // ROWS, ROWS * row_bytes(K))
    cs, ss = [], []
    at = 0
    for q in range(quads):
        n = min(4, chunks - 4 * q)
        ss.append(b[:, :, at:at + 256])
        cs.append(b[:, :, at + 256:at + 256 + n * 1024])
        at += 256 + n * 1024
    c = torch.cat(cs, dim=-1).reshape(-1, N // ROWS, chunks, 4, ROWS, 16).permute(0, 1, 4, 2, 3, 5)
    s = torch.cat(ss, dim=-1).reshape(-1, N // ROWS, quads, 4, ROWS, 4).permute(0, 1, 4, 2, 5, 3)
    lead = bank.shape[:-2]
    return (c.reshape(*lead, N, chunks * CHUNK // 2)[..., :K // 2].contiguous(),
            s.reshape(*lead, N, quads * QUAD // GROUP)[..., :K // GROUP].contiguous())


def unpack_w13(bank: torch.Tensor, H: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) [..., 2I, .] of a gate-up bank: the inverse of pack_w13."""
    codes, scales = unpack_w2(bank, H)
    N = int(bank.shape[-2])

    def part(t):
        t = t.unflatten(-2, (N // 2 // ROWS, 2, ROWS))
        return t.transpose(-4, -3).flatten(-4, -2).contiguous()

    return part(codes), part(scales)


def _empty(shape: tuple, device, pin: bool) -> torch.Tensor:
    if pin:
        try:
            return torch.empty(shape, dtype=torch.uint8, device=device, pin_memory=True)
        except RuntimeError:  # no device runtime, or out of page-locked memory
            pass
    return torch.empty(shape, dtype=torch.uint8, device=device)


def _has_kernel(w: torch.Tensor, gate_up: bool) -> bool:
    """Whether native.quantize_mx4 takes these weights."""
    return w.is_cuda and w.dtype in (torch.bfloat16, torch.float32) and w.is_contiguous() and \
        w.data_ptr() % 16 == 0 and int(w.shape[1]) % (64 if gate_up else ROWS) == 0 and int(w.shape[2]) <= 1 << 23


def pack_experts(w13: torch.Tensor, w2: torch.Tensor, *, pin_memory: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """4-bit banks of bf16 (or f32) experts w13 [E, 2I, H], w2 [E, H, I], an
    expert at a time: what SlotMoELayer registers for 4-bit experts.  pin_memory:
    into page-locked memory (host weights) where there is some, for the host store
    to adopt."""
    if w13.dim() != 3 or w2.dim() != 3 or w13.shape[0] != w2.shape[0]:
        raise ValueError("experts are [E, 2I, H] and [E, H, I]")
    if int(w2.shape[1]) != int(w13.shape[2]) or 2 * int(w2.shape[2]) != int(w13.shape[1]):
        raise ValueError(f"w13 {tuple(w13.shape)} and w2 {tuple(w2.shape)} are not one layer's")
    out = []
    for w, pack in ((w13, pack_w13), (w2, pack_w2)):
        bank = _empty((*w.shape[:2], row_bytes(int(w.shape[2]))), w.device, pin_memory)
        if _has_kernel(w, pack is pack_w13):
            from vllm_moe_offload_amd import native  # which needs this module

            with torch.cuda.device(w.device):
                native.quantize_mx4(w.detach(), bank, gate_up=pack is pack_w13)
            out.append(bank)
            continue
        for e in range(int(w.shape[0])):
            bank[e] = pack(*quantize(w[e]))
        out.append(bank)
    return out[0], out[1]
