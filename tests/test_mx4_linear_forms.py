"""The rule that gives each product with one 4-bit matrix its kernel form, on the CPU: the
forms that the sizes of the GPU tests are for, and the refusals of the entry that tells."""

import ctypes

import pytest

from tests.test_gpu_mx4_linear_tiles import CASES, SPLIT


@pytest.mark.parametrize("kind,rows,columns,T,K,N", CASES + SPLIT)
def test_the_cases_reach_their_form(kind, rows, columns, T, K, N):
    from vllm_moe_offload_amd import native

    form = native.mx4_linear_form(kind.removesuffix("-f32"), T, K, N, out_f32=kind.endswith("-f32"), cu_count=256)
    assert form == (rows, columns, (kind, rows, columns, T, K, N) in SPLIT)


def test_every_form_has_cases():
    assert {(r, c) for _, r, c, *_ in SPLIT} == {(16, 32), (16, 64), (32, 64), (16, 128)}
    forms = {(kind, rows, columns) for kind, rows, columns, *_ in CASES}
    assert forms == {("bf16", 32, 256), ("bf16", 64, 256), ("bf16", 128, 256),
                     *(("mx8", r, c) for r, c in ((64, 64), (64, 128), (128, 128), (128, 256), (256, 256))),
                     *(("mx8-f32", r, c) for r, c in ((64, 64), (64, 128), (128, 128))),
                     *(("mx4", r, c) for r, c in ((64, 64), (64, 128), (128, 128), (256, 256)))}


@pytest.mark.parametrize("kind", ["bf16", "mx8", "mx4"])
def test_few_rows_split_k(kind):
    from vllm_moe_offload_amd import native

    form = lambda *size: native.mx4_linear_form(kind, *size, cu_count=256)
    assert form(1, 2048, 5120) == form(16, 2048, 16384) == (16, 32, True)
    assert form(16, 2048, 50000) == (16, 128, True)
    assert form(33, 2048, 5120) == (16, 64, True)
    assert form(64, 7168, 7168) == (32, 64, True)
    assert form(128, 2048, 5120)[2] == (kind == "bf16")
    for T, K, N in ((1 << 30, 32, 16), (65_536 * 32 + 5, 32, 16), (1 << 20, 1 << 23, 1 << 20)):
        assert not form(T, K, N)[2]


def test_refusals():
    from vllm_moe_offload_amd import native

    lib = native.load_library()
    out = (ctypes.c_int * 3)()
    call = lambda rows=2, T=4, K=64, N=32, cus=256, form=out: lib.lmoe_mx4_linear_form(rows, 0, T, K, N, cus, form)
    assert call() == 0 and list(out) == [16, 32, 1]
    assert [call(T=0), call(T=-1), call(K=0), call(N=0), call(cus=-1), call(form=None)] == [1000] * 6
    assert [call(K=48), call(N=24), call(K=(1 << 23) + 32)] == [1001] * 3
    assert call(rows=3) == call(rows=-1) == lib.lmoe_mx4_linear(None, None, 3, 4, 64, 32, *[None] * 2, 0, None, None, 0, None) != 0
