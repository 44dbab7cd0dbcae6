"""CPU checks of the 8-bit and expert operators: every refusal that the C ABI and the binding decide on the host, before
anything reaches a GPU, and the sizes that the queries report."""
import pytest
import torch

from wush_int4_kernel_b200 import capi

BAD, UNSUPPORTED, WORKSPACE = capi.WUSH_ERR_INVALID_ARGUMENT, capi.WUSH_ERR_UNSUPPORTED, capi.WUSH_ERR_WORKSPACE
P = 1 << 20            # an aligned address that nothing touches: every call below is refused before a launch


@pytest.fixture(scope="module")
def lib():
    return capi.load()


@pytest.mark.parametrize("args", [
    (P, 7, 4, 64, P, P), (P, -1, 4, 64, P, P),                      # dtype
    (P, capi.BF16, 4, 60, P, P), (P, capi.BF16, 4, 0, P, P), (P, capi.BF16, -1, 64, P, P),
    (P, capi.BF16, 4, capi.W8A8_MAX_K + 16, P, P),
    (None, capi.BF16, 4, 64, P, P), (P, capi.BF16, 4, 64, None, P), (P, capi.BF16, 4, 64, P, None),
    (P + 2, capi.BF16, 4, 64, P, P), (P, capi.BF16, 4, 64, P + 8, P), (P, capi.F32, 4, 64, P, P + 2),
])
def test_quant_int8_refusals(lib, args):
    assert lib.wush_quant_int8(*args, None) == BAD
    assert b"quant_int8" in lib.wush_last_error()


@pytest.mark.parametrize("change", [
    dict(K=40), dict(K=0), dict(K=capi.W8A8_MAX_K + 16), dict(M=-1), dict(N=-1), dict(M=1 << 31), dict(N=1 << 31),
    dict(xq=None), dict(xs=None), dict(wq=None), dict(ws=None), dict(y=None), dict(xq=P + 4), dict(wq=P + 8), dict(xs=P + 2),
    dict(bias=P + 1), dict(y=P + 2), dict(out=-1), dict(out=9),
])
def test_w8a8_gemm_refusals(lib, change):
    a = dict(xq=P, xs=P, wq=P, ws=P, bias=None, M=4, N=64, K=64, y=P, out=capi.F16) | change
    assert lib.wush_w8a8_gemm(a["xq"], a["xs"], a["wq"], a["ws"], a["bias"], a["M"], a["N"], a["K"], a["y"], a["out"], None, 0,
                              None) == BAD


def test_w8a8_empty_is_fine(lib):
    assert lib.wush_w8a8_gemm(None, None, None, None, None, 0, 64, 64, None, capi.F16, None, 0, None) == 0
    assert lib.wush_w8a8_gemm(None, None, None, None, None, 4, 0, 64, None, capi.F16, None, 0, None) == 0
    assert lib.wush_quant_int8(None, capi.BF16, 0, 64, None, None, None) == 0
    assert lib.wush_w8a8_gemm_workspace_bytes(0, 1) == 0 == lib.wush_w8a8_gemm_workspace_bytes(5, 0)
    assert lib.wush_w8a8_linear_workspace_bytes(0, 64) == 0 == lib.wush_w8a8_linear_workspace_bytes(4, 0)
    assert lib.wush_w8a8_expert_ffn_workspace_bytes(0, 64, 64, 4, 2) == 0


def test_w8a8_linear_refusals(lib):
    need = lib.wush_w8a8_linear_workspace_bytes(5, 64)
    assert need >= 5 * 64 + 5 * 4
    call = lambda x=P, dt=capi.BF16, work=P, n=need: lib.wush_w8a8_linear(x, dt, P, P, None, 5, 64, 64, P, work, n, None)  # noqa: E731
    assert call(dt=capi.F32) == BAD and call(x=None) == BAD and call(x=P + 2) == BAD
    assert call(work=None) == WORKSPACE and call(n=need - 1) == WORKSPACE and str(need).encode() in lib.wush_last_error()


@pytest.mark.parametrize("change", [
    dict(bytes=2), dict(k=0), dict(k=capi.EXPERT_MAX_K + 1), dict(E=0), dict(E=capi.EXPERT_MAX + 1), dict(T=-1), dict(ids=None),
    dict(pos=None), dict(offsets=None), dict(ids=P + 4), dict(pos=P + 2), dict(offsets=P + 1)])
def test_expert_sort_refusals(lib, change):
    a = dict(ids=P, bytes=8, T=4, k=2, E=8, pos=P, offsets=P) | change
    assert lib.wush_expert_sort(a["ids"], a["bytes"], a["T"], a["k"], a["E"], a["pos"], a["offsets"], None) == BAD


def test_expert_entries_limit(lib):
    assert lib.wush_expert_sort(P, 8, 1 << 30, 2, 8, P, P, None) == UNSUPPORTED
    assert lib.wush_expert_combine(P, capi.BF16, capi.BF16, 1 << 30, 64, P, 2, None, P, None) == UNSUPPORTED


@pytest.mark.parametrize("change", [
    dict(dt=3), dict(T=-1), dict(H=0), dict(k=0), dict(E=0), dict(x=None), dict(pos=None), dict(off=None), dict(out=None),
    dict(x=P + 1), dict(out=P + 1), dict(pos=P + 2), dict(off=P + 2)])
def test_expert_moves_refusals(lib, change):
    a = dict(x=P, dt=capi.BF16, T=4, H=32, pos=P, k=2, off=P, E=8, out=P) | change
    assert lib.wush_expert_gather(a["x"], a["dt"], a["T"], a["H"], a["pos"], a["k"], a["off"], a["E"], a["out"], None) == BAD
    assert lib.wush_expert_gather_quant_int8(a["x"], a["dt"], a["T"], a["H"], a["pos"], a["k"], a["off"], a["E"], a["out"], P, None) == BAD
    assert lib.wush_expert_combine_grad(a["x"], P, a["dt"], a["T"], a["H"], a["pos"], a["k"], a["off"], a["E"], P, a["out"], P, None) == BAD
    if not {"off", "E"} & set(change):
        assert lib.wush_expert_combine(a["x"], a["dt"], a["dt"], a["T"], a["H"], a["pos"], a["k"], None, a["out"], None) == BAD


def test_expert_combine_types(lib):
    for dt, out in ((capi.BF16, capi.F16), (capi.F16, capi.F32), (capi.F32, 3), (capi.F32, -1)):
        assert lib.wush_expert_combine(P, dt, out, 4, 32, P, 2, None, P, None) == BAD


def test_expert_gather_quant_needs_sixteen(lib):
    assert lib.wush_expert_gather_quant_int8(P, capi.BF16, 4, 40, P, 2, P, 8, P, P, None) == BAD


@pytest.mark.parametrize("change", [dict(K=40), dict(E=0), dict(E=capi.EXPERT_MAX + 1), dict(off=None), dict(wq=P + 4), dict(rows=-1)])
def test_grouped_refusals(lib, change):
    a = dict(wq=P, off=P, rows=8, E=4, N=32, K=64) | change
    assert lib.wush_w8a8_grouped_gemm(P, P, a["wq"], P, a["off"], a["rows"], a["E"], a["N"], a["K"], P, capi.F16, None, 0, None) == BAD
    assert lib.wush_w8a8_grouped_gated(P, P, a["wq"], P, a["off"], a["rows"], a["E"], a["N"], a["K"], P, None, 0, None) == BAD


def test_expert_ffn_refusals(lib):
    need = lib.wush_w8a8_expert_ffn_workspace_bytes(4, 64, 32, 8, 2)
    base = dict(x=P, dt=capi.BF16, ids=P, ib=8, w=P, w13q=P, H=64, inner=32, E=8, k=2, y=P, work=P, n=need)

    def call(**change):
        a = base | change
        return lib.wush_w8a8_expert_ffn(a["x"], a["dt"], a["ids"], a["ib"], a["w"], a["w13q"], P, P, P, 4, a["H"], a["inner"], a["E"], a["k"],
                                        a["y"], a["work"], a["n"], None)
    for change in (dict(dt=capi.F32), dict(ib=1), dict(H=40), dict(inner=8), dict(k=0), dict(E=0), dict(x=None), dict(ids=None),
                   dict(w=None), dict(y=None), dict(x=P + 2), dict(y=P + 8), dict(w13q=None), dict(w13q=P + 8), dict(work=P + 8)):
        assert call(**change) == BAD, change
    assert call(work=None) == WORKSPACE and call(n=need - 1) == WORKSPACE


def test_binding_refuses_cpu_tensors():
    from my_int4 import _C

    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    ids, pos, off = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(9, dtype=torch.int32)
    w = torch.zeros(4, 2)
    for call in (lambda: _C.quant_int8(x), lambda: _C.w8a8_gemm(q, s, q, s), lambda: _C.w8a8_linear(x, q, s),
                 lambda: _C.expert_sort(ids, 8), lambda: _C.expert_gather(x, pos, off), lambda: _C.expert_gather_quant_int8(x, pos, off),
                 lambda: _C.expert_combine(x, pos, w), lambda: _C.expert_combine_grad(x, x, pos, off, w),
                 lambda: _C.w8a8_grouped_gemm(q, s, q[None], s[None], off), lambda: _C.w8a8_grouped_gated(q, s, q[None], s[None], off),
                 lambda: _C.w8a8_expert_ffn(x, ids, w, q[None], s[None], q[None], s[None])):
        with pytest.raises(RuntimeError):
            call()


def test_header_constants_of_the_8_bit_operators():
    import os
    import re

    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "wush_int4.h")).read()
    value = lambda name: int(re.search(rf"\b{name}\s*=?\s*(\d+)", header).group(1))  # noqa: E731
    assert [value("WUSH_BF16"), value("WUSH_F16"), value("WUSH_F32")] == [capi.BF16, capi.F16, capi.F32]
    assert [value("#define WUSH_W8A8_MAX_K".split()[1]), value("WUSH_EXPERT_MAX"), value("WUSH_EXPERT_MAX_K")] == \
        [capi.W8A8_MAX_K, capi.EXPERT_MAX, capi.EXPERT_MAX_K]


def test_division_of_work_covers_every_stage_once(lib):
    """Both kernels' pieces, walked on the host: every stage of every tile once, every piece a slot of its own."""
    import ctypes
    import random

    rng = random.Random(5)
    shapes = [(0, 1), (1, 1), (1, 1000), (147, 3), (148, 1), (149, 64), (448, 64), (192, 33), (64, 64), (3, 2), (1000, 9), (224, 32), (75, 31)]
    shapes += [(int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 9))) for _ in range(400)]
    cuts = [0, 0]
    for kernel, ctas in ((0, 148), (1, 74), (0, 132), (1, 66)):
        for tiles, steps in shapes:
            cover, cut = (ctypes.c_int * max(1, tiles * steps))(), ctypes.c_int(-1)
            assert lib.wush_debug_w8a8_cover(kernel, tiles, steps, ctas, cover, ctypes.byref(cut)) == 0, (kernel, tiles, steps, ctas)
            assert all(v == 1 for v in cover[:tiles * steps]), (kernel, tiles, steps, ctas)
            cuts[kernel] += cut.value
    assert cuts[0] > 1000 and cuts[1] > 100
