"""GPU tests of the 8-bit and expert operators against plain definitions in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32, e(t) = finfo(t).eps / 2 of the result's type.  A product is the exact integer
sum rounded to fp32, times the rounded product of two scales: three roundings, then one to the result's type, whose
subnormals (fp16) add at most half of 2^-24.  The other bounds count the roundings of the formula in the same way, where the
test uses them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY16 = 2.0 ** -25
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def e(t):
    return torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def C():
    assert torch.cuda.is_available()
    from my_int4 import _C
    _C.init()
    yield _C
    import ctypes

    from wush_int4_kernel_b200 import capi
    flag = ctypes.c_int(-1)
    capi.check(capi.load().wush_device_flag(ctypes.byref(flag)), "device flag")
    assert (flag.value >> 16) & 0xff == 0, f"a bounded wait of an 8-bit product gave up (role code {(flag.value >> 16) & 0xff})"


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, g, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def codes(*shape, g):
    return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def scales(*shape, g, width):
    return (torch.rand(*shape, generator=g, device="cuda") + 0.5) / (127 * 40 * width ** 0.5) ** 0.5


def quant64(x):
    """Codes and scales of the definition; torch.round is ties-to-even."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * x / top), 0.0), (top / 127).squeeze(-1)


def within(y, want, bound):
    err = (y.double() - want).abs()
    worst = (err / bound.clamp(min=1e-300)).max().item() if err.numel() else 0.0
    assert torch.isfinite(y.double()).all() and worst <= 1.0, f"{worst} of the bound"


# ---- quantiser -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,K", [(1, 16), (1, 8192), (3, 48), (7, 1040), (300, 512), (700, 4112), (2, 33024), (1, 131072), (400, 40000)])
def test_quant_int8_codes_are_the_definition(C, dtype, rows, K):
    g = gen(rows * 7 + K)
    x = randn(rows, K, g=g) * torch.exp(2 * randn(rows, 1, g=g))
    x[:, :: 5] *= 0.01
    x = x.to(dtype)
    q, s = C.quant_int8(x)
    q64, s64 = quant64(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and s.shape == (rows,)
    assert torch.equal(q.double(), q64)
    within(s, s64, s64 * 2 * U)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quant_int8_every_value_against_every_maximum(C, dtype):
    """All mantissas of x against many maxima: every exact tie of the grid occurs (x = amax / 2 gives 63.5, for one)."""
    m = 8 if dtype == torch.bfloat16 else 11
    tops = torch.arange(2 ** (m - 1), 2 ** m, 1 if m == 8 else 7, device="cuda").double()
    base = torch.arange(0, 2 ** m, device="cuda").double()
    x = torch.cat([base * 2.0 ** -p for p in range(0, 9)])
    x = x[None, :].expand(tops.numel(), -1)
    x = torch.where(x <= tops[:, None], x, -x / 2)
    x = torch.where(x.abs() <= tops[:, None], x, 0.0)
    x = torch.cat((tops[:, None], x, x.new_zeros(x.shape[0], -(x.shape[1] + 1) % 16)), 1).to(dtype)
    q, _ = C.quant_int8(x.contiguous())
    q64, _ = quant64(x)
    tie = (127 * x.double() / tops[:, None]).frac().abs() == 0.5
    assert tie.sum() > 100 and torch.equal(q.double(), q64)


def test_quant_int8_special_rows(C):
    inf, nan = float("inf"), float("nan")
    for dtype in TYPES:
        x = torch.zeros(8, 64, device="cuda")
        x[1, 3] = inf
        x[2, 5] = nan
        x[3] = 1.0
        x[4, 0] = torch.finfo(dtype).max
        x[4, 1:] = torch.finfo(dtype).max / 3
        x[5, 0], x[5, 1] = -inf, nan
        x[6, 7] = torch.finfo(dtype).smallest_normal * 2
        x[6, 8] = -torch.finfo(dtype).smallest_normal
        x[7, 9] = -0.0
        xd = x.to(dtype)
        if dtype == torch.bfloat16:
            xd[7, 10] = 2.0 ** -133        # the smallest subnormal
        q, s = C.quant_int8(xd)
        assert s[0] == 0 and not q[0].any()
        assert s[1] == inf and not q[1].any()
        assert torch.isnan(s[2]) and torch.isnan(s[5]) and not q[2].any() and not q[5].any()
        assert (q[3] == 127).all()
        assert q[4, 0] == 127 and (q[4, 1:] == 42).all()
        assert q[6, 7] == 127 and q[6, 8] == -64               # 63.5, a tie, goes to the even 64
        if dtype == torch.bfloat16:
            assert q[7, 10] == 127 and q[7].abs().sum() == 127


@pytest.mark.parametrize("rows,K", [(1, 1024), (513, 1408), (5, 70000 // 16 * 16)])
def test_quant_int8_fp32_rows(C, rows, K):
    x = randn(rows, K, g=gen(K))
    q, s = C.quant_int8(x)
    top = x.double().abs().amax(-1)
    within(s, top / 127, top / 127 * U)
    v = 127 * x.double() / top[:, None]
    assert ((q.double() - v).abs() <= 0.5 + v.abs() * 3 * U).all()


def test_quant_int8_shapes(C):
    x = randn(2, 3, 64, g=gen(1), dtype=torch.bfloat16)
    q, s = C.quant_int8(x)
    assert q.shape == (2, 3, 64) and s.shape == (2, 3)
    q, s = C.quant_int8(x[:0])
    assert q.shape == (0, 3, 64) and s.shape == (0, 3)
    q1, s1 = C.quant_int8(x[0, 0])
    assert q1.shape == (64,) and s1.shape == ()
    for bad in (x[..., ::2], x[..., :40].contiguous(), x.double(), x.transpose(0, 1)):
        with pytest.raises(RuntimeError):
            C.quant_int8(bad)


# ---- product -------------------------------------------------------------------------------------------------------------

def product64(xq, xs, wq, ws):
    return (xq.double() @ wq.double().T) * xs.double()[:, None] * ws.double()


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 16), (1, 128, 128), (1, 4096, 4096), (2, 130, 272), (3, 5003, 4112), (5, 640, 8192), (15, 257, 1040), (16, 1024, 512),
    (17, 1024, 512), (31, 999, 2064), (32, 256, 16384), (33, 384, 640), (63, 127, 144), (64, 8192, 1024), (65, 256, 256),
    (100, 1000, 2000), (128, 512, 512), (129, 513, 528), (255, 640, 1024), (256, 256, 256), (257, 258, 272), (300, 2048, 4096),
    (513, 1026, 1008), (1000, 3001, 720), (2100, 512, 2048),
    # long K: tiles of the last wave cut along K, few of them, many of them, with narrow and odd edges
    (65, 130, 16384), (100, 1000, 12304), (129, 513, 8192), (300, 4099, 8192), (333, 2048, 28672), (300, 20000, 6160)])
def test_w8a8_gemm(C, M, N, K, out):
    g = gen(M * 31 + N * 7 + K)
    xq, wq = codes(M, K, g=g), codes(N, K, g=g)
    xs, ws = scales(M, g=g, width=K), scales(N, g=g, width=K)
    y = C.w8a8_gemm(xq, xs, wq, ws, None, out)
    want = product64(xq, xs, wq, ws)
    assert y.dtype == out and y.shape == (M, N)
    within(y, want, want.abs() * (e(out) + 4 * U) + TINY16)
    bias = randn(N, g=g)
    y = C.w8a8_gemm(xq, xs, wq, ws, bias, out)
    both = want + bias.double()
    within(y, both, want.abs() * 4 * U + both.abs() * (e(out) + 2 * U) + TINY16)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_w8a8_gemm_largest_sums(C, M):
    """All codes at the limit and the longest K: the int32 sums reach 127 * 127 * 131072 = 2.11e9 < 2^31."""
    K, N = 131072, 130
    xq = torch.full((M, K), 127, dtype=torch.int8, device="cuda")
    wq = torch.full((N, K), 127, dtype=torch.int8, device="cuda")
    wq[1::2] = -127
    one = torch.full((M,), 2.0 ** -16, device="cuda")
    y = C.w8a8_gemm(xq, one, wq, torch.ones(N, device="cuda"), None, torch.float16)
    want = torch.tensor(127 * 127 * 131072 / 65536.0, device="cuda").double().expand(M, N) * torch.where(torch.arange(N, device="cuda") % 2 == 0, 1, -1)
    within(y, want, want.abs() * (e(torch.float16) + 4 * U))


def test_w8a8_gemm_shapes_and_refusals(C):
    g = gen(2)
    xq, xs, wq, ws = codes(2, 3, 64, g=g), scales(2, 3, g=g, width=64), codes(32, 64, g=g), scales(32, g=g, width=64)
    y = C.w8a8_gemm(xq, xs, wq, ws)
    assert y.shape == (2, 3, 32) and y.dtype == torch.float16
    assert torch.equal(y.view(6, 32), C.w8a8_gemm(xq.view(6, 64), xs.view(6), wq, ws))
    assert C.w8a8_gemm(xq[:0], xs[:0], wq, ws).shape == (0, 3, 32)
    assert C.w8a8_gemm(xq, xs, wq[:0], ws[:0]).shape == (2, 3, 0)
    for args in ((xq, xs[0], wq, ws), (xq, xs, wq[:, :48].contiguous(), ws), (xq, xs, wq, ws[:31]), (xq, xs.half(), wq, ws),
                 (xq.to(torch.uint8), xs, wq, ws), (xq, xs, wq, ws, ws[:31]), (xq, xs, wq, ws, ws.half()), (xq, xs, wq, ws, None, torch.float64),
                 (xq, xs, wq.T, ws), (xq.cpu(), xs, wq, ws), (xq, xs, wq.cpu(), ws)):
        with pytest.raises(RuntimeError):
            C.w8a8_gemm(*args)


def test_w8a8_non_finite_rows(C):
    """A row with an infinity or a NaN answers NaN, its neighbours are untouched."""
    from wush_int4_kernel_b200.linear import W8A8Linear
    g = gen(3)
    lin = W8A8Linear.from_weight(randn(96, 128, g=g))
    x = randn(5, 128, g=g, dtype=torch.bfloat16)
    clean = lin(x)
    x[1, 7], x[3, 100] = float("inf"), float("nan")
    y = lin(x)
    assert torch.isnan(y[[1, 3]]).all() and torch.equal(y[[0, 2, 4]], clean[[0, 2, 4]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K,bias", [(1, 512, 1024, False), (1, 4100, 8192, True), (4, 77, 48, True), (24, 1000, 4096, False), (70, 640, 512, True),
                                        (600, 1281, 1024, True), (3, 200, 40000, False)])
def test_linear_is_quantiser_then_product(C, dtype, M, N, K, bias):
    from wush_int4_kernel_b200.linear import W8A8Linear
    g = gen(M + N + K)
    lin = W8A8Linear.from_weight(randn(N, K, g=g, dtype=dtype) * 0.05, randn(N, g=g) if bias else None)
    assert (lin.in_features, lin.out_features) == (K, N)
    x = randn(M, K, g=g, dtype=dtype)
    xq, xs = C.quant_int8(x)
    want = C.w8a8_gemm(xq, xs, lin.wq, lin.ws, lin.bias, dtype)
    for _ in range(3):
        assert torch.equal(lin(x), want)
    assert torch.equal(lin(x.view(M, 1, K)), want.view(M, 1, N))


# ---- order ---------------------------------------------------------------------------------------------------------------

def order64(ids, E):
    """pos and offsets of the definition, on the host."""
    a = ids.cpu().numpy().reshape(-1)
    pos, offsets = np.full(a.shape, -1, np.int32), np.zeros(E + 1, np.int32)
    for i in range(E):
        at = np.nonzero(a == i)[0]
        pos[at] = offsets[i] + np.arange(at.size)
        offsets[i + 1] = offsets[i] + at.size
    return torch.from_numpy(pos.reshape(ids.shape)).cuda(), torch.from_numpy(offsets).cuda()


def ids_of(T, k, E, g, drop=0.1, dtype=torch.int64):
    ids = torch.randint(0, E, (T, k), generator=g, device="cuda")
    ids = torch.where(torch.rand(T, k, generator=g, device="cuda") < drop, -1, ids)
    return ids.to(dtype)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (1, 8, 64), (5, 3, 1024), (64, 8, 128), (333, 7, 60), (512, 8, 256), (513, 8, 256),
                                   (4097, 1, 3), (9000, 8, 256), (20000, 3, 1000), (1000, 64, 33)])
def test_expert_sort(C, T, k, E, dtype):
    ids = ids_of(T, k, E, gen(T + k + E), dtype=dtype)
    pos, offsets = C.expert_sort(ids, E)
    want_pos, want_offsets = order64(ids, E)
    assert pos.dtype == offsets.dtype == torch.int32
    assert torch.equal(pos, want_pos) and torch.equal(offsets, want_offsets)


def test_expert_sort_extremes(C):
    E = 16
    for T, k in ((700, 8), (40, 2)):
        one = torch.full((T, k), 11, device="cuda")
        pos, offsets = C.expert_sort(one, E)
        assert torch.equal(pos.view(-1), torch.arange(T * k, device="cuda", dtype=torch.int32))
        assert offsets.tolist() == [0] * 12 + [T * k] * 5
        odd = torch.tensor([-1, E, -(1 << 40), (1 << 40) + 3, (1 << 63) - 1], device="cuda")
        none = odd[torch.arange(T * k, device="cuda") % 5].view(T, k)
        pos, offsets = C.expert_sort(none, E)
        assert (pos == -1).all() and not offsets.any()
    for ids, n in ((one, 0), (one, 1025), (one.float(), 4), (one[0], 4), (one.t(), 4), (one.cpu(), 4)):
        with pytest.raises(RuntimeError):
            C.expert_sort(ids, n)


ORDER_CASES = [(1, 1, 1, 1), (1, 8, 64, 2048), (6, 2, 3, 7), (64, 8, 128, 2048), (50, 5, 60, 1001), (333, 9, 17, 136), (2000, 3, 8, 516),
               (5, 64, 8, 40), (257, 4, 256, 4096)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,E,H", ORDER_CASES)
def test_expert_moves(C, T, k, E, H, dtype):
    g = gen(T + k + E + H)
    ids = ids_of(T, k, E, g)
    pos, offsets = C.expert_sort(ids, E)
    used = int(offsets[-1])
    x = randn(T, H, g=g, dtype=dtype)
    rows = C.expert_gather(x, pos, offsets)
    want = torch.zeros(T * k, H, device="cuda", dtype=dtype)
    t_of = torch.arange(T, device="cuda").repeat_interleave(k)
    here = pos.view(-1) >= 0
    want[pos.view(-1)[here].long()] = x[t_of[here]]
    assert torch.equal(rows, want)
    # the rows behind the last entry and the weights of absent entries hold NaN: neither may be read
    ys = randn(T * k, H, g=g, dtype=dtype)
    ys[used:] = float("nan")
    w = torch.where(pos >= 0, randn(T, k, g=g), float("nan"))
    dy = randn(T, H, g=g, dtype=dtype)
    y = C.expert_combine(ys, pos, w)
    picked = torch.where(pos.unsqueeze(-1) >= 0, ys.double()[pos.clamp(min=0).long()], 0.0)
    w64 = torch.where(pos >= 0, w.double(), 0.0).unsqueeze(-1)
    terms = picked * w64
    within(y, terms.sum(1), terms.abs().sum(1) * k * U + terms.sum(1).abs() * (e(dtype) + 2 * U) + TINY16)
    plain = C.expert_combine(ys, pos)
    within(plain, picked.sum(1), picked.abs().sum(1) * k * U + picked.sum(1).abs() * (e(dtype) + 2 * U) + TINY16)
    if dtype == torch.float32:
        for out in (torch.bfloat16, torch.float16):
            y = C.expert_combine(ys, pos, w, out)
            assert y.dtype == out
            within(y, terms.sum(1), terms.abs().sum(1) * (k + 1) * U + terms.sum(1).abs() * (e(out) + 2 * U) + TINY16)
    d_rows, d_w = C.expert_combine_grad(dy, ys, pos, offsets, w)
    want = torch.zeros(T * k, H, device="cuda", dtype=torch.float64)
    want[pos.view(-1)[here].long()] = (w64 * dy.double().unsqueeze(1)).reshape(T * k, H)[here]
    within(d_rows, want, want.abs() * (e(dtype) + 2 * U) + TINY16)
    assert not d_rows[used:].any()
    products = picked * dy.double().unsqueeze(1)
    within(d_w, products.sum(-1), products.abs().sum(-1) * (H / 32 + 24) * U + 1e-300)
    assert not d_w[pos < 0].any()
    if H % 16 == 0:
        q, s = C.expert_gather_quant_int8(x, pos, offsets)
        q1, s1 = C.quant_int8(x)
        wq, wsc = torch.zeros_like(q), torch.zeros_like(s)
        wq[pos.view(-1)[here].long()], wsc[pos.view(-1)[here].long()] = q1[t_of[here]], s1[t_of[here]]
        assert torch.equal(q, wq) and torch.equal(s, wsc)


@pytest.mark.parametrize("dtype", TYPES)
def test_expert_moves_at_odd_addresses(C, dtype):
    """Pointers that are aligned to one element only take the narrow path and give the same answers."""
    T, k, E, H = 37, 3, 5, 64
    g = gen(9)
    pos, offsets = C.expert_sort(ids_of(T, k, E, g), E)
    w = randn(T, k, g=g)

    def shifted(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)
    x, ys = randn(T, H, g=g, dtype=dtype), randn(T * k, H, g=g, dtype=dtype)
    assert torch.equal(C.expert_gather(shifted(x), pos, offsets), C.expert_gather(x, pos, offsets))
    assert torch.equal(C.expert_combine(shifted(ys), pos, w), C.expert_combine(ys, pos, w))
    a, b = C.expert_combine_grad(shifted(x), ys, pos, offsets, w), C.expert_combine_grad(x, ys, pos, offsets, w)
    assert torch.equal(a[0], b[0])
    prod = (ys.double()[pos.clamp(min=0).long()] * x.double().unsqueeze(1)).abs().sum(-1)
    assert ((a[1] - b[1]).abs().double() <= prod * 2 * 26 * U).all()          # another order of the same sum


def test_expert_moves_all_dropped_and_empty(C):
    for T in (0, 5):
        pos, offsets = C.expert_sort(torch.full((T, 2), -1, device="cuda"), 4)
        x = randn(T, 32, g=gen(1), dtype=torch.bfloat16)
        nan = torch.full((T * 2, 32), float("nan"), device="cuda", dtype=torch.bfloat16)
        w = torch.ones(T, 2, device="cuda")
        assert not C.expert_gather(x, pos, offsets).any() and not C.expert_combine(nan, pos, w).any()
        d_rows, d_w = C.expert_combine_grad(x, nan, pos, offsets, w)
        assert not d_rows.any() and not d_w.any()
        q, s = C.expert_gather_quant_int8(x, pos, offsets)
        assert not q.any() and not s.any()


def test_expert_moves_refuse(C):
    T, k, E, H = 6, 2, 4, 32
    g = gen(4)
    pos, offsets = C.expert_sort(ids_of(T, k, E, g), E)
    x, ys, w = randn(T, H, g=g, dtype=torch.bfloat16), randn(T * k, H, g=g, dtype=torch.bfloat16), randn(T, k, g=g)
    for call in (lambda: C.expert_gather(x[:5], pos, offsets), lambda: C.expert_gather(x.t(), pos, offsets),
                 lambda: C.expert_gather(x, pos.long(), offsets), lambda: C.expert_gather(x, pos, offsets.long()),
                 lambda: C.expert_gather(x.double(), pos, offsets), lambda: C.expert_gather(x, pos.cpu(), offsets),
                 lambda: C.expert_combine(ys[:-1], pos, w), lambda: C.expert_combine(ys, pos, w.half()),
                 lambda: C.expert_combine(ys, pos, w[:, :1]), lambda: C.expert_combine(ys, pos, w, torch.float32), lambda: C.expert_combine(ys, pos.view(-1), None),
                 lambda: C.expert_combine_grad(x.float(), ys, pos, offsets, w), lambda: C.expert_combine_grad(x[:, :16], ys, pos, offsets, w),
                 lambda: C.expert_gather_quant_int8(x[:, :24].contiguous(), pos, offsets)):
        with pytest.raises(RuntimeError):
            call()


def test_route_gradients(C):
    """Autograd of the two moves: against the formula through plain indexing, and against differences."""
    from wush_int4_kernel_b200.experts import ExpertRoute
    T, k, E, H = 9, 3, 4, 20
    g = gen(5)
    ids = ids_of(T, k, E, g, drop=0.2)
    route = ExpertRoute.sort(ids, E)
    x0, w0, scale = randn(T, H, g=g), randn(T, k, g=g), randn(T * k, H, g=g)

    def loss(x, w):
        return (route.combine(route.gather(x) * scale, w) ** 2).sum()

    def plain(x, w):
        here = (route.pos >= 0).unsqueeze(-1)
        at = route.pos.clamp(min=0).long()
        y = torch.where(here, x.unsqueeze(1) * scale.double()[at], 0.0) * torch.where(here, w.unsqueeze(-1), 0.0)
        return (y.sum(1) ** 2).sum()
    x, w = x0.clone().requires_grad_(), w0.clone().requires_grad_()
    loss(x, w).backward()
    x64, w64 = x0.double().requires_grad_(), w0.double().requires_grad_()
    plain(x64, w64).backward()
    for a, b in ((x.grad, x64.grad), (w.grad, w64.grad)):
        assert (a.double() - b).norm() <= b.norm() * 64 * U * k
    # a central difference of step h in 64 bits along a random direction: error h^2 / 6 of a third derivative, and the loss is
    # a polynomial of degree two in each of x and w, so along x alone it has none; 2^-20 covers the gradient's own roundings
    dirs = randn(T, H, g=g).double()
    h = 1e-3
    diff = (plain(x0.double() + h * dirs, w0.double()) - plain(x0.double() - h * dirs, w0.double())) / (2 * h)
    assert abs((x.grad.double() * dirs).sum() - diff) <= 2.0 ** -20 * (x.grad.double() * dirs).abs().sum() + 1e-9
    # a gradient that arrives expanded, and one input only
    xo = x0.clone().requires_grad_()
    route.gather(xo).sum().backward()
    assert torch.equal(xo.grad, (route.pos >= 0).sum(1, keepdim=True).float().expand(T, H))
    wo = w0.clone().requires_grad_()
    route.combine(scale, wo).sum().backward()
    want = torch.where(route.pos >= 0, scale.double().sum(-1)[route.pos.clamp(min=0).long()], 0.0)
    assert ((wo.grad.double() - want).abs() <= scale.double().abs().sum(-1).max() * 26 * U).all()


# ---- experts' products -----------------------------------------------------------------------------------------------------

def grouped_case(sizes, tail, N, K, g):
    E, R = len(sizes), sum(sizes) + tail
    offsets = torch.tensor([0] + list(np.cumsum(sizes)), dtype=torch.int32, device="cuda")
    xq, xs = codes(R, K, g=g), scales(R, g=g, width=K)
    xs[sum(sizes):] = float("nan")                        # rows of no expert: not read
    return xq, xs, codes(E, N, K, g=g), scales(E, N, g=g, width=K), offsets


SIZES = [([1], 0), ([0, 0, 3, 0], 2), ([5, 0, 1, 17, 2], 0), ([16, 33, 64, 65], 7), ([0, 300, 0, 129, 1], 40), ([700, 2, 256, 255], 0),
         ([1] * 40, 3), ([0] * 60 + [40] + [0] * 40, 5), ([0, 0], 6)]


@pytest.mark.parametrize("N,K", [(128, 128), (1000, 272), (77, 1040), (2048, 1024)])
@pytest.mark.parametrize("sizes,tail", SIZES)
def test_grouped_gemm(C, sizes, tail, N, K):
    xq, xs, wq, ws, offsets = grouped_case(sizes, tail, N, K, gen(sum(sizes) + N + K))
    for out in TYPES:
        y = C.w8a8_grouped_gemm(xq, xs, wq, ws, offsets, out)
        assert y.shape == (xq.shape[0], N) and y.dtype == out and not y[sum(sizes):].any()
        a = 0
        for i, n in enumerate(sizes):
            want = product64(xq[a:a + n], xs[a:a + n], wq[i], ws[i])
            within(y[a:a + n], want, want.abs() * (e(out) + 4 * U) + TINY16)
            a += n


@pytest.mark.parametrize("inner,K", [(64, 128), (500, 272), (37, 1040), (1024, 2048)])
@pytest.mark.parametrize("sizes,tail", SIZES)
def test_grouped_gated(C, sizes, tail, inner, K):
    """g and u carry 3 u each; silu has a relative condition of at most 1 + |g|; __expf (2 + 1.173 |g| units in the last place,
    of 2 u each), the sum, the quotient and the last product add 4 + 2.4 |g| + 1 + 4 + 1 of u; beyond |g| = 80 the exponential
    leaves the range of fp32 and 1e-30 |u| covers the rest."""
    xq, xs, wq, ws, offsets = grouped_case(sizes, tail, 2 * inner, K, gen(sum(sizes) + inner + K))
    h = C.w8a8_grouped_gated(xq, xs, wq, ws, offsets)
    assert h.shape == (xq.shape[0], inner) and h.dtype == torch.float32 and not h[sum(sizes):].any()
    a = 0
    for i, n in enumerate(sizes):
        g, u = product64(xq[a:a + n], xs[a:a + n], wq[i], ws[i]).chunk(2, dim=-1)
        want = g * torch.sigmoid(g) * u
        within(h[a:a + n], want, want.abs() * (5.4 * g.abs() + 3 + 3 + 10 + 2) * U + 1e-30 * (1 + u.abs()))
        a += n


@pytest.mark.parametrize("sizes,tail", [([100, 0, 300, 71], 5), ([512], 0), ([1, 700], 3), ([90] * 6, 0)])
def test_grouped_long_k(C, sizes, tail):
    """Enough stages for the last wave's tiles to be cut along K."""
    N, K = 520, 8208
    xq, xs, wq, ws, offsets = grouped_case(sizes, tail, N, K, gen(sum(sizes)))
    y = C.w8a8_grouped_gemm(xq, xs, wq, ws, offsets)
    h = C.w8a8_grouped_gated(xq, xs, wq, ws, offsets)
    assert not y[sum(sizes):].any() and not h[sum(sizes):].any()
    a = 0
    for i, n in enumerate(sizes):
        want = product64(xq[a:a + n], xs[a:a + n], wq[i], ws[i])
        within(y[a:a + n], want, want.abs() * (e(torch.float16) + 4 * U) + TINY16)
        g, u = want.chunk(2, dim=-1)
        want = g * torch.sigmoid(g) * u
        within(h[a:a + n], want, want.abs() * (5.4 * g.abs() + 3 + 3 + 10 + 2) * U + 1e-30 * (1 + u.abs()))
        a += n


def test_gated_extreme_gates(C):
    """Gates far out on both sides: silu(g) is g or 0, never NaN."""
    K, inner = 128, 8
    wq = torch.zeros(1, 2 * inner, K, dtype=torch.int8, device="cuda")
    wq[0, :inner] = torch.tensor([127, -127, 1, -1, 0, 64, -64, 8], device="cuda", dtype=torch.int8)[:, None]
    wq[0, inner:] = 1
    xq = torch.full((1, K), 127, dtype=torch.int8, device="cuda")
    h = C.w8a8_grouped_gated(xq, torch.ones(1, device="cuda"), wq, torch.ones(1, 2 * inner, device="cuda"),
                             torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    g = wq[0, :inner, 0].double() * 127 * K
    assert torch.isfinite(h).all() and torch.equal(h[0].double(), torch.where(g > 0, g, 0.0) * 127 * K)


def test_grouped_offsets_outside_the_rows_are_cut(C):
    """Offsets that leave the rows are cut to them: nothing outside is read, and rows inside keep their answers."""
    xq, xs, wq, ws, _ = grouped_case([20, 30], 0, 64, 128, gen(8))
    y = C.w8a8_grouped_gemm(xq, xs, wq, ws, torch.tensor([-7, 20, 5000], dtype=torch.int32, device="cuda"))
    assert torch.equal(y, C.w8a8_grouped_gemm(xq, xs, wq, ws, torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")))
    # descending ones: every row belongs to at most one expert, the first that reaches it
    for bad, good in (([0, 50, 20, 50], [0, 50, 50, 50]), ([30, 10, 50, 0], [30, 30, 50, 50]), ([50, 0, 0, 0], [50] * 4)):
        wq3, ws3 = torch.cat((wq, wq[:1])), torch.cat((ws, ws[:1]))
        as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        y, want = (C.w8a8_grouped_gemm(xq, xs, wq3, ws3, as_int(v)) for v in (bad, good))
        a, b = good[0], good[-1]
        assert torch.equal(y[a:b], want[a:b])
    pos = torch.tensor([[0, 99], [-5, 1 << 30]], dtype=torch.int32, device="cuda")
    x = randn(2, 128, g=gen(1), dtype=torch.bfloat16)
    rows = C.expert_gather(x, pos, torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    assert torch.equal(rows[0], x[0]) and not rows[1:].any()
    y = C.expert_combine(rows, pos)
    assert torch.equal(y[0], x[0]) and not y[1].any()


def test_grouped_most_experts(C):
    """1024 experts, most of them without a row, through every operator that takes offsets."""
    from wush_int4_kernel_b200.experts import W8A8Experts
    g = gen(77)
    E, H, inner = 1024, 64, 32
    block = W8A8Experts.from_weights(randn(E, 2 * inner, H, g=g) * H ** -0.5, randn(E, H, inner, g=g) * inner ** -0.5)
    for T, k in ((3, 2), (40, 64), (700, 64)):
        ids = torch.randint(0, E, (T, k), generator=g, device="cuda") // 3 * 3
        x, w = randn(T, H, g=g, dtype=torch.bfloat16), torch.softmax(randn(T, k, g=g), -1)
        assert torch.equal(block(x, ids, w), block.by_operators(x, ids, w))
        pos, offsets = C.expert_sort(ids, E)
        want = order64(ids, E)
        assert torch.equal(pos, want[0]) and torch.equal(offsets, want[1])
        xq, xs = C.expert_gather_quant_int8(x, pos, offsets)
        y = C.w8a8_grouped_gemm(xq, xs, block.w13q, block.w13s, offsets, torch.float32)
        owner = ids.view(-1)[pos.view(-1).argsort()]                     # expert of each row
        want = torch.einsum("rk,rnk->rn", xq.double(), block.w13q[owner].double()) * xs.double()[:, None] * block.w13s[owner].double()
        within(y, want, want.abs() * 4 * U)


def test_grouped_refuse(C):
    xq, xs, wq, ws, offsets = grouped_case([3, 4], 0, 32, 64, gen(8))
    for args in ((xq, xs, wq, ws, offsets[:-1]), (xq, xs, wq[0], ws, offsets), (xq, xs, wq, ws[:, :-1], offsets),
                 (xq, xs[:-1], wq, ws, offsets), (xq, xs, wq, ws, offsets.long()), (xq[:, :48], xs, wq, ws, offsets),
                 (xq.cpu(), xs, wq, ws, offsets)):
        with pytest.raises(RuntimeError):
            C.w8a8_grouped_gemm(*args)
        with pytest.raises(RuntimeError):
            C.w8a8_grouped_gated(*args)
    with pytest.raises(RuntimeError):
        C.w8a8_grouped_gated(xq, xs, wq[:, :31].contiguous(), ws[:, :31].contiguous(), offsets)


FFN_CASES = [(1, 64, 32, 4, 2, 0.0), (1, 2048, 1024, 64, 8, 0.0), (7, 272, 80, 5, 3, 0.3), (48, 512, 704, 32, 4, 0.0), (300, 1024, 512, 8, 2, 0.1),
             (1200, 512, 272, 16, 6, 0.05), (2, 128, 64, 4, 1, 1.0),
             (2100, 1024, 64, 8, 8, 0.02)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,inner,E,k,drop", FFN_CASES)
def test_expert_block(C, T, H, inner, E, k, drop, dtype):
    """One call against the composition of the operators, bit for bit, and the composition's last two steps against 64 bits."""
    from wush_int4_kernel_b200.experts import ExpertRoute, W8A8Experts
    g = gen(T + H + inner)
    block = W8A8Experts.from_weights(randn(E, 2 * inner, H, g=g, dtype=dtype) * H ** -0.5, randn(E, H, inner, g=g, dtype=dtype) * inner ** -0.5)
    x, ids = randn(T, H, g=g, dtype=dtype), ids_of(T, k, E, g, drop=drop)
    w = torch.softmax(randn(T, k, g=g), -1)
    y = block(x, ids, w)
    assert y.shape == (T, H) and y.dtype == dtype
    assert torch.equal(y, block.by_operators(x, ids, w))
    assert torch.equal(block(x.view(T, 1, H), ids.view(T, 1, k), w.view(T, 1, k)), y.view(T, 1, H))
    assert torch.equal(block(x, ids.int(), w), y)
    # against 64 bits, with the codes of h taken from the operators (a code of h may differ at a tie of the grid)
    route = ExpertRoute.sort(ids, E)
    xq, xs = route.gather_quant_int8(x)
    h = C.w8a8_grouped_gated(xq, xs, block.w13q, block.w13s, route.offsets)
    hq, hs = C.quant_int8(h)
    o64 = torch.zeros(T * k, H, device="cuda", dtype=torch.float64)
    at = route.offsets.tolist()
    for i in range(E):
        o64[at[i]:at[i + 1]] = product64(hq[at[i]:at[i + 1]], hs[at[i]:at[i + 1]], block.w2q[i], block.w2s[i])
    terms = torch.where(route.pos.unsqueeze(-1) >= 0, o64[route.pos.clamp(min=0).long()] * w.double().unsqueeze(-1), 0.0)
    rounded = e(dtype) if 4 * T * k * H > 64 << 20 else 0.0               # the outputs of the experts, where they leave fp32
    bound = terms.abs().sum(1) * (rounded + (k + 4) * U) + terms.sum(1).abs() * e(dtype) * 1.01 + TINY16 * (k + 1)
    within(y, terms.sum(1), bound)


def test_same_expert_twice_and_no_token(C):
    """A token that names one expert several times counts as often; a block without tokens has no rows."""
    from wush_int4_kernel_b200.experts import ExpertRoute, W8A8Experts
    g = gen(21)
    E, H, inner, T = 4, 64, 32, 50
    block = W8A8Experts.from_weights(randn(E, 2 * inner, H, g=g) * H ** -0.5, randn(E, H, inner, g=g) * inner ** -0.5)
    x = randn(T, H, g=g, dtype=torch.bfloat16)
    ids = torch.randint(0, E, (T, 1), generator=g, device="cuda").expand(T, 3)
    w = torch.rand(T, 3, generator=g, device="cuda")
    y, once = block(x, ids, w), block(x, ids[:, :1], w.sum(1, keepdim=True))
    # the same term three times, summed in fp32 in three steps or one, then one rounding each
    assert ((y.double() - once.double()).abs() <= once.double().abs() * (2 * e(torch.bfloat16) + 8 * U) + 1e-30).all()
    route = ExpertRoute.sort(ids, E)
    assert torch.equal(route.pos.sort(dim=0)[0].view(-1).sort()[0], torch.arange(3 * T, device="cuda", dtype=torch.int32))
    none = block(x[:0], ids[:0], w[:0])
    assert none.shape == (0, H) and none.dtype == torch.bfloat16
    wide = randn(T, 2 * H, g=g, dtype=torch.bfloat16)[:, :H]               # rows with a stride: copied
    assert torch.equal(block(wide, ids, w), block(wide.contiguous(), ids, w))


def test_blocks_one_after_another(C):
    """Calls that follow each other without a pause on the same workspace addresses, each on data of its own."""
    from wush_int4_kernel_b200.experts import W8A8Experts
    g = gen(41)
    E, H, inner = 16, 1024, 528
    block = W8A8Experts.from_weights(randn(E, 2 * inner, H, g=g, dtype=torch.bfloat16) * H ** -0.5,
                                     randn(E, H, inner, g=g, dtype=torch.bfloat16) * inner ** -0.5)
    for T, k in ((2, 4), (60, 4), (300, 2), (900, 5)):
        sets = [(randn(T, H, g=g, dtype=torch.bfloat16), ids_of(T, k, E, g), torch.softmax(randn(T, k, g=g), -1)) for _ in range(12)]
        want = [block.by_operators(*s) for s in sets]
        torch.cuda.synchronize()
        got = [block(*s) for _ in range(3) for s in sets]
        for i, y in enumerate(got):
            assert torch.equal(y, want[i % len(sets)]), (T, k, i)


def test_a_large_block_in_a_graph(C):
    """The other kernels of the chain (sort in a cluster, CTA pairs, tiles cut along K) captured, replayed on new inputs."""
    from wush_int4_kernel_b200.experts import W8A8Experts
    g = gen(31)
    E, H, inner, T, k = 8, 512, 6160, 900, 4
    block = W8A8Experts.from_weights(randn(E, 2 * inner, H, g=g, dtype=torch.bfloat16) * H ** -0.5,
                                     randn(E, H, inner, g=g, dtype=torch.bfloat16) * inner ** -0.5)
    held = [randn(T, H, g=g, dtype=torch.float16), ids_of(T, k, E, g), torch.softmax(randn(T, k, g=g), -1)]
    block(*held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(*held)
    for seed in (1, 2):
        s = gen(seed)
        new = [randn(T, H, g=s, dtype=torch.float16), ids_of(T, k, E, s), torch.softmax(randn(T, k, g=s), -1)]
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, block(*new)) and torch.equal(out, block.by_operators(*new))


def test_a_step_of_a_block_with_both_widths(C):
    """As used together: a 4-bit projection, an 8-bit projection of its result, and the expert block, in one captured graph
    that is replayed on new inputs, beside a second graph and eager calls on another stream."""
    from wush_int4_kernel_b200 import synth
    from wush_int4_kernel_b200.experts import W8A8Experts
    from wush_int4_kernel_b200.linear import W4A4Linear, W8A8Linear
    g = gen(11)
    H, inner, E, k = 512, 256, 8, 2
    layer = synth.make_layer(H, H, seed=3, device="cuda", quantiser=C.quant_int4)
    four = W4A4Linear(layer.t_bf16, layer.wq, layer.ws)
    eight = W8A8Linear.from_weight(randn(H, H, g=g, dtype=torch.float16) * H ** -0.5)
    block = W8A8Experts.from_weights(randn(E, 2 * inner, H, g=g) * H ** -0.5, randn(E, H, inner, g=g) * inner ** -0.5)

    def step(x, ids, w):
        return block(eight(four(x)), ids, w)

    def inputs(T, seed):
        s = gen(seed)
        return [randn(T, H, g=s, dtype=torch.bfloat16), ids_of(T, k, E, s, drop=0.1), torch.softmax(randn(T, k, g=s), -1)]
    graphs = []
    for T in (3, 150):
        held = inputs(T, T)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*held)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*held)
        graphs.append((T, held, graph, out))
    other = torch.cuda.Stream()
    for seed in (21, 22, 23):
        wants = []
        for T, held, graph, out in graphs:
            new = inputs(T, seed + T)
            for a, b in zip(held, new):
                a.copy_(b)
            wants.append(step(*new))
        other.wait_stream(torch.cuda.current_stream())
        new = inputs(40, seed)
        torch.cuda.synchronize()
        want40 = step(*new)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            got40 = step(*new)
        for (T, held, graph, out), want in zip(graphs, wants):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got40, want40)
        for (T, held, graph, out), want in zip(graphs, wants):
            assert torch.equal(out, want)
