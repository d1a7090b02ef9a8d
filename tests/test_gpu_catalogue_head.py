"""The catalogue head (8-bit rows, their product, drawing an item, distillation) against plain 64-bit forms on the CPU."""
import math

import numpy as np
import pytest
import torch

import star_gcn_amd._lib as L
from star_gcn_amd import functional as SF
from star_gcn_amd import ops
from star_gcn_amd.recommend import CatalogueHead

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- rows to codes -----------------------------------------------------------------------------------------------------


def quant_reference(h, w, norm, eps):
    y = h.double()
    if norm:
        y = y / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double()
    scale = (y.abs().amax(1) / 127).float()
    bad = ~torch.isfinite(y).all(1) | ~torch.isfinite(scale)
    s = scale.double()[:, None]
    codes = torch.where(s > 0, (y / s).round().clamp(-127, 127), torch.zeros_like(y))
    codes[bad] = 0
    scale[bad] = math.nan
    return codes.to(torch.int8), scale


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_more_rows_than_one_launch_takes(dtype):
    rows = (1 << 21) + 70
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(rows, 6, generator=g, device=DEV).to(dtype)[:, :5]
    r = torch.randn(rows, 7, generator=g, device=DEV).to(dtype)[:, 2:]
    w = torch.rand(5, generator=g, device=DEV).to(dtype)
    codes, scale, h = ops.rms_norm_i8(x, w, residual=r)
    assert torch.equal(h, x + r)
    for cut in (slice(0, 64), slice((1 << 21) - 64, (1 << 21) + 64), slice(rows - 70, rows)):
        check_codes((codes[cut], scale[cut]), quant_reference(h[cut].cpu(), w.cpu(), True, 1e-6))


def check_codes(got, want):
    # both sides decide in 64 bits: a code differs only where the quotient lies within ~1e-13 of a tie, and the scale only
    # where the 64-bit value lies that near to the middle of two fp32 numbers; none does in these fixed inputs
    assert torch.equal(got[0].cpu(), want[0])
    assert torch.equal(got[1].cpu().nan_to_num(-1.0), want[1].nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 3, 7, 64, 75, 250, 256, 257, 511, 513, 1000, 1025, 2049, 4097, 8200, 16384])
def test_rms_norm_codes(dtype, dim):
    g = gen(dim)
    for rows in (1, 5, 130):
        x, r = (torch.randn(rows, dim, generator=g).to(dtype) for _ in range(2))
        w = (1 + 0.3 * torch.randn(dim, generator=g))
        h = (x.double() + r.double()).to(dtype)
        for weight in (w.to(dtype), w, None):
            codes, scale, hh = ops.rms_norm_i8(x.to(DEV), None if weight is None else weight.to(DEV), residual=r.to(DEV))
            assert torch.equal(hh.cpu(), h)
            check_codes((codes, scale), quant_reference(h, weight, True, 1e-6))
        xd = x.to(DEV)
        codes, scale, hh = ops.rms_norm_i8(xd, w.to(DEV), eps=0.5)
        assert hh.data_ptr() == xd.data_ptr()
        check_codes((codes, scale), quant_reference(x, w, True, 0.5))
        check_codes(ops.quantize_rows(xd), quant_reference(x, None, False, 0.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_strided_rows_and_slices(dtype):
    big = torch.randn(40, 300, generator=gen(3)).to(dtype).to(DEV)
    for x in (big[:, :77], big[:, 5:82], big[::3, 1:], big[:7].t(), big[:1].expand(4, 300)):
        check_codes(ops.quantize_rows(x), quant_reference(x.cpu(), None, False, 0.0))
    r = big[3:, 100:177]
    codes, scale, h = ops.rms_norm_i8(big[:37, :77], None, residual=r)
    assert torch.equal(h, (big[:37, :77].float() + r.float()).to(dtype))
    check_codes((codes, scale), quant_reference(h.cpu(), None, True, 1e-6))


def test_codes_of_ties_zeros_and_extreme_rows():
    k = torch.arange(-127, 127).float() + 0.5
    rows = [torch.cat([s * k, torch.tensor([127.0 * s])]) for s in (1.0, 3.0, 5.0, 0.375, 7 * 2.0 ** -60, 2.0 ** 100, 11 * 2.0 ** -140)]
    x = torch.stack(rows + [torch.zeros(255), torch.full((255,), 3.4028234663852886e38), torch.full((255,), 1e-45)])
    check_codes(ops.quantize_rows(x.to(DEV)), quant_reference(x, None, False, 0.0))
    check_codes(ops.rms_norm_i8(x.to(DEV))[:2], quant_reference(x, None, True, 1e-6))
    assert ops.quantize_rows(x.to(DEV))[1][7].item() == 0.0


def test_zeros_have_scale_zero_whatever_eps():
    x = torch.zeros(3, 100, device=DEV)
    x[1] = 2.0
    codes, scale, _ = ops.rms_norm_i8(x, eps=0.0)
    assert scale.tolist() == [0.0, float(np.float32(1.0 / 127)), 0.0] and (codes[1] == 127).all() and (codes[::2] == 0).all()


def test_the_sum_may_replace_the_residual():
    x, r = (torch.randn(70, 300, generator=gen(k)).to(DEV) for k in (1, 2))
    want = ops.rms_norm_i8(x, None, residual=r)
    codes, scale = torch.empty(70, 300, dtype=torch.int8, device=DEV), torch.empty(70, device=DEV)
    args = lambda ldr: (L.ptr(codes), L.ptr(scale), L.ptr(r), L.ptr(x), 300, L.ptr(r), ldr, None, 0, 70, 300, 0, 1, 1e-6, L.stream_ptr())      # noqa: E731
    assert L.lib().sg_quant_rows_i8_hip(*args(301)) == -1      # rows with gaps cannot be replaced by a sum without
    L.check(L.lib().sg_quant_rows_i8_hip(*args(300)))
    assert torch.equal(r, want[2]) and torch.equal(codes, want[0]) and torch.equal(scale, want[1])


@pytest.mark.parametrize("norm", [False, True])
def test_a_row_that_is_not_finite_has_no_codes_and_harms_no_other(norm):
    x = torch.randn(9, 333, generator=gen(1))
    x[1, 5], x[3, 332], x[5, 0] = INF, -INF, math.nan
    got = ops.rms_norm_i8(x.to(DEV))[:2] if norm else ops.quantize_rows(x.to(DEV))
    check_codes(got, quant_reference(x, None, norm, 1e-6))
    assert got[1].isnan().nonzero().flatten().tolist() == [1, 3, 5]
    out = ops.gemm_i8(*got, *ops.quantize_rows(torch.randn(20, 333, generator=gen(2)).to(DEV)))
    assert out.isnan().any(1).nonzero().flatten().tolist() == [1, 3, 5] and out[1].isnan().all()


# ---- the product ---------------------------------------------------------------------------------------------------------

ACTS = {None: lambda v: v, "leaky": lambda v: torch.where(v > 0, v, 0.2 * v), "relu": torch.relu, "sigmoid": torch.sigmoid,
        "tanh": torch.tanh}


def check_product(a, sa, b, sb, bias, act, out):
    exact = a.double() @ b.double().t()
    t = exact * sa.double()[:, None] * sb.double()
    v = t if bias is None else t + bias.double()
    ref = ACTS[act](v)
    # the sum to fp32, its products with the two scales (the second fused with the bias): three roundings of half a step each;
    # the activations' slopes are at most 1 and sigmoid / tanh themselves are good to 4 steps; then one rounding to the type
    tol = 2.0 ** -24 * (2 * t.abs() + v.abs()) * 1.01 + (8 * 2.0 ** -24 * ref.abs() + 2.0 ** -24 if act in ("sigmoid", "tanh") else 2.0 ** -24 * ref.abs())
    fi = torch.finfo(out.dtype)
    tol = tol + (fi.eps / 2 * ref.abs() + fi.smallest_normal * fi.eps if out.dtype != torch.float32 else 0)
    err = (out.double().to(ref.device) - ref).abs()
    assert (err <= tol * 1.01 + 1e-45).all(), float((err - tol).max())


def codes(rows, k, g, hi=128):
    return torch.randint(-128, hi, (rows, k), generator=g, dtype=torch.int8 if hi < 128 else torch.int16).to(torch.int8)


def product_case(M, N, K, dtype=torch.float32, bias=True, act=None, seed=0):
    g = gen(seed + M * 1000003 + N * 1009 + K)
    a, b = codes(M, K, g), codes(N, K, g)
    sa, sb = torch.rand(M, generator=g) + 0.1, torch.rand(N, generator=g) * 0.01
    bi = torch.randn(N, generator=g) if bias else None
    out = ops.gemm_i8(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV), bias=None if bi is None else bi.to(DEV), act=act, slope=0.2,
                      out_dtype=dtype)
    assert out.dtype == dtype and out.shape == (M, N)
    check_product(a, sa, b, sb, bi, act, out)


@pytest.mark.parametrize("M", [1, 2, 3, 5, 17, 31, 32, 33, 64, 65, 127, 128, 129, 257, 300])
@pytest.mark.parametrize("N", [1, 31, 129, 1000])
def test_product_of_odd_sizes(M, N):
    for K in (1, 15, 16, 17, 63, 64, 65, 128, 250, 256, 272):
        product_case(M, N, K, bias=K % 2 == 0)


@pytest.mark.parametrize("M,N,K", [(1, 5, 8192), (1, 10677, 256), (4, 3, 131071), (7, 300, 5000), (40, 130, 4096), (200, 70, 20000),
                                   (513, 515, 1024), (1, 1, 131071), (300, 2500, 4100), (1025, 1030, 2048)])
def test_product_of_long_rows_and_few(M, N, K):
    product_case(M, N, K)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", list(ACTS))
def test_product_types_and_activations(dtype, act):
    for M, N, K in ((3, 50, 64), (130, 200, 250), (260, 520, 1024)):
        product_case(M, N, K, dtype=dtype, act=act)


@pytest.mark.parametrize("M,N", [(2000, 2050), (2049, 4099), (4000, 4100)])      # 128 x 128, 128 x 256 and 256 x 256 tiles
@pytest.mark.parametrize("K", [64, 200, 250, 256, 512, 528, 600, 640, 1040])
def test_product_of_large_matrices(M, N, K):
    g = torch.Generator(device=DEV).manual_seed(K)
    a, b = (torch.randint(-128, 128, (n, K), generator=g, device=DEV, dtype=torch.int16).to(torch.int8) for n in (M, N))
    sa, sb, bias = (torch.rand(n, generator=g, device=DEV) + 0.1 for n in (M, N, N))
    for dtype, act in ((torch.float32, None), (torch.bfloat16, None), (torch.float16, "tanh")):
        s = 1.0 if dtype != torch.float16 else 1e-5
        out = ops.gemm_i8(a, sa * s, b, sb, bias=bias, act=act, slope=0.2, out_dtype=dtype)
        check_product(a, sa * s, b, sb, bias, act, out)
    wide = torch.zeros(M, N + 9, device=DEV)
    ops.gemm_i8(a, sa, b, sb, out=wide[:, 4:N + 4])
    check_product(a, sa, b, sb, None, None, wide[:, 4:N + 4])
    assert (wide[:, :4] == 0).all() and (wide[:, N + 4:] == 0).all()


def test_product_larger_than_the_infinity_cache():
    g = torch.Generator(device=DEV).manual_seed(1)
    a, b = (torch.randint(-128, 128, (n, 96), generator=g, device=DEV, dtype=torch.int16).to(torch.int8) for n in (8200, 8208))
    sa, sb = (torch.rand(n, generator=g, device=DEV) for n in (8200, 8208))
    out = ops.gemm_i8(a, sa, b, sb)
    for rows in (slice(0, 300), slice(4000, 4300), slice(7950, 8200)):
        check_product(a[rows], sa[rows], b, sb, None, None, out[rows])


def test_product_at_the_integers_limit():
    for K in (131071,):
        a = torch.full((2, K), -128, dtype=torch.int8, device=DEV)
        one = torch.ones(2, device=DEV)
        out = ops.gemm_i8(a, one, a, one)
        assert (out.double() == float(np.float32(128 * 128 * K))).all()


def test_product_of_nothing():
    z = lambda *s: torch.zeros(*s, dtype=torch.int8, device=DEV)      # noqa: E731
    v = lambda n: torch.ones(n, device=DEV)      # noqa: E731
    assert ops.gemm_i8(z(0, 8), v(0), z(3, 8), v(3)).shape == (0, 3)
    assert ops.gemm_i8(z(3, 8), v(3), z(0, 8), v(0)).shape == (3, 0)
    bias = torch.tensor([-1.0, 2.0], device=DEV)
    assert ops.gemm_i8(z(3, 0), v(3), z(2, 0), v(2), bias=bias, act="relu").tolist() == [[0.0, 2.0]] * 3


@pytest.mark.parametrize("off", [0, 1, 16, 24])
@pytest.mark.parametrize("M", [2, 40, 200])
def test_product_of_strided_operands_into_a_slice(off, M):
    g = gen(off)
    A, B = codes(M, 600, g).to(DEV), codes(150, 608, g).to(DEV)
    a, b = A[:, off:off + 320], B[:, off:off + 320]
    sa, sb = torch.rand(M, generator=g), torch.rand(150, generator=g)
    wide = torch.full((M + 1, 200), 7.0, device=DEV)
    out = ops.gemm_i8(a, sa.to(DEV), b, sb.to(DEV), out=wide[:M, 20:170])
    assert out.data_ptr() == wide[:, 20:].data_ptr()
    check_product(a.cpu(), sa, b.cpu(), sb, None, None, out)
    assert (wide[:, :20] == 7).all() and (wide[:, 170:] == 7).all() and (wide[M] == 7).all()
    t = ops.gemm_i8(A[:, ::2], sa.to(DEV), B[:, :600:2], sb.to(DEV))
    check_product(A[:, ::2].cpu(), sa, B[:, :600:2].cpu(), sb, None, None, t)


def test_product_is_the_same_however_the_rows_are_batched():
    g = gen(11)
    a, b = codes(300, 4096, g).to(DEV), codes(257, 4096, g).to(DEV)
    sa, sb = torch.rand(300, generator=g).to(DEV), torch.rand(257, generator=g).to(DEV)
    whole = ops.gemm_i8(a, sa, b, sb)
    for m in (1, 2, 8, 33, 129):
        assert torch.equal(ops.gemm_i8(a[:m], sa[:m], b, sb), whole[:m])


# ---- drawing -------------------------------------------------------------------------------------------------------------


def draw_reference(l, u, T=1.0, k=0, p=1.0, m=0.0):
    """One row in 64 bits -> (id, prob, how near u comes to the border of another item)."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    if l.size == 0 or l.max() == -np.inf:
        return -1, 0.0, 1.0
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        w = np.where(l == l.max(), 1.0, np.exp((l - l.max()) / T) if T > 0 else 0.0)
    order = np.argsort(-l, kind="stable")
    order = order[l[order] > -np.inf]
    if not T > 0 or not p > 0 or not m <= 1:
        order = order[:1]
    if 0 < k < order.size:
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        order = order[:int(np.searchsorted(c, p * c[-1], side="left")) + 1]
    if m <= 1:
        order = order[w[order] >= m]
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    at = min(int(np.searchsorted(c, u * c[-1], side="right")), kept.size - 1)
    near = np.abs(c / c[-1] - u).min()
    return int(kept[at]), float(w[kept[at]] / c[-1]), near


def check_draw(l, u, **kw):
    par = {k: (v.to(DEV) if torch.is_tensor(v) else v) for k, v in kw.items()}
    ids, prob = ops.sample_rows(l if l.is_cuda else l.to(DEV), u.to(DEV), **par)
    assert ids.dtype == torch.int32 and prob.dtype == torch.float32
    ids, prob = ids.cpu().numpy(), prob.cpu().numpy()
    names = {"temperature": "T", "top_k": "k", "top_p": "p", "min_p": "m"}
    for i, row in enumerate(l.float().cpu().numpy()):
        par = {names[k]: (v[i].item() if torch.is_tensor(v) else v) for k, v in kw.items()}
        want, wp, near = draw_reference(row, float(u[i]), **par)
        assert ids[i] == want or near < 1e-12, (i, ids[i], want, wp, near)
        if ids[i] == want:
            # a weight is within half of 2^-s, s = min(51, 62 - log2 n), and 1e-14 of its value; one rounding to fp32
            assert abs(prob[i] - wp) <= wp * (2.0 ** -24 + 1e-13) + 2.0 ** -38, (i, prob[i], wp)


SETTINGS = [dict(), dict(temperature=0.5), dict(top_k=1), dict(top_k=7), dict(top_k=1000000), dict(top_p=0.9), dict(top_p=0.3, temperature=2.0),
            dict(min_p=0.1), dict(top_k=50, top_p=0.8), dict(top_k=40, top_p=0.95, min_p=0.05, temperature=0.7), dict(temperature=0.0),
            dict(top_p=0.0), dict(min_p=1.0), dict(min_p=1.5), dict(temperature=50.0, top_p=0.999), dict(temperature=0.01)]


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 255, 1000, 1682, 4097, 10677, 16385, 70000])
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_draw(n, kw):
    g = gen(n)
    for dtype in DTYPES:
        l = (2.0 * torch.randn(6, n, generator=g)).to(dtype)
        l[torch.rand(6, n, generator=g) < 0.05] = -INF
        u = torch.rand(6, generator=g)
        u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
        check_draw(l, u, **kw)


@pytest.mark.parametrize("kw", [dict(top_k=5), dict(top_p=0.5), dict(top_k=100, top_p=0.77), dict(top_k=300, top_p=0.4, min_p=0.2), dict()], ids=str)
@pytest.mark.parametrize("n", [9, 700, 5000, 40000])
def test_draw_among_equal_scores(kw, n):
    g = gen(n)
    rows = [torch.zeros(n), torch.full((n,), -3.4028234663852886e38), torch.randint(0, 3, (n,), generator=g).float(),
            torch.where(torch.rand(n, generator=g) < 0.5, 0.0, -0.0), torch.arange(n).float() % 2, -(torch.arange(n) // 7).float() * 0.01]
    for u in (0.0, 0.37, 0.99):
        check_draw(torch.stack(rows), torch.full((len(rows),), u), **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.2, top_k=9, top_p=0.9)], ids=str)
@pytest.mark.parametrize("n", [5, 300, 20000])
def test_draw_of_masked_infinite_and_nan_rows(kw, n):
    low = -3.4028234663852886e38
    l = torch.randn(8, n, generator=gen(n))
    l[0] = -INF                                            # nothing left
    l[1, :] = -INF
    l[1, n - 1] = -50.0                                    # one item left
    l[2, ::2] = low                                        # the type's lowest value as a mask
    l[3] = math.nan
    l[4, 1::2] = math.nan
    l[5, 2] = INF                                          # the only possible item
    l[6, 1] = l[6, 4] = INF
    l[7] = l[7] * 1e-42
    check_draw(l, torch.tensor([0.3, 0.9, 0.5, 0.1, 0.99, 0.4, 0.7, 0.2]), **kw)
    ids, prob = ops.sample_rows(l.to(DEV), torch.full((8,), 0.5, device=DEV), **kw)
    assert ids[0].item() == ids[3].item() == -1 and prob[0].item() == prob[3].item() == 0.0 and ids[1].item() == n - 1


def test_draw_with_settings_of_each_row():
    g = gen(5)
    l = 3 * torch.randn(32, 3000, generator=g)
    check_draw(l, torch.rand(32, generator=g), temperature=torch.linspace(0.0, 2.0, 32), top_k=torch.arange(32, dtype=torch.int32) * 5 - 5,
               top_p=torch.linspace(0.2, 1.2, 32), min_p=torch.linspace(0.0, 1.1, 32))
    check_draw(l, torch.rand(32, generator=g), top_k=torch.arange(32))


@pytest.mark.parametrize("n", [300, 40000])
def test_draw_at_extreme_temperatures(n):
    l = torch.randn(4, n, generator=gen(n))
    l[1, 5] = INF
    l[2] *= 1e38
    l[3] *= 1e-38
    u = torch.tensor([0.2, 0.4, 0.6, 0.8])
    for T in (5e-324, 1e-320, 1e-300, 1e-45, 1e30, 1e300):
        for kw in (dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.5, top_k=50, top_p=0.5)):
            check_draw(l, u, temperature=T, **kw)
    check_draw(l, u, temperature=torch.tensor([1e-45, 1e-40, 3e38, 1e-10]), top_p=0.9)
    # every finite score alike, unless an infinite one (row 1's, and where 1e38 overflows row 2's) leaves the others nothing
    ids, prob = ops.sample_rows(l.to(DEV), u.to(DEV), temperature=INF)
    for i, row in enumerate(l):
        alike = ((row == INF) if (row == INF).any() else row > -INF).nonzero().flatten()
        assert ids[i].item() == alike[int(alike.numel() * float(u[i]))] and abs(prob[i].item() * alike.numel() - 1) < 1e-6


def test_draw_with_settings_on_the_device():
    l, u = torch.randn(5, 400, generator=gen(1)), torch.rand(5, generator=gen(2))
    want = ops.sample_rows(l.to(DEV), u.to(DEV), temperature=0.5, top_k=30, top_p=0.75)
    one = lambda v, t: torch.tensor(v, dtype=t, device=DEV)      # noqa: E731
    got = ops.sample_rows(l.to(DEV), u.to(DEV), temperature=one(0.5, torch.float64), top_k=one(30, torch.int64), top_p=one(0.75, torch.float16))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    many = ops.sample_rows(l.to(DEV), u.to(DEV), top_k=torch.full((5,), (1 << 32) + 1, device=DEV))
    assert torch.equal(many[0], ops.sample_rows(l.to(DEV), u.to(DEV))[0])
    assert torch.equal(ops.sample_rows(l.to(DEV), u.to(DEV), top_k=1 << 40)[0], many[0])


def test_draw_from_slices_and_transposed_scores():
    big = (2 * torch.randn(20, 5003, generator=gen(9))).to(DEV)
    u = torch.rand(20, generator=gen(10))
    check_draw(big[:, 3:], u, top_p=0.9)
    check_draw(big[::2, 1:4000], u[:10], top_k=20)
    check_draw(big[:, :20].t(), u, top_k=4)
    check_draw(big.half()[:, 1:4002], u, top_k=20, top_p=0.5)
    assert ops.sample_rows(big[:, :0], u.to(DEV))[0].tolist() == [-1] * 20
    assert ops.sample_rows(big[:0], u[:0].to(DEV))[0].shape == (0,)


@pytest.mark.parametrize("rows,n", [(1, 1000003), (3, 300000), (70, 100001), (300, 20001)])
def test_draw_from_long_rows(rows, n):
    g = gen(n)
    l = 2 * torch.randn(rows, n, generator=g) - torch.rand(n, generator=g).log()
    l[torch.rand(rows, n, generator=g) < 0.02] = -INF
    l[-1] = torch.randint(0, 50, (n,), generator=g).float() * 0.1
    u = torch.rand(rows, generator=g)
    for kw in (dict(), dict(top_p=0.95), dict(top_k=500), dict(top_k=20000, top_p=0.7, min_p=1e-3), dict(min_p=0.01)):
        check_draw(l, u, **kw)


@pytest.mark.parametrize("n", [8191, 12289, 16383, 16384])
def test_draw_from_the_longest_rows_of_one_workgroup(n):
    g = gen(n)
    for dtype in DTYPES:
        l = (2 * torch.randn(3, n, generator=g)).to(dtype)
        for kw in (dict(), dict(top_k=900, top_p=0.9), dict(top_p=0.999)):
            check_draw(l, torch.rand(3, generator=g), **kw)


def test_draw_from_more_rows_than_one_launch_takes():
    rows = (1 << 22) + 40
    g = torch.Generator(device=DEV).manual_seed(6)
    logits = torch.randn(rows, 4, generator=g, device=DEV)[:, :3]
    u, t, p, m = (torch.rand(rows, generator=g, device=DEV) for _ in range(4))
    k = torch.randint(0, 4, (rows,), generator=g, device=DEV)
    ids, prob = ops.sample_rows(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    for cut in (slice(0, 64), slice((1 << 22) - 64, (1 << 22) + 40)):
        i, q = ops.sample_rows(logits[cut], u[cut], temperature=t[cut], top_k=k[cut], top_p=p[cut], min_p=m[cut])
        assert torch.equal(ids[cut], i) and torch.equal(prob[cut], q)
    assert ((ids >= 0) & (ids < 3)).all()


def test_draws_follow_the_kept_distribution():
    l = torch.tensor([0.0, 1.0, 2.0, -1.0, 1.5], device=DEV)
    n = 200000
    u = (torch.arange(n, device=DEV) + 0.5) / n
    ids, prob = ops.sample_rows(l.expand(n, 5), u.float(), top_k=3)
    p = torch.softmax(l[[1, 2, 4]].double(), 0).cpu()
    for item, want in zip((1, 2, 4), p):
        assert abs((ids == item).double().mean().item() - want) < 2e-5      # u is a grid of steps of 5e-6
        assert abs(prob[ids == item][0].item() - want) < 1e-6
    assert not ((ids == 0) | (ids == 3)).any()


# ---- distillation ------------------------------------------------------------------------------------------------------


def distill_reference(s, t, ids, scale, T):
    """-> (loss, gradient, q + p): the gradient is the difference of q and p, times scale * T."""
    s = s.double().detach().requires_grad_(True)
    n = s.shape[1]
    terms, size = [], torch.zeros(s.shape, dtype=torch.float64)
    for r in range(s.shape[0]):
        keep = (ids[r] >= 0) & (ids[r] < n) & (t[r] > -INF)
        if not keep.any() or not (s[r] > -INF).any():
            continue
        p = torch.softmax(t[r][keep].double() / T, 0)
        live = p > 0
        log_q = torch.log_softmax(s[r] / T, 0)
        size[r] = log_q.detach().exp().index_add(0, ids[r][keep].long(), p)
        log_q = log_q[ids[r][keep].long()]
        terms.append((p[live] * (p[live].log() - log_q[live])).sum())
    loss = scale * T * T * torch.stack(terms).sum() if terms else s.sum() * 0
    if not terms:
        return torch.tensor(0.0, dtype=torch.float64), torch.zeros_like(s), size
    loss.backward()
    return loss.detach(), s.grad, size


def check_distill(s, t, ids, scale=0.25, T=2.0, up=1.5):
    x = (s if s.is_cuda else s.to(DEV)).detach().requires_grad_(True)
    loss = SF.distill_loss(x, t.to(DEV), ids.to(DEV), scale, temperature=T)
    grad, = torch.autograd.grad(loss * up, x)
    want, wg, size = distill_reference(s.cpu(), t.cpu(), ids.cpu(), scale, T)
    rows = s.shape[0]
    # log of an fp32 sum of exps (each good to 2e-6 where it matters: an exponent of up to ~30 rounded to fp32), a row's total
    # share is 1; then one rounding of each row's loss and of the sum
    if torch.isfinite(want):
        assert abs(loss.item() - want.item()) <= 3e-6 * scale * T * T * rows + 2.0 ** -22 * abs(want.item()), (loss.item(), want.item())
    else:
        assert loss.item() == want.item()
    f, fi = scale * T * up, torch.finfo(s.dtype)
    # q = exp2(d c) / sum: d exact to 2^-24, c and d c rounded, |d c| <= 40 where q matters: 40 * 2 * 2^-24 * ln 2 = 3.3e-6 of q,
    # the sum as much again at worst, v_exp_f32 and the products 5 * 2^-24: 7e-6 of q; p 2^-22 of p.  q - p cancels where the
    # student is close, so the bound is on q + p and not on the difference; then the type's rounding
    tol = f * (7e-6 * size + 2.0 ** -120) + fi.eps / 2 * (wg * up).abs() + fi.smallest_normal * fi.eps
    err = (grad.double().cpu() - wg * up).abs()
    assert grad.dtype == s.dtype and (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 63, 250, 1024, 1682, 4099, 10677, 40001])
def test_distill_value_and_gradient(dtype, n):
    g = gen(n)
    for rows, k in ((1, 1), (5, min(n, 10)), (3, min(n, 300))):
        s = (2 * torch.randn(rows, n, generator=g)).to(dtype)
        t = 3 * torch.randn(rows, k, generator=g)
        ids = torch.stack([torch.randperm(n, generator=g)[:k] for _ in range(rows)]).int()
        for T in (1.0, 3.5):
            check_distill(s, t, ids, T=T)


@pytest.mark.parametrize("rows,n", [(2, 1000001), (300, 9000), (40, 100000)])
def test_distill_of_long_rows(rows, n):
    g = gen(n)
    s = 2 * torch.randn(rows, n, generator=g)
    v, i = (s + torch.randn(rows, n, generator=g)).topk(64, dim=1)
    check_distill(s, v, i.int(), T=1.0)


@pytest.mark.parametrize("rows,n,dtype", [(34, 1000003, torch.float32), (900, 90001, torch.bfloat16), (520, 65536, torch.float32)])
def test_distill_of_gradients_larger_than_the_cache(rows, n, dtype):
    g = torch.Generator(device=DEV).manual_seed(n)
    s = (2 * torch.randn(rows, n, generator=g, device=DEV)).to(dtype)
    t = torch.randn(rows, 20, generator=g, device=DEV)
    ids = torch.randint(0, n, (rows, 20), generator=g, device=DEV)
    x = s.requires_grad_(True)
    loss = SF.distill_loss(x, t, ids, 1.0 / rows, temperature=1.5)
    grad, = torch.autograd.grad(loss, x)
    f, fi = 1.5 / rows, torch.finfo(dtype)
    for r in range(0, rows, 7):
        q = torch.softmax(s[r].detach().double() / 1.5, 0)
        p = torch.zeros_like(q).index_add_(0, ids[r], torch.softmax(t[r].double() / 1.5, 0))
        want = f * (q - p)
        # the bound of check_distill
        assert ((grad[r].double() - want).abs() <= f * 7e-6 * (q + p) + fi.eps / 2 * want.abs() + fi.smallest_normal * fi.eps).all(), r


def test_distill_gradient_against_differences():
    g = gen(2)
    s = torch.randn(1, 40, generator=g).to(DEV)
    t, ids = torch.randn(1, 6, generator=g).to(DEV), torch.tensor([[3, 9, 0, 39, 17, 20]], dtype=torch.int32, device=DEV)
    x = s.clone().requires_grad_(True)
    SF.distill_loss(x, t, ids, 1.0).backward()
    h = 0.05
    for j in (0, 3, 5, 20, 39):
        d = torch.zeros_like(s)
        d[0, j] = h
        diff = (SF.distill_loss(s + d, t, ids, 1.0).item() - SF.distill_loss(s - d, t, ids, 1.0).item()) / (2 * h)
        # the loss is good to 4e-6 (the test above) on either side; its third derivative, a cumulant of an indicator, is below 0.1
        assert abs(diff - x.grad[0, j].item()) <= 4e-6 / h + 0.1 * h * h / 6


def test_distill_of_padding_masks_and_items_named_twice():
    g = gen(4)
    s = torch.randn(9, 500, generator=g)
    t = torch.randn(9, 12, generator=g)
    ids = torch.stack([torch.randperm(500, generator=g)[:12] for _ in range(9)]).int()
    ids[0, 3:] = -1
    ids[1] = -1                                            # nothing to fit
    t[2] = -INF                                            # nothing to fit
    t[3, 5:] = -INF
    s[4] = -INF                                            # nothing to fit it with
    ids[5, 4] = ids[5, 0]
    ids[5, 7] = ids[5, 0]
    ids[6] = ids[6, 0]                                     # one item, named 12 times
    ids[7, 2], ids[7, 9] = 500, 2147483647                 # out of range: padding
    s[8, :100] = -INF
    ids[8] = torch.arange(200, 212)
    check_distill(s, t, ids)
    far = ids.long()
    far[0, 5], far[7, 2] = (1 << 32) + 7, -(1 << 40)       # no item, in 64 bits either
    check_distill(s, t, far)
    x = s.to(DEV).requires_grad_(True)
    loss = SF.distill_loss(x, t.to(DEV), ids.to(DEV), 1.0)
    loss.backward()
    assert torch.isfinite(loss) and (x.grad[[1, 2, 4]] == 0).all() and torch.isfinite(x.grad).all()
    low = s.clone()
    low[8, :100] = -3.4028234663852886e38
    low[4] = -3.4028234663852886e38
    check_distill(low, t, ids)
    only = SF.distill_loss(x[1:3], t[1:3].to(DEV), ids[1:3].to(DEV), 1.0)
    assert only.item() == 0.0
    masked = s[:1].clone()
    masked[0, ids[0, 1].long()] = -INF                     # the teacher wants what the student may not give
    assert SF.distill_loss(masked.to(DEV), t[:1].to(DEV), ids[:1].to(DEV), 1.0).item() == INF


def test_distill_passes_nan_on_and_keeps_it_to_its_row():
    s, t = torch.randn(3, 50, generator=gen(8)), torch.randn(3, 4, generator=gen(9))
    s[1, 7] = math.nan
    ids = torch.arange(12, dtype=torch.int32).view(3, 4)
    x = s.to(DEV).requires_grad_(True)
    loss = SF.distill_loss(x, t.to(DEV), ids.to(DEV), 1.0)
    loss.backward()
    assert loss.isnan() and x.grad[1].isnan().all() and torch.isfinite(x.grad[[0, 2]]).all()


def test_distill_of_slices_and_of_no_rows():
    big = torch.randn(30, 700, generator=gen(6)).to(DEV)
    t, ids = torch.randn(10, 5, generator=gen(7)), torch.arange(50, dtype=torch.int64).view(10, 5)
    check_distill(big[::3, 11:411], t, ids)
    check_distill(big.bfloat16()[:10, 1:78], t, ids)
    check_distill(big[:60, :10].t()[:10, :], t, ids % 30)
    x = big[:0].clone().requires_grad_(True)
    loss = SF.distill_loss(x, t[:0].to(DEV), ids[:0].to(DEV), 1.0)
    loss.backward()
    assert loss.item() == 0.0 and x.grad.shape == (0, 700)
    x = big[:2].clone().requires_grad_(True)
    loss = SF.distill_loss(x, t[:2, :0].to(DEV), ids[:2, :0].to(DEV), 1.0)
    loss.backward()
    assert loss.item() == 0.0 and (x.grad == 0).all()


def test_distill_has_no_second_derivative():
    x = torch.randn(2, 9, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(SF.distill_loss(x, torch.zeros(2, 1, device=DEV), torch.zeros(2, 1, dtype=torch.int32, device=DEV), 1.0), x,
                             create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---- together, as they are used ------------------------------------------------------------------------------------------


def test_head_scores_and_draws():
    g = gen(12)
    users, items = torch.randn(70, 64, generator=g), torch.randn(1682, 64, generator=g)
    w, bias, res = 1 + 0.1 * torch.randn(64, generator=g), torch.randn(1682, generator=g), torch.randn(70, 64, generator=g)
    head = CatalogueHead(items.to(DEV), bias=bias.to(DEV), norm_weight=w.to(DEV))
    s = head.scores(users.to(DEV), residual=res.to(DEV))
    h = (users.double() + res.double()).float().double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * w.double()
    ref = y @ items.double().t() + bias.double()
    su, si = y.abs().amax(1) / 127, items.double().abs().amax(1) / 127
    bound = 0.5 * (torch.outer(y.abs().sum(1), si) + torch.outer(su, items.double().abs().sum(1))) + 64 * torch.outer(su, si) / 4
    assert ((s.double().cpu() - ref).abs() <= bound + 1e-5).all()
    seen = (torch.arange(70).repeat_interleave(100).to(DEV), torch.randint(0, 1682, (7000,), generator=g).to(DEV))
    ids, prob = head.draw(users.to(DEV), torch.rand(70, generator=g).to(DEV), temperature=0.5, top_k=20, residual=res.to(DEV), seen=seen)
    masked = s.clone()
    masked[seen] = -INF
    top = masked.topk(20, dim=1).indices
    assert (top == ids[:, None].long()).any(1).all() and (prob > 0).all()
    assert not ((seen[0] * 1682 + seen[1])[:, None] == (torch.arange(70, device=DEV) * 1682 + ids)[None]).any()


def test_network_answers_out_of_the_catalogue():
    import star_gcn_amd.model as M
    import star_gcn_amd.synthetic as S
    torch.manual_seed(0)
    graph, eu, ei, _ = S.make_graph("tiny")
    net = M.Net(graph, "user", "movie", embed_units=32, agg_units=(32,), out_units=(32,), nblocks=2, use_dae=True).to(DEV).eval()
    plan = net.make_plan(graph, rating_node_pairs=np.stack([eu, ei]), device=DEV)
    with torch.no_grad():
        preds, _, _ = net.run(plan)
        users, items = net.rating_rows(plan)
    pu, pi = plan["idx"][-1]["rating"]["user"], plan["idx"][-1]["rating"]["movie"]
    dot = (users.double()[torch.from_numpy(np.asarray(pu)).long().to(DEV)] * items.double()[torch.from_numpy(np.asarray(pi)).long().to(DEV)]).sum(1)
    assert (dot - preds[-1].view(-1).double()).abs().max() <= 1e-5 * dot.abs().max()
    head = CatalogueHead(items)
    ids, prob = head.draw(users, torch.rand(users.shape[0], device=DEV), temperature=1e-4, top_p=0.9)
    assert ids.min() >= 0 and ids.max() < items.shape[0] and (prob > 0).all()


def test_student_learns_the_teachers_order():
    g = gen(21)
    users, items = torch.randn(64, 16, generator=g).to(DEV), torch.randn(200, 16, generator=g).to(DEV)
    t, ids = (users @ items.t()).topk(10, dim=1)
    w = torch.zeros(200, 16, device=DEV, requires_grad=True)
    for _ in range(3):
        loss = SF.distill_loss(SF.linear(users, w), t, ids, 1.0 / 64, temperature=2.0)
        grad, = torch.autograd.grad(loss, w)
        s = (users.double() @ w.detach().double().t())
        _, gs, _ = distill_reference(s.cpu(), t.cpu(), ids.cpu(), 1.0 / 64, 2.0)
        want = gs.t().to(DEV) @ users.double()
        assert (grad.double() - want).abs().max() <= 2e-5 * want.abs().max()
        w = (w.detach() - grad).requires_grad_(True)


# ---- streams and graphs ------------------------------------------------------------------------------------------------


def head_pass(x, r, items, u, t, i):
    codes, scale, h = ops.rms_norm_i8(x, None, residual=r)
    s = ops.gemm_i8(codes, scale, *items)
    ids, prob = ops.sample_rows(s, u, top_k=50, top_p=0.9)
    y = s.detach().requires_grad_(True)
    loss = SF.distill_loss(y, t, i, 0.1, temperature=2.0)
    grad, = torch.autograd.grad(loss, y)
    return h, codes, scale, s, ids, prob, loss.detach(), grad


def test_captured_passes_follow_their_inputs_at_every_replay():
    items = ops.quantize_rows(torch.randn(20011, 256, generator=gen(31)).to(DEV))
    shapes = [(3, 256), (3, 256)]
    bufs = [torch.empty(s, device=DEV) for s in shapes] + [torch.empty(3, device=DEV), torch.empty(3, 8, device=DEV)]
    ids = torch.randint(0, 20011, (3, 8), generator=gen(32), dtype=torch.int32).to(DEV)

    def fill(seed):
        for b in bufs:
            b.copy_(torch.rand(b.shape, generator=gen(seed)) if b.dim() == 1 else torch.randn(b.shape, generator=gen(seed)))

    def call():
        return head_pass(bufs[0], bufs[1], items, bufs[2], bufs[3], ids)

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                     # two graphs: neither may use the other's scratch memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for seed in range(1, 5):
        fill(seed)
        want = [v.clone() for v in call()]
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
            call()
        torch.cuda.synchronize()
        for graph, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    items = ops.quantize_rows(torch.randn(5000, 128, generator=gen(41)).to(DEV))
    args = []
    for seed in (1, 2):
        g = gen(seed)
        args.append([torch.randn(4, 128, generator=g).to(DEV), torch.randn(4, 128, generator=g).to(DEV), items, torch.rand(4, generator=g).to(DEV),
                     torch.randn(4, 8, generator=g).to(DEV), torch.randint(0, 5000, (4, 8), generator=g).to(DEV)])
    want = [head_pass(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = []
    for _ in range(5):
        for st, a in zip(streams, args):
            with torch.cuda.stream(st):
                got.append(head_pass(*a))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for a, b in zip(out, want[i % 2]):
            assert torch.equal(a, b)


# ---- refusals ------------------------------------------------------------------------------------------------------------


def test_refusals_on_tensors():
    x = torch.randn(4, 8, device=DEV)
    c, s = ops.quantize_rows(x)
    bad = [lambda: ops.quantize_rows(x.cpu()), lambda: ops.quantize_rows(x.double()), lambda: ops.quantize_rows(x[0]),
           lambda: ops.quantize_rows(x[:, :0]), lambda: ops.quantize_rows(torch.zeros(1, 16385, device=DEV)),
           lambda: ops.rms_norm_i8(x, x[0, :7]), lambda: ops.rms_norm_i8(x, x[0].half()), lambda: ops.rms_norm_i8(x, residual=x[:3]),
           lambda: ops.rms_norm_i8(x, residual=x.half()), lambda: ops.rms_norm_i8(x, eps=-1.0), lambda: ops.rms_norm_i8(x, eps=math.nan),
           lambda: ops.gemm_i8(x, s, c, s), lambda: ops.gemm_i8(c, s[:3], c, s), lambda: ops.gemm_i8(c, s, c[:, :7], s),
           lambda: ops.gemm_i8(c, s.double(), c, s), lambda: ops.gemm_i8(c, s, c, s, bias=s[:2]), lambda: ops.gemm_i8(c, s, c, s, act="elu"),
           lambda: ops.gemm_i8(c, s, c, s, out=torch.empty(4, 5, device=DEV)), lambda: ops.gemm_i8(c, s, c, s, out_dtype=torch.int32),
           lambda: ops.gemm_i8(c, s, c, s, out=torch.empty(5, 4, device=DEV).t()[:, :4]), lambda: ops.gemm_i8(c, s, c, s.cpu()),
           lambda: ops.gemm_i8(torch.zeros(1, 131072, dtype=torch.int8, device=DEV), s[:1], torch.zeros(1, 131072, dtype=torch.int8, device=DEV), s[:1]),
           lambda: ops.sample_rows(x, s[:3]), lambda: ops.sample_rows(x, s.double()), lambda: ops.sample_rows(x.double(), s),
           lambda: ops.sample_rows(x, s, temperature=-1.0), lambda: ops.sample_rows(x, s, top_k=-1), lambda: ops.sample_rows(x, s, top_p=math.nan),
           lambda: ops.sample_rows(x, s, min_p=-0.5), lambda: ops.sample_rows(x, s, temperature=s[:2]), lambda: ops.sample_rows(x, s, top_k=torch.ones(4, device=DEV)),
           lambda: ops.sample_rows(x, s, top_k=2.5), lambda: ops.sample_rows(x, s, top_p=s.cpu()), lambda: ops.sample_rows(x, s, top_p=s > 0),
           lambda: SF.distill_loss(x, x, x, 1.0), lambda: SF.distill_loss(x, c, c.int(), 1.0),
           lambda: SF.distill_loss(x, x[:3], c[:3].int(), 1.0), lambda: SF.distill_loss(x, x, c[:, :4].int(), 1.0),
           lambda: SF.distill_loss(x.double(), x, c.int(), 1.0), lambda: SF.distill_loss(x, x, c.int(), 1.0, temperature=0.0),
           lambda: SF.distill_loss(x, torch.zeros(4, 1025, device=DEV), torch.zeros(4, 1025, dtype=torch.int32, device=DEV), 1.0),
           lambda: SF.distill_loss(x[:, :0], x[:, :1], c[:, :1].int(), 1.0), lambda: CatalogueHead(x).scores(x, residual=x)]
    for i, f in enumerate(bad):
        with pytest.raises(L.StarGCNError):
            f()
            pytest.fail("call %d was not refused" % i)


def test_distill_bwd_refuses_what_is_not_of_its_forward():
    x, t = torch.randn(4, 50, device=DEV), torch.randn(4, 6, device=DEV)
    ids = torch.randint(0, 50, (4, 6), device=DEV)
    loss, saved = ops.distill_fwd(x, t, ids, 1.0)
    one = torch.ones((), device=DEV)
    grad = ops.distill_bwd(one, x, saved, ids, 1.0)
    assert grad.shape == x.shape
    bad = [(one, torch.randn(5, 50, device=DEV), saved, ids), (one, x, saved[:-1], ids), (one, x, saved.double(), ids), (one, x, saved[None], ids),
           (one, x, torch.cat([saved, saved])[::2], ids), (one, x, saved, ids[:, :5]), (one, x, saved, ids[:3]), (one, x, saved, ids[0]),
           (one, x, saved, torch.cat([ids, ids], 1)), (torch.ones(2, device=DEV), x, saved, ids), (one[None][:0], x, saved, ids),
           (one, x.double(), saved, ids), (one, x[0], saved, ids), (one, x, saved.cpu(), ids), (one, x, saved, ids.float()),
           (one, torch.randn(4, 20000, device=DEV), saved, ids)]
    for i, (g, s, v, j) in enumerate(bad):
        with pytest.raises(L.StarGCNError):
            ops.distill_bwd(g, s, v, j, 1.0)
            pytest.fail("call %d was not refused" % i)


def test_seen_pairs_outside_the_scores_name_nothing():
    g = gen(14)
    users, items = torch.randn(5, 32, generator=g).to(DEV), torch.randn(200, 32, generator=g).to(DEV)
    head = CatalogueHead(items)
    u = torch.rand(5, generator=g).to(DEV)
    i64 = lambda v: torch.tensor(v, device=DEV)      # noqa: E731
    s = head.scores(users)
    for rows, cols in (([0, 0, 4, 4], [3, 3, 199, 0]), ([0, -1, 5, 1 << 40, 2, 2, 2, 3], [-1, 4, 7, 7, 200, 1 << 40, -(1 << 40), 9]), ([], [])):
        masked = s.clone()
        for r, c in zip(rows, cols):
            if 0 <= r < 5 and 0 <= c < 200:
                masked[r, c] = -INF
        seen = (i64(rows).long(), i64(cols).long())
        for kw in (dict(), dict(top_k=1)):
            want, got = ops.sample_rows(masked, u, **kw), head.draw(users, u, seen=seen, **kw)
            assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    best = s.argmax(1)
    second, _ = head.draw(users, u, top_k=1, seen=(torch.arange(5, device=DEV).int(), best.int()))
    assert (second != best).all()
    every = (torch.arange(5, device=DEV)[:, None], torch.arange(200, device=DEV))      # every pair
    ids, prob = head.draw(users, u, seen=every)
    assert (ids == -1).all() and (prob == 0).all()
    lost = users.clone()
    lost[0, 1] = math.nan                                  # scores of NaN stay what is never drawn
    ids, prob = head.draw(lost, u, seen=(i64([-1, 0]), i64([-1, 2])))
    assert ids[0] == -1 and (ids[1:] >= 0).all()
    rows = torch.arange(5)
    on_host, _ = head.draw(users, u, top_k=1, seen=(rows, best.cpu()))
    assert torch.equal(on_host, second)
    for bad in ((best, best[:3]), (best, best.float()), (best > 0, best)):
        with pytest.raises(L.StarGCNError):
            head.draw(users, u, seen=bad)


@pytest.mark.parametrize("kind", ["pairs", "full", "resident"])
def test_network_answers_with_items_of_the_graph(kind):
    import star_gcn_amd.model as M
    import star_gcn_amd.synthetic as S
    from star_gcn_amd.resident import ResidentPlan
    torch.manual_seed(1)
    graph, eu, ei, _ = S.make_graph("tiny")
    net = M.Net(graph, "user", "movie", embed_units=32, agg_units=(32,), out_units=(32,), nblocks=2, use_dae=True).to(DEV).eval()
    every = net.make_plan(graph, full_node_ids=graph.node_ids_dict, device=DEV)
    with torch.no_grad():
        all_users, all_items = net.rating_rows(every)
    order = np.random.default_rng(5).permutation(eu.size)[:60]       # some of the pairs, in no order
    pairs = np.stack([eu[order], ei[order]])
    plan = {"pairs": lambda: net.make_plan(graph, rating_node_pairs=pairs, device=DEV), "full": lambda: every,
            "resident": lambda: ResidentPlan(net, graph, device=DEV).set_batch(rating_node_pairs=pairs, remove_batch_edges=False)}[kind]()
    with torch.no_grad():
        users, items = net.rating_rows(plan)
    user_ids, item_ids = net.rating_ids(plan)
    assert user_ids.shape == users.shape[:1] and item_ids.shape == items.shape[:1] and item_ids.dtype == torch.int64
    if kind == "pairs":
        assert sorted(item_ids.tolist()) == sorted(set(pairs[1].tolist())) and item_ids.tolist() != sorted(item_ids.tolist())
        assert sorted(user_ids.tolist()) == sorted(set(pairs[0].tolist()))
    # the rows are those of the nodes that the ids name: the whole neighbourhood is aggregated either way, only sums' orders differ
    for rows, ids, ref in ((users, user_ids, all_users), (items, item_ids, all_items)):
        assert (rows - ref[ids]).abs().max() <= 2e-5 * ref.abs().max()
    head = CatalogueHead(items, item_ids=item_ids)
    s = head.scores(users)
    best = item_ids[s.argmax(1)]
    u = torch.rand(users.shape[0], device=DEV)
    rows = torch.arange(users.shape[0], device=DEV)
    ids, _ = head.draw(users, u, top_k=1)
    assert ids.dtype == torch.int64 and torch.equal(ids, best)
    # the best item masked by its id: the second is drawn.  Items that the catalogue lacks, and no items, mask nothing
    lacking = sorted(set(range(2000)) - set(item_ids.tolist()))[:3]
    seen = (torch.cat([rows, rows[:3], rows[:1]]), torch.cat([best, torch.tensor(lacking + [-1], device=DEV)]))
    ids, _ = head.draw(users, u, top_k=1, seen=seen)
    assert torch.equal(ids, item_ids[s.topk(2, dim=1).indices[:, 1]])
    every_item = (rows[:, None], item_ids[None].int())
    ids, prob = head.draw(users, u, seen=every_item)
    assert (ids == -1).all() and (prob == 0).all()


def test_item_ids_are_checked():
    x = torch.randn(4, 8, device=DEV)
    ids = torch.tensor([7, 1 << 40, 0, 3], device=DEV)
    got, _ = CatalogueHead(x, item_ids=ids).draw(x, torch.rand(4, device=DEV), top_k=1, seen=(torch.zeros(1, dtype=torch.int64, device=DEV), ids[1:2]))
    assert all(v in ids.tolist() for v in got.tolist()) and got[0] != 1 << 40
    none, prob = CatalogueHead(x[:0], item_ids=ids[:0]).draw(x, torch.rand(4, device=DEV), seen=(ids[:1], ids[:1]))
    assert none.tolist() == [-1] * 4 and none.dtype == torch.int64
    small, _ = CatalogueHead(x, item_ids=torch.tensor([9, 8, 7, 6], dtype=torch.int32, device=DEV)).draw(x, torch.rand(4, device=DEV))
    assert small.dtype == torch.int32
    for bad in (ids[:3], ids.cpu(), ids.float(), ids[None], torch.tensor([1, 2, 2, 3], device=DEV), torch.tensor([1, 2, -2, 3], device=DEV)):
        with pytest.raises(L.StarGCNError):
            CatalogueHead(x, item_ids=bad)


def test_draw_with_top_k_of_every_integer_type():
    l, u = torch.randn(6, 300, generator=gen(61)).to(DEV), torch.rand(6, generator=gen(62)).to(DEV)
    k = [0, 1, 5, 100, 127, 64]
    want = ops.sample_rows(l, u, top_k=torch.tensor(k, dtype=torch.int32, device=DEV))
    for t in (torch.int8, torch.uint8, torch.int16, torch.int64):
        got = ops.sample_rows(l, u, top_k=torch.tensor(k, dtype=t, device=DEV))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), t
    every = ops.sample_rows(l, u)
    for t, low in ((torch.int64, -(1 << 32) + 5), (torch.int64, -(1 << 63)), (torch.int32, -(1 << 31)), (torch.int8, -128), (torch.int64, 1 << 40)):
        top_k = torch.full((6,), low, dtype=t, device=DEV)
        got = ops.sample_rows(l, u, top_k=top_k)
        assert (top_k == low).all()                        # the caller's tensor stays as it is
        assert torch.equal(got[0], every[0]) and torch.equal(got[1], every[1]), low
    for bad in (INF, -INF, math.nan, 2.5, -(1 << 70), -1, "5", None):
        with pytest.raises(L.StarGCNError):
            ops.sample_rows(l, u, top_k=bad)


def test_distill_ids_of_every_integer_type():
    s, t = torch.randn(3, 100, generator=gen(63)).to(DEV), torch.randn(3, 4, generator=gen(64)).to(DEV)
    ids = torch.randint(0, 100, (3, 4), generator=gen(65))
    want = SF.distill_loss(s, t, ids.int().to(DEV), 1.0)
    for dt in (torch.int8, torch.uint8, torch.int16, torch.int64):
        assert torch.equal(SF.distill_loss(s, t, ids.to(dt).to(DEV), 1.0), want), dt


@pytest.mark.parametrize("T", [2.0 ** -63, 1e-10, 1e-3, 0.5, 1e3, 1e10, 2.0 ** 63])
def test_distill_at_every_temperature(T):
    g = gen(71)
    for dtype in DTYPES:
        s = (2 * torch.randn(6, 333, generator=g)).to(dtype)
        t = s.float().gather(1, torch.arange(12).expand(6, 12)) + torch.randn(6, 12, generator=g)
        ids = torch.stack([torch.randperm(333, generator=g)[:12] for _ in range(6)]).int()
        s[4, 10:40] = -INF
        s[5] = 0.25                                        # all alike
        ids[4] = torch.arange(50, 62)
        if dtype == torch.float16 and T >= 1e10:
            # scale T q is about 1e10 / 6 / 333 = 5e6: past 65520 the nearest fp16 number is infinity
            x = s.to(DEV).requires_grad_(True)
            grad, = torch.autograd.grad(SF.distill_loss(x, t.to(DEV), ids.to(DEV), 1.0 / 6, temperature=T), x)
            _, want, size = distill_reference(s, t, ids, 1.0 / 6, T)
            past = want.abs() - T / 6 * 7e-6 * size > 65520
            assert past.sum() > 1900 and torch.equal(grad.cpu().double()[past], torch.sign(want)[past] * INF) and (grad[4, 10:40] == 0).all()
            continue
        check_distill(s, t, ids, scale=1.0 / 6, T=T)


@pytest.mark.parametrize("T", [0.3, 0.5, 2.0])
def test_distill_towards_items_masked_by_the_lowest_value(T):
    g = gen(72)
    s, t = torch.randn(4, 200, generator=g), torch.randn(4, 6, generator=g)
    ids = torch.stack([torch.randperm(200, generator=g)[:6] for _ in range(4)]).int()
    s[1, ids[1, 2].long()] = -3.4028234663852886e38        # the loss is as large as the score, and finite
    s[2, ids[2].long()] = -3.4028234663852886e38
    check_distill(s, t, ids, scale=1.0 / 8, T=T)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["two levels", "few levels", "rising", "falling", "rising, masked"])
def test_distill_sums_of_long_rows_of_a_large_batch(dtype, kind):
    # 1024 rows: a row is not split, and a thread adds hundreds of vectors, whose roundings all go the same way where terms repeat
    rows, n = 1024, 400000
    g = torch.Generator(device=DEV).manual_seed(3)
    i = torch.arange(n, device=DEV)
    row = {"two levels": torch.randint(0, 2, (n,), generator=g, device=DEV), "few levels": torch.randint(0, 50, (n,), generator=g, device=DEV) * 0.1,
           "rising": (i // 1024) * 1e-4, "falling": 1.0 - (i // 1024) * 1e-4,
           "rising, masked": ((i // 1024) * 1e-4).masked_fill(i % 3 == 0, -INF)}[kind].to(dtype)
    s = row.expand(rows, n).contiguous()
    t, ids = torch.zeros(rows, 4, device=DEV), (torch.arange(4, device=DEV) * 3 + 1).expand(rows, 4).contiguous()
    x = s.requires_grad_(True)
    loss = SF.distill_loss(x, t, ids, 1.0 / rows)
    grad, = torch.autograd.grad(loss, x)
    z = row.double()
    q = torch.softmax(z, 0)
    log_q = torch.log_softmax(z, 0)[ids[0]]
    # the rows are alike.  A term: exponents up to 4 log2(e), rounded twice (4 * 2^-24 * 2 * ln 2 * 1.45 = 5e-7), v_exp_f32 one step
    # (1.2e-7); a vector's terms pairwise, three half steps (1.8e-7); the waves' joins and the inverse a few more half steps: 1.5e-6
    assert abs(loss.item() - (-math.log(4.0) - log_q.mean().item())) <= 1.5e-6 + 2.0 ** -22 * abs(log_q.mean().item())
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[ids[0]] = False
    fi = torch.finfo(dtype)
    for r in (0, 511, 1023):
        # the gradient's own exponent and products as much again, and the type's rounding
        err = (grad[r].double() * rows - q).abs()[rest]
        assert (err <= (3e-6 + fi.eps / 2) * q[rest] + rows * fi.smallest_normal * fi.eps).all(), float((err / q[rest]).max())


def peak_and_tail(n, x, dtype, peak):
    """One score of 0 and n - 1 of x -> scores, the weight of a tail item and of all (the peak's is 1), what the tail's weights may be
    off by together: half a unit of their fixed point each."""
    l = torch.full((1, n), x, dtype=dtype, device=DEV)
    l[0, peak] = 0.0
    w = math.exp(float(l[0, (peak + 1) % n]))
    unit = max(63 - math.ceil(math.log2(n)), 0) if n <= 1 << 20 else 51
    return l, w, 1.0 + (n - 1) * w, n * 2.0 ** -(min(unit, 51) + 1)


@pytest.mark.parametrize("n,x,dtype", [(1 << 20, -25.0, torch.float32), (1 << 20, -31.0, torch.float32), ((1 << 20) + 1, -31.0, torch.float32),
                                       (10000000, -27.0, torch.float32), (10000000, -27.2, torch.float32), (10000000, -16.0, torch.float16),
                                       (1 << 26, -26.0, torch.bfloat16), (1 << 28, -24.25, torch.bfloat16), (1 << 28, -19.0, torch.float16)])
def test_draw_of_a_flat_tail_that_holds_what_one_unit_of_weight_does_not(n, x, dtype):
    peak = n // 3
    l, w, total, off = peak_and_tail(n, x, dtype, peak)
    assert off <= 2.0 ** -24 * 1.01
    first, last = peak * w / total, (peak * w + 1.0) / total      # the shares between which the peak is drawn
    margin = off / total + 2.0 ** -24                      # and u itself is rounded to fp32
    us = [first / 2, first + 1.5 * margin, 0.5 * (first + last), last - 1.5 * margin, 0.5 * (1.0 + last)]
    want = [first > 4 * margin, True, True, True, 1 - last > 4 * margin]
    for u, sure, inside in zip(us, want, (False, True, True, True, False)):
        if not sure:
            continue
        ids, prob = ops.sample_rows(l, torch.tensor([u], device=DEV))
        assert (ids.item() == peak) == inside, (u, ids.item())
        if inside:
            assert abs(prob.item() - 1.0 / total) <= off / total + 2.0 ** -24
        else:
            # an item of the tail, as far along as u asks for: its weight is off by half a unit
            assert 0 <= ids.item() < n and abs(prob.item() - w / total) <= 2 * off / n + 2.0 ** -24 * w / total
            at = float(np.float32(u)) * total / w
            if u > last:
                at = (float(np.float32(u)) * total - 1.0) / w + 1
            assert abs(ids.item() - at) <= 2 * off / w + 2 + n * 1e-9


@pytest.mark.parametrize("n", [(1 << 20) + 1, 3000000, 10000000])
def test_draw_among_millions_of_equal_scores(n):
    # the weight of all of them passes 2^64; ranks and shares are known without a sum
    l = torch.zeros(4, n, device=DEV, dtype=torch.float16)
    l[1] = 1.5
    l[1, n // 2:] = -INF
    l[2, ::2] = math.nan
    l[3, 7] = INF
    u = torch.tensor([0.75, 0.75, 0.75, 0.75], device=DEV)
    live = [n, n // 2, n // 2, 1]
    index = [lambda r: r, lambda r: r, lambda r: 2 * r + 1, lambda r: 7]
    for kw, keep in ((dict(), lambda m: m), (dict(top_k=1000001), lambda m: min(m, 1000001)), (dict(top_p=0.5), lambda m: math.ceil(m * 0.5)),
                     (dict(top_k=600000, top_p=0.25), lambda m: math.ceil(min(m, 600000) * 0.25)), (dict(min_p=1.0), lambda m: m)):
        ids, prob = ops.sample_rows(l, u, **kw)
        for i in range(4):
            m = keep(live[i])
            assert ids[i].item() == index[i](int(0.75 * m)), (kw, i)
            assert abs(prob[i].item() * m - 1) <= 2.0 ** -23, (kw, i)


@pytest.mark.parametrize("n,dtype", [(1 << 20, torch.float32), ((1 << 20) + 1, torch.float32), (3000001, torch.bfloat16), (3000000, torch.float32)])
def test_draw_from_rows_of_millions(n, dtype):
    g = gen(n)
    l = torch.randn(3, n, generator=g).to(dtype)
    l[1] = (0.3 * torch.randn(n, generator=g)).to(dtype)
    l[2, torch.rand(n, generator=g) < 0.5] = -INF
    u = torch.rand(3, generator=g)
    for kw in (dict(), dict(top_p=0.95), dict(top_k=700), dict(top_k=40000, top_p=0.7, min_p=1e-3), dict(min_p=0.01, temperature=0.5)):
        check_draw(l, u, **kw)


@pytest.mark.parametrize("M,N,K", [(1, 40, 64), (3, 50, 8192), (130, 300, 250), (600, 2100, 64), (2050, 4099, 80), (4096, 4096, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_product_with_scales_over_the_whole_range(M, N, K, dtype):
    g = torch.Generator(device=DEV).manual_seed(K)
    a, b = (torch.randint(-128, 128, (n, K), generator=g, device=DEV, dtype=torch.int16).to(torch.int8) for n in (M, N))
    a[0], b[0] = 0, 0                                      # sums of nothing stay 0 whatever the scales
    # exponents over all of fp32's, subnormal ones among them; most rows next to each other differ by far
    sa, sb = (torch.ldexp(torch.rand(n, generator=g, device=DEV) + 0.5, torch.randint(-148, 127, (n,), generator=g, device=DEV)) for n in (M, N))
    sa[0], sb[N // 2] = 3e38, 3e38
    sa[M // 2] = 1.7e29
    sb[1], sb[2] = -1e-30, 0.0
    bias = torch.randn(N, generator=g, device=DEV)
    for c, act in ((bias, None), (None, None), (bias, "leaky")):
        out = ops.gemm_i8(a, sa, b, sb, bias=c, act=act, slope=0.2, out_dtype=dtype).double()
        exact = a.double() @ b.double().t().contiguous()
        t = exact * sa.double()[:, None] * sb.double()
        v = t if c is None else t + c.double()
        ref = ACTS[act](v)
        # check_product's roundings; below the normal numbers a rounding is at most half the least number instead (the product
        # with sb and the sum with the bias are one)
        fi = torch.finfo(dtype)
        tol = 1.01 * (2.0 ** -24 * (2 * t.abs() + v.abs() + ref.abs()) + 2.0 ** -149) + (0 if dtype == torch.float32 else fi.eps / 2 * ref.abs() + fi.smallest_normal * fi.eps)
        edge = fi.max * (1 + fi.eps / 4)                   # the border between the largest number and infinity
        # what the activation takes is an fp32 number already: 0.2 times an infinity is one, 0.2 times what it stands for need not be
        room = 2.0 ** 128 * (1 - 2.0 ** -25) - v.abs()
        small = (ref.abs() + tol < edge) & (room > 2.0 ** 105)
        past = (ref.abs() - tol >= edge) | (room < -(2.0 ** 105))
        assert ((out - ref).abs() <= tol)[small].all(), float(((out - ref).abs() - tol)[small].max())
        assert (out[past] == torch.sign(ref[past]) * INF).all() and not out.isnan().any()
        assert small.any() and (past.any() or M * N < 1000)


@pytest.mark.parametrize("rows,n,dtype", [(33000, 16390, torch.bfloat16), (16385, 20001, torch.float32)])
def test_draw_from_more_long_rows_than_one_batch(rows, n, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows)
    l = (2 * torch.randn(rows, n, generator=g, device=DEV)).to(dtype)
    u, t, p, m = (torch.rand(rows, generator=g, device=DEV) for _ in range(4))
    k = torch.randint(0, 3000, (rows,), generator=g, device=DEV)
    for kw in (dict(), dict(top_p=p), dict(temperature=0.5 + t, top_k=k, top_p=p, min_p=0.01 * m)):
        ids, prob = ops.sample_rows(l, u, **kw)
        for lo, hi in ((0, 40), (16370, min(16420, rows)), (rows - 9, rows)):
            cut = {name: v[lo:hi] for name, v in kw.items()}
            i, q = ops.sample_rows(l[lo:hi], u[lo:hi], **cut)
            assert torch.equal(ids[lo:hi], i) and torch.equal(prob[lo:hi], q)


def test_captured_head_follows_its_inputs_at_every_replay():
    g = gen(91)
    items, item_ids = torch.randn(1500, 48, generator=g).to(DEV), torch.randperm(9000, generator=g)[:1500].to(DEV)
    head = CatalogueHead(items, item_ids=item_ids, norm_weight=torch.ones(48, device=DEV))
    users, u = torch.empty(9, 48, device=DEV), torch.empty(9, device=DEV)
    rows, seen = torch.empty(40, dtype=torch.int64, device=DEV), torch.empty(40, dtype=torch.int64, device=DEV)

    def fill(seed):
        users.copy_(torch.randn(9, 48, generator=gen(seed)))
        u.copy_(torch.rand(9, generator=gen(seed + 100)))
        rows.copy_(torch.randint(-1, 10, (40,), generator=gen(seed + 200)))
        seen.copy_(torch.randint(-1, 9001, (40,), generator=gen(seed + 300)))
        seen[:9] = item_ids[head.scores(users).argmax(1)]
        rows[:9] = torch.arange(9, device=DEV)

    def call():
        return head.draw(users, u, temperature=0.2, top_k=30, top_p=0.95, seen=(rows, seen))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(1, 6):
        fill(seed)
        want = [v.clone() for v in call()]
        graph.replay()
        call()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        best = seen[:9]
        assert (out[0] != best).all() and torch.isin(out[0], item_ids).all()


@pytest.mark.parametrize("n", [1682, 16385, 40000, (1 << 20) + 7])
def test_captured_draws_of_every_length(n):
    l, u = torch.empty(5, n, device=DEV), torch.empty(5, device=DEV)
    par = dict(temperature=torch.empty(5, device=DEV), top_k=torch.empty(5, dtype=torch.int64, device=DEV), top_p=torch.empty(5, device=DEV),
               min_p=torch.empty(5, device=DEV))

    def fill(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        l.normal_(generator=g)
        for v in (u, par["temperature"], par["top_p"], par["min_p"]):
            v.uniform_(generator=g)
        par["top_k"].random_(0, n, generator=g)

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample_rows(l, u, **par)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for kw in (par, dict(), dict(top_p=0.7)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, kw, ops.sample_rows(l, u, **kw)))
    for seed in range(1, 5):
        fill(seed)
        for graph, kw, out in graphs:
            want = [v.clone() for v in ops.sample_rows(l, u, **kw)]
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
