"""The 8-bit decoder-layer operators (quantised rows, products of whole numbers, head norms with rotation, cache append) against their formulas in 64 bits.

Tolerances count roundings. U = 2^-24 is a rounding to fp32, eps / 2 one to the 16-bit result type. A sum of squares of n values in fp32 is at most n U off
(relative, all terms positive), the norm's factor half of that and three roundings more."""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16]


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def K():
    from openvino_b200.ops import cuda as ops
    ops.lib()
    return ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def within(got, want, bound, what=""):
    """|got - want| <= bound element by element; NaN where the formula has NaN."""
    got, want = got.double().cpu(), want.double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(want)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), what
    off = ((got - want).abs() - bound)[~nan]
    assert off.numel() == 0 or float(off.max()) <= 0, "%s: %.3g beyond the bound" % (what, float(off.max()))


# ------------------------------------------------------------------------------------------------ quantised rows
def codes_of(y32):
    """The definition in fp32 arithmetic of numpy, which rounds every operation once: codes, scale, sum."""
    y = y32.cpu().float().numpy()
    a = np.abs(y).max(1, keepdims=True)
    with np.errstate(all="ignore"):
        f = np.float32(127.0) / a
        q = np.rint(y * f)
        q = np.where(a < np.float32(2.0 ** -119), 0, q)
        ok = np.isfinite(a)
        q = np.where(ok, q, 0)
        scale = np.where(ok, np.where(a < np.float32(2.0 ** -119), np.float32(0), a / np.float32(127.0)), np.float32(np.nan))
    return torch.from_numpy(q.astype(np.int8)), torch.from_numpy(scale[:, 0]), torch.from_numpy(q.sum(1).astype(np.int32))


WIDTHS = [(1, 1), (3, 7), (5, 8), (2, 130), (9, 512), (6, 520), (7, 1024), (130, 1333), (4, 4096), (3, 6152), (2, 14336), (2, 28672), (1, 33000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", WIDTHS)
def test_rows_are_quantised_to_the_bit(K, rows, cols, dtype):
    x = (torch.randn((rows, cols), generator=gen(cols), device="cuda") * 3).to(dtype)
    r = K.quantize_rows(x)
    K.check_status("quantize_rows")
    q, scale, total = codes_of(x)
    assert torch.equal(r.q.cpu(), q) and torch.equal(r.scales.cpu(), scale) and torch.equal(r.sums.cpu(), total)
    assert r.q.stride(0) % 16 == 0 and r.dtype == dtype and r.shape == (rows, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [24, 27, 2048])
def test_rows_with_nothing_tiny_and_not_finite_values(K, cols):
    x = torch.randn((8, cols), generator=gen(3), device="cuda").bfloat16()
    x[0] = 0
    x[1] *= 2.0 ** -125                     # below the floor: zero
    x[2] = 0
    x[2, 5] = 2.0 ** -119                   # the smallest row that counts
    x[3, 7] = math.nan
    x[4, 2] = math.inf
    x[5, 1] = -math.inf
    x[6] = torch.finfo(torch.bfloat16).max  # 127 / a is tiny, the codes are 127
    r = K.quantize_rows(x)
    q, scale, total = codes_of(x)
    assert torch.equal(r.q.cpu(), q) and torch.equal(r.sums.cpu(), total)
    assert torch.equal(r.scales.cpu().isnan(), scale.isnan()) and torch.equal(r.scales.cpu().nan_to_num(0), scale.nan_to_num(0))
    assert r.scales[0] == 0 and r.scales[1] == 0 and r.scales[2] > 0 and r.scales[3:6].isnan().all() and (r.q[6] == 127).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", WIDTHS)
def test_normed_rows_are_quantised(K, rows, cols, dtype):
    x = (torch.randn((rows, cols), generator=gen(cols + 1), device="cuda") * 2).to(dtype)
    gamma = (1 + 0.3 * torch.randn(cols, generator=gen(2), device="cuda")).to(dtype)
    r = K.quantize_rows(x, norm=(gamma, 1e-3))
    y = x.double() * torch.rsqrt(x.double().pow(2).mean(1, keepdim=True) + 1e-3) * gamma.double()
    a = y.abs().amax(1, keepdim=True)
    rel = (cols / 2 + 8) * U                # of every normed value and of the largest: the factor's error and two products
    within(r.scales, (a / 127)[:, 0], (a / 127)[:, 0] * (rel + 2 * U), "scale")
    within(r.q, y * 127 / a, 0.5 + 127 * (2 * rel + 4 * U), "codes")
    assert torch.equal(r.sums, r.q.sum(1, dtype=torch.int32))
    pick = torch.tensor([rows - 1, 0, rows - 1, rows, -1], dtype=torch.int32, device="cuda")        # indices outside read row 0
    p = K.quantize_rows(x, norm=(gamma, 1e-3, pick))
    rows_of = [rows - 1, 0, rows - 1, 0, 0]
    assert torch.equal(p.q, r.q[rows_of]) and torch.equal(p.scales, r.scales[rows_of]) and torch.equal(p.sums, r.sums[rows_of])


@pytest.mark.gpu
def test_rows_of_other_strides(K):
    x = torch.randn((6, 200), generator=gen(1), device="cuda").bfloat16()
    for view in (x[::2], x[:, 3:90], x[:, 8:136], x[1:2].expand(4, 200), x[2:, 1:2], x[:0]):
        r = K.quantize_rows(view)
        q, scale, total = codes_of(view) if view.shape[0] else (torch.empty((0, 200), dtype=torch.int8), torch.empty(0), torch.empty(0, dtype=torch.int32))
        assert torch.equal(r.q.cpu(), q) and torch.equal(r.scales.cpu(), scale) and torch.equal(r.sums.cpu(), total)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 515])
@pytest.mark.parametrize("cols", [1, 7, 9, 16, 23, 100, 513, 1030, 2049, 4097, 8200, 16401, 32767, 32769])
def test_rows_at_any_place(K, rows, cols):
    """Views that start at every 16-bit place of a 16-byte piece, with odd and even pitches: the codes of the rows, and with a norm the same bits wherever they lie."""
    norm_want = None
    for off in range(9):
        wide = torch.full((rows, cols + 9 + off % 2), math.nan, device="cuda", dtype=torch.bfloat16)
        view = wide[:, off:off + cols]
        view.copy_(torch.randn((rows, cols), generator=gen(cols), device="cuda"))
        r = K.quantize_rows(view)
        q, scale, total = codes_of(view)
        assert torch.equal(r.q.cpu(), q) and torch.equal(r.scales.cpu(), scale) and torch.equal(r.sums.cpu(), total)
        gamma = torch.empty(cols + 8, device="cuda", dtype=torch.bfloat16)[off % 8:off % 8 + cols]
        gamma.copy_(1 + 0.3 * torch.randn(cols, generator=gen(2), device="cuda"))
        n = K.quantize_rows(view, norm=(gamma, 1e-3))
        norm_want = norm_want or n
        assert torch.equal(n.q, norm_want.q) and torch.equal(n.scales, norm_want.scales) and torch.equal(n.sums, norm_want.sums)
    K.check_status("quantize_rows")


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(300, 514), (300, 520), (700, 1024), (513, 1003)])
def test_residuals_of_many_tokens(K, T, N):
    """The residual in rows of other pitches than the result's, of any alignment, and in the result's own place."""
    Kd = 256
    w, s, z = weight(N, Kd, "signed_zp", 3)
    rows = K.quantize_rows(torch.randn((T, Kd), generator=gen(T), device="cuda").bfloat16())
    for pw in (K.PackedWeight.from_ir_i8(w, s), K.PackedWeight.from_ir_i8(w, s, z)):
        plain = K.gemm(rows, pw, out_f32=True)
        for off, pad in ((0, 0), (0, 8), (3, 5), (8, 16)):
            wide = torch.randn((T, N + off + pad), generator=gen(N), device="cuda").bfloat16()
            res, keep = wide[:, off:off + N], wide.clone()
            want = (plain + res.float()).bfloat16()
            assert torch.equal(K.gemm(rows, pw, residual=res), want) and torch.equal(wide, keep)
            assert torch.equal(K.gemm(rows, pw, residual=res, out=res), want)
            keep[:, off:off + N] = want
            assert torch.equal(wide, keep)
    K.check_status("gemm_i8")


# ------------------------------------------------------------------------------------------------ products
def weight(N, Kd, form, seed):
    g = gen(seed)
    if form == "unsigned":
        w = torch.randint(0, 256, (N, Kd), generator=g, device="cuda", dtype=torch.uint8)
        z = torch.randint(0, 256, (N,), generator=g, device="cuda", dtype=torch.uint8)
    else:
        w = torch.randint(-128, 128, (N, Kd), generator=g, device="cuda", dtype=torch.int8)
        z = torch.randint(-128, 128, (N,), generator=g, device="cuda", dtype=torch.int8) if form == "signed_zp" else None
    s = ((0.5 + torch.rand(N, generator=g, device="cuda")) / (74 * math.sqrt(Kd))).half()
    return w, s, z


def value64(rows, w, s, z, bias=None):
    """The product's value before its activation, and the size that its fp32 roundings (conversion, two scales, their product, the bias) refer to."""
    w64 = w.double() - (0 if z is None else z.double()[:, None])
    v = rows.q.double() @ w64.T * rows.scales.double()[:, None] * s.double()
    size = v.abs()
    if bias is not None:
        v = v + bias.double()
        size = torch.maximum(size, v.abs())
    return v, 5 * U * size


SIZES = [(1, 128, 128), (1, 1, 1), (2, 130, 33), (3, 257, 500), (7, 1000, 1333), (8, 384, 4096), (16, 512, 640), (17, 4096, 2048), (33, 640, 14336), (64, 1024, 4096),
         (100, 300, 777), (129, 256, 128), (200, 2048, 1024), (255, 128, 256), (256, 384, 384), (257, 1000, 130), (333, 512, 4096), (600, 130, 300), (1000, 2560, 512),
         (2049, 384, 256)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", ["signed", "signed_zp", "unsigned"])
@pytest.mark.parametrize("T,N,Kd", SIZES)
def test_product(K, T, N, Kd, form, dtype):
    x = torch.randn((T, Kd), generator=gen(T), device="cuda").to(dtype)
    w, s, z = weight(N, Kd, form, N)
    bias = torch.randn(N, generator=gen(5), device="cuda").to(dtype)
    residual = torch.randn((T, N), generator=gen(6), device="cuda").to(dtype)
    rows = K.quantize_rows(x)
    plain, biased = K.PackedWeight.from_ir_i8(w, s, z), K.PackedWeight.from_ir_i8(w, s, z, bias=bias)
    # fp32 out: only the roundings of the epilogue
    v, off = value64(rows, w, s, z)
    within(K.gemm(rows, plain, out_f32=True), v, off, "fp32 out")
    v, off = value64(rows, w, s, z, bias)
    got = K.gemm(x, biased, residual=residual)
    want = v + residual.double()
    within(got, want, off + U * want.abs() + half_eps(dtype) * (want.abs() + off) + 2.0 ** -25, "bias and residual")
    assert torch.equal(K.gemm(rows, biased, residual=residual), got)         # rows quantised before, the same bits
    h = residual.clone()
    assert torch.equal(K.gemm(x, biased, out=h, residual=h), got) and torch.equal(h, got)      # in place
    K.check_status("gemm_i8")


def test_product_activation_bounds():
    """The bounds of the next test: derivatives of the activations are at most 1.13 (gelu), 1.1 (silu)."""
    v = torch.linspace(-20, 20, 200001, dtype=torch.float64)
    for f in (torch.nn.functional.gelu, torch.nn.functional.silu, lambda t: torch.nn.functional.gelu(t, approximate="tanh")):
        y = f(v)
        assert ((y[1:] - y[:-1]) / (v[1:] - v[:-1])).abs().max() < 1.14


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,N,Kd", [(1, 256, 500), (5, 384, 4096), (40, 512, 256), (150, 640, 1000), (300, 256, 512), (700, 1280, 640)])
def test_product_activations(K, T, N, Kd, dtype):
    F = torch.nn.functional
    x = torch.randn((T, Kd), generator=gen(T), device="cuda").to(dtype)
    w, s, z = weight(N, Kd, "unsigned", N)
    s = s * 2
    pw, rows = K.PackedWeight.from_ir_i8(w, s, z), K.quantize_rows(x)
    v, off = value64(rows, w, s, z)
    forms = [(K.ACT_GELU_ERF, F.gelu, {}), (K.ACT_RELU, F.relu, {}), (K.ACT_SILU, F.silu, {}), (K.ACT_GELU_TANH, lambda t: F.gelu(t, approximate="tanh"), {}),
             (K.ACT_RELU2, lambda t: F.relu(t) ** 2, {}), (K.ACT_SOFTCAP, lambda t: 3 * torch.tanh(t / 3), {"cap": 3.0})]
    for act, f, more in forms:
        want = f(v)
        # what the epilogue's functions may add: errors of exp, tanh and erf of some 2^-21 of the value (of the cap), beside the argument's error
        slope = 1.14 if act != K.ACT_RELU2 else 2 * v.abs() + 1
        own = 2.0 ** -20 * (v.abs() + (3 if act == K.ACT_SOFTCAP else 0)) + (3 * U * want.abs() if act == K.ACT_RELU2 else 0)
        bound = off * slope + own
        within(K.gemm(rows, pw, act=act, **more), want, bound + half_eps(dtype) * (want.abs() + bound) + 2.0 ** -25, "activation %d" % act)
    tiles = v.view(T, -1, 2, 64)
    offs = off.view(T, -1, 2, 64)
    gate, up = tiles[:, :, 0], tiles[:, :, 1]
    want = F.silu(gate) * up
    bound = (1.14 * offs[:, :, 0] + 2.0 ** -20 * gate.abs()) * up.abs() + offs[:, :, 1] * gate.abs() + 2 * U * want.abs()
    within(K.gemm(x, pw, act=K.ACT_SWIGLU), want.reshape(T, -1), (bound + half_eps(dtype) * (want.abs() + bound) + 2.0 ** -25).reshape(T, -1), "swiglu")
    g, u = gate.clamp(max=0.7), up.clamp(-0.7, 0.7)
    want = g * torch.sigmoid(1.702 * g) * (u + 1)
    bound = (1.3 * offs[:, :, 0] + 2.0 ** -20 * g.abs()) * 1.7 + offs[:, :, 1] * g.abs() + 4 * U * want.abs()
    within(K.gemm(rows, pw, act=K.ACT_GLU_LIMITED, glu=(0.7, 1.702, 1.0)), want.reshape(T, -1), (bound + half_eps(dtype) * (want.abs() + bound) + 2.0 ** -25).reshape(T, -1), "glu")
    K.check_status("gemm_i8")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6, 300])
def test_rows_that_are_not_finite_show_behind_every_activation(K, T):
    x = torch.randn((T, 256), generator=gen(T), device="cuda").bfloat16()
    x[T - 1, 7] = math.nan
    w, s, z = weight(256, 256, "unsigned", 1)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    for act in range(K.ACT_NONE, K.ACT_SOFTCAP + 1):
        got = K.gemm(x, pw, act=act, glu=(7.0, 1.7, 1.0), cap=3.0)
        assert got[T - 1].isnan().all() and got[:T - 1].isfinite().all(), act


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 300])
def test_activations_at_the_ends_of_their_range(K, T):
    """Scales that carry the arguments from 2^-12 to 2^60: what saturates does so, what is small keeps its digits."""
    F, N, Kd = torch.nn.functional, 256, 64
    x = torch.randn((T, Kd), generator=gen(T), device="cuda").bfloat16()
    w, s, _ = weight(N, Kd, "signed", 1)
    s = torch.exp2(torch.linspace(-20, 52, N, device="cuda"))
    pw, rows = K.PackedWeight.from_ir_i8(w, s), K.quantize_rows(x)
    v, off = value64(rows, w, s, None)
    for act, f, more in ((K.ACT_SILU, F.silu, {}), (K.ACT_GELU_TANH, lambda t: F.gelu(t, approximate="tanh"), {}), (K.ACT_SOFTCAP, lambda t: 30 * torch.tanh(t / 30), {"cap": 30.0})):
        want = f(v)
        # 2^-20 of the value, or where it vanishes of the argument's share that an exponential leaves (of the cap, once it is felt)
        own = 2.0 ** -20 * (torch.minimum(v.abs(), torch.tensor(30.0, device="cuda", dtype=torch.float64)) + (want.abs()))
        bound = off.clamp(max=1e30) * 1.14 + own
        bound = torch.where(v.abs() > 1e6, want.abs() * 2.0 ** -20 + 2.0 ** -25, bound)
        got = K.gemm(rows, pw, act=act, out_f32=True, **more).double()
        assert got.isfinite().all()
        within(got, want, bound + 2.0 ** -25, "activation %d" % act)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 4, 20, 300])
def test_product_with_the_norm_in_front(K, T):
    N, Kd, dtype = 640, 2048, torch.bfloat16
    x = torch.randn((T, Kd), generator=gen(T), device="cuda").to(dtype)
    gamma = (1 + 0.2 * torch.randn(Kd, generator=gen(2), device="cuda")).to(dtype)
    w, s, z = weight(N, Kd, "signed", N)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    rows = K.quantize_rows(x, norm=(gamma, 1e-5))
    assert torch.equal(K.gemm(x, pw, norm=(gamma, 1e-5)), K.gemm(rows, pw))
    pick = torch.tensor([T - 1, 0, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(K.gemm(x, pw, norm=(gamma, 1e-5, pick)), K.gemm(rows, pw)[[T - 1, 0, 0]])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 5, 600])
def test_results_in_the_place_of_the_rows(K, T):
    """x + W norm(x) written over x: rows are quantised before the first result is stored."""
    Kd = 4096
    x = torch.randn((T, Kd), generator=gen(T), device="cuda").bfloat16()
    gamma = (1 + 0.2 * torch.randn(Kd, generator=gen(2), device="cuda")).bfloat16()
    w, s, z = weight(Kd, Kd, "signed_zp", 3)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    want = K.gemm(K.quantize_rows(x, norm=(gamma, 1e-5)), pw, residual=x)
    for _ in range(8):
        h = x.clone()
        assert torch.equal(K.gemm(h, pw, out=h, residual=h, norm=(gamma, 1e-5)), want)
    many = torch.cat([x, x])[:T + 1].contiguous()           # one row of several, picked by its index, over another
    pick = torch.zeros(1, dtype=torch.int32, device="cuda")
    one = K.gemm(many, pw, norm=(gamma, 1e-5, pick))
    assert torch.equal(K.gemm(many, pw, out=many[:1], norm=(gamma, 1e-5, pick)), one)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,Kd", [(1, 128, 65536), (20, 130, 65536), (300, 256, 65536)])
def test_largest_sums_stay_exact(K, T, N, Kd):
    x = torch.ones((T, Kd), device="cuda", dtype=torch.bfloat16)
    w = torch.full((N, Kd), 255, dtype=torch.uint8, device="cuda")
    w[::2] = 0
    z = torch.zeros(N, dtype=torch.uint8, device="cuda")
    z[::2] = 255
    s = torch.full((N,), 2.0 ** -20, device="cuda")
    got = K.gemm(x, K.PackedWeight.from_ir_i8(w, s, z), out_f32=True)
    rows = K.quantize_rows(x)
    v, off = value64(rows, w, s, z)
    within(got, v, off)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 9, 70, 500])
def test_rows_that_are_not_finite_stay_to_themselves(K, T):
    x = torch.randn((T + 2, 384), generator=gen(T), device="cuda").bfloat16()
    w, s, z = weight(200, 384, "unsigned", 1)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    clean = K.gemm(x, pw)
    x[0, 3], x[T + 1, 0] = math.nan, math.inf
    got = K.gemm(x, pw)
    assert got[0].isnan().all() and got[T + 1].isnan().all() and torch.equal(got[1:T + 1], clean[1:T + 1])
    x[0] = 0
    assert (K.gemm(x, pw)[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(1, 77), (5, 384), (40, 130), (300, 384), (600, 200)])
def test_views_and_rows_behind_the_last(K, T, N):
    """Rows that the call does not have, and columns beside its own, stay as they were; outputs and residuals of any pitch and alignment."""
    Kd = 300
    x = torch.randn((T, Kd), generator=gen(T), device="cuda").half()
    w, s, z = weight(N, Kd, "signed", N)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    want = K.gemm(x, pw)
    for lead, dtype in ((0, torch.float16), (1, torch.float16), (3, torch.float32), (4, torch.float32)):
        big = torch.full((T + 3, N + 9), 7.0, dtype=dtype, device="cuda")
        got = K.gemm(x, pw, out=big[1:T + 1, lead:lead + N], out_f32=dtype == torch.float32)
        assert torch.equal(got.half(), want)
        big[1:T + 1, lead:lead + N] = 7
        assert (big == 7).all()
    res = torch.randn((T, N + 3), generator=gen(9), device="cuda").half()[:, 1:N + 1]
    assert torch.equal(K.gemm(x, pw, residual=res), K.gemm(x, pw, residual=res.contiguous()))
    wide = torch.zeros((T, Kd + 5), dtype=torch.float16, device="cuda")
    wide[:, 2:Kd + 2] = x
    assert torch.equal(K.gemm(wide[:, 2:Kd + 2], pw), want)
    wt = torch.zeros((N, 2 * Kd), dtype=torch.int8, device="cuda")
    wt[:, 5:Kd + 5] = w
    assert torch.equal(K.gemm(x, K.PackedWeight.from_ir_i8(wt[:, 5:Kd + 5], s, z)), want)
    assert torch.equal(K.gemm(x, K.PackedWeight.from_ir_i8(w.t().contiguous().t(), s, z)), want)
    assert K.gemm(x[:0], pw).shape == (0, N)
    K.check_status("gemm_i8")


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,Kd", [(1, 6144, 4096), (16, 4096, 14336), (64, 4096, 4096), (500, 1024, 2048)])
def test_products_on_two_streams_and_in_graphs(K, T, N, Kd):
    xs = [torch.randn((T, Kd), generator=gen(i), device="cuda").bfloat16() for i in range(2)]
    w, s, z = weight(N, Kd, "unsigned", N)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    want = [K.gemm(x, pw) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    outs = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(K.gemm(xs[i], pw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])
    graphs, got = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(K.gemm(x, pw))
        graphs.append(g)
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs[0].copy_(xs[1])                      # a replay reads what its inputs hold then
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[1])
    K.check_status("gemm_i8")


# ------------------------------------------------------------------------------------------------ head norms and rotation
def rope64(x, w, positions, inv_freq, eps, interleaved, mult=1.0):
    """x [..., H, D] with positions [...]: the value in 64 bits and the bound of its fp32 arithmetic before the last rounding."""
    y, D, rot = x.double(), x.shape[-1], 2 * inv_freq.numel()
    rel = 0.0
    if w is not None:
        y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
        rel = (D / 2 + 8) * U
    angle = (positions.double().unsqueeze(-1) * inv_freq.double()).unsqueeze(-2)
    c, s = torch.cos(angle) * mult, torch.sin(angle) * mult
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    p, q, size = a * c - b * s, b * c + a * s, (a.abs() + b.abs()) * abs(mult)
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat([u, v], -1))
    # cos and sin: the angle in turns is rounded once (2^-25 of a turn, 2 pi 2^-25 in radians), their own error 2 ulp, the factor one rounding; then products and a sum
    off = torch.cat([join(size, size) * (rel + 2 * math.pi * 2.0 ** -25 + 8 * U), y[..., rot:].abs() * rel], -1)
    return torch.cat([join(p, q), y[..., rot:]], -1), off


def check_heads(got, x, w, positions, inv_freq, eps, interleaved, mult=1.0):
    want, off = rope64(x, w, positions, inv_freq, eps, interleaved, mult)
    within(got, want, off + half_eps(x.dtype) * (want.abs() + off) + 2.0 ** -25, "heads")


def freqs(rot, theta=10000.0):
    return (theta ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / max(rot, 1))).float()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hkv,D,rot", [(1, 1, 1, 1, 64, 64), (2, 5, 12, 12, 64, 32), (1, 37, 32, 8, 128, 128), (3, 200, 9, 3, 80, 40), (2, 300, 16, 2, 96, 96), (1, 33, 8, 1, 256, 64),
                                              (1, 7, 5, 2, 2, 2), (2, 9, 4, 4, 20, 20), (1, 11, 6, 3, 100, 50), (1, 6, 3, 1, 320, 128), (1, 530, 70, 5, 128, 0), (1, 4, 2, 2, 8, 8)])
def test_heads(K, B, S, Hq, Hkv, D, rot, interleaved, dtype):
    g = gen(D)
    q, k = ((torch.randn((B, S, H, D), generator=g, device="cuda") * 2).to(dtype) for H in (Hq, Hkv))
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2))
    pos = torch.randint(0, 130000, (B, S), generator=g, device="cuda", dtype=torch.int32)
    f = freqs(rot)
    for nq, nk in ((wq, wk), (None, None), (wq, None), (None, wk)):
        qo, ko = K.qk_norm_rope(q, k, pos, f, q_norm=nq, k_norm=nk, eps=1e-3, interleaved=interleaved)
        check_heads(qo, q, nq, pos, f, 1e-3, interleaved)
        check_heads(ko, k, nk, pos, f, 1e-3, interleaved)
    qo2, ko2 = K.qk_norm_rope(q, k, pos[0], f, wq, wk, interleaved=interleaved, mult=1.25)       # positions that the batch shares
    check_heads(qo2, q, wq, pos[:1].expand(B, S), f, 1e-6, interleaved, 1.25)
    check_heads(ko2, k, wk, pos[:1].expand(B, S), f, 1e-6, interleaved, 1.25)
    qi, ki = q.clone(), k.clone()                                                                # in place
    K.qk_norm_rope(qi, ki, pos[0], f, wq, wk, interleaved=interleaved, mult=1.25, q_out=qi, k_out=ki)
    assert torch.equal(qi, qo2) and torch.equal(ki, ko2)
    # [B, H, S, D] in memory, and heads of a fused projection
    qt, kt = q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(1, 2).contiguous().transpose(1, 2)
    got = K.qk_norm_rope(qt, kt, pos[0], f, wq, wk, interleaved=interleaved, mult=1.25)
    assert torch.equal(got[0], qo2) and torch.equal(got[1], ko2)
    fused = torch.cat([torch.zeros((B, S, 3), dtype=dtype, device="cuda"), q.flatten(2), k.flatten(2)], -1)
    fq, fk = fused[..., 3:3 + Hq * D].unflatten(-1, (Hq, D)), fused[..., 3 + Hq * D:].unflatten(-1, (Hkv, D))
    got = K.qk_norm_rope(fq, fk, pos[0], f, wq, wk, interleaved=interleaved, mult=1.25)
    if D % 8 == 0 and rot % 8 == 0 and D <= 256:            # other alignment, other kernel: the norm's sum has another order
        check_heads(got[0], q, wq, pos[:1].expand(B, S), f, 1e-6, interleaved, 1.25)
    else:
        assert torch.equal(got[0], qo2) and torch.equal(got[1], ko2)
    K.check_status("qk_norm_rope")


@pytest.mark.gpu
def test_heads_far_positions_and_values_that_are_not_finite(K):
    q = torch.randn((1, 6, 2, 128), generator=gen(1), device="cuda").bfloat16()
    k = torch.randn((1, 6, 1, 128), generator=gen(2), device="cuda").bfloat16()
    pos = torch.tensor([0, 1, 131071, 10 ** 6, 2 ** 31 - 1, -5], dtype=torch.int32, device="cuda")
    f = freqs(128, 500000.0)
    qo, ko = K.qk_norm_rope(q, k, pos, f)
    check_heads(qo, q, None, pos[None], f, 0, False)
    check_heads(ko, k, None, pos[None], f, 0, False)
    assert torch.equal(qo[0, 0], q[0, 0])                   # position 0 turns nothing
    q[0, 1, 0, 100] = math.nan
    k[0, 2, 0, 3] = math.inf
    w = torch.ones(128, device="cuda").bfloat16()
    qn, kn = K.qk_norm_rope(q, k, pos, f[:32], w, None)      # the first 64 dimensions turn
    assert qn[0, 1, 0].isnan().all() and qn[0, 1, 1].isfinite().all() and qn[0, 2:].isfinite().all()
    assert not kn[0, 2, 0, [3, 35]].isfinite().any() and kn[0, 2, 0, 64:].isfinite().all() and torch.equal(kn[0, :, 0, 64:], k[0, :, 0, 64:])
    z = torch.zeros_like(q)                                 # a head of zeros stays zero
    qz, _ = K.qk_norm_rope(z, k, pos, f, w, w)
    assert (qz == 0).all()


def u8_rows(values):
    """The byte cache's arithmetic in 64 bits: scale and zero point are rounded to fp16 before they are used."""
    mn, mx = values.amin(-1, keepdim=True), values.amax(-1, keepdim=True)
    return mn, mx


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,Hq,Hkv,D,rot,bs,interleaved,norms", [(1, 32, 8, 128, 128, 16, False, True), (64, 32, 8, 128, 128, 16, False, True), (3, 4, 2, 64, 32, 4, True, True),
                                                                 (700, 8, 8, 128, 64, 16, False, False), (40, 6, 3, 80, 80, 16, True, False), (19, 7, 1, 100, 20, 8, False, True),
                                                                 (600, 64, 8, 128, 128, 32, False, True), (5, 2, 1, 256, 256, 1, False, True)])
def test_append(K, T, Hq, Hkv, D, rot, bs, interleaved, norms, dtype):
    g = gen(T)
    pitch = (Hq + 2 * Hkv) * D
    qkv = (torch.randn((T, pitch), generator=g, device="cuda") * 2).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) if norms else None for _ in range(2))
    pos = torch.randint(0, 5000, (T,), generator=g, device="cuda", dtype=torch.int32)
    blocks = T // bs + 3
    slots = torch.randperm(blocks * bs, generator=g, device="cuda")[:T].to(torch.int32)
    dropped = torch.arange(T, device="cuda") % 5 == 3
    slots[dropped] = -1
    f = freqs(rot)
    kc, vc = (torch.full((blocks, Hkv, bs, D), 9.0, dtype=dtype, device="cuda") for _ in range(2))
    q_out = torch.full((T, Hq * D + 8), 5.0, dtype=dtype, device="cuda")
    before = qkv.clone()
    K.qk_norm_rope_kv_write(qkv, pos, slots, kc, vc, f, Hq, Hkv, D, bs, wq, wk, 1e-5, interleaved, q_out=q_out[:, :Hq * D])
    K.check_status("append")
    assert torch.equal(qkv, before) and (q_out[:, Hq * D:] == 5).all()
    heads = qkv.view(T, Hq + 2 * Hkv, D)
    check_heads(q_out[:, :Hq * D].reshape(T, Hq, D), heads[:, :Hq], wq, pos, f, 1e-5, interleaved)
    kept = ~dropped
    blk, at = slots[kept].long() // bs, slots[kept].long() % bs
    check_heads(kc[blk, :, at], heads[kept, Hq:Hq + Hkv], wk, pos[kept], f, 1e-5, interleaved)
    assert torch.equal(vc[blk, :, at], heads[kept, Hq + Hkv:])
    for c in (kc, vc):                                       # slots of no token stay as they were
        c[blk, :, at] = 9
        assert (c == 9).all()
    # queries in place: the same bits; keys and values of the projection stay
    K.qk_norm_rope_kv_write(qkv, pos, slots, kc, vc, f, Hq, Hkv, D, bs, wq, wk, 1e-5, interleaved)
    assert torch.equal(qkv[:, :Hq * D], q_out[:, :Hq * D]) and torch.equal(qkv[:, Hq * D:], before[:, Hq * D:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,D,rot,interleaved", [(1, 128, 128, False), (50, 128, 64, True), (600, 64, 64, False), (9, 96, 32, False), (5, 256, 256, True)])
def test_append_to_bytes(K, T, D, rot, interleaved, dtype):
    Hq, Hkv, bs, g = 4, 2, 16, gen(T)
    qkv = (torch.randn((T, (Hq + 2 * Hkv) * D), generator=g, device="cuda") * 2).to(dtype)
    qkv[0] = 0                                               # a row without a range
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2))
    pos = torch.arange(T, device="cuda", dtype=torch.int32) + 70
    slots = torch.randperm((T // bs + 2) * bs, generator=g, device="cuda")[:T].to(torch.int32)
    f = freqs(rot)
    kc, vc = (torch.full((T // bs + 2, Hkv, bs, D), 77, dtype=torch.uint8, device="cuda") for _ in range(2))
    km, vm = (torch.full((T // bs + 2, Hkv, bs, 2), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    q_out = torch.empty((T, Hq * D), dtype=dtype, device="cuda")
    K.qk_norm_rope_kv_write(qkv, pos, slots, kc, vc, f, Hq, Hkv, D, bs, wq, wk, 1e-5, interleaved, q_out=q_out, k_meta=km, v_meta=vm)
    K.check_status("append to bytes")
    heads, blk, at = qkv.view(T, Hq + 2 * Hkv, D), slots.long() // bs, slots.long() % bs
    check_heads(q_out.view(T, Hq, D), heads[:, :Hq], wq, pos, f, 1e-5, interleaved)
    keys, off = rope64(heads[:, Hq:Hq + Hkv], wk, pos, f, 1e-5, interleaved)
    for cache, meta, want, err in ((kc, km, keys, off), (vc, vm, heads[:, Hq + Hkv:].double(), torch.zeros_like(off))):
        rows, m = cache[blk, :, at].double(), meta[blk, :, at].double()
        scale, zp = m[..., :1], m[..., 1:]
        span = want.amax(-1, keepdim=True) - want.amin(-1, keepdim=True)
        e = err.amax(-1, keepdim=True)
        flat = span == 0
        within(scale, torch.where(flat, 1.0, span / 255), (2 * e / 255 + span / 255 * 8 * U) * (1 + 2.0 ** -10) + span / 255 * 2.0 ** -11 + 2.0 ** -25, "scale")
        # a code is off by half a step, and the fp16 scale and zero point can push the ends of a row over 0 or 255: 255 * 2^-11 of the scale's rounding and
        # up to 256 * 2^-11 of the zero point's
        within((rows - zp) * scale, want, scale * (0.5 + 255 * 2.0 ** -11 + 256 * 2.0 ** -11) + e + 8 * U * want.abs(), "values")
    kc[blk, :, at], vc[blk, :, at], km[blk, :, at], vm[blk, :, at] = 77, 77, 7, 7
    assert (kc == 77).all() and (vc == 77).all() and (km == 7).all() and (vm == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", [(1036, 3, 1, 128, 128), (2300, 12, 4, 64, 32), (1500, 5, 3, 80, 40), (1200, 9, 2, 256, 64), (4700, 2, 2, 96, 96)])
def test_many_tokens(K, T, Hq, Hkv, D, rot, interleaved, dtype):
    """From 1036 tokens on a warp works on whole tokens, in a form of the kernel of its own."""
    test_heads(K, 2, T // 2, Hq, Hkv, D, rot, interleaved, dtype)
    test_append(K, T, Hq, Hkv, D, rot, 16, interleaved, D != 64, dtype)
    test_append_to_bytes(K, T, D, rot, interleaved, dtype)


@pytest.mark.gpu
def test_slots_behind_the_cache_are_not_written(K):
    qkv = torch.randn((3, 4 * 64), generator=gen(1), device="cuda").bfloat16()
    big = torch.zeros((6, 1, 4, 64), dtype=torch.bfloat16, device="cuda")
    kc, vc = big[:2], torch.zeros_like(big[:2])
    slots = torch.tensor([5, 8, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    K.qk_norm_rope_kv_write(qkv, torch.arange(3, device="cuda", dtype=torch.int32), slots, kc, vc, freqs(64), 2, 1, 64, 4)
    assert K.read_status() == 5 and K.read_status() == 0
    assert (big[2:] == 0).all() and (kc[1, 0, 1] != 0).any() and (kc[0] == 0).all()


@pytest.mark.gpu
def test_append_agrees_with_the_older_writer(K):
    """Without norms, halves of whole heads and near positions, the rows are those of rope_kv_write up to the rounding of its angle in 32 bits."""
    T, Hq, Hkv, D, bs = 33, 8, 2, 128, 16
    qkv = torch.randn((T, (Hq + 2 * Hkv) * D), generator=gen(1), device="cuda").bfloat16()
    pos, slots = torch.arange(T, device="cuda", dtype=torch.int32), torch.arange(T, device="cuda", dtype=torch.int32) + 5
    caches = [torch.zeros((4, Hkv, bs, D), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    a, b = qkv.clone(), qkv.clone()
    K.rope_kv_write(a, pos, slots, caches[0], caches[1], Hq, Hkv, D, 10000.0, bs)
    K.qk_norm_rope_kv_write(b, pos, slots, caches[2], caches[3], freqs(D), Hq, Hkv, D, bs)
    for x, y in ((a[:, :Hq * D], b[:, :Hq * D]), (caches[0], caches[2])):
        # two roundings to bf16 of values that differ by 33 * 2^-22 of a pair's size at most
        assert ((x.double() - y.double()).abs() <= 2 * half_eps(torch.bfloat16) * x.double().abs() + 2.0 ** -15).all()
    assert torch.equal(caches[1], caches[3])


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("seqs,new,past", [(5, 1, 37), (3, 20, 0), (2, 70, 33)])
def test_front_of_a_layer(K, seqs, new, past):
    """Norm and quantisation, projection, head norms and rotation into the cache, attention over the pages, output projection with its residual: as a
    serving step runs them, against the same layer in 64 bits from the same codes."""
    H, Hq, Hkv, D, bs, eps, dtype = 512, 4, 2, 128, 16, 1e-5, torch.bfloat16
    T, g = seqs * new, gen(seqs)
    h = torch.randn((T, H), generator=g, device="cuda").to(dtype)
    gamma, wq, wk = ((1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(dtype) for n in (H, D, D))
    (w1, s1, z1), (w2, s2, z2) = weight((Hq + 2 * Hkv) * D, H, "unsigned", 1), weight(H, Hq * D, "signed", 2)
    per = -(-(past + new) // bs)
    order = torch.randperm(seqs * per + 1, generator=g, device="cuda")[:seqs * per].reshape(seqs, per)
    kc, vc = (torch.randn((seqs * per + 1, Hkv, bs, D), generator=g, device="cuda").to(dtype) for _ in range(2))
    at = torch.arange(past, past + new, device="cuda")
    pos = at.repeat(seqs).to(torch.int32)
    slots = (order[:, at // bs] * bs + at % bs).reshape(-1).to(torch.int32)
    f = freqs(D)
    rows = K.quantize_rows(h, norm=(gamma, eps))
    qkv = K.gemm(rows, K.PackedWeight.from_ir_i8(w1, s1, z1))
    raw = qkv.clone()
    K.qk_norm_rope_kv_write(qkv, pos, slots, kc, vc, f, Hq, Hkv, D, bs, wq, wk, eps)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    att = K.paged_attention(qkv, kc, vc, i32([past] * seqs), i32([i * new for i in range(seqs + 1)]), order.reshape(-1).to(torch.int32),
                            i32([i * per for i in range(seqs + 1)]), Hq, Hkv, D, max_context_len=past + new, max_q_len=new, block_size=bs)
    rows2 = K.quantize_rows(att)
    out = K.gemm(rows2, K.PackedWeight.from_ir_i8(w2, s2, z2), residual=h)
    K.check_status("layer")
    v, off = value64(rows, w1, s1, z1)
    within(raw, v, off + half_eps(dtype) * (v.abs() + off) + 2.0 ** -25, "projection")
    heads = raw.view(T, -1, D)
    q64, k64 = rope64(heads[:, :Hq], wq, pos, f, eps, False)[0], rope64(heads[:, Hq:Hq + Hkv], wk, pos, f, eps, False)[0]
    flat = lambda c: c.transpose(1, 2).reshape(-1, Hkv, D)
    att64 = torch.empty((T, Hq, D), dtype=torch.float64, device="cuda")
    for i in range(seqs):
        ctx = torch.arange(past + new, device="cuda")
        sl = order[i, ctx // bs] * bs + ctx % bs
        keys, vals = flat(kc)[sl].double(), flat(vc)[sl].double()
        keys[past:], vals[past:] = k64[i * new:(i + 1) * new], heads[i * new:(i + 1) * new, Hq + Hkv:].double()
        keys, vals = (t.repeat_interleave(Hq // Hkv, 1) for t in (keys, vals))
        sc = torch.einsum("qhd,khd->hqk", q64[i * new:(i + 1) * new], keys) / math.sqrt(D)
        mask = ctx[None, :] > torch.arange(past, past + new, device="cuda")[:, None]
        att64[i * new:(i + 1) * new] = torch.einsum("hqk,khd->qhd", sc.masked_fill(mask, -math.inf).softmax(-1), vals)
    # attention in bf16: its rounded queries, keys, probabilities and results are half a step off each, 2-norm
    assert float((att.double() - att64.reshape(T, -1)).norm() / att64.norm()) < 4 * half_eps(dtype)
    v, off = value64(rows2, w2, s2, z2)
    want = v + h.double()
    within(out, want, off + U * want.abs() + half_eps(dtype) * (want.abs() + off) + 2.0 ** -25, "output projection")


# ------------------------------------------------------------------------------------------------ refusals, before anything is launched
def cpu_weight():
    from openvino_b200.ops import cuda as K
    return K.PackedWeight(K.W_I8, torch.zeros(16384, dtype=torch.uint8), 128, 64, torch.ones(128), None, 64, None, tiled=True)


@pytest.mark.parametrize("call", [
    lambda K, x, w: K.gemm(x[0], w), lambda K, x, w: K.gemm(x.float(), w), lambda K, x, w: K.gemm(x[:, :63], w), lambda K, x, w: K.gemm(x, w, comm=object()),
    lambda K, x, w: K.gemm(x, w, splits=2), lambda K, x, w: K.gemm(x, w, block_t=16), lambda K, x, w: K.gemm(x, w, act=K.ACT_GLU_LIMITED),
    lambda K, x, w: K.gemm(x, w, out=torch.zeros((4, 127)).bfloat16()), lambda K, x, w: K.gemm(x, w, out=torch.zeros((4, 128))),
    lambda K, x, w: K.gemm(x, w, out=torch.zeros((4, 256)).bfloat16()[:, ::2]), lambda K, x, w: K.gemm(x, w, out=torch.zeros((1, 128)).bfloat16().expand(4, 128)),
    lambda K, x, w: K.gemm(x, w, residual=torch.zeros((4, 128)).half()), lambda K, x, w: K.gemm(x, w, residual=torch.zeros((3, 128)).bfloat16()),
    lambda K, x, w: K.gemm(K.QuantizedRows(torch.zeros((4, 64), dtype=torch.int8), torch.ones(4), torch.zeros(4, dtype=torch.int32), torch.bfloat16), w, norm=(x[0], 1e-5)),
    lambda K, x, w: K.gemm(x, w),                                                                          # not on a device
    lambda K, x, w: K.quantize_rows(x.float()), lambda K, x, w: K.quantize_rows(x[0]), lambda K, x, w: K.quantize_rows(x.t()), lambda K, x, w: K.quantize_rows(x[:, :0]),
    lambda K, x, w: K.quantize_rows(x, norm=(x[0, :63], 1e-5)), lambda K, x, w: K.quantize_rows(x, norm=(x[0].float(), 1e-5)),
    lambda K, x, w: K.quantize_rows(x, norm=(x[0], 1e-5, torch.zeros(3, dtype=torch.int64))), lambda K, x, w: K.quantize_rows(x),
    lambda K, x, w: K.PackedWeight.from_ir_i8(torch.zeros((4, 4)), torch.ones(4)), lambda K, x, w: K.PackedWeight.from_ir_i8(torch.zeros((4, 4), dtype=torch.int8), torch.ones(3)),
    lambda K, x, w: K.PackedWeight.from_ir_i8(torch.zeros((0, 4), dtype=torch.int8), torch.ones(0)),
    lambda K, x, w: K.PackedWeight.from_ir_i8(torch.zeros((1, 65537), dtype=torch.int8), torch.ones(1)),
    lambda K, x, w: K.PackedWeight.from_ir_i8(torch.zeros((4, 4), dtype=torch.int8), torch.ones(4), torch.zeros(4, dtype=torch.uint8)),
    lambda K, x, w: K.PackedWeight.from_ir_i8(torch.zeros((4, 4), dtype=torch.int8), torch.ones(4), bias=torch.zeros(4)),
    lambda K, x, w: K.PackedWeight.from_ir_i8(torch.zeros((4, 4), dtype=torch.int8), torch.ones(4)),
])
def test_products_are_refused(call):
    from openvino_b200.ops import cuda as K
    with pytest.raises(ValueError):
        call(K, torch.zeros((4, 64)).bfloat16(), cpu_weight())


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros((4, 64), dtype=torch.uint8)), dict(q=torch.zeros(64, dtype=torch.int8)), dict(q=torch.zeros((4, 60), dtype=torch.int8)),
    dict(q=torch.zeros((64, 4), dtype=torch.int8).t()), dict(q=torch.zeros((1, 64), dtype=torch.int8).expand(4, 64)), dict(scales=torch.ones(3)), dict(scales=torch.ones(4).half()),
    dict(scales=torch.ones((4, 1))), dict(scales=torch.ones(8)[::2]), dict(sums=torch.zeros(4)), dict(sums=torch.zeros(5, dtype=torch.int32)), dict(dtype=torch.float32),
])
def test_quantised_rows_hold_together(change):
    from openvino_b200.ops import cuda as K
    good = dict(q=torch.zeros((4, 64), dtype=torch.int8), scales=torch.ones(4), sums=torch.zeros(4, dtype=torch.int32), dtype=torch.bfloat16)
    assert K.QuantizedRows(**good).shape == (4, 64)
    with pytest.raises(ValueError):
        K.QuantizedRows(**dict(good, **change))


HEADS = dict(q=torch.zeros((1, 4, 2, 64)).half(), k=torch.zeros((1, 4, 1, 64)).half(), positions=torch.zeros(4, dtype=torch.int32), inv_freq=torch.ones(32))
APPEND = dict(qkv=torch.zeros((4, 256)).half(), positions=torch.zeros(4, dtype=torch.int32), slot_map=torch.zeros(4, dtype=torch.int32), k_cache=torch.zeros((3, 1, 16, 64)).half(),
              v_cache=torch.zeros((3, 1, 16, 64)).half(), inv_freq=torch.ones(32), Hq=2, Hkv=1, D=64, block_size=16)


@pytest.mark.parametrize("name,change", [
    ("heads", dict(q=torch.zeros((1, 4, 2, 64)))), ("heads", dict(k=torch.zeros((1, 4, 1, 64)).bfloat16())), ("heads", dict(k=torch.zeros((1, 5, 1, 64)).half())),
    ("heads", dict(q=torch.zeros((4, 2, 64)).half())), ("heads", dict(positions=torch.zeros(4, dtype=torch.int64))), ("heads", dict(positions=torch.zeros(3, dtype=torch.int32))),
    ("heads", dict(inv_freq=torch.ones(33))), ("heads", dict(inv_freq=torch.ones(32).half())), ("heads", dict(q_norm=torch.ones(64))), ("heads", dict(k_norm=torch.ones(63).half())),
    ("heads", {}),                                                                                        # not on a device
    ("append", dict(qkv=torch.zeros((4, 255)).half())), ("append", dict(qkv=torch.zeros((4, 256)))), ("append", dict(slot_map=torch.zeros(3, dtype=torch.int32))),
    ("append", dict(positions=torch.zeros(4, dtype=torch.int64))), ("append", dict(k_cache=torch.zeros((3, 1, 16, 64)).bfloat16())), ("append", dict(v_cache=torch.zeros((2, 1, 16, 64)).half())),
    ("append", dict(block_size=8)), ("append", dict(k_cache=torch.zeros((3, 1, 16, 64), dtype=torch.uint8), v_cache=torch.zeros((3, 1, 16, 64), dtype=torch.uint8))),
    ("append", dict(q_out=torch.zeros((4, 127)).half())), ("append", dict(q_out=torch.zeros((1, 128)).half().expand(4, 128))), ("append", dict(qkv=torch.zeros((1, 256)).half().expand(4, 256))),
    ("append", dict(Hkv=0)), ("append", {}),
])
def test_heads_are_refused(name, change):
    from openvino_b200.ops import cuda as K
    fn, args = (K.qk_norm_rope, HEADS) if name == "heads" else (K.qk_norm_rope_kv_write, APPEND)
    with pytest.raises(ValueError):
        fn(**dict(args, **change))


def test_the_library_refuses_what_it_cannot_run():
    """The C entry points themselves: arguments are looked at before anything touches a device."""
    import ctypes as C
    from openvino_b200.ops import cuda as K
    l = K.lib()
    buf = (C.c_uint8 * 4096)()
    p = (C.addressof(buf) + 255) // 256 * 256
    good = dict(x=p, x_scale=p, x_sum=p, w=p, w_scale=p, out=p, T=1, N=128, K=64, ldx=64, ldo=128)
    for change in (dict(x=None), dict(T=0), dict(N=-1), dict(K=65537, ldx=65552), dict(ldx=48), dict(ldx=72), dict(x=p + 8), dict(w=p + 16), dict(act=9), dict(act=4, N=130, ldo=130),
                   dict(act=4, bias=p), dict(out_f32=1, residual=p, ldr=128), dict(ldo=127), dict(residual=p, ldr=100)):
        a = K.GemmI8Args(**dict(good, **change))
        assert l.ovb_gemm_i8(C.byref(a), None) < 0, change
    good = dict(x=p, q=p, scale=p, sum=p, ldx=64, rows=1, cols=64, ldq=64)
    for change in (dict(q=None), dict(rows=0), dict(cols=0), dict(ldq=63), dict(ldx=-1), dict(row_idx=p)):
        assert l.ovb_quantize_rows(C.byref(K.QuantRowsArgs(**dict(good, **change))), None) < 0, change
    good = dict(q=p, k=p, q_out=p, k_out=p, positions=p, inv_freq=p, B=1, S=1, Hq=1, Hkv=1, D=64, rot=64)
    for change in (dict(q=None), dict(S=0), dict(D=63), dict(D=8192), dict(rot=66), dict(rot=3), dict(inv_freq=None), dict(k_out=None), dict(v=p), dict(kv_u8=1),
                   dict(k_cache=p, v=p, v_cache=p, slot_map=p, slots=16), dict(k_cache=p, v_cache=p, slot_map=p, slots=16, block_size=16),
                   dict(k_cache=p, v=p, v_cache=p, slot_map=p, slots=16, block_size=16, kv_u8=1),
                   dict(k_cache=p, v=p, v_cache=p, k_meta=p, v_meta=p, slot_map=p, slots=16, block_size=16, kv_u8=1, D=60, rot=60)):
        assert l.ovb_qk_norm_rope(C.byref(K.QkRopeArgs(**dict(good, **change))), None) < 0, change
    assert l.ovb_pack_i8(None, 0, p, 1, 1, C.c_int64(1), None) < 0
    assert l.ovb_pack_i8(C.c_void_p(p), 0, C.c_void_p(p + 4), 1, 1, C.c_int64(1), None) < 0
