"""8-bit decoder-layer operators where their kernels' shares, paths and operands are uneven.

Tolerances count roundings as in test_int8_layer.py: U = 2^-24 is one to fp32, eps / 2 one to the 16-bit result type."""
import math

import pytest
import torch

U = 2.0 ** -24


@pytest.fixture(scope="module")
def K():
    from openvino_b200.ops import cuda as ops
    ops.lib()
    return ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def weight(N, Kd, zero_points, seed):
    g = gen(seed)
    w = torch.randint(-128, 128, (N, Kd), generator=g, device="cuda", dtype=torch.int8)
    z = torch.randint(-128, 128, (N,), generator=g, device="cuda", dtype=torch.int8) if zero_points else None
    return w, ((0.5 + torch.rand(N, generator=g, device="cuda")) / (74 * math.sqrt(Kd))).half(), z


def value64(rows, w, s, z):
    """The product's value, and what its fp32 roundings (conversion, two scales and their product) may take it off."""
    v = rows.q.double() @ (w.double() - (0 if z is None else z.double()[:, None])).T * rows.scales.double()[:, None] * s.double()
    return v, 4 * U * v.abs()


# ------------------------------------------------------------------------------------------------ one token, K shared by a cluster
# down projections whose blocks of 128 columns do not divide by the CTAs of a cluster, a small one, and widths that end inside a block
UNEVEN = [(4096, 11008), (896, 4864), (1536, 8960), (2048, 5632), (4096, 2304), (128, 1920), (384, 1928), (130, 3848)]


@pytest.mark.gpu
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("N,Kd", UNEVEN)
def test_one_token_with_uneven_shares(K, N, Kd, zero_points):
    """The row quantised in the product and before it: the same bits, and the formula's values."""
    w, s, z = weight(N, Kd, zero_points, N)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    for seed in range(3):
        x = torch.randn((1, Kd), generator=gen(seed), device="cuda").bfloat16()
        rows = K.quantize_rows(x)
        got = K.gemm(x, pw, out_f32=True)
        v, off = value64(rows, w, s, z)
        assert bool(((got.double() - v).abs() <= off).all())
        assert torch.equal(got, K.gemm(rows, pw, out_f32=True))
        residual = torch.randn((1, N), generator=gen(9), device="cuda").bfloat16()
        assert torch.equal(K.gemm(x, pw, residual=residual), K.gemm(rows, pw, residual=residual))
    K.check_status("gemm_i8")


@pytest.mark.gpu
@pytest.mark.parametrize("N,Kd", [(256, 1920), (11008 * 2 // 128 * 128, 2304), (1920, 4864)])
@pytest.mark.parametrize("zero_points", [False, True])
def test_one_token_gated_with_uneven_shares(K, N, Kd, zero_points):
    w, s, z = weight(N, Kd, zero_points, N)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    x = torch.randn((1, Kd), generator=gen(1), device="cuda").half()
    assert torch.equal(K.gemm(x, pw, act=K.ACT_SWIGLU), K.gemm(K.quantize_rows(x), pw, act=K.ACT_SWIGLU))
    K.check_status("gemm_i8")


@pytest.mark.gpu
@pytest.mark.parametrize("N", [128, 640, 4096])
def test_one_token_with_every_number_of_blocks(K, N):
    """K from 1 to 128 blocks of 128 columns, whole and with a last block of 72."""
    w, s, z = weight(N, 16384, True, N)
    x = torch.randn((1, 16384), generator=gen(2), device="cuda").bfloat16()
    wrong = []
    for blocks in range(1, 129):
        for Kd in (128 * blocks, 128 * blocks - 56):
            pw = K.PackedWeight.from_ir_i8(w[:, :Kd], s, z)
            row = x[:, :Kd]
            if not torch.equal(K.gemm(row, pw, out_f32=True), K.gemm(K.quantize_rows(row), pw, out_f32=True)):
                wrong.append(Kd)
    K.check_status("gemm_i8")
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("N,Kd", UNEVEN)
def test_one_normed_token_with_uneven_shares(K, N, Kd):
    """The norm's factor is in the scale alone: the codes are the same wherever the row is quantised, and sums of squares of n terms in two orders are 2 n U apart at
    most, their roots half of that, next to eight roundings on each side."""
    w, s, z = weight(N, Kd, True, N)
    pw = K.PackedWeight.from_ir_i8(w, s, z)
    x = torch.randn((1, Kd), generator=gen(4), device="cuda").bfloat16()
    gamma = (1 + 0.3 * torch.randn(Kd, generator=gen(5), device="cuda")).bfloat16()
    rows = K.quantize_rows(x, norm=(gamma, 1e-5))
    v, off = value64(rows, w, s, z)
    got = K.gemm(x, pw, out_f32=True, norm=(gamma, 1e-5))
    assert bool(((got.double() - v).abs() <= off + (Kd + 16) * U * v.abs()).all())
    many = torch.cat([torch.full_like(x, math.nan), x])                  # picked from several by its index
    pick = torch.ones(1, dtype=torch.int32, device="cuda")
    assert torch.equal(K.gemm(many, pw, out_f32=True, norm=(gamma, 1e-5, pick)), got)
    K.check_status("gemm_i8")
