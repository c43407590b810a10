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


# ------------------------------------------------------------------------------------------------ outputs that share memory (host)
def elements(t):
    """Addresses of all elements, in elements of the tensor's storage."""
    at = torch.tensor(t.storage_offset())
    for n, st in zip(t.shape, t.stride()):
        at = at.unsqueeze(-1) + torch.arange(n) * st
    return set(at.reshape(-1).tolist())


def views(B, S, D, H, other):
    """Views [B, S, H, D] of one buffer: fused rows, in several orders of dimensions, at several places."""
    buf = torch.zeros(4 * B * S * (H + other) * D + 64)
    W = (H + other) * D
    for off in (0, D, H * D, other * D, W, B * S * H * D, B * S * W, 7):
        yield buf.as_strided((B, S, H, D), (S * W, W, D, 1), off)
        yield buf.as_strided((B, S, H, D), (S * H * D, D, S * D, 1), off)
        yield buf.as_strided((B, S, H, D), (S * H * D, H * D, D, 1), off)
        yield buf.as_strided((B, S, H, D), (W, B * W, D, 1), off)


@pytest.mark.parametrize("B,S,D", [(1, 1, 4), (1, 3, 4), (2, 1, 4), (2, 3, 4)])
def test_places_apart_are_told_by_strides(B, S, D):
    """`_apart` never calls views apart that share an element, and knows the parts of fused rows."""
    from openvino_b200.ops import cuda as K
    seen = 0
    for a in views(B, S, D, 2, 3):
        base = a.untyped_storage().data_ptr()
        mine = elements(a)
        whole = torch.empty(0).set_(a.untyped_storage())
        for st, off in {(v.stride(), v.storage_offset()) for v in views(B, S, D, 3, 2)}:
            b = whole.as_strided((B, S, 3, D), st, off)
            assert b.untyped_storage().data_ptr() == base
            if K._apart(a, b):
                seen += 1
                assert not mine & elements(b), (a.stride(), a.storage_offset(), st, off)
    assert seen
    fused = torch.zeros((B, S, 8 * D))
    q, k, v = (fused[..., c * D:(c + n) * D].view(B, S, n, D) for c, n in ((0, 4), (4, 2), (6, 2)))
    assert K._apart(q, k) and K._apart(k, q) and K._apart(v, q) and K._apart(k, v) and not K._apart(q, q) and not K._apart(q, fused[..., 3 * D:5 * D].view(B, S, 2, D))


@pytest.mark.gpu
def test_outputs_that_share_memory_are_refused(K):
    g = gen(1)
    rows = torch.randn((2, 5, 8 * 64), generator=g, device="cuda").bfloat16()
    part = lambda t, c, n: t[..., c * 64:(c + n) * 64].view(2, 5, n, 64)
    q, k = part(rows, 0, 4), part(rows, 4, 4)
    pos, f = torch.arange(5, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
    want = [t.clone() for t in K.qk_norm_rope(q, k, pos, f)]
    other = torch.empty_like(rows)
    for q_out, k_out in ((k, None), (None, q), (k, q), (q, q), (part(rows, 1, 4), None), (None, part(rows, 3, 4)), (part(other, 0, 4), part(other, 3, 4)), (part(other, 0, 4), part(other, 0, 4)),
                         (q, part(rows, 3, 4)), (k.clone().flip(0)[:0], None)):
        with pytest.raises(ValueError):
            K.qk_norm_rope(q, k, pos, f, q_out=q_out, k_out=k_out)
    with pytest.raises(ValueError):
        K.qk_norm_rope(q, q, pos, f, q_out=q, k_out=part(other, 0, 4))                  # keys that are read while the queries in their place are written
    got = K.qk_norm_rope(q, k, pos, f, q_out=part(other, 0, 4), k_out=part(other, 4, 4))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    same = rows.clone()
    K.qk_norm_rope(part(same, 0, 4), part(same, 4, 4), pos, f, q_out=part(same, 0, 4), k_out=part(same, 4, 4))
    assert torch.equal(part(same, 0, 4), want[0]) and torch.equal(part(same, 4, 4), want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 6])
def test_append_keeps_queries_off_the_heads_it_reads(K, T):
    g, Hq, Hkv, D = gen(2), 4, 2, 64
    wide = torch.randn((T, 16 * D), generator=g, device="cuda").bfloat16()
    pos, slots, f = torch.arange(T, dtype=torch.int32, device="cuda"), torch.arange(T, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda")
    kc, vc = (torch.zeros((1, Hkv, 16, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    run = lambda rows, q_out: K.qk_norm_rope_kv_write(rows, pos, slots, kc, vc, f, Hq, Hkv, D, 16, q_out=q_out)
    want = torch.empty((T, Hq * D), dtype=torch.bfloat16, device="cuda")
    run(wide[:, :8 * D], want)
    for at in (1, 4, 6, 7):                                                             # over keys, values and a part of the queries
        with pytest.raises(ValueError):
            run(wide[:, :8 * D], wide[:, at * D:(at + 4) * D])
    for at in (0, 8, 12):                                                               # the queries' place, columns behind the heads
        rows = wide.clone()
        run(rows[:, :8 * D], rows[:, at * D:(at + 4) * D])
        assert torch.equal(rows[:, at * D:(at + 4) * D], want)
    rows = torch.cat([wide, wide])
    run(rows[:T, :8 * D], rows[T:, :4 * D])                                             # rows behind the last
    assert torch.equal(rows[T:, :4 * D], want)


# ------------------------------------------------------------------------------------------------ launches that are counted
def kernels_of(call):
    """Kernel nodes of a captured call."""
    from cuda.bindings import runtime as rt
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
    raw = rt.cudaGraph_t(g.raw_cuda_graph())
    err, nodes, n = rt.cudaGraphGetNodes(raw, 0)
    assert int(err) == 0
    err, nodes, n = rt.cudaGraphGetNodes(raw, n)
    assert int(err) == 0
    kinds = [rt.cudaGraphNodeGetType(node) for node in nodes[:n]]
    return sum(kind == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for _, kind in kinds)


@pytest.mark.gpu
@pytest.mark.parametrize("N,Kd", [(256, 512), (4096, 16384), (4224, 16384), (28672, 4096), (128, 500), (128, 16392)])
@pytest.mark.parametrize("T", [1, 2, 300])
def test_launches_are_told(K, T, N, Kd):
    w = torch.randint(-128, 128, (N, Kd), generator=gen(1), device="cuda", dtype=torch.int8)
    pw = K.PackedWeight.from_ir_i8(w, torch.full((N,), 0.01, device="cuda"))
    x = torch.randn((T, Kd), generator=gen(2), device="cuda").bfloat16()
    assert kernels_of(lambda: K.gemm(x, pw)) == K.gemm_i8_launches(T, pw)


# ------------------------------------------------------------------------------------------------ operands that do not belong together (host)
def test_quantised_rows_are_refused_where_rows_are_expected():
    from openvino_b200.ops import cuda as K
    rows = K.QuantizedRows(torch.zeros((4, 64), dtype=torch.int8), torch.ones(4), torch.zeros(4, dtype=torch.int32), torch.bfloat16)
    for mode in (K.W_BF16, K.W_U8, K.W_F32):
        with pytest.raises(ValueError):
            K.gemm(rows, K.PackedWeight(mode, torch.zeros((128, 64)).bfloat16(), 128, 64))
    with pytest.raises(ValueError):
        K.quantize_rows(rows)


def test_packed_structures_are_as_long_as_the_librarys():
    """The formats that calls are packed with, and the same structures field by field."""
    import ctypes as C
    from openvino_b200.ops import cuda as K
    for packed, fields in ((K._QUANT_ROWS, K.QuantRowsArgs), (K._GEMM_I8, K.GemmI8Args), (K._QK_ROPE, K.QkRopeArgs)):
        assert packed.size == C.sizeof(fields)
        values = [i + 1 for i in range(len(fields._fields_))]
        raw = fields.from_buffer_copy(packed.pack(*values))
        assert [getattr(raw, f[0]) for f in fields._fields_] == values


# ------------------------------------------------------------------------------------------------ rows whichever kernel quantises them
@pytest.mark.gpu
@pytest.mark.parametrize("cols", [700, 2048, 4100, 8192, 14336])
def test_rows_among_few_and_many(K, cols):
    """From 512 rows on other kernels quantise them. Without a norm the bits are the same; with one the codes and their sums are, and the scales are as far apart as two
    sums of squares of `cols` terms may be, 2 cols U, half of that behind the root, next to eight roundings on each side."""
    x = torch.randn((512, cols), generator=gen(cols), device="cuda").bfloat16()
    gamma = (1 + 0.3 * torch.randn(cols, generator=gen(2), device="cuda")).bfloat16()
    for norm in (None, (gamma, 1e-5)):
        few, many, one = K.quantize_rows(x[:511], norm=norm), K.quantize_rows(x, norm=norm), K.quantize_rows(x[7:8], norm=norm)
        assert torch.equal(few.q, many.q[:511]) and torch.equal(few.sums, many.sums[:511]) and torch.equal(one.q, many.q[7:8])
        if norm is None:
            assert torch.equal(few.scales, many.scales[:511])
        else:
            assert bool(((few.scales - many.scales[:511]).double().abs() <= (cols + 16) * U * few.scales.double()).all())
    K.check_status("quantize_rows")
