"""Compressed weights whose graphs leave something out: zero points (missing ones are 0), a scale for every channel, or that hold unusual ones."""
import numpy as np
import pytest
import torch

import openvino_b200 as ov
from openvino_b200 import opset as ops
from openvino_b200 import properties as props
from openvino_b200._tensor import Tensor
from openvino_b200._types import Type
from openvino_b200.models import llama, ov_builders
from openvino_b200.models.llm_config import TINY_LLAMA
from openvino_b200.models.ov_builders import build_llama
from openvino_b200.runtime import llm_import

SMALL = TINY_LLAMA.with_(vocab_size=320)
RANGES = {"u4": (0, 16), "u8": (0, 256), "i8": (-128, 128)}


def product(kind, N, Kd, zero_point=None, one_scale=False, seed=3):
    """(model of one product with a compressed weight, the weight's values in 64 bits, what is added up without zero points)."""
    rng = np.random.default_rng(seed)
    q = rng.integers(*RANGES[kind], (N, Kd))
    s = np.full((1, 1), 0.0123, np.float16) if one_scale else ((0.5 + rng.random((N, 1))) / 100).astype(np.float16)
    x = ops.parameter([-1, Kd], "f32", "x")
    qt = Tensor(q.astype(np.float32)).astype(getattr(Type, kind)) if kind == "u4" else q.astype(np.uint8 if kind == "u8" else np.int8)
    w = ops.convert(ops.constant(qt), "f16")
    if zero_point is not None:
        w = ops.subtract(w, ops.constant(np.asarray(zero_point, np.float16)))
    w = ops.convert(ops.multiply(w, ops.constant(s)), "f32")
    z = 0.0 if zero_point is None else np.asarray(zero_point, np.float64)
    return ov.Model([ops.result(ops.matmul(x, w.output(0), False, True))], [x], "product"), (q - z) * s.astype(np.float64)


def check(m, w64, rows, precision, group):
    """The compiled product against the formula. Four roundings to 16 bits at most between the inputs and a result (row, scale, weight, result; the sums are held in
    32 bits); with quantised rows a value is half a step of a / 127 off, a the row's largest."""
    Kd = w64.shape[1]
    x = np.abs(np.random.default_rng(rows).standard_normal((rows, Kd))).astype(np.float32) + 0.25       # (one sign: a wrong zero point cannot cancel)
    cm = ov.Core().compile_model(m, "CUDA", {props.hint.inference_precision: precision, props.hint.dynamic_quantization_group_size: group})
    got = cm(x)[0].astype(np.float64)
    want = x.astype(np.float64) @ w64.T
    size = x.astype(np.float64) @ np.abs(w64).T
    eps = 2.0 ** -8 if precision == "bf16" else 2.0 ** -11
    bound = (4 * eps + 2.0 ** -11) * size
    if group:
        bound += x.max(1, keepdims=True) / 254 * (1 + 4 * eps) * np.abs(w64).sum(1)
    worst = float((np.abs(got - want) / bound).max())
    assert worst <= 1
    return cm


@pytest.mark.parametrize("kind", RANGES)
def test_missing_zero_points_are_zero_on_the_host(kind):
    m, w64 = product(kind, 24, 64)
    x = np.random.default_rng(1).standard_normal((5, 64)).astype(np.float32)
    assert np.abs(ov.Core().compile_model(m, "CPU")(x)[0] - x @ w64.T).max() < 2.0 ** -9 * (np.abs(x) @ np.abs(w64).T).max()


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["bf16", "f16"])
@pytest.mark.parametrize("group", [0, -1])
@pytest.mark.parametrize("kind,N,Kd", [("u8", 160, 128), ("u8", 75, 96), ("i8", 160, 128), ("i8", 75, 96), ("u4", 128, 128)])
def test_missing_zero_points_are_zero(kind, N, Kd, group, precision):
    m, w64 = product(kind, N, Kd)
    for rows in (1, 13):
        check(m, w64, rows, precision, group)


def without_zero_points(monkeypatch):
    """Weights of built decoders lose the Subtract of their zero points."""
    subtract = ov_builders.ops.subtract

    def bare(a, b):
        node = a.get_node() if hasattr(a, "get_node") else a
        return a if node.get_type_name() == "Convert" and node.input_value(0).get_element_type() in (Type.u4, Type.u8) else subtract(a, b)
    monkeypatch.setattr(ov_builders.ops, "subtract", bare)


@pytest.mark.parametrize("compress", ["int8", "int4"])
def test_missing_zero_points_are_zero_in_the_serving_import(compress, monkeypatch):
    without_zero_points(monkeypatch)
    cfg = SMALL.with_(group_size=0 if compress == "int8" else 128)
    _, parts = llm_import.analyze(build_llama(cfg, llama.random_float_state(cfg, seed=1, std=0.05), compress=compress))
    linears = list(parts["lin"].values()) + [parts["lm_head"]]
    assert all(v.compressed and not v.zp.any() and v.zp.shape == v.scales.shape for v in linears)


# ------------------------------------------------------------------------------------------------ zero points that are not whole numbers of the weight's type
def test_zero_points_between_whole_numbers_are_not_served(monkeypatch):
    subtract = ov_builders.ops.subtract

    def between(a, b):
        node = b.get_node() if hasattr(b, "get_node") else b
        if node.get_type_name() != "Convert" or node.input_value(0).get_element_type() != Type.u8:
            return subtract(a, b)
        z = np.float16(node.input_value(0).get_node().get_tensor_view().to_float32()) + np.float16(0.5)
        return subtract(a, ov_builders.constant(z))
    monkeypatch.setattr(ov_builders.ops, "subtract", between)
    cfg = SMALL.with_(group_size=0)
    with pytest.raises(llm_import.NotAnLlm, match="whole numbers"):
        llm_import.analyze(build_llama(cfg, llama.random_float_state(cfg, seed=1, std=0.05), compress="int8"))


@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, -1])
@pytest.mark.parametrize("kind,zero_point", [("u8", 127.5), ("u8", -3.0), ("u8", 300.0), ("i8", 0.5), ("i8", 130.0), ("u4", 7.5)])
def test_zero_points_outside_the_weights_type(kind, zero_point, group):
    """Such weights are multiplied as the graph says, expanded."""
    m, w64 = product(kind, 128, 128, zero_point)
    cm = check(m, w64, 13, "bf16", group)
    assert all(st["packed"] is None for st in cm.program.ctx.cache.values() if isinstance(st, dict) and "packed" in st)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, -1])
@pytest.mark.parametrize("kind,zero_point", [("u8", 0.0), ("u8", 255.0), ("i8", -128.0), ("i8", 127.0), ("u4", 15.0)])
def test_zero_points_at_the_ends_of_the_weights_type(kind, zero_point, group):
    m, w64 = product(kind, 128, 128, zero_point)
    check(m, w64, 13, "bf16", group)


# ------------------------------------------------------------------------------------------------ one scale for the whole weight
@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, -1])
@pytest.mark.parametrize("kind,N,Kd", [("u8", 160, 128), ("u8", 75, 96), ("i8", 75, 96), ("u4", 128, 128)])
@pytest.mark.parametrize("zero_point", [None, 5.0])
def test_one_scale_for_a_whole_weight(kind, N, Kd, zero_point, group):
    m, w64 = product(kind, N, Kd, zero_point, one_scale=True)
    for rows in (1, 13):
        check(m, w64, rows, "bf16", group)


def test_one_scale_for_a_whole_weight_in_the_serving_import(monkeypatch):
    multiply = ov_builders.ops.multiply

    def single(a, b, **kw):
        node = b.get_node() if hasattr(b, "get_node") else b
        if node.get_type_name() != "Constant" or not node.get_friendly_name().endswith("/scale"):
            return multiply(a, b, **kw)
        return multiply(a, ov_builders.constant(np.full((1, 1, 1), 0.01, np.float16)))
    monkeypatch.setattr(ov_builders.ops, "multiply", single)
    cfg = SMALL.with_(group_size=0)
    _, parts = llm_import.analyze(build_llama(cfg, llama.random_float_state(cfg, seed=1, std=0.05), compress="int8"))
    for v in list(parts["lin"].values()) + [parts["lm_head"]]:
        assert v.whole_rows and v.scales.shape == (v.N, 1) and bool((v.scales == float(np.float16(0.01))).all()) and v.zp.shape == (v.N, 1)


# ------------------------------------------------------------------------------------------------ weights, scales and zero points that are inputs
@pytest.mark.parametrize("inputs", [("w",), ("s",), ("z",), ("w", "s", "z"), ()])
def test_inputs_of_compressed_products_are_those_of_the_call(inputs):
    """The body of a folded block is called with the weights of one block after the other; nothing that was expanded for one call serves another."""
    from openvino_b200.runtime.cuda_plugin import GraphProgram
    rng = np.random.default_rng(5)
    N, Kd = 24, 64

    def values():
        return {"w": rng.integers(0, 256, (N, Kd)).astype(np.uint8), "s": (rng.random((N, 1)) / 50).astype(np.float32), "z": rng.integers(100, 150, (N, 1)).astype(np.uint8)}
    fixed = values()
    x = ops.parameter([-1, Kd], "f32", "x")
    nodes = {n: ops.parameter(list(v.shape), "f32" if n == "s" else "u8", n) if n in inputs else ops.constant(v) for n, v in fixed.items()}
    fc = ops.fully_connected_compressed(x, nodes["w"], ops.constant(np.zeros(0, np.float32)), nodes["s"], nodes["z"])
    prog = GraphProgram(ov.Model([ops.result(fc)], [x] + [nodes[n] for n in inputs], "block"), "cpu")
    for _ in range(3):
        v = {**fixed, **{n: t for n, t in values().items() if n in inputs}}
        a = rng.standard_normal((5, Kd)).astype(np.float32)
        got = prog.run([torch.from_numpy(a)] + [torch.from_numpy(v[n]) for n in inputs])[0].numpy()
        w64 = (v["w"].astype(np.float64) - v["z"]) * v["s"]
        assert np.abs(got - a @ w64.T).max() <= (Kd + 4) * 2.0 ** -24 * (np.abs(a) @ np.abs(w64).T).max()
