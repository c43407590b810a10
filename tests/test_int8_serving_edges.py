"""Serving program: single tokens whose products share K unevenly, decoders whose rotations are not those of all heads."""
import numpy as np
import pytest
import torch

import openvino_b200 as ov
from openvino_b200.models import llama, ov_builders
from openvino_b200.models.llm_config import TINY_LLAMA
from openvino_b200.models.ov_builders import build_llama
from openvino_b200.runtime import llm_import
from test_int8_serving import INT8_LOGITS, SMALL, executor, feed_of, off, paged, prefill


# ------------------------------------------------------------------------------------------------ single tokens whose products share K unevenly
@pytest.mark.gpu
@pytest.mark.parametrize("ffn", [1920, 1152, 4864])
def test_decode_steps_with_uneven_shares(ffn):
    """The down projection's blocks of 128 columns (15, 9 and 38) do not divide by the CTAs that share them."""
    from openvino_b200.ops import cuda as K
    cfg = TINY_LLAMA.with_(weight_format="int8", int8_activations=True, group_size=0, ffn_size=ffn)
    state = llama.random_float_state(cfg, seed=5, std=0.05)
    eff = {k: v.cuda() for k, v in llama.effective_state(cfg, state).items()}
    ex = executor(cfg, state, use_cuda_graphs=False)
    ids = torch.randint(0, cfg.vocab_size, (43,), generator=torch.Generator().manual_seed(1))
    want = llama.reference_logits(cfg, eff, ids.cuda())
    assert off(prefill(ex, ids[:40].numpy()), want[39]) < INT8_LOGITS
    for i in (40, 41, 42):
        assert off(prefill(ex, ids[i:i + 1].numpy(), i), want[i]) < INT8_LOGITS
    K.check_status("executor")


# ------------------------------------------------------------------------------------------------ heads that the position does not rotate
# the calls of _rope while a decoder of two layers is built: queries and keys of the first, then of the second
@pytest.mark.parametrize("left_out", [(2, 3), (0, 1), (1, 3), (0, 2), (3,), (0, 1, 2, 3)])
@pytest.mark.parametrize("in_pages", [False, True])
@pytest.mark.parametrize("norms", [False, True])
def test_heads_that_do_not_turn_are_refused(left_out, in_pages, norms, monkeypatch):
    cfg = SMALL.with_(qk_norm=norms)
    rope, count = ov_builders._rope, iter(range(100))
    monkeypatch.setattr(ov_builders, "_rope", lambda x, c, s, D: x if next(count) in left_out else rope(x, c, s, D))
    m = build_llama(cfg, llama.random_float_state(cfg, seed=1, std=0.05))
    with pytest.raises(llm_import.NotAnLlm, match="does not rotate"):
        llm_import.analyze(paged(m) if in_pages else m)


# ------------------------------------------------------------------------------------------------ cosines and sines that are not of one angle
def with_sine(monkeypatch, change):
    sin = ov_builders.ops.sin
    monkeypatch.setattr(ov_builders.ops, "sin", lambda a: change(sin, a))


@pytest.mark.parametrize("name,change", [
    ("factor of the sine", lambda sin, a: ov_builders.ops.multiply(sin(a), ov_builders.constant(np.array(1.5, np.float32)))),
    ("other direction", lambda sin, a: ov_builders.ops.negative(sin(a))),
    ("factor of its angles", lambda sin, a: sin(ov_builders.ops.divide(a, ov_builders.constant(np.array(2.0, np.float32))))),
    ("angles the other way", lambda sin, a: sin(ov_builders.ops.negative(a))),
])
@pytest.mark.parametrize("in_pages", [False, True])
def test_sines_that_do_not_belong_to_the_cosines_are_refused(name, change, in_pages, monkeypatch):
    with_sine(monkeypatch, change)
    m = build_llama(SMALL, llama.random_float_state(SMALL, seed=1, std=0.05))
    with pytest.raises(llm_import.NotAnLlm, match="sine"):
        llm_import.analyze(paged(m) if in_pages else m)


def test_rotations_the_other_way_are_read(monkeypatch):
    """Cosines and sines of negative angles: a table of negative frequencies, as the graph computes it."""
    cos, sin = ov_builders.ops.cos, ov_builders.ops.sin
    monkeypatch.setattr(ov_builders.ops, "cos", lambda a: cos(ov_builders.ops.negative(a)))
    monkeypatch.setattr(ov_builders.ops, "sin", lambda a: sin(ov_builders.ops.negative(a)))
    state = llama.random_float_state(SMALL, seed=4, std=0.05)
    m = build_llama(SMALL, state)
    got, _ = llm_import.analyze(m)
    assert np.allclose(got.inv_freq(), -np.array(SMALL.inv_freq()), rtol=1e-3) and not got.plain_rotation
    ids = np.array([[5, 9, 200, 17, 3]], dtype=np.int64)
    want = llama.reference_logits(SMALL.with_(rope_inv_freq=got.rope_inv_freq), {k: v.float() for k, v in state.items()}, torch.tensor(ids[0])).numpy()
    assert np.abs(ov.Core().compile_model(m, "CPU")(feed_of(ids))[0][0] - want).max() < 1e-3 * np.abs(want).max()


# ------------------------------------------------------------------------------------------------ launches of a step
@pytest.mark.gpu
@pytest.mark.parametrize("hidden,ffn,vocab", [(256, 512, 512), (4096, 8448, 512), (256, 512, 262208)])
def test_launches_of_a_step_are_counted(hidden, ffn, vocab):
    """The kernels of a step of one token and of several: those of the same decoder in 16 bits, and what its products launch more or less. Weights above 64 MB are
    not multiplied in the launch that quantises their row. (The attention is the same in both: its launches cancel.)"""
    from openvino_b200.ops import cuda as K
    from openvino_b200.runtime.cuda_llm import CudaLlmExecutor, LlmWeights, StepShape
    from test_int8_edges import kernels_of
    kernels, counted = {}, {}
    for name, more in (("whole numbers", dict(weight_format="int8", int8_activations=True, group_size=0)), ("16 bits", dict(weight_format="bf16"))):
        cfg = TINY_LLAMA.with_(qk_norm=True, hidden_size=hidden, ffn_size=ffn, vocab_size=vocab, **more)
        ex = CudaLlmExecutor(cfg, LlmWeights.random(cfg, "cuda"), num_kv_blocks=64, max_batch_tokens=16, max_seqs=4, use_cuda_graphs=False)
        for n in (1, 9):
            ids = np.arange(n)
            prefill(ex, ids)
            before = ex.kernel_launches
            ex._forward(ex.prefill, StepShape(n, 1, n, n))
            counted[name, n] = ex.kernel_launches - before
            kernels[name, n] = kernels_of(lambda: ex._forward(ex.prefill, StepShape(n, 1, n, n)))
    for n in (1, 9):
        assert counted["whole numbers", n] - counted["16 bits", n] == kernels["whole numbers", n] - kernels["16 bits", n]
    K.check_status("executor")


# ------------------------------------------------------------------------------------------------ biases
@pytest.mark.parametrize("which", ["q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"])
@pytest.mark.parametrize("compress", [None, "int8"])
@pytest.mark.parametrize("value", [0.0, 0.7])
def test_projections_with_biases_are_refused(which, compress, value, monkeypatch):
    """The serving program adds none; one of zeros adds nothing, where the graph's form lets it be seen."""
    matmul = ov_builders.ops.matmul

    def biased(*a, **kw):
        r = matmul(*a, **kw)
        if not str(kw.get("name") or "").endswith(which):
            return r
        return ov_builders.ops.add(r, ov_builders.constant(np.full((1, 1, r.output(0).get_partial_shape()[2].get_length()), value, np.float32)))
    monkeypatch.setattr(ov_builders.ops, "matmul", biased)
    m = build_llama(SMALL.with_(group_size=0), llama.random_float_state(SMALL, seed=1, std=0.05), compress=compress)
    if value == 0.0 and which in ("q_proj", "k_proj", "v_proj"):
        assert llm_import.analyze(m)[0].num_layers == 2
    elif value:
        with pytest.raises(llm_import.NotAnLlm):
            llm_import.analyze(m)


# ------------------------------------------------------------------------------------------------ neighbours paired
def neighbours(x, cos, sin, D):
    """The rotation of neighbouring pairs as graphs write it, from the builder's tables of halves side by side."""
    ops, _i64 = ov_builders.ops, ov_builders._i64
    cut = lambda t, b, e, step=1: ops.slice(t, _i64([b]), _i64([e]), _i64([step]), _i64([3])).output(0)
    S = x.get_partial_shape()[3].get_length()
    if D < S:
        return ops.concat([neighbours(cut(x, 0, D), cos, sin, D), cut(x, D, S)], 3).output(0)

    def spread(t):                              # [f0, f1, ..] -> [f0, f0, f1, f1, ..]
        half = ops.unsqueeze(cut(t, 0, D // 2), _i64([4])).output(0)
        return ops.reshape(ops.concat([half, half], 4), _i64([0, 0, 0, D]), True).output(0)
    odd, even = cut(x, 1, D, 2), cut(x, 0, D, 2)
    turned = ops.concat([ops.unsqueeze(ops.negative(odd), _i64([4])).output(0), ops.unsqueeze(even, _i64([4])).output(0)], 4)
    return ops.add(ops.multiply(x, spread(cos)), ops.multiply(ops.reshape(turned, _i64([0, x.get_partial_shape()[1].get_length(), -1, D]), True), spread(sin))).output(0)


@pytest.mark.parametrize("more", [{}, dict(rotary_dim=64), dict(qk_norm=True, rope_scale=1.25)])
@pytest.mark.parametrize("in_pages", [False, True])
def test_rotations_of_neighbours_are_recognised(more, in_pages, monkeypatch):
    monkeypatch.setattr(ov_builders, "_rope", neighbours)
    cfg = SMALL.with_(**more)
    state = llama.random_float_state(cfg, seed=4, std=0.05)
    m = build_llama(cfg, state)
    ids = np.array([[5, 9, 200, 17, 3]], dtype=np.int64)
    want = llama.reference_logits(cfg.with_(rope_interleaved=True), {k: v.float() for k, v in state.items()}, torch.tensor(ids[0])).numpy()
    assert np.abs(ov.Core().compile_model(m, "CPU")(feed_of(ids))[0][0] - want).max() < 1e-3 * np.abs(want).max()
    got, _ = llm_import.analyze(paged(m) if in_pages else m)
    assert got.rope_interleaved and got.rotary_dim == cfg.rotary_dim and got.qk_norm == cfg.qk_norm and abs(got.rope_scale - cfg.rope_scale) < 1e-6
    assert np.allclose(got.inv_freq(), cfg.inv_freq(), rtol=1e-3)
