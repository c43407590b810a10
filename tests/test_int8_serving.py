"""8-bit products, head norms and other rotations in the serving program and in compiled graphs: import from graphs (host), executor and device (GPU)."""
import numpy as np
import pytest
import torch

import openvino_b200 as ov
from openvino_b200 import passes
from openvino_b200 import properties as props
from openvino_b200.models import llama, ov_builders
from openvino_b200.models.llm_config import TINY_LLAMA, TINY_MOE
from openvino_b200.models.ov_builders import build_llama
from openvino_b200.runtime import llm_import

SMALL = TINY_LLAMA.with_(vocab_size=320)
SCALED = tuple(float(f) for f in np.float32([500000.0 ** (-2.0 * i / 128) / (1.0 if i < 20 else 8.0) for i in range(64)]))
FORMS = {
    "head_norms": dict(qk_norm=True, qk_norm_eps=1e-3),
    "partial": dict(rotary_dim=64, rope_theta=10000.0),
    "scaled": dict(rope_inv_freq=SCALED),
    "all": dict(qk_norm=True, qk_norm_eps=1e-6, rotary_dim=32, rope_inv_freq=tuple(f / 4 for f in SCALED[:16])),
}
# relative error (2-norm) of logits of the 16-bit program against fp32, as in test_llm_engine.py
BF16_LOGITS = 3e-2
# What a product's quantised rows add: steps of a / 127 with a about 3.5 times the rows' rms, an error of 1 / sqrt(12) of a step. Nine products in a row
# (two layers and the vocabulary), errors added up in the worst case.
INT8_PRODUCT = 3.5 / 127 / 12 ** 0.5
INT8_LOGITS = BF16_LOGITS + 9 * INT8_PRODUCT


def paged(m):
    mgr = passes.Manager()
    mgr.register_pass(passes.SDPAToPagedAttention())
    mgr.run_passes(m)
    return m


def feed_of(ids):
    return {"input_ids": ids, "attention_mask": np.ones_like(ids), "position_ids": np.arange(ids.shape[1], dtype=np.int64)[None], "beam_idx": np.zeros(1, np.int32)}


# ------------------------------------------------------------------------------------------------ import
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("in_pages", [False, True])
def test_head_norms_and_rotations_are_recognised(form, in_pages, tmp_path):
    cfg = SMALL.with_(**FORMS[form])
    state = llama.random_float_state(cfg, seed=4, std=0.05)
    m = build_llama(cfg, state)
    # the graph computes what the reference model computes
    ids = np.array([[5, 9, 200, 17, 3]], dtype=np.int64)
    want = llama.reference_logits(cfg, {k: v.float() for k, v in state.items()}, torch.tensor(ids[0])).numpy()
    logits = ov.Core().compile_model(m, "CPU")(feed_of(ids))[0]
    assert np.abs(logits[0] - want).max() < 1e-3 * np.abs(want).max()
    if in_pages:
        paged(m)
    for i, n in enumerate(m.get_ops()):
        if n.get_type_name() not in ("Parameter", "Result"):
            n.set_friendly_name("op_%d" % i)
    ov.save_model(m, str(tmp_path / "m.xml"), compress_to_fp16=False)
    got, parts = llm_import.analyze(ov.Core().read_model(str(tmp_path / "m.xml")))
    assert (got.num_layers, got.num_heads, got.num_kv_heads, got.head_dim) == (2, 4, 2, 128)
    assert got.qk_norm == cfg.qk_norm and got.rotary_dim == cfg.rotary_dim and not got.rope_interleaved and not got.plain_rotation
    assert np.allclose(got.inv_freq(), cfg.inv_freq(), rtol=1e-3)
    assert (got.rope_inv_freq is not None) == (cfg.rope_inv_freq is not None)
    if cfg.qk_norm:
        assert abs(got.qk_norm_eps - cfg.qk_norm_eps) < 1e-9
        for l in range(2):
            for key in ("q_norm", "k_norm"):
                assert torch.allclose(parts["norms"][(l, key)], state["layers.%d.%s" % (l, key)].float())


@pytest.mark.parametrize("in_pages", [False, True])
def test_factors_of_the_rotation_are_recognised(in_pages):
    cfg = SMALL.with_(rope_scale=1.25)
    state = llama.random_float_state(cfg, seed=4, std=0.05)
    m = build_llama(cfg, state)
    ids = np.array([[5, 9, 200, 17, 3]], dtype=np.int64)
    want = llama.reference_logits(cfg, {k: v.float() for k, v in state.items()}, torch.tensor(ids[0])).numpy()
    assert np.abs(ov.Core().compile_model(m, "CPU")(feed_of(ids))[0][0] - want).max() < 1e-3 * np.abs(want).max()
    got, _ = llm_import.analyze(paged(m) if in_pages else m)
    assert abs(got.rope_scale - 1.25) < 1e-6 and got.rope_inv_freq is None and not got.plain_rotation


def test_angles_with_a_factor_are_another_table(monkeypatch):
    """positions * frequencies / 4: as if the frequencies were a quarter."""
    cos, sin = ov_builders.ops.cos, ov_builders.ops.sin
    quarter = lambda a: ov_builders.ops.divide(a, ov_builders.constant(np.array(4.0, dtype=np.float32)))
    monkeypatch.setattr(ov_builders.ops, "cos", lambda a: cos(quarter(a)))
    monkeypatch.setattr(ov_builders.ops, "sin", lambda a: sin(quarter(a)))
    got, _ = llm_import.analyze(build_llama(SMALL, llama.random_float_state(SMALL, seed=1, std=0.05)))
    assert got.rope_scale == 1.0 and np.allclose(got.inv_freq(), np.array(SMALL.inv_freq()) / 4, rtol=1e-3)


def test_norms_behind_the_rotation_are_refused(monkeypatch):
    rope = ov_builders._rope
    count = iter(range(100))
    monkeypatch.setattr(ov_builders, "_rope", lambda x, c, s, D: ov_builders._rms(rope(x, c, s, D), np.full(128, 1.5, np.float32), 1e-6, "late%d" % next(count)))
    with pytest.raises(llm_import.NotAnLlm, match="behind the rotation"):
        llm_import.analyze(build_llama(SMALL, llama.random_float_state(SMALL, seed=1, std=0.05)))


def test_rotations_and_epsilons_that_differ_are_refused(monkeypatch):
    state = llama.random_float_state(SMALL.with_(qk_norm=True), seed=1, std=0.05)
    rope, rms, calls = ov_builders._rope, ov_builders._rms, []

    def other(x, c, s, D):
        calls.append(1)
        f = ov_builders.constant(np.array(1.0 if len(calls) <= 2 else 1.5, dtype=np.float32))           # the second layer's cos and sin
        return rope(x, ov_builders.ops.multiply(c, f).output(0), ov_builders.ops.multiply(s, f).output(0), D)
    with monkeypatch.context() as m:
        m.setattr(ov_builders, "_rope", other)
        with pytest.raises(llm_import.NotAnLlm, match="rotations that differ"):
            llm_import.analyze(build_llama(SMALL, state))
    monkeypatch.setattr(ov_builders, "_rms", lambda x, g, eps, name: rms(x, g, 1e-3 if name.endswith("k_norm") else eps, name))
    with pytest.raises(llm_import.NotAnLlm, match="epsilon"):
        llm_import.analyze(build_llama(SMALL.with_(qk_norm=True), state))


def test_plain_decoders_keep_their_configuration():
    got, parts = llm_import.analyze(build_llama(SMALL, llama.random_float_state(SMALL, seed=1, std=0.05)))
    assert got.plain_rotation and not got.int8_activations and got.rope_inv_freq is None and (0, "q_norm") not in parts["norms"]
    assert abs(got.rope_theta / SMALL.rope_theta - 1) < 1e-3


def test_weights_with_one_scale_per_row_are_told_from_groups():
    state = llama.random_float_state(SMALL, seed=1, std=0.05)
    rows = llm_import.analyze(build_llama(SMALL.with_(group_size=0), state, compress="int8"))[1]["lin"]
    groups = llm_import.analyze(build_llama(SMALL, state, compress="int8"))[1]["lin"]
    fours = llm_import.analyze(build_llama(SMALL.with_(group_size=0), state, compress="int4"))[1]["lin"]
    assert all(v.whole_rows for v in rows.values()) and not any(v.whole_rows for v in groups.values()) and not any(v.whole_rows for v in fours.values())


@pytest.mark.parametrize("value,K,on", [(0, 64, False), (None, 64, False), ("0", 64, False), (-1, 64, True), (2 ** 64 - 1, 64, True), ("64", 64, True), (32, 64, False), (63, 64, False)])
def test_group_sizes_that_ask_for_whole_rows(value, K, on):
    assert llm_import.quantizes_rows(value, K) == on


def test_the_option_is_typed():
    from openvino_b200.runtime.cuda_plugin import CudaConfig
    name = props.hint.dynamic_quantization_group_size
    c = CudaConfig()
    assert c[name] == 0
    c.set_user_property({name: str(2 ** 64 - 1)})
    assert c[name] == 2 ** 64 - 1
    with pytest.raises(ValueError):
        c.set_user_property({name: -2})


def test_whole_number_products_are_not_summed_over_ranks():
    cfg = SMALL.with_(group_size=0)
    got, parts = llm_import.analyze(build_llama(cfg, llama.random_float_state(cfg, seed=1, std=0.05), compress="int8"))
    with pytest.raises(llm_import.NotAnLlm):
        llm_import.build_weights(got.with_(int8_activations=True), parts, "cpu", 0, 2)


# ------------------------------------------------------------------------------------------------ executor
def prefill(ex, ids, start=0, blocks=(3, 4, 5, 6, 7, 8, 9, 10)):
    """One sequence's tokens behind ``start`` earlier ones, in scattered blocks; logits of the last."""
    from openvino_b200.runtime.cuda_llm import StepShape
    n, sb = len(ids), ex.prefill
    v = {name: sb.view(name, host=0).numpy() for name in sb.offsets}
    at = np.arange(start, start + n)
    v["ids"][:n], v["positions"][:n] = ids, at
    v["slot_map"][:n] = np.array(blocks)[at // 16] * 16 + at % 16
    v["tok_src"][:n], v["tok_dst"][0], v["logit_idx"][0], v["past_lens"][0] = -1, -1, n - 1, start
    nb = -(-(start + n) // 16)
    v["subsequence_begins"][:2], v["block_indices_begins"][:2] = [0, n], [0, nb]
    v["block_indices"][:nb] = blocks[:nb]
    ex.upload(sb)
    ex.run(sb, StepShape(n, 1, n, start + n))
    torch.cuda.synchronize()
    return sb.logits[0].float()


def executor(cfg, state, **kw):
    from openvino_b200.runtime.cuda_llm import CudaLlmExecutor, LlmWeights
    return CudaLlmExecutor(cfg, LlmWeights.from_float(cfg, state, "cuda"), num_kv_blocks=64, max_batch_tokens=128, max_seqs=4, **kw)


def off(a, b):
    return float((a - b).norm() / b.norm())


EXECUTORS = {
    "head_norms": (dict(qk_norm=True, weight_format="bf16"), BF16_LOGITS),
    "interleaved": (dict(rope_interleaved=True, rotary_dim=64, weight_format="int4"), BF16_LOGITS),
    "scaled_norms_int4": (dict(qk_norm=True, rope_inv_freq=SCALED), BF16_LOGITS),
    "scaled_turns": (dict(rope_scale=1.25, rope_inv_freq=SCALED, weight_format="bf16"), BF16_LOGITS),
    "int8": (dict(weight_format="int8", int8_activations=True, group_size=0), INT8_LOGITS),
    "int8_head_norms": (dict(weight_format="int8", int8_activations=True, group_size=0, qk_norm=True, qk_norm_eps=1e-6), INT8_LOGITS),
}


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "u8"])
@pytest.mark.parametrize("name", EXECUTORS)
def test_logits_of_prefills_chunks_and_single_tokens(name, kv):
    from openvino_b200.ops import cuda as K
    more, bound = EXECUTORS[name]
    cfg = TINY_LLAMA.with_(**more)
    state = llama.random_float_state(cfg, seed=5, std=0.05)
    eff = {k: v.cuda() for k, v in llama.effective_state(cfg, state).items()}
    ex = executor(cfg, state, use_cuda_graphs=False, kv_cache_precision=kv)
    assert not ex._is_native()
    ids = torch.randint(0, cfg.vocab_size, (57,), generator=torch.Generator().manual_seed(1))
    want = llama.reference_logits(cfg, eff, ids.cuda())
    # a byte cache adds its own steps, of (max - min) / 255, about 6 rms / 255 / sqrt(12) of keys and values
    bound = bound + (4 * 6 / 255 / 12 ** 0.5 if kv == "u8" else 0)
    assert off(prefill(ex, ids[:40].numpy()), want[39]) < bound
    assert off(prefill(ex, ids[40:56].numpy(), 40), want[55]) < bound           # a chunk behind them
    assert off(prefill(ex, ids[56:].numpy(), 56), want[56]) < bound             # one token
    K.check_status("executor")


@pytest.mark.gpu
@pytest.mark.parametrize("more", [dict(weight_format="int8", int8_activations=True, group_size=0), dict(qk_norm=True, rope_inv_freq=SCALED)])
def test_experts(more):
    """Decoders with experts: their products in whole numbers, and head norms in front of their attention."""
    from openvino_b200.ops import cuda as K
    cfg = TINY_MOE.with_(**more)
    state = llama.random_float_state(cfg, seed=5, std=0.05)
    eff = {k: v.cuda() for k, v in llama.effective_state(cfg, state).items()}
    ex = executor(cfg, state, use_cuda_graphs=False)
    ids = torch.randint(0, cfg.vocab_size, (41,), generator=torch.Generator().manual_seed(2))
    want = llama.reference_logits(cfg, eff, ids.cuda())
    bound = INT8_LOGITS if cfg.int8_activations else BF16_LOGITS
    assert ex.int8 == cfg.int8_activations
    assert off(prefill(ex, ids[:40].numpy()), want[39]) < bound
    assert off(prefill(ex, ids[40:].numpy(), 40), want[40]) < bound
    K.check_status("experts")


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["int8_head_norms", "scaled_norms_int4"])
def test_generation_with_captured_steps(name):
    """Prompts of several lengths through the batching pipeline, decode steps as CUDA graphs: every token is the reference's best under the same earlier
    tokens or as close to it as the logits are known."""
    from openvino_b200.genai.pipeline import ContinuousBatchingPipeline, GenerationConfig
    from openvino_b200.genai.scheduler import SchedulerConfig
    from openvino_b200.ops import cuda as K
    more, bound = EXECUTORS[name]
    cfg = TINY_LLAMA.with_(**more)
    state = llama.random_float_state(cfg, seed=3, std=0.05)
    eff = {k: v.cuda() for k, v in llama.effective_state(cfg, state).items()}
    pipe = ContinuousBatchingPipeline(executor(cfg, state), SchedulerConfig(max_num_batched_tokens=48, max_num_seqs=4, num_kv_blocks=64))
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (5, 37, 70, 16)]
    res = pipe.generate(prompts, GenerationConfig(max_new_tokens=6))
    K.check_status("llm")
    assert pipe.metrics.decode_steps >= 5
    for p, r in zip(prompts, res):
        logits = llama.reference_logits(cfg, eff, torch.tensor(p + r.tokens[:-1], device="cuda"))
        for i, tok in enumerate(r.tokens):
            row = logits[len(p) - 1 + i]
            # both logits may be off: their errors are of `bound` rms each on average, eight times that for the difference of two single ones
            assert row[tok] >= row.max() - 8 * bound * row.square().mean().sqrt(), (i, tok, int(row.argmax()))


@pytest.mark.gpu
def test_a_captured_decode_step_replays_with_new_inputs():
    """The same decode step eagerly and from its graph, twice with other tokens."""
    from openvino_b200.runtime.cuda_llm import StepShape
    cfg = TINY_LLAMA.with_(weight_format="int8", int8_activations=True, group_size=0, qk_norm=True)
    state = llama.random_float_state(cfg, seed=6, std=0.05)
    ids = np.random.default_rng(0).integers(0, cfg.vocab_size, 30)
    rows = {}
    for graphs in (False, True):
        ex = executor(cfg, state, use_cuda_graphs=graphs)
        prefill(ex, ids)
        sb, out = ex.decode, []
        for step, tok in enumerate((7, 300, 41)):
            v = {n: sb.view(n, host=0).numpy() for n in sb.offsets}
            at = 30 + step
            v["ids"][0], v["positions"][0], v["slot_map"][0], v["past_lens"][0] = tok, at, (3 + at // 16) * 16 + at % 16, at
            v["tok_src"][0], v["tok_dst"][0], v["logit_idx"][0] = -1, -1, 0
            v["subsequence_begins"][:2], v["block_indices_begins"][:2], v["block_indices"][:3] = [0, 1], [0, 3], [3, 4, 5]
            ex.upload(sb)
            ex.run(sb, StepShape(1, 1, 1, at + 1))
            torch.cuda.synchronize()
            out.append(sb.logits[0].clone())
        rows[graphs] = out
    assert all(torch.equal(a, b) for a, b in zip(rows[False], rows[True]))
    assert not torch.equal(rows[True][0], rows[True][1])


# ------------------------------------------------------------------------------------------------ device
@pytest.mark.gpu
@pytest.mark.parametrize("in_pages", [False, True])
def test_serving_program_from_a_graph(in_pages):
    from openvino_b200.ops import cuda as K
    cfg = SMALL.with_(group_size=0, qk_norm=True)
    state = llama.random_float_state(cfg, seed=8, std=0.05)
    m = build_llama(cfg, state, compress="int8")
    if in_pages:
        paged(m)
    core = ov.Core()
    eff = {k: v.cuda() for k, v in llama.effective_state(cfg.with_(weight_format="int8"), state).items()}
    ids = np.random.default_rng(1).integers(0, cfg.vocab_size, 40)
    want = llama.reference_logits(cfg, eff, torch.tensor(ids, device="cuda"))[-1]
    for group, int8 in ((0, False), (-1, True), (256, False), (2 ** 64 - 1, True)):
        cm = core.compile_model(m, "CUDA", {props.cuda.serving_program: True, props.hint.dynamic_quantization_group_size: group})
        ex, _ = cm.create_llm_executor(max_num_seqs=2, max_num_batched_tokens=64, max_model_len=256)
        assert ex.int8 == int8 and ex.cfg.qk_norm and (ex.w.layers[0].qkv.mode == K.W_I8) == int8
        assert off(prefill(ex, ids, blocks=tuple(range(3, 11))), want) < (INT8_LOGITS if int8 else BF16_LOGITS)
    K.check_status("serving")


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["f16", "bf16"])
@pytest.mark.parametrize("signed", [False, True])
def test_compiled_graph_quantises_its_rows(precision, signed):
    """A two-layer perceptron with compressed weights: in whole numbers with the option, as before without it."""
    from openvino_b200 import opset as ops
    rng = np.random.default_rng(2)
    x = ops.parameter([-1, 96], "f32", "x")

    def dense(inp, N, Kd):
        q = rng.integers(0, 256, (N, 1, Kd)).astype(np.uint8)
        z = rng.integers(100, 150, (N, 1, 1)).astype(np.uint8)
        if signed:
            q, z = (q.astype(np.int32) - 128).astype(np.int8), (z.astype(np.int32) - 128).astype(np.int8)
        s = ((0.5 + rng.random((N, 1, 1))) / (74 * Kd ** 0.5)).astype(np.float16)
        w = ops.multiply(ops.subtract(ops.convert(ops.constant(q), "f16"), ops.convert(ops.constant(z), "f16")), ops.constant(s))
        w = ops.convert(ops.reshape(w, ops.constant(np.array([N, Kd], np.int64)), False), "f32")
        y = ops.matmul(inp, w.output(0), False, True)
        return ops.add(y, ops.constant(rng.standard_normal((1, N)).astype(np.float32)))

    m = ov.Model([ops.result(dense(ops.relu(dense(x, 160, 96)), 75, 160))], [x], "mlp")
    core = ov.Core()
    feed = rng.standard_normal((13, 96)).astype(np.float32)
    want = torch.from_numpy(core.compile_model(m, "CPU")(feed)[0].copy())
    eps = 2.0 ** -8 if precision == "bf16" else 2.0 ** -11
    errors = {}
    for group in (0, -1, 128):
        cm = core.compile_model(m, "CUDA", {props.hint.inference_precision: precision, props.hint.dynamic_quantization_group_size: group})
        req = cm.create_infer_request()
        got = [torch.from_numpy(req.infer([feed])[0].copy()) for _ in range(3)]            # eager, captured, replayed
        assert torch.equal(got[0], got[1]) and torch.equal(got[1], got[2])
        packed = [st["packed"].mode for st in cm.program.ctx.cache.values() if isinstance(st, dict) and st.get("packed") is not None]
        assert packed.count(5) == {0: 0, -1: 2, 128: 1}[group]                              # rows of 96 and of 160 values
        errors[group] = off(got[0], want)
        # two products in a row: inputs, weights, activations and results rounded to 16 bits, quantised rows
        assert errors[group] < 8 * eps + {0: 0, -1: 2, 128: 1}[group] * INT8_PRODUCT
    assert errors[-1] > errors[0]
