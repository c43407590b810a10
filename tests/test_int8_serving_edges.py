"""8-bit products in the serving program where shares of K are uneven."""
import pytest
import torch

from openvino_b200.models import llama
from openvino_b200.models.llm_config import TINY_LLAMA
from test_int8_serving import INT8_LOGITS, executor, off, prefill


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
