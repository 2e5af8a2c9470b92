"""An expired wait of a kernel reaches the user: the engine reports the error
word that the kernel sets (here the test sets it) instead of going on with
unfinished results."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def engine(cuda_device):
    from test1_b200 import SlideFSDP, SlideFSDPConfig
    from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM
    from test1_b200.ops import native

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=1000, hidden_size=256, intermediate_size=512, num_hidden_layers=1,
                      num_attention_heads=2, num_key_value_heads=1)
    eng = SlideFSDP(LlamaForCausalLM(cfg, device="meta"), SlideFSDPConfig(dtype=torch.bfloat16, device=cuda_device))
    yield eng
    native.gemm_error(reset=True)
    eng.close()


@pytest.mark.parametrize("training", [False, True])
def test_expired_wait_is_reported(training, engine):
    from test1_b200 import PreferenceObjective
    from test1_b200.ops import native

    ids = torch.randint(0, 1000, (2, 128))
    step = (lambda: engine(input_ids=ids, labels=ids, objective=PreferenceObjective())) if training else \
        (lambda: engine.token_logprobs(ids, ids))  # noqa: E731
    step()
    engine.wait_for_updates()
    native.error_word().fill_(131)
    step()
    with pytest.raises(RuntimeError, match="131"):
        engine.wait_for_updates()
    for after in (lambda: engine(input_ids=ids, labels=ids), lambda: engine.token_logprobs(ids, ids)):
        with pytest.raises(RuntimeError, match="131"):
            after()
