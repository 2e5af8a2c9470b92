"""What the engine refuses of an objective's inputs, it refuses before anything
of the step has started: the calls after it run as before."""
import pytest
import torch

from test1_b200 import PolicyObjective, PreferenceObjective, SlideFSDPConfig
from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM
from test1_b200.slide_fsdp import SlideFSDP


@pytest.fixture
def engine():
    torch.manual_seed(0)
    eng = SlideFSDP(LlamaForCausalLM(LlamaConfig.tiny(), device="meta"), SlideFSDPConfig(dtype=torch.float32, device="cpu"))
    yield eng
    eng.close()


IDS = torch.arange(32).view(2, 16)


@pytest.mark.parametrize("bad", [dict(temperature=0.0), dict(temperature=float("inf")), dict(temperature=float("nan")),
                                 dict(labels=IDS[:1]), dict(labels=IDS[:, :8]), dict(labels=IDS.t()),
                                 dict(labels=IDS.reshape(-1))])
def test_refused_logprobs_leave_the_engine_usable(bad, engine):
    want = engine.token_logprobs(IDS, IDS)
    with pytest.raises(ValueError):
        engine.token_logprobs(**{**dict(input_ids=IDS, labels=IDS), **bad})
    assert torch.equal(engine.token_logprobs(IDS, IDS), want)


@pytest.mark.parametrize("labels", [IDS[:1], IDS[:, :8], IDS.t()])
def test_refused_labels_leave_the_engine_usable(labels, engine):
    with pytest.raises(ValueError):
        engine(input_ids=IDS, labels=labels, objective=PreferenceObjective())
    assert bool(torch.isfinite(engine(input_ids=IDS, labels=IDS, objective=PreferenceObjective()).loss))


@pytest.mark.parametrize("extra", [dict(old_logps=torch.zeros(2, 16)), dict(advantages=torch.zeros(2))])
def test_inputs_that_a_preference_objective_does_not_take(extra, engine):
    with pytest.raises(ValueError, match="does not take"):
        engine(input_ids=IDS, labels=IDS, objective=PreferenceObjective(), **extra)
    assert engine.completed_steps == 0


def test_label_smoothing_of_other_kinds_is_pointed_out(recwarn):
    PreferenceObjective(kind="sigmoid", label_smoothing=0.1)
    PreferenceObjective(kind="hinge")
    assert not [w for w in recwarn if "label_smoothing" in str(w.message)]
    for kind in ("hinge", "ipo"):
        with pytest.warns(UserWarning, match="label_smoothing"):
            PreferenceObjective(kind=kind, label_smoothing=0.1)
