"""Answer generation and distillation at the ends of what their calls take: the
least temperature, on the CPU."""
import math

import pytest
import torch

from test1_b200 import DistillationObjective, PolicyObjective, ops

LEAST = 2.0 ** -126


def test_temperatures_whose_inverse_fp32_does_not_have_are_refused():
    z, u, ids = torch.zeros(2, 8), torch.zeros(2), torch.zeros(2, 3, dtype=torch.int64)
    for tau in (LEAST * (1 - 2.0 ** -40), 1e-40, 1e-310):
        for call in (lambda: ops.topk_logprobs(z, 2, tau), lambda: ops.sample_tokens(z, u, tau),
                     lambda: ops.linear_topk_logprob_fwd(z, z, ids, tau),
                     lambda: ops.linear_topk_logprob_bwd(u[:, None].expand(2, 3), z, z, ids, u, z, z, tau),
                     lambda: DistillationObjective(temperature=tau), lambda: PolicyObjective(temperature=tau)):
            with pytest.raises(ValueError, match="2\\^-126"):
                call()


def test_the_least_temperature():
    """The largest logits have all the probability, each the same of it."""
    z = torch.tensor([[0.0, -1.0, 0.0, -1e-30]])
    logp, ids = ops.topk_logprobs(z, 3, LEAST)
    assert ids.tolist() == [[0, 2, 3]] and abs(float(logp[0, 0]) + math.log(2)) < 1e-6
    assert float(logp[0, 0]) == float(logp[0, 1]) and float(logp[0, 2]) < -1e7
    for u, token in ((0.0, 0), (0.49, 0), (0.51, 2), (0.99, 2)):
        assert int(ops.sample_tokens(z, torch.tensor([u]), LEAST)[0]) == token
