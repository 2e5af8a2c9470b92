"""Edges of the plain loss operators: what the kernels do there, they do."""
import pytest
import torch

from test1_b200 import ops


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("kl_coef", [0.0, 0.1])
def test_policy_loss_of_no_sequences(reduction, kl_coef):
    none, ids = torch.zeros(0), torch.zeros(0, dtype=torch.int64)
    loss, dlogp, stats = ops.policy_loss_fwd_bwd(none, none, none if kl_coef else None, none, ids, 8, kl_coef=kl_coef,
                                                 reduction=reduction)
    assert float(loss) == 0 and dlogp.shape == (0,) and stats.tolist() == [0.0, 0.0]
