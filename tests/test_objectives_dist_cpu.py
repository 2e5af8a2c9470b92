"""Objectives on two gloo ranks against one process: every rank's loss is that
of its own batch, the gradients are their mean over the ranks (AdamW on the HF
model, as in the cross-entropy test)."""
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

from tests._objective_worker import STEPS, batch, run
from tests.test_objectives_cpu import _hf_loss, _label_logps


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


@pytest.mark.parametrize("kind,mode,grad", [("preference", "full", "gpu_reduce"), ("policy", "shard", "gpu_reduce"),
                                            ("policy", "full", "cpu_reduce")])
def test_two_ranks_match_autograd(tmp_path, kind, mode, grad):
    transformers = pytest.importorskip("transformers")
    from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM

    world, out, port = 2, str(tmp_path / "res"), _free_port()
    ctx = mp.get_context("spawn")
    procs = [ctx.Process(target=run, args=(r, world, port, kind, mode, grad, out)) for r in range(world)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=300)
    errs = [f for f in os.listdir(tmp_path) if ".err" in f]
    assert not errs, open(os.path.join(tmp_path, errs[0])).read()
    res = [torch.load(out + f".{r}") for r in range(world)]

    cfg = LlamaConfig.tiny()
    torch.manual_seed(0)
    ours = LlamaForCausalLM(cfg)
    hf = transformers.LlamaForCausalLM(cfg.to_hf()).float()
    hf.load_state_dict({n: p.detach().clone() for n, p in ours.named_parameters()})
    opt = torch.optim.AdamW(hf.parameters(), lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    data = [batch(cfg, r) for r in range(world)]
    with torch.no_grad():
        refs = [_label_logps(hf, ids, labels)[0] for ids, labels, _, _ in data]
    for r in range(world):
        assert torch.allclose(res[r]["ref"], refs[r], atol=2e-5)
    for step in range(STEPS):
        opt.zero_grad()
        for r, (ids, labels, adv, noise) in enumerate(data):
            lp, tg = _label_logps(hf, ids, labels)
            loss = _hf_loss(kind, lp, tg, refs[r], refs[r] + noise, adv)
            (loss / world).backward()
            assert abs(res[r]["losses"][step] - float(loss.detach())) < 1e-4 * max(1.0, abs(float(loss.detach())))
        opt.step()
    for n, p in hf.named_parameters():
        d = (res[0]["master"][n].view(p.shape) - p.detach()).abs()
        # Adam moves an element of ~0 gradient by up to lr on rounding alone
        assert (d > 1e-4).float().mean().item() < 2e-3, n
