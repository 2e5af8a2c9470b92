"""Generation and distillation on two gloo ranks against one process: a rank
whose answers end early keeps step with the other; every rank's loss is that of
its own batch, the gradients are their mean over the ranks."""
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

import _lists_oracle as oracle
from tests._distillation_worker import K, NEW, STEPS, lists, prompts, run


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _greedy(hf, ids, new):
    for _ in range(new):
        with torch.no_grad():
            ids = torch.cat([ids, hf(input_ids=ids).logits[:, -1].argmax(-1, keepdim=True)], 1)
    return ids


@pytest.mark.parametrize("mode,grad", [("full", "gpu_reduce"), ("shard", "cpu_reduce")])
def test_two_ranks(tmp_path, mode, grad):
    transformers = pytest.importorskip("transformers")
    from test1_b200 import ops
    from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM

    cfg = LlamaConfig.tiny()
    torch.manual_seed(0)
    ours = LlamaForCausalLM(cfg)
    hf = transformers.LlamaForCausalLM(cfg.to_hf()).float()
    hf.load_state_dict({n: p.detach().clone() for n, p in ours.named_parameters()})
    free = [_greedy(hf, prompts(cfg, r), NEW) for r in range(2)]
    eos = int(free[0][0, 8])  # the first rank's first answer ends with its second token
    world, out, port = 2, str(tmp_path / "res"), _free_port()
    ctx = mp.get_context("spawn")
    procs = [ctx.Process(target=run, args=(r, world, port, mode, grad, eos, out)) for r in range(world)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=300)
    errs = [f for f in os.listdir(tmp_path) if ".err" in f]
    assert not errs, open(os.path.join(tmp_path, errs[0])).read()
    res = [torch.load(out + f".{r}") for r in range(world)]
    opt = torch.optim.AdamW(hf.parameters(), lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    for r in range(world):
        assert res[r]["refused"] == 2  # answers of other lengths than the other rank's
        a = res[r]["answers"]
        for b in range(2):
            answer = free[r][b, 7:].tolist()
            n = answer.index(eos) + 1 if eos in answer else NEW
            assert int(a["lengths"][b]) == 7 + n and a["labels"][b, 7:7 + n].tolist() == answer[:n]
            assert bool((a["labels"][b, 7 + n:] == -100).all())
        with torch.no_grad():
            want, _ = torch.log_softmax(hf(input_ids=a["input_ids"]).logits, -1).topk(K, -1)
        assert torch.allclose(res[r]["top"][0], want, atol=2e-5)
    for step in range(STEPS):
        opt.zero_grad()
        for r in range(world):
            a = res[r]["answers"]
            logps, ids = lists(cfg, r, a["input_ids"].shape)
            keep = ops.shift_labels(a["labels"]).view(*a["labels"].shape, 1) >= 0
            lp = torch.log_softmax(hf(input_ids=a["input_ids"]).logits, -1).gather(2, ids).reshape(-1, K)
            loss, grad_lp, _, _ = oracle.distillation(lp.detach(), logps.view(-1, K), torch.where(keep, ids, -1).view(-1, K),
                                                      "forward", True)
            (lp * (grad_lp.float() / world)).sum().backward()
            assert abs(res[r]["losses"][step] - float(loss)) < 1e-4 * max(1.0, float(loss))
        opt.step()
    for n, p in hf.named_parameters():
        d = (res[0]["master"][n].view(p.shape) - p.detach()).abs()
        # Adam moves an element of ~0 gradient by up to lr on rounding alone
        assert (d > 1e-4).float().mean().item() < 2e-3, n
