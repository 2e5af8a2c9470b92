"""Worker of the two-rank objective test (gloo, CPU)."""
import os
import sys
import traceback

import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

B, S, STEPS = 4, 24, 2


def batch(cfg, rank):
    """Ids, labels with prompts and padding of the rank's own lengths, advantages."""
    g = torch.Generator().manual_seed(50 + rank)
    ids = torch.randint(0, cfg.vocab_size, (B, S), generator=g)
    labels = ids.clone()
    labels[:, :5 + 4 * rank] = -100
    labels[1, 16:] = -100
    return ids, labels, torch.randn(B, generator=g), 0.05 * torch.randn(B, S, generator=g)


def run(rank, world, port, kind, mode, grad, out_path):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), LOCAL_WORLD_SIZE=str(world), LOCAL_RANK=str(rank),
                      T1_QUIET="1")
    try:
        from datetime import timedelta

        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=120))
        from test1_b200 import PolicyObjective, PreferenceObjective, SlideFSDPConfig
        from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM
        from test1_b200.slide_fsdp import SlideFSDP

        cfg = LlamaConfig.tiny()
        torch.manual_seed(0)
        eng = SlideFSDP(LlamaForCausalLM(cfg), SlideFSDPConfig(dtype=torch.float32, device="cpu", lr=1e-3, weight_decay=0.01,
                                                               param_transfer_mode=mode, grad_sync_mode=grad))
        ids, labels, adv, noise = batch(cfg, rank)
        ref = eng.token_logprobs(ids, labels)
        losses = []
        for _ in range(STEPS):
            if kind == "preference":
                out = eng(input_ids=ids, labels=labels, objective=PreferenceObjective(beta=0.3), ref_logps=ref)
            else:
                out = eng(input_ids=ids, labels=labels, objective=PolicyObjective(kl_coef=0.1), ref_logps=ref,
                          old_logps=ref + noise, advantages=adv)
            losses.append(float(out.loss))
        eng.wait_for_updates()
        dist.barrier()
        res = {"losses": losses, "ref": ref}
        if rank == 0:
            res["master"] = {n: t.clone() for n, t in eng.named_master_tensors()}
        torch.save(res, out_path + f".{rank}")
        dist.barrier()
        eng.close()
        dist.destroy_process_group()
    except Exception:
        with open(out_path + f".err{rank}", "w") as f:
            f.write(traceback.format_exc())
        raise
