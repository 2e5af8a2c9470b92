"""Worker of the two-rank generation and distillation test (gloo, CPU)."""
import os
import sys
import traceback

import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

STEPS, NEW, K = 2, 5, 6


def prompts(cfg, rank):
    return torch.randint(0, cfg.vocab_size, (2, 7), generator=torch.Generator().manual_seed(60 + rank))


def lists(cfg, rank, shape):
    g = torch.Generator().manual_seed(70 + rank)
    return torch.log_softmax(2 * torch.randn(*shape, cfg.vocab_size, generator=g), -1).topk(K, -1)


def run(rank, world, port, mode, grad, eos, out_path):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), LOCAL_WORLD_SIZE=str(world), LOCAL_RANK=str(rank),
                      T1_QUIET="1")
    try:
        from datetime import timedelta

        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=120))
        from test1_b200 import DistillationObjective, SlideFSDPConfig
        from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM
        from test1_b200.slide_fsdp import SlideFSDP

        cfg = LlamaConfig.tiny()
        torch.manual_seed(0)
        eng = SlideFSDP(LlamaForCausalLM(cfg), SlideFSDPConfig(dtype=torch.float32, device="cpu", lr=1e-3, weight_decay=0.01,
                                                               param_transfer_mode=mode, grad_sync_mode=grad))
        answers = eng.generate(prompts(cfg, rank), NEW, top_k=1, eos_token_id=eos)
        refused = 0
        for new, end in [(NEW + rank, eos), (NEW, eos if rank else None)]:
            try:
                eng.generate(prompts(cfg, rank), new, top_k=1, eos_token_id=end)
            except ValueError:
                refused += 1
        top = eng.top_logprobs(answers.input_ids, K)
        logps, ids = lists(cfg, rank, answers.input_ids.shape)
        losses = []
        for _ in range(STEPS):
            out = eng(input_ids=answers.input_ids, labels=answers.labels, objective=DistillationObjective(),
                      teacher_logps=logps, teacher_ids=ids)
            losses.append(float(out.loss))
        eng.wait_for_updates()
        dist.barrier()
        res = {"losses": losses, "answers": vars(answers), "top": top, "refused": refused}
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
