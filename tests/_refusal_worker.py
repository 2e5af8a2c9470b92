"""Worker of the test of refused arguments on two ranks (gloo, CPU)."""
import os
import sys
import traceback

import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def run(rank, world, port, out_path):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), LOCAL_WORLD_SIZE=str(world), LOCAL_RANK=str(rank),
                      T1_QUIET="1")
    try:
        from datetime import timedelta

        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=20))
        from test1_b200 import SlideFSDPConfig
        from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM
        from test1_b200.slide_fsdp import SlideFSDP

        cfg = LlamaConfig.tiny()
        torch.manual_seed(0)
        eng = SlideFSDP(LlamaForCausalLM(cfg), SlideFSDPConfig(dtype=torch.float32, device="cpu"))
        good = torch.randint(0, cfg.vocab_size, (2, 7))
        said = []
        for bad in (dict(input_ids=good + cfg.vocab_size), dict(input_ids=good[0]), dict(lengths=torch.tensor([8, 1])),
                    dict(max_new_tokens=0), dict(max_new_tokens=2.5), dict(top_p=0.0), dict(temperature=0.0),
                    dict(lengths="2")):
            for which in range(world):
                kw = dict(dict(input_ids=good, max_new_tokens=3), **(bad if rank == which else {}))
                try:
                    eng.generate(**kw)
                    said.append("taken")
                except (ValueError, TypeError, AttributeError) as e:
                    said.append("another" if "another rank" in str(e) else "own")
        a = eng.generate(good, 3)  # all keep step after all that
        torch.save({"said": said, "shape": tuple(a.input_ids.shape)}, out_path + f".{rank}")
        dist.barrier()
        eng.close()
        dist.destroy_process_group()
    except Exception:
        with open(out_path + f".err{rank}", "w") as f:
            f.write(traceback.format_exc())
        raise
