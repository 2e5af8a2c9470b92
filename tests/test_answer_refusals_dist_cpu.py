"""generate on two gloo ranks where one rank's arguments are refused: both raise,
none waits for the other, and the next call runs."""
import os

import torch
import torch.multiprocessing as mp

from test_distillation_dist_cpu import _free_port
from tests._refusal_worker import run


def test_a_refusal_on_one_rank_is_one_on_all(tmp_path):
    world, out, port = 2, str(tmp_path / "res"), _free_port()
    ctx = mp.get_context("spawn")
    procs = [ctx.Process(target=run, args=(r, world, port, out)) for r in range(world)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=300)
    errs = [f for f in os.listdir(tmp_path) if ".err" in f]
    assert not errs, open(os.path.join(tmp_path, errs[0])).read()
    res = [torch.load(out + f".{r}") for r in range(world)]
    assert res[0]["said"] == ["own", "another"] * 8 and res[1]["said"] == ["another", "own"] * 8
    assert res[0]["shape"] == res[1]["shape"] == (2, 10)
