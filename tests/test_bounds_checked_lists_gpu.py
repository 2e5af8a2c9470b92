"""The operators on rows of logits and lists of tokens in the bounds-checked
build: no index out of range at small, odd and long sizes, and the results of
the normal build."""
import os
import subprocess
import sys

import pytest
from test_bounds_checked_gpu import ROOT, _checked_built

pytestmark = pytest.mark.gpu

SCRIPT = r"""
import hashlib, os, sys, torch
sys.path.insert(0, os.environ["T1_ROOT"])
from test1_b200 import _native, ops

C = _native.cuda()
assert C.bounds_checked == (os.environ["T1_BOUNDS_CHECK"] == "1")
C.bounds_errors(True)
g = torch.Generator(device="cuda").manual_seed(0)
rand = lambda *n: torch.randn(*n, device="cuda", generator=g)
digest = hashlib.sha256()

def done(what, *tensors):
    torch.cuda.synchronize()
    errs = C.bounds_errors(True)
    assert not errs, (what, errs)
    for t in tensors:
        digest.update(t.contiguous().reshape(-1).view(torch.uint8).cpu().numpy().tobytes())

for B, V in [(1, 1), (3, 2), (5, 33), (7, 1000), (4, 8193), (3, 20011), (2, 128256), (1, 262145)]:
    for z in (rand(B, V), rand(B, V).bfloat16(), rand(B, V).round(), torch.full((B, V), -2.0, device="cuda")):
        u = torch.rand(B, device="cuda", generator=g)
        for k in (1, min(V, 300)):
            done((B, V, k), *ops.topk_logprobs(z, k))
        for kw in (dict(), dict(top_k=40), dict(top_k=2000), dict(top_p=0.9), dict(top_p=0.9, min_p=0.3), dict(min_p=0.1)):
            done((B, V, kw), *ops.sample_tokens(z, u, **kw))
for T, H, V, K in [(1, 64, 257, 1), (2, 8, 5, 5), (16, 2056, 1500, 512), (33, 72, 255, 7), (129, 264, 1000, 33),
                   (300, 520, 4097, 64), (600, 1024, 50021, 40), (300, 64, 600, 512), (5000, 64, 120011, 9)]:
    x, w, up = rand(T, H).bfloat16(), (rand(V, H) * 2 / H ** 0.5).bfloat16(), rand(T, K)
    ids = torch.randint(-2, V + 2, (T, K), device="cuda", generator=g)
    ids[1::3] = -100
    done((T, H, V), ops.linear_logits(x, w))
    for i in (ids, torch.full_like(ids, -1)):
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        logp, lse = ops.linear_topk_logprob_fwd(x, w, i)
        ops.linear_topk_logprob_bwd(up, x, w, i, lse, dx, dw)
        done((T, H, V, K), logp, lse, dx, dw)
for T, K in [(1, 1), (3, 7), (40, 32), (257, 8), (100, 64), (1000, 65), (70, 512), (5000, 20)]:
    b = torch.log_softmax(rand(T, K + 1), 1)[:, :K].contiguous()
    a = torch.log_softmax(rand(T, K + 1), 1)[:, :K].contiguous()
    ids = torch.where(rand(T, K) < 1, torch.arange(K, device="cuda"), -1)
    for kind in ops.DISTILLATION_KINDS:
        for tail in (True, False):
            done((T, K), *ops.distillation_loss_fwd_bwd(a, b, ids, kind=kind, tail=tail))
print("digest", digest.hexdigest())
"""


@pytest.mark.skipif(not _checked_built(), reason="bounds-checked build absent (T1_BUILD_CHECKED=1)")
def test_checked_build_is_clean_and_agrees():
    digests = []
    for checked in "10":
        env = dict(os.environ, T1_BOUNDS_CHECK=checked, T1_ROOT=ROOT, T1_QUIET="1")
        r = subprocess.run([sys.executable, "-c", SCRIPT], env=env, capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
        digests.append(r.stdout.split()[-1])
    assert digests[0] == digests[1]
