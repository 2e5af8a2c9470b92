"""The log-probability and loss operators in the bounds-checked build: no
index out of range at small, odd and packed sizes, and the results of the
normal build."""
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
        digest.update(t.reshape(-1).view(torch.uint8).cpu().numpy().tobytes())

for T, H, V in [(1, 64, 257), (2, 8, 5), (1, 256, 1), (8, 1032, 5003), (16, 2056, 1500), (5, 8192, 600), (33, 72, 255),
                (129, 264, 1000), (300, 520, 4097), (513, 256, 20011), (257, 2048, 520), (700, 1032, 30011),
                (1500, 2048, 8001), (5000, 64, 128256)]:
    x, w, up = rand(T, H).bfloat16(), (rand(V, H) * 2 / H ** 0.5).bfloat16(), rand(T)
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    t[1::3] = -100
    for tt in (t, torch.full_like(t, -100)):
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        logp, lse = ops.linear_logprob_fwd(x, w, tt)
        ops.linear_logprob_bwd(up, x, w, tt, lse, dx, dw)
        done((T, H, V), logp, lse, dx, dw)
for B, S in [(2, 1), (2, 7), (4, 33), (6, 255), (4, 4097), (2, 20001), (300, 5), (2048, 3), (40, 1024), (5000, 8), (5000, 33)]:
    T = B * S
    ids = torch.where(rand(T) < 0.5, 3, -100)
    lp, old, ref = rand(T), rand(T), rand(T)
    done((B, S), *ops.preference_loss_fwd_bwd(lp, ref, ids, S))
    for adv in (rand(B), rand(T)):
        for reduction in ("token", "sequence"):
            done((B, S), *ops.policy_loss_fwd_bwd(lp, old, ref, adv, ids, S, kl_coef=0.1, reduction=reduction))
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
