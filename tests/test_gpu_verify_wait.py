"""Verification when the CTAs of a sequence wait for one another in vain: in front of the first sums, between rows, at the draw; in all of them at once, in one, after which the
others' next wait runs out, or in one warp of each. The sequence is answered as one that has no answer, sequences of a single CTA as ever, and the device goes on working."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = r"""
import torch
import warpdecode_b200 as wd


def call(n_seqs, vocab, with_draft, dtype=torch.float32):
    x = torch.zeros(3 * n_seqs, vocab, dtype=dtype, device="cuda")
    x[:, 5] = 30.0
    d = x.clone()
    rows = torch.arange(3 * n_seqs)
    tokens = torch.full((3 * n_seqs,), 5, dtype=torch.int32, device="cuda")
    u = torch.where(rows % 3 == 0, 0.5, 0.25).cuda()
    path, count, following = (torch.full((n,), -7, dtype=torch.int32, device="cuda") for n in (3 * n_seqs, n_seqs, n_seqs))
    torch.cuda.synchronize()
    wd.verify_drafts(x.data_ptr(), 3 * n_seqs, vocab, tokens.data_ptr(), u.data_ptr(), path.data_ptr(), count.data_ptr(), following.data_ptr(), n_seqs=n_seqs,
                     draft_ptr=d.data_ptr() if with_draft else None, type=wd.TYPE_F32 if dtype == torch.float32 else wd.TYPE_BF16)
    torch.cuda.synchronize()
    return path.tolist(), count.tolist(), following.tolist()


for with_draft in (False, True):
    for n_seqs, vocab, dtype in ((1, 40000, torch.float32), (2, 131072, torch.bfloat16), (1, 500009, torch.float32)):
        assert call(n_seqs, vocab, with_draft, dtype) == ([-1] * 3 * n_seqs, [-1] * n_seqs, [-1] * n_seqs), (with_draft, n_seqs, vocab)
    assert call(2, 100, with_draft) == ([0, 1, 2] * 2, [3] * 2, [5] * 2)
print("as expected")
"""


@pytest.mark.parametrize("stop_at", ["0", "3", "0:0", "1:3", "2:-1:3", "3:0:0", "3:7", "3:-1:5"])         # three rows, then the draw
def test_a_wait_that_runs_out_is_no_answer(stop_at):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", PROGRAM], env={**os.environ, "WD_VERIFY_STOP_AT": stop_at, "PYTHONPATH": root}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as expected" in r.stdout, r.stdout + r.stderr
