"""The exchange of a row that several CTAs share: the order of its barriers in the source, and calls one behind the other on the device."""
import os
import re

import numpy as np
import pytest

import warpdecode_b200 as wd


def test_shared_memory_of_another_block_is_waited_for():
    """A block's shared memory may be written by another one only when all of the cluster are known to run."""
    text = open(os.path.join(wd.HERE, "csrc", "wd_score.cu")).read()
    code = re.sub(r"//[^\n]*", "", text)
    arrive, wait, remote = (code.index(w) for w in ("barrier.cluster.arrive", "barrier.cluster.wait", "map_shared_rank"))
    assert arrive < wait < remote
    assert code.index("cp.async.wait_group") < wait            # the wait is behind the row's reads, where it costs nothing


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(1, 16384), (1, 32768), (3, 65536), (18, 65536), (37, 65537), (74, 16390), (148, 16384)])      # clusters of 2, 4 and 8
def test_shared_rows_one_behind_the_other(rows, vocab):
    import torch

    g = torch.Generator().manual_seed(vocab + rows)
    x = torch.randn(rows, vocab, generator=g) * 3
    t = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    want = torch.log_softmax(x.double(), dim=1)
    order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :7].to(torch.int32).numpy()
    xd, td = x.cuda(), t.cuda()
    outs = [[torch.full((rows,), 9.0, device="cuda") for _ in range(2)] + [torch.full((rows, 7), 9, dtype=torch.int32, device="cuda"), torch.full((rows, 7), 9.0, device="cuda")]
            for _ in range(40)]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    for i, (lp, h, ids, best) in enumerate(outs):
        wd.token_logprobs(xd.data_ptr(), rows, vocab, td.data_ptr(), lp.data_ptr(), h.data_ptr(), 7, ids.data_ptr(), best.data_ptr(), stream=streams[i % 4].cuda_stream)
    torch.cuda.synchronize()
    lp = want.gather(1, t.long()[:, None])[:, 0].numpy()
    h = -(want * want.exp()).sum(dim=1).numpy()
    tol = 2.0 ** -16 + 40 * 2.0 ** -22        # sums of e^y of 2^18 terms at most, and the values' own steps of F32
    for o in outs:
        assert np.abs(o[0].cpu().double().numpy() - lp).max() <= tol and np.abs(o[1].cpu().double().numpy() - h).max() <= tol
        assert np.array_equal(o[2].cpu().numpy(), order)
        for a, b in zip(o, outs[0]):
            assert torch.equal(a, b)
