"""Each attention kernel by its name, in windows and on rows that are told apart by nothing else: that the sizes run where they are meant to."""
import numpy as np
import pytest
import torch

from test_gpu_kv_cache import TYPES, Pair

pytestmark = pytest.mark.gpu
FEW, PROMPT, RUNS = "kv_attend_kernel", "kv_prompt_kernel", "kv_prompt_kernel, kv_prompt_join_kernel"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim,page,codes", [(32, 16, 0), (64, 64, 1), (96, 32, 0), (128, 128, 1), (256, 16, 0)])
@pytest.mark.parametrize("heads,seqs,before,count,window,kernel", [(4, 3, 700, 2, 100, FEW), (4, 2, 3000, 3, 1500, FEW), (16, 1, 5500, 560, 4500, RUNS), (16, 1, 6000, 500, 5000, RUNS),
                                                                   (16, 2, 500, 1300, 200, PROMPT), (16, 2, 100, 1300, 1000, PROMPT), (16, 2, 130, 1300, 0, PROMPT)])
def test_windows_on_the_kernel_they_are_meant_for(heads, seqs, before, count, window, kernel, dim, page, codes, dtype):
    p = Pair(heads, 2, dim, page, codes, dtype, n_pages=seqs * ((before + count) // page + 1), max_seqs=4, max_context=7000, layers=1)
    ids = list(range(seqs))[::-1]
    if before:
        p.step(ids, [before + i for i in ids])
    p.step(ids, [count] * seqs)
    q = p.rand(seqs * count, heads, dim, size=1.5)
    qd = q.cuda()
    out = torch.full_like(qd, 3.0)
    p.kv.attend(0, qd.data_ptr(), out.data_ptr(), TYPES[dtype][1], window=window)
    torch.cuda.synchronize()
    assert p.kv.kernel_name() == kernel and p.kv.status() == 0
    got, rows = out.double().cpu().numpy(), np.unique(np.linspace(0, count - 1, 9).astype(int))
    tol = p.tolerance(q, ids, layer=0) + (2048 if dtype == "f32" else 4096) * 2.0 ** -23 * (kernel != FEW)        # (sums on tensor cores)
    for i, s in enumerate(ids):
        want = p.ref[0].attend(s, q[i * count:(i + 1) * count].double().numpy(), dim ** -0.5, window, rows=rows)
        values = np.abs(p.ref[0].numbers(s)[1]).max()
        assert np.abs(got[i * count + rows] - want).max() <= tol * values
