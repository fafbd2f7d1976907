"""The answers of wd_kv_attend over its queries."""
import pytest
import torch

import warpdecode_b200 as wd
from test_gpu_kv_cache import Pair

pytestmark = pytest.mark.gpu


def test_the_output_over_queries_of_another_stride_is_refused():
    """A row's answer would lie on another row's queries."""
    kv = wd.KvCache(1, 8, 2, 64, 8, 2, 100)
    x = torch.zeros(8, 8, 64, device="cuda")
    kv.begin([0], [3])
    kv.append(0, x.data_ptr(), x.data_ptr())
    for q_stride, out_stride in ((600, 0), (0, 600), (513, 514)):
        with pytest.raises(wd.WdError, match="stride"):
            kv.attend(0, x.data_ptr(), x.data_ptr(), q_stride=q_stride, out_stride=out_stride)
    torch.cuda.synchronize()


@pytest.mark.parametrize("counts", [[2, 1], [900, 700]])        # the kernel for few rows, and the one for prompts
@pytest.mark.parametrize("width", [512, 520, 515])
def test_in_place_with_a_stride(counts, width):
    p = Pair(8, 2, 64, 16, 0, "f32", layers=1)
    p.step([0, 1], [70, 30])
    p.step([0, 1], counts)
    n = sum(counts)
    x = p.rand(n, width).cuda()
    q, rest = x[:, :512].reshape(n, 8, 64).contiguous(), x[:, 512:].clone()
    want = torch.empty_like(q)
    p.kv.attend(0, q.data_ptr(), want.data_ptr())
    p.kv.attend(0, x.data_ptr(), x.data_ptr(), q_stride=width, out_stride=0 if width == 512 else width)
    torch.cuda.synchronize()
    assert torch.equal(x[:, :512].reshape(n, 8, 64), want) and torch.equal(x[:, 512:], rest)
