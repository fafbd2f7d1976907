"""Verification where what is left of the target lies next to nothing for most tokens, and the draft's largest probability is many times the target's."""
import numpy as np
import pytest
import torch

import verify_oracle
from test_gpu_verify import call, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,gone", [(400001, 300), (1000001, 300), (1000001, 1000)])
def test_a_draft_that_has_one_token_for_many(vocab, gone):
    """The draft has `gone` tokens' share at token 0; of the others half are a little above what the target has, half as much below: by less than what sums of F32 are off, by more
    than 2^-18 of the draft's terms. They are 2^-16 to 2^-19 of what is left."""
    off = np.float32(1.6 * 2.0 ** -18 / gone)
    x, y = np.where(np.arange(vocab) % 2 == 0, off, -off).astype(np.float32), np.zeros(vocab, np.float32)
    x[:gone + 1] = 0.0
    y[1:gone + 1] = -np.inf
    y[0] = np.log(gone + 1.0)
    left = np.maximum(verify_oracle.softmax(x, 1.0) - verify_oracle.softmax(y, 1.0), 0.0)
    sums = np.cumsum(left)
    sums /= sums[-1]
    target, draft = (torch.tensor(np.stack([v, v]), device="cuda") for v in (x, y))
    for token in range(gone // 10, gone, gone // 10 + 1):
        border = np.float32(sums[token])                # (the numbers are 2^-25 from the border at most, 2^-26 at least with few exceptions: the sums are 64 bits)
        for u in (np.nextafter(border, np.float32(0)), np.nextafter(border, np.float32(1))):
            want = int(np.nonzero(sums > np.float64(u))[0][0])
            assert want == token + (np.float64(u) >= sums[token])
            path, count, following = call(target, ints([0, 0]), None, torch.tensor([u, 0.5], device="cuda"), draft)
            assert count[0] == 1 and following[0] == want


def test_where_nothing_is_left():
    """Target and draft are certain of one token and alike; another one that was not drawn from them is turned down, and then nothing is left: the sibling that would have been
    accepted in front of it is not, and the token behind is the target's."""
    x = torch.full((3, 300), -60000.0, device="cuda")
    x[:, 17] = 1.0
    half = torch.full((3,), 0.5, device="cuda")
    for tokens, count in (([0, 3, 17], 1), ([0, 17, 3], 2)):
        path, n, following = call(x, ints(tokens), ints([-1, 0, 0]), half, x.clone())
        assert n[0] == count and following[0] == 17 and path.tolist() == ([0, -1, -1] if count == 1 else [0, 1, -1])


@pytest.mark.parametrize("with_draft", [True, False])
def test_the_least_probability(with_draft):
    """2^-995 of the largest is one, 2^-1010 is none: by the number 0 the first that is one is drawn."""
    x = torch.full((1, 700), -700.0, device="cuda")
    x[0, 400:], x[0, 600] = -690.0, 0.0
    assert call(x, ints([0]), None, torch.zeros(1, device="cuda"), x.clone() if with_draft else None)[2][0] == 400
