"""What the rotary positions refuse, on the host alone."""
import numpy as np
import pytest

import warpdecode_b200 as wd


@pytest.mark.parametrize("kw", [dict(), dict(rotary_dim=32), dict(rotary_dim=2), dict(sections=(8, 12, 12)), dict(sections=(0, 32)), dict(sections=(8, 8, 8, 8), neighbours=True),
                                dict(inv_freq=np.ones(32)), dict(rotary_dim=6, inv_freq=[0.0, -1.0, 2.0]), dict(factor=0.0), dict(inv_freq=np.ones(32), theta=-1.0)])
def test_takes(kw):
    r = wd.Rope(64, **kw)
    r.close()
    r.close()


@pytest.mark.parametrize("kw", [dict(rotary_dim=66), dict(rotary_dim=3), dict(rotary_dim=-2), dict(theta=0.0), dict(theta=-1.0), dict(theta=float("nan")), dict(theta=float("inf")),
                                dict(factor=float("inf")), dict(sections=(8, 8)), dict(sections=(40, -8)), dict(sections=(33, 0)), dict(sections=(16, 8, 4, 5)),
                                dict(inv_freq=np.full(32, np.nan)), dict(inv_freq=np.full(32, np.inf))])
def test_refuses(kw):
    with pytest.raises(wd.WdError, match="rotary positions"):
        wd.Rope(64, **kw)


@pytest.mark.parametrize("head_dim", [0, 1, -64, 258])
def test_refuses_a_head(head_dim):
    with pytest.raises(wd.WdError, match="rotary positions"):
        wd.Rope(head_dim)


def test_refuses_what_python_sees():
    for kw in (dict(sections=(32,)), dict(sections=(8, 8, 8, 4, 4)), dict(inv_freq=np.ones(31)), dict(inv_freq=np.ones((2, 16))), dict(rotary_dim=2 ** 32 + 64), dict(sections=(2 ** 32, 32))):
        with pytest.raises(ValueError):
            wd.Rope(64, **kw)


def test_needs_a_device():
    kv = wd.KvCache(2, 8, 2, 64, 12, 5, 100, page_tokens=16, device=-1)
    kv.begin([0], [4])
    with pytest.raises(wd.WdError, match="without a device"):
        kv.append_rope(0, wd.Rope(64), 16, 16)
    for kw in (dict(layer=2 ** 32), dict(type=2 ** 32), dict(q_stride=2 ** 64), dict(v_stride=2 ** 64 + 512)):
        with pytest.raises(ValueError):
            kv.append_rope(kw.pop("layer", 0), wd.Rope(64), 16, 16, **kw)


def test_attention_of_a_tree_needs_a_device():
    kv = wd.KvCache(2, 8, 2, 64, 12, 5, 100, page_tokens=16, device=-1)
    kv.begin([0], [4])
    with pytest.raises(wd.WdError, match="without a device"):
        kv.attend_tree(0, 16, 16, 16)
    for kw in (dict(layer=2 ** 32), dict(type=2 ** 32), dict(window=2 ** 32), dict(q_stride=2 ** 64)):
        with pytest.raises(ValueError):
            kv.attend_tree(kw.pop("layer", 0), 16, 16, 16, **kw)
