"""Numbers beyond 32 bits are refused by the Python calls, not cut to some other number."""
import pytest

import warpdecode_b200 as wd

BIG = 2 ** 32


def cache(**kw):
    c = dict(n_layers=2, n_heads=8, n_kv_heads=2, head_dim=64, n_pages=12, max_seqs=5, max_context=100, page_tokens=16, device=-1)
    c.update(kw)
    return wd.KvCache(**c)


@pytest.mark.parametrize("which", ["n_layers", "n_heads", "n_kv_heads", "head_dim", "n_pages", "max_seqs", "max_context", "page_tokens", "device"])
def test_a_geometry(which):
    for more in (BIG, -BIG):
        with pytest.raises(ValueError):
            cache(**{which: {"n_layers": 2, "n_heads": 8, "n_kv_heads": 2, "head_dim": 64, "n_pages": 12, "max_seqs": 5, "max_context": 100,
                             "page_tokens": 16, "device": -1}[which] + more})


def test_calls_on_sequences():
    kv = cache()
    kv.begin([0], [20])
    for call in (lambda: kv.truncate(BIG, 3), lambda: kv.truncate(0, BIG + 3), lambda: kv.keep(BIG, 0, [1]), lambda: kv.keep(0, BIG, [1]), lambda: kv.fork(BIG, [1]),
                 lambda: kv.length(BIG), lambda: kv.pages(BIG), lambda: kv.append(BIG, 16, 16), lambda: kv.append(0, 16, 16, BIG), lambda: kv.append(0, 16, 16, k_stride=2 ** 64),
                 lambda: kv.attend(BIG, 16, 16), lambda: kv.attend(0, 16, 16, window=BIG), lambda: kv.attend(0, 16, 16, out_stride=2 ** 64 + 512),
                 lambda: kv.read(BIG, [0], [0], [1], 16, 16)):
        with pytest.raises(ValueError):
            call()
    assert kv.length(0) == 20 and kv.length(1) == 0


def test_scores():
    for bad in (dict(rows=BIG), dict(vocab=BIG + 8), dict(n_top=BIG), dict(stride=2 ** 64)):
        a = dict(logits_ptr=1024, rows=0, vocab=8, tokens_ptr=1024, logprob_ptr=1024)
        a.update(bad)
        with pytest.raises(ValueError):
            wd.token_logprobs(**a)
