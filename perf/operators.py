"""The work that a program gives the 8-bit key/value cache and the scoring of tokens, as cases that can be prepared, run and timed.

Four kinds of call stand behind the cases:

  attend   attention of a step's rows over a cache in 8 bits: one token of each sequence, the few tokens of a speculative
           verify, a chunk of a prompt
  append   the keys and values of a step's rows go into the cache and are read back (an export, a check, a prefix handed on)
  pages    fork: one sequence becomes several that share its pages, and each gets room for its next token; keep: the
           accepted tokens of a draft tree (or what an eviction leaves of a context) move together
  score    log probabilities of given tokens, the entropy, the likeliest alternatives

A cache holds codes (int8, or e4m3) with one float scale for each page of tokens, kv head, and keys or values. Tokens that
come into a page that holds some already may make its scale grow; the codes that are there are then rounded anew:
s' = max(s, amax / limit), c' = round(c s / s').
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = {"int8": 127.0, "e4m3": 448.0}


# ---- cases ------------------------------------------------------------------------------------------------------------
def _attend(name, seqs, shortest, longest, count, heads, kv_heads, head_dim, page, codes, dtype, window=0):
    return dict(name=name, kind="attend", seqs=seqs, shortest=shortest, longest=longest, count=count, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, page=page, codes=codes, dtype=dtype, window=window)


def _append(name, seqs, before, count, kv_heads, head_dim, page, codes, dtype):
    return dict(name=name, kind="append", seqs=seqs, before=before, count=count, kv_heads=kv_heads, head_dim=head_dim, page=page, codes=codes, dtype=dtype)


def _pages(name, what, layers, length, forks, first, kept, kv_heads, head_dim, page, codes, dtype):
    return dict(name=name, kind="pages", what=what, layers=layers, length=length, forks=forks, first=first, kept=kept, kv_heads=kv_heads,
                head_dim=head_dim, page=page, codes=codes, dtype=dtype)


def _score(name, rows, vocab, top, dtype):
    return dict(name=name, kind="score", rows=rows, vocab=vocab, top=top, dtype=dtype)


def listed():
    return [
        # one token of a short chat on a small model: the call is latency
        _attend("attend_short_1", 1, 131, 131, 1, 16, 4, 64, 16, "int8", "f32"),
        # one token after a few thousand, the full-attention layer beside the MoE block of the 48-layer model
        _attend("attend_gated_1", 1, 4097, 4097, 1, 16, 2, 256, 64, "int8", "f32"),
        # four tokens of a speculative verify on a few sequences, a layer that sees the last 1,000 tokens
        _attend("attend_verify_4", 6, 700, 5000, 4, 32, 8, 128, 32, "int8", "f32", window=1000),
        # a batch that is being served, lengths all over the place, the dense decoder's heads
        _attend("attend_batch_64", 64, 90, 8000, 1, 32, 8, 64, 32, "int8", "bf16"),
        # one very long context, a step at a time
        _attend("attend_long_1", 1, 131089, 131089, 1, 32, 8, 128, 128, "e4m3", "f16"),
        # a chunk of a prompt behind a prefix that is cached
        _attend("attend_prompt", 1, 5011, 5011, 4000, 32, 8, 64, 64, "int8", "bf16"),
        # the next token of every sequence of a batch
        _append("append_step_64", 64, 1003, 1, 8, 128, 64, "int8", "f32"),
        # a prompt
        _append("append_prompt", 1, 45, 8191, 8, 128, 64, "e4m3", "bf16"),
        # parallel samples of one prompt: the page that is not full is copied for each of them
        _pages("fork_32", "fork", 16, 1500, 32, 0, 0, 8, 64, 64, "int8", "bf16"),
        # an eviction: a bit over half of a context stays
        _pages("keep_half", "keep", 16, 6000, 1, 100, 3301, 8, 64, 64, "int8", "bf16"),
        # a speculative verify step: four tokens to judge
        _score("score_verify_4", 4, 151936, 5, "f32"),
        # a text to be scored
        _score("score_text", 1000, 128256, 20, "f32"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return int(min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choices(["attend", "prompt", "append", "fork", "keep", "score"], [4, 3, 2, 1, 1, 3])[0]
    head_dim, page, codes, dtype = rng.choice([32, 64, 64, 96, 128, 128, 256]), rng.choice([16, 32, 64, 128]), rng.choice(["int8", "int8", "e4m3"]), rng.choice(["f32", "f32", "f16", "bf16"])
    while True:
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8])
        window = rng.choice([0, 0, 0, _spread(rng, 1, 4096)])
        if kind == "attend":
            longest = _spread(rng, 5, 131072)
            count = rng.choice([1, 1, 1, 2, 3, 4, rng.randint(5, 24)])
            c = _attend(None, _spread(rng, 1, 96), max(count, longest // rng.randint(1, 50)), max(count, longest), count, heads, kv_heads, head_dim, page, codes, dtype, window)
            if c["seqs"] * c["longest"] * kv_heads * head_dim <= 1.4e8 and c["seqs"] * heads * count * c["longest"] <= 1e8:
                break
        elif kind == "prompt":
            count = _spread(rng, 25, 4096)
            before = rng.choice([0, 0, _spread(rng, 1, 3000)])
            seqs = rng.choice([1, 1, 2, 3])
            c = _attend(None, seqs, count + before // 3, count + before, count, heads, kv_heads, head_dim, page, codes, dtype, window)
            if seqs * heads * head_dim * count * (count + before) <= 2.5e10 and seqs * heads * count * (count + before) <= 6.4e8:
                break
        elif kind == "append":
            c = _append(None, _spread(rng, 1, 128), rng.choice([0, _spread(rng, 1, 2000)]), rng.choice([1, 1, _spread(rng, 2, 8192)]), kv_heads, head_dim, page, codes, dtype)
            if c["seqs"] * (c["before"] + c["count"]) * kv_heads * head_dim <= 1.6e8 and c["seqs"] * c["count"] * kv_heads * head_dim <= 8.4e6:
                break
        elif kind == "fork":
            c = _pages(None, "fork", rng.randint(1, 24), _spread(rng, 3, 3000), _spread(rng, 1, 64), 0, 0, kv_heads, head_dim, page, codes, dtype)
            if c["length"] % page and c["forks"] * c["layers"] * page * kv_heads * head_dim <= 1.7e7:
                break
        elif kind == "keep":
            length = _spread(rng, 8, 8000)
            first = rng.randint(0, length - 4)
            c = _pages(None, "keep", rng.randint(1, 24), length, 1, first, rng.randint(1, length - first - 1), kv_heads, head_dim, page, codes, dtype)
            if length * c["layers"] * kv_heads * head_dim <= 5e7:
                break
        else:
            c = _score(None, _spread(rng, 1, 1000), _spread(rng, 1000, 152064), rng.randint(0, 24), dtype)
            if c["rows"] * c["vocab"] <= 1.28e8:
                break
    c.pop("name")
    return c


def _lengths(c):
    """The sequences' lengths with the step's tokens in them: from the shortest to the longest, by a curve that has more short ones."""
    n = c["seqs"]
    if c["kind"] == "append":
        return [c["before"] + c["count"] + (i * 7) % c["page"] if c["before"] else c["count"] for i in range(n)]
    lo, hi = c["shortest"], c["longest"]
    return [hi if n == 1 else round(lo + (hi - lo) * (i / (n - 1)) ** 2) for i in range(n)]


def work(c):
    if c["kind"] == "score":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["rows"] * (c["vocab"] * size + 12 + 8 * c["top"]), "flops": 4.0 * c["rows"] * c["vocab"]}
    size, hd, page = 4 if c["dtype"] == "f32" else 2, c["kv_heads"] * c["head_dim"], c["page"]
    if c["kind"] == "attend":
        b = f = 0.0
        for n in _lengths(c):
            seen = n if not c["window"] else min(n, c["window"] + c["count"] - 1)
            b += 2 * seen * hd + 8 * c["kv_heads"] * (-(-seen // page)) + 2 * c["count"] * c["heads"] * c["head_dim"] * size
            full = c["count"] * (n - c["count"]) + c["count"] * (c["count"] + 1) / 2
            if c["window"]:
                full = sum(min(p + 1, c["window"]) for p in range(n - c["count"], n))
            f += 4.0 * c["head_dim"] * c["heads"] * full
        return {"bytes": b, "flops": f}
    if c["kind"] == "append":
        # the rows in, their codes out, the codes of the pages that they lie in back and out as numbers
        old = sum((n - c["count"]) % page for n in _lengths(c))
        rows = c["seqs"] * c["count"]
        return {"bytes": 2.0 * hd * (rows * (size + 1) + (rows + old) * (1 + size)), "flops": 2.0 * hd * 8 * rows}
    if c["what"] == "fork":
        old = c["length"] % page
        return {"bytes": 2.0 * hd * c["layers"] * old * (1 + c["forks"] * (1 + 1 + size)), "flops": 2.0 * hd * c["layers"] * c["forks"] * old}
    return {"bytes": 2.0 * hd * c["layers"] * c["kept"] * (1 + 1 + 1 + size), "flops": 2.0 * hd * c["layers"] * c["kept"] * 2}


# ---- the plain cache: codes [layer][page][token][kv head][head dim], scales [layer][page][kv head][2] ----------------------
def _codes_of(q, codes):
    """Quotients in 64 bits -> the codes' values, to the nearest, ties to even."""
    if codes == "int8":
        return torch.round(q).clamp_(-127, 127)
    a = q.abs()
    e = torch.floor(torch.log2(a.clamp(min=2.0 ** -6)))
    e = torch.where(torch.exp2(e) > a, e - 1, e).clamp_(min=-6)
    step = torch.exp2(e - 3)
    return torch.sign(q) * (torch.round(a / step) * step).clamp_(max=448)


def _held(v, codes):
    return v.to(torch.int8 if codes == "int8" else torch.float8_e4m3fn)


def _quantise(x, scale, codes):
    """x [..., token, head, dim] by scale [..., 1, head, 1]."""
    s = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    return _codes_of(x.double() / s, codes)


def _grown(x, mask, scale, codes):
    """The scale after tokens x [page, token, head, dim] (those in mask [page, token]) have come: [page, head]."""
    amax = torch.where(mask[:, :, None, None], x.abs(), torch.zeros_like(x)).amax(dim=(1, 3)).float()
    limit = torch.full_like(amax, LIMIT[codes])
    s = torch.where(amax > 0, torch.clamp(amax / limit, min=2.0 ** -100), amax)
    return torch.maximum(scale, s)


def _put(held, scale, x, mask, codes):
    """Tokens x (in mask) go into pages that hold `held` [page, token, head, dim] with `scale` [page, head]: the new codes' values and scales."""
    new = _grown(x, mask, scale, codes)
    ratio_s = new[:, None, :, None]
    old = _quantise(held.double() * scale.double()[:, None, :, None], ratio_s, codes)
    return torch.where(mask[:, :, None, None], _quantise(x, ratio_s, codes), old), new


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7fffffff)


def _rows(c, n, gen, outliers=True):
    """Keys or values of n tokens, [n, kv heads, head dim], in the rows' type: channels of different size, now and then a large token."""
    x = torch.randn(n, c["kv_heads"], c["head_dim"], device="cuda", generator=gen)
    x *= 0.5 + torch.rand(c["kv_heads"], c["head_dim"], device="cuda", generator=gen)
    if outliers:
        x *= 1.0 + 3.0 * (torch.rand(n, 1, 1, device="cuda", generator=gen) < 0.02)
    return x.to(TYPES[c["dtype"]])


def _into_pages(x, starts, counts, page, n_pages):
    """Rows [sum(counts), head, dim] of sequences that begin at `starts` -> ([seq * n_pages, page, head, dim], mask [seq * n_pages, page])."""
    dev = x.device
    counts_t, starts_t = torch.tensor(counts, device=dev), torch.tensor(starts, device=dev)
    seq = torch.repeat_interleave(torch.arange(len(counts), device=dev), counts_t)
    first = torch.cumsum(counts_t, 0) - counts_t
    at = seq * n_pages * page + starts_t[seq] + torch.arange(x.shape[0], device=dev) - first[seq]
    out = torch.zeros(len(counts) * n_pages * page, *x.shape[1:], dtype=x.dtype, device=dev)
    mask = torch.zeros(len(counts) * n_pages * page, dtype=torch.bool, device=dev)
    out[at] = x
    mask[at] = True
    return out.reshape(-1, page, *x.shape[1:]), mask.reshape(-1, page)


def _fill(c, old, before, n_pages):
    """A plain layer with `before` tokens in each sequence: codes and scales for keys and values, [seq * n_pages, ...]."""
    got = []
    for x in old:
        x, mask = _into_pages(x, [0] * len(before), before, c["page"], n_pages)
        zero = torch.zeros(x.shape[0], c["kv_heads"], device="cuda")
        v, s = _put(torch.zeros_like(x, dtype=torch.int8), zero, x.float(), mask, c["codes"])
        got += [_held(v, c["codes"]), s]
        del x, mask, v
    return got


def _cache(c, layers, lengths, extra):
    """The framework's cache with room for the sequences and `extra` pages."""
    import warpdecode_b200 as wd

    pages = sum(-(-n // c["page"]) for n in lengths)
    seqs = len(lengths) + (c["forks"] if c["kind"] == "pages" else 0)
    return wd.KvCache(layers, c.get("heads", c["kv_heads"]), c["kv_heads"], c["head_dim"], pages + extra, seqs, max(lengths) + c["page"],
                      page_tokens=c["page"], codes=wd.KV_INT8 if c["codes"] == "int8" else wd.KV_E4M3)


def _type(c):
    import warpdecode_b200 as wd

    return {"f32": wd.TYPE_F32, "f16": wd.TYPE_F16, "bf16": wd.TYPE_BF16}[c["dtype"]]


# ---- preparation ----------------------------------------------------------------------------------------------------------
def _prepare_steps(c, seed):
    """A cache that holds all but the step's tokens, and the step's rows."""
    gen, lengths, n, page = _gen(seed), _lengths(c), c["count"], c["page"]
    before = [v - n for v in lengths]
    old = [_rows(c, sum(before), gen) for _ in range(2)]
    new = [_rows(c, n * len(lengths), gen) for _ in range(2)]
    n_pages = -(-max(lengths) // page)
    s = dict(case=c, lengths=lengths, n_pages=n_pages, new=new)
    if c["kind"] == "attend":
        s["q"] = (1.5 * torch.randn(n * len(lengths), c["heads"], c["head_dim"], device="cuda", generator=gen)).to(TYPES[c["dtype"]])
        s["out"] = torch.empty_like(s["q"])
    else:
        rows = sum((v - n) % page + n for v in lengths)
        s["back"] = [torch.empty(rows, c["kv_heads"], c["head_dim"], dtype=TYPES[c["dtype"]], device="cuda") for _ in range(2)]
        s["firsts"] = [(v - n) // page * page for v in lengths]
        s["counts"] = [v - f for v, f in zip(lengths, s["firsts"])]
    if own:
        kv = s["kv"] = _cache(c, 1, lengths, 0)
        ids = s["ids"] = list(range(len(lengths)))
        kv.begin(ids, before)
        if sum(before):
            kv.append(0, old[0].data_ptr(), old[1].data_ptr(), _type(c))
        kv.begin(ids, [n] * len(ids))
        if c["kind"] == "attend":
            kv.append(0, new[0].data_ptr(), new[1].data_ptr(), _type(c))
        torch.cuda.synchronize()
        return s
    layer = _fill(c, old, before, n_pages)
    if c["kind"] == "attend":
        for i in (0, 1):
            x, mask = _into_pages(new[i], before, [n] * len(lengths), page, n_pages)
            v, layer[2 * i + 1] = _put(layer[2 * i].float(), layer[2 * i + 1], x.float(), mask, c["codes"])
            layer[2 * i] = _held(v, c["codes"])
            del x, mask, v
    # the pages lie in any order, as those of a cache that has been in use
    order = torch.randperm(len(lengths) * n_pages, device="cuda", generator=gen)
    s["table"] = torch.argsort(order).reshape(len(lengths), n_pages)
    s["k"], s["ks"], s["v"], s["vs"] = (x.view(torch.uint8)[order].view(x.dtype) if x.element_size() == 1 else x[order] for x in layer)
    return s


def _prepare_pages(c, seed):
    gen, page, n = _gen(seed), c["page"], c["length"]
    old = [[_rows(c, n, gen) for _ in range(2)] for _ in range(c["layers"])]
    n_pages = -(-n // page)
    rows = c["forks"] * (n % page) if c["what"] == "fork" else c["kept"]
    s = dict(case=c, back=[torch.empty(c["layers"], rows, c["kv_heads"], c["head_dim"], dtype=TYPES[c["dtype"]], device="cuda") for _ in range(2)])
    keep = torch.sort(torch.randperm(n - c["first"], device="cuda", generator=gen)[: c["kept"]]).values
    s["keep"] = keep.cpu().numpy().astype("int32")
    if own:
        kv = s["kv"] = _cache(c, c["layers"], [n], c["forks"] + n_pages + 1)
        kv.begin([0], [n])
        for l, x in enumerate(old):
            kv.append(l, x[0].data_ptr(), x[1].data_ptr(), _type(c))
        s["ids"] = list(range(1, 1 + c["forks"]))
        torch.cuda.synchronize()
        return s
    layers = [_fill(c, x, [n], n_pages) for x in old]
    s["k"], s["ks"], s["v"], s["vs"] = (torch.stack([l[i].view(torch.uint8) if l[i].element_size() == 1 else l[i] for l in layers]).view(layers[0][i].dtype) for i in range(4))
    s["at"] = keep + c["first"]
    return s


def _prepare_score(c, seed):
    gen = _gen(seed)
    n = c["rows"]
    x = torch.randn(n, c["vocab"], device="cuda", generator=gen) * (1.0 + 2.0 * torch.rand(n, 1, device="cuda", generator=gen))
    x[:, -(c["vocab"] // 200):] = -math.inf  # rows of the head that stand for no token
    # a few tokens stand out, and the given one is mostly among them
    likely = torch.randint(0, c["vocab"] - c["vocab"] // 200, (n, 6), device="cuda", generator=gen)
    x.scatter_add_(1, likely, 12.0 * torch.rand(n, 6, device="cuda", generator=gen))
    s = dict(case=c, logits=x.to(TYPES[c["dtype"]]), tokens=likely[:, 0].to(torch.int32).contiguous())
    s["logprob"], s["entropy"] = (torch.empty(n, device="cuda") for _ in range(2))
    if c["top"]:
        s["ids"], s["best"] = torch.empty(n, c["top"], dtype=torch.int32, device="cuda"), torch.empty(n, c["top"], device="cuda")
    return s


def prepare(case, seed):
    state = {"attend": _prepare_steps, "append": _prepare_steps, "pages": _prepare_pages, "score": _prepare_score}[case["kind"]](case, seed)
    torch.cuda.synchronize()
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def _dense(s, which, kind):
    """Keys or values of the sequences as numbers, [seq, kv head, token, dim]."""
    codes, scale = (s["k"], s["ks"]) if which == 0 else (s["v"], s["vs"])
    x = codes.view(torch.uint8)[s["table"]].view(codes.dtype).to(kind) * scale[s["table"]].to(kind)[:, :, None, :, None]
    n, p, t, h, d = x.shape
    return x.reshape(n, p * t, h, d).permute(0, 2, 1, 3)


def _attention(s, kind):
    c, dev = s["case"], s["q"].device
    n, kvh, hd, m = c["seqs"], c["kv_heads"], c["head_dim"], c["count"]
    g = c["heads"] // kvh
    k = _dense(s, 0, kind)
    q = s["q"].to(kind).reshape(n, m, kvh, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, g * m, hd)
    x = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    del k, q
    at = (torch.tensor(s["lengths"], device=dev)[:, None] - m + torch.arange(m, device=dev))[:, :, None]
    token = torch.arange(x.shape[3], device=dev)
    seen = token <= at
    if c["window"]:
        seen &= token > at - c["window"]
    x = x.reshape(n, kvh, g, m, -1).masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(dim=4, keepdim=True))
    total = x.sum(dim=4, keepdim=True)
    o = torch.matmul(x.reshape(n, kvh, g * m, -1), _dense(s, 1, kind)).reshape(n, kvh, g, m, hd) / total
    return o.permute(0, 3, 1, 2, 4).reshape(n * m, c["heads"], hd)


def _appended(s, kind):
    """The tokens of the pages that the step's rows lie in, as numbers; the pages of the state stay as they are."""
    c = s["case"]
    page, n, lengths = c["page"], c["count"], s["lengths"]
    dev = s["new"][0].device
    starts = [v - n for v in lengths]
    counts, firsts = torch.tensor(s["counts"], device=dev), torch.tensor(s["firsts"], device=dev)
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=dev), counts)
    offset = torch.arange(seq.shape[0], device=dev) - (torch.cumsum(counts, 0) - counts)[seq]
    at = seq * s["n_pages"] * page + firsts[seq] + offset
    touched = torch.unique_consecutive(at // page)
    out = []
    for i, (codes, scale) in enumerate(((s["k"], s["ks"]), (s["v"], s["vs"]))):
        x, mask = _into_pages(s["new"][i], starts, [n] * len(lengths), page, s["n_pages"])
        rows = s["table"].reshape(-1)[touched]
        v, new = _put(codes.view(torch.uint8)[rows].view(codes.dtype).float(), scale[rows], x[touched].float(), mask[touched], c["codes"])
        v = (v.to(kind) * new.to(kind)[:, None, :, None]).reshape(-1, c["kv_heads"], c["head_dim"])
        place = torch.searchsorted(touched, at // page) * page + at % page
        out.append(v[place])
    return out


def _copied(s, kind):
    """What the forks, or the sequence that kept some of its tokens, hold: their copied page, or the kept tokens."""
    c = s["case"]
    page, n, dev = c["page"], c["length"], s["k"].device
    if c["what"] == "fork":
        at = torch.arange(n // page * page, n, device=dev).repeat(c["forks"])
        new = [x[:, at // page] for x in (s["ks"], s["vs"])]
        old = new
    else:
        # a page takes the largest scale among those that its tokens come from
        at = s["at"]
        to = c["first"] + torch.arange(c["kept"], device=dev)
        old = [x[:, at // page] for x in (s["ks"], s["vs"])]
        new = []
        for x, o in zip((s["ks"], s["vs"]), old):
            y = torch.zeros_like(x)
            if c["first"] % page:
                y[:, c["first"] // page] = x[:, c["first"] // page]
            y.scatter_reduce_(1, (to // page)[None, :, None].expand_as(o), o, "amax", include_self=True)
            new.append(y[:, to // page])
    out = []
    for codes, o, w in zip((s["k"], s["v"]), old, new):
        v = codes.view(torch.uint8)[:, at // page, at % page].view(codes.dtype).double()
        v = _quantise(v * o.double()[:, :, :, None], w[:, :, :, None], c["codes"])
        out.append(v.to(kind) * w.to(kind)[:, :, :, None])
    return out


def _scores(s, kind):
    c, x = s["case"], s["logits"].to(kind)
    top = x.amax(dim=1, keepdim=True)
    x = x - top
    e = torch.exp(x)
    total = e.sum(dim=1)
    lse = torch.log(total)
    entropy = lse - torch.where(e > 0, x * e, torch.zeros_like(x)).sum(dim=1) / total
    logprob = x.gather(1, s["tokens"].long()[:, None])[:, 0] - lse
    if not c["top"]:
        return logprob, entropy, None, None
    best, ids = torch.sort(x, dim=1, descending=True, stable=True)
    return logprob, entropy, ids[:, : c["top"]].to(torch.int32), best[:, : c["top"]] - lse[:, None]


def _run_own(s):
    c = s["case"]
    if c["kind"] == "attend":
        s["kv"].attend(0, s["q"].data_ptr(), s["out"].data_ptr(), _type(c), window=c["window"])
        return s["out"]
    if c["kind"] == "append":
        s["kv"].append(0, s["new"][0].data_ptr(), s["new"][1].data_ptr(), _type(c))
        s["kv"].read(0, s["ids"], s["firsts"], s["counts"], s["back"][0].data_ptr(), s["back"][1].data_ptr(), _type(c))
        return s["back"]
    if c["kind"] == "pages":
        kv, n, page = s["kv"], c["length"], c["page"]
        kv.fork(0, s["ids"])
        if c["what"] == "fork":
            kv.begin(s["ids"], [1] * c["forks"])
            kv.read(-1, s["ids"], [n // page * page] * c["forks"], [n % page] * c["forks"], s["back"][0].data_ptr(), s["back"][1].data_ptr(), _type(c))
        else:
            kv.keep(1, c["first"], s["keep"])
            kv.read(-1, s["ids"], [c["first"]], [c["kept"]], s["back"][0].data_ptr(), s["back"][1].data_ptr(), _type(c))
        kv.free(s["ids"])
        return s["back"]
    import warpdecode_b200 as wd

    top = c["top"]
    wd.token_logprobs(s["logits"].data_ptr(), c["rows"], c["vocab"], s["tokens"].data_ptr(), s["logprob"].data_ptr(), s["entropy"].data_ptr(), top,
                      s["ids"].data_ptr() if top else None, s["best"].data_ptr() if top else None, _type(c))
    return [s["logprob"], s["entropy"]] + ([s["ids"], s["best"]] if top else [])


def _values(s, kind):
    c = s["case"]
    if c["kind"] == "attend":
        return _attention(s, kind)
    if c["kind"] == "append":
        return _appended(s, kind)
    if c["kind"] == "pages":
        return _copied(s, kind)
    return [x for x in _scores(s, kind) if x is not None]


def run(state):
    if own:
        return _run_own(state)
    got = _values(state, torch.float32)
    c = state["case"]
    if c["kind"] == "score":
        return got
    return got.to(TYPES[c["dtype"]]) if c["kind"] == "attend" else [x.to(TYPES[c["dtype"]]) for x in got]


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    """The operators' definitions in 64 bits, sequence by sequence, head by head and page by page, on the inputs of prepare()."""
    global own
    held, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = held
    c = case
    if c["kind"] == "attend":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        m, g = c["count"], c["heads"] // c["kv_heads"]
        for i, n in enumerate(s["lengths"]):
            pages = s["table"][i, : -(-n // c["page"])]
            position = torch.arange(n - m, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None, :]
            hidden = (j > position) | ((j <= position - c["window"]) if c["window"] else (j < 0))
            for h in range(c["kv_heads"]):
                k = (s["k"].view(torch.uint8)[pages][:, :, h].view(s["k"].dtype).double() * s["ks"][pages, h].double()[:, None, None]).reshape(-1, c["head_dim"])[:n]
                v = (s["v"].view(torch.uint8)[pages][:, :, h].view(s["v"].dtype).double() * s["vs"][pages, h].double()[:, None, None]).reshape(-1, c["head_dim"])[:n]
                for a in range(h * g, (h + 1) * g):
                    z = (s["q"][i * m:(i + 1) * m, a].double() @ k.T / math.sqrt(c["head_dim"])).masked_fill(hidden, -math.inf)
                    out[i * m:(i + 1) * m, a] = torch.softmax(z, dim=1) @ v
        return out
    if c["kind"] == "score":
        x = s["logits"]
        got = [torch.empty(c["rows"], dtype=torch.float64, device="cuda") for _ in range(2)]
        best = torch.empty(c["rows"], c["top"], dtype=torch.float64, device="cuda")
        for at in range(0, c["rows"], 64):
            p = torch.log_softmax(x[at:at + 64].double(), dim=1)
            got[0][at:at + 64] = p.gather(1, s["tokens"][at:at + 64].long()[:, None])[:, 0]
            got[1][at:at + 64] = -torch.where(p > -math.inf, p * p.exp(), torch.zeros_like(p)).sum(dim=1)
            if c["top"]:
                best[at:at + 64] = p.sort(dim=1, descending=True).values[:, : c["top"]]
        return got + ([None, best] if c["top"] else [])
    if c["kind"] == "append":
        if c["seqs"] * -(-c["count"] // c["page"]) > 1500:
            return None
        outs = []
        for which, (codes, scale) in enumerate(((s["k"], s["ks"]), (s["v"], s["vs"]))):
            parts = []
            for i, n in enumerate(s["lengths"]):
                begin = n - c["count"]
                for p in range(s["firsts"][i] // c["page"], -(-n // c["page"])):
                    lo, hi = max(begin, p * c["page"]), min(n, (p + 1) * c["page"])
                    old = lo - p * c["page"]
                    x = s["new"][which][i * c["count"] + lo - begin:i * c["count"] + hi - begin].double()
                    row = s["table"][i, p]
                    s0 = scale[row].double()
                    s1 = torch.maximum(s0, (x.abs().amax(dim=(0, 2)) / LIMIT[c["codes"]]).float().double())
                    both = torch.cat([codes.view(torch.uint8)[row, :old].view(codes.dtype).double() * s0[None, :, None], x])
                    z = both / s1[None, :, None]
                    if c["codes"] == "int8":
                        z = torch.round(z)
                    else:
                        _, e = torch.frexp(z)  # z = m 2^e with m in [1/2, 1): 4 bits from 2^(e - 1) on down to 2^-9
                        u = torch.ldexp(torch.ones_like(z), torch.clamp(e - 4, min=-9))
                        z = torch.round(z / u) * u
                    parts.append(z * s1[None, :, None])
            outs.append(torch.cat(parts))
        return outs
    outs = []
    for codes, scale in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        page, n = c["page"], c["length"]
        if c["what"] == "fork":
            p = n // page
            one = codes.view(torch.uint8)[:, p, : n % page].view(codes.dtype).double() * scale[:, p].double()[:, None, :, None]
            outs.append(torch.cat([one] * c["forks"], dim=1))
            continue
        parts, index = [], s["at"].tolist()
        for p in range(c["first"] // page, -(-(c["first"] + c["kept"]) // page)):
            mine = index[max(0, p * page - c["first"]):(p + 1) * page - c["first"]]
            sources = sorted({j // page for j in mine} | ({p} if c["first"] > p * page else set()))
            s1 = scale[:, sources].amax(dim=1).double()
            i = torch.tensor(mine, device="cuda")
            z = codes.view(torch.uint8)[:, i // page, i % page].view(codes.dtype).double() * scale[:, i // page].double()[:, :, :, None] / s1[:, None, :, None]
            if c["codes"] == "int8":
                z = torch.round(z)
            else:
                _, e = torch.frexp(z)
                u = torch.ldexp(torch.ones_like(z), torch.clamp(e - 4, min=-9))
                z = torch.round(z / u) * u
            parts.append(z * s1[:, None, :, None])
        outs.append(torch.cat(parts, dim=1))
    return outs
