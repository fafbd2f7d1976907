"""The work that a step of speculative decoding gives the rotation of heads into the 8-bit cache, attention over a tree of drafts and their
verification, as cases that can be prepared, run and timed.

Three kinds of call stand behind the cases:

  place    the heads' norms and the rotary positions of a step's queries and keys, the keys and values into the cache's pages on the way
  tree     attention of a step's rows over the cache where each sequence's rows are a tree of drafted tokens
  verify   which drafted tokens the target's probabilities accept, given random numbers, and the token behind them

A cache holds codes (int8, or e4m3) with one float scale for each page of tokens, kv head, and keys or values. Tokens that come into a page that
holds some already may make its scale grow; the codes that are there are then rounded anew: s' = max(s, amax / limit), c' = round(c s / s').
A rotated key is rounded to F32 once and becomes a code from there.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = {"int8": 127.0, "e4m3": 448.0}
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------------------------------
def _place(name, seqs, before, count, heads, kv_heads, head_dim, rotary, page, codes, dtype, norm=True, neighbours=False, axes=1):
    return dict(name=name, kind="place", seqs=seqs, before=before, count=count, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rotary=rotary, page=page,
                codes=codes, dtype=dtype, norm=norm, neighbours=neighbours, axes=axes)


def _tree(name, seqs, shortest, longest, count, heads, kv_heads, head_dim, page, codes, dtype, window=0):
    return dict(name=name, kind="tree", seqs=seqs, shortest=shortest, longest=longest, count=count, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                codes=codes, dtype=dtype, window=window)


def _verify(name, seqs, count, vocab, draft, chain, dtype):
    return dict(name=name, kind="verify", seqs=seqs, count=count, vocab=vocab, draft=draft, chain=chain, dtype=dtype)


def listed():
    return [
        # the next token of one sequence, a full-attention layer beside the MoE block: a quarter of a head's elements is rotated
        _place("place_gated_1", 1, 4096, 1, 16, 2, 256, 64, 64, "int8", "f32"),
        # the next token of every sequence of a batch
        _place("place_step_64", 64, 1003, 1, 32, 8, 128, 128, 64, "int8", "bf16"),
        # a prompt's chunk on the dense decoder's heads, no norms
        _place("place_prompt", 1, 45, 4000, 32, 8, 64, 64, 64, "int8", "bf16", norm=False),
        # pictures in a prompt: positions in time, height and width
        _place("place_images", 1, 0, 5003, 32, 8, 128, 128, 128, "e4m3", "bf16", axes=3),
        # a small tree behind a short chat: the call is latency
        _tree("tree_short_1", 1, 144, 144, 13, 16, 4, 64, 16, "int8", "f32"),
        # a batch whose sequences each verify a tree
        _tree("tree_batch_16", 16, 300, 6000, 26, 32, 8, 128, 64, "int8", "bf16"),
        # a layer that sees the last 1,000 positions
        _tree("tree_window_6", 6, 700, 5000, 45, 16, 2, 256, 32, "int8", "f32", window=1000),
        # a large tree behind one very long context
        _tree("tree_long_1", 1, 131089, 131089, 64, 32, 8, 128, 128, "e4m3", "f16"),
        # four tokens of a draft model, one sequence
        _verify("verify_chain_1", 1, 5, 151936, True, True, "f32"),
        # the same for a batch
        _verify("verify_chain_64", 64, 5, 151936, True, True, "f32"),
        # a tree of likely tokens (draft heads, n-grams)
        _verify("verify_tree_1", 1, 64, 128256, False, False, "bf16"),
        # trees whose branches a draft model has drawn
        _verify("verify_tree_16", 16, 26, 128256, True, False, "bf16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return int(min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["place", "tree", "verify"])
    head_dim, page, codes, dtype = rng.choice([32, 64, 64, 96, 128, 128, 256]), rng.choice([16, 32, 64, 128]), rng.choice(["int8", "int8", "e4m3"]), rng.choice(["f32", "f16", "bf16", "bf16"])
    while True:
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8])
        if kind == "place":
            rotary = rng.choice([head_dim, head_dim, head_dim // 2])
            c = _place(None, _spread(rng, 1, 128), rng.choice([0, _spread(rng, 1, 100000)]), rng.choice([1, 1, rng.randint(2, 24), _spread(rng, 2, 8192)]), heads, kv_heads, head_dim,
                       rotary, page, codes, dtype, norm=rng.random() < 0.6, neighbours=rng.random() < 0.3, axes=rng.choice([1, 1, 1, 2, 3, 4]))
            if c["seqs"] * (c["before"] + c["count"]) * kv_heads * head_dim <= 1.6e8 and c["seqs"] * c["count"] * (heads + 2 * kv_heads) * head_dim <= 3e7:
                break
        elif kind == "tree":
            longest, count = _spread(rng, 5, 131072), rng.choice([1, rng.randint(2, 24), _spread(rng, 8, 128)])
            c = _tree(None, _spread(rng, 1, 64), max(count, longest // rng.randint(1, 50)), max(count, longest), count, heads, kv_heads, head_dim, page, codes, dtype,
                      rng.choice([0, 0, 0, _spread(rng, 1, 4096)]))
            if c["seqs"] * c["longest"] * kv_heads * head_dim <= 1.4e8 and c["seqs"] * heads * count * c["longest"] <= 2.7e8:
                break
        else:
            chain = rng.random() < 0.5
            c = _verify(None, _spread(rng, 1, 64), rng.randint(1, 9) if chain else _spread(rng, 3, 100), _spread(rng, 1000, 152064), rng.random() < 0.6, chain, dtype)
            if c["seqs"] * c["count"] * c["vocab"] <= (1.0 if c["draft"] else 2.0) * 5.4e7:
                break
    c.pop("name")
    return c


def _lengths(c):
    """The sequences' lengths with the step's tokens in them: from the shortest to the longest, by a curve that has more short ones."""
    n = c["seqs"]
    if c["kind"] == "place":
        return [c["before"] + c["count"] + (i * 7) % c["page"] if c["before"] else c["count"] for i in range(n)]
    lo, hi = c["shortest"], c["longest"]
    return [hi if n == 1 else round(lo + (hi - lo) * (i / (n - 1)) ** 2) for i in range(n)]


def _visited(c):
    """Rows of the target that a verification has to look at, on the average of these inputs: a drafted chain is followed by 0.7 a token, a tree 0.8 a level."""
    if c["chain"]:
        return sum(0.7 ** i for i in range(c["count"]))
    return sum(0.8 ** i for i in range(1 + int(math.log2(c["count"]))))


def work(c):
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "verify":
        rows = c["seqs"] * _visited(c)
        return {"bytes": rows * c["vocab"] * size * (2 if c["draft"] else 1) + c["seqs"] * c["count"] * 16, "flops": 8.0 * rows * c["vocab"]}
    hd, page = c["kv_heads"] * c["head_dim"], c["page"]
    rows = c["seqs"] * c["count"]
    if c["kind"] == "place":
        # the rows in, q and the codes out, the codes of the pages that they lie in back and out as numbers
        old = sum((n - c["count"]) % page for n in _lengths(c))
        q = 2 * rows * c["heads"] * c["head_dim"] * size + 4 * rows * c["axes"]
        return {"bytes": q + 2.0 * hd * (rows * (size + 1) + (rows + old) * (1 + size)), "flops": 10.0 * rows * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]}
    b = f = 0.0
    for n in _lengths(c):
        seen = n if not c["window"] else min(n, c["window"] + c["count"] - 1)
        b += 2 * seen * hd + 8 * c["kv_heads"] * (-(-seen // page)) + 2 * c["count"] * c["heads"] * c["head_dim"] * size + 4 * c["count"]
        f += 4.0 * c["head_dim"] * c["heads"] * c["count"] * min(n - c["count"] + 4, c["window"] or n)
    return {"bytes": b, "flops": f}


# ---- trees ----------------------------------------------------------------------------------------------------------------
def _parents(count, rng):
    """A tree of drafts: eight branches at most at the first token, four further on, most of them early."""
    parents, room = [-1], [0] * 8
    for i in range(1, count):
        at = int(len(room) * rng.random() ** 1.5)
        parents.append(room.pop(at))
        room += [i] * 4
        if len(room) > 60:
            room = room[-60:]
    return parents


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


# ---- the plain cache: codes [seq * pages][token][kv head][head dim], scales [seq * pages][kv head] ------------------------------
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


def _put(held, scale, x, mask, codes):
    """Tokens x (in mask) go into pages that hold `held` [page, token, head, dim] with `scale` [page, head]: the new codes' values and scales."""
    amax = torch.where(mask[:, :, None, None], x.abs(), torch.zeros_like(x)).amax(dim=(1, 3)).float()
    need = torch.where(amax > 0, torch.clamp(amax / torch.full_like(amax, LIMIT[codes]), min=2.0 ** -100), amax)
    new = torch.maximum(scale, need)
    s = torch.where(new > 0, new, torch.ones_like(new)).double()[:, None, :, None]
    old = _codes_of(held.double() * scale.double()[:, None, :, None] / s, codes)
    return torch.where(mask[:, :, None, None], _codes_of(x.double() / s, codes), old), new


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7fffffff)


def _rows(c, n, heads, gen):
    """Heads of n tokens, [n, heads, head dim], in the rows' type: channels of different size, now and then a large token."""
    x = torch.randn(n, heads, c["head_dim"], device="cuda", generator=gen)
    x *= 0.5 + torch.rand(heads, c["head_dim"], device="cuda", generator=gen)
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


def _type(c):
    import warpdecode_b200 as wd

    return {"f32": wd.TYPE_F32, "f16": wd.TYPE_F16, "bf16": wd.TYPE_BF16}[c["dtype"]]


def _cache(c, lengths):
    """The framework's cache with room for the sequences."""
    import warpdecode_b200 as wd

    pages = sum(-(-n // c["page"]) for n in lengths)
    return wd.KvCache(1, c["heads"], c["kv_heads"], c["head_dim"], pages, len(lengths), max(lengths), page_tokens=c["page"],
                      codes=wd.KV_INT8 if c["codes"] == "int8" else wd.KV_E4M3)


# ---- preparation ----------------------------------------------------------------------------------------------------------
def _sections(c):
    """Pairs of each axis."""
    pairs, n = c["rotary"] // 2, c["axes"]
    return [pairs // n + (i < pairs % n) for i in range(n)]


def _positions(c, lengths):
    """[rows, axes]. One axis: the tokens' places. Several: places of text, then pictures of 40 columns."""
    out = []
    for n in lengths:
        at = torch.arange(n - c["count"], n)
        if c["axes"] == 1:
            out.append(at[:, None])
            continue
        i = (at - 100).clamp(min=0)
        grid = [100 + i // 1600, 100 + i // 40 % 40, 100 + i % 40, 100 + i // 400]
        out.append(torch.stack([torch.where(at < 100, at, g) for g in grid[: c["axes"]]], dim=1))
    return torch.cat(out).to(torch.int32).cuda().contiguous()


def _prepare_steps(c, seed):
    """A cache that holds all but the step's tokens (and them too, for attention), and the step's rows."""
    gen, lengths, n, page = _gen(seed), _lengths(c), c["count"], c["page"]
    before = [v - n for v in lengths]
    rows = n * len(lengths)
    old = [_rows(c, sum(before), c["kv_heads"], gen) for _ in range(2)]
    new = [_rows(c, rows, c["kv_heads"], gen) for _ in range(2)]
    n_pages = -(-max(lengths) // page)
    s = dict(case=c, lengths=lengths, n_pages=n_pages, new=new)
    if c["kind"] == "tree":
        s["q"] = (1.5 * torch.randn(rows, c["heads"], c["head_dim"], device="cuda", generator=gen)).to(TYPES[c["dtype"]])
        s["out"] = torch.empty_like(s["q"])
        rng = random.Random(seed)
        parents = [_parents(n, rng) for _ in lengths]
        s["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda").reshape(-1)
        s["levels"] = 1 + max(max(_depths(p)) for p in parents)
    else:
        s["q"] = _rows(c, rows, c["heads"], gen)
        s["out"] = torch.empty_like(s["q"])
        s["norms"] = [1.0 + 0.2 * torch.randn(c["head_dim"], device="cuda", generator=gen) for _ in range(2)] if c["norm"] else None
        s["positions"] = _positions(c, lengths)
        back = sum((v - n) % page + n for v in lengths)
        s["back"] = [torch.empty(back, c["kv_heads"], c["head_dim"], dtype=TYPES[c["dtype"]], device="cuda") for _ in range(2)]
        s["firsts"] = [(v - n) // page * page for v in lengths]
        s["counts"] = [v - f for v, f in zip(lengths, s["firsts"])]
    if own:
        import warpdecode_b200 as wd

        kv = s["kv"] = _cache(c, lengths)
        ids = s["ids"] = list(range(len(lengths)))
        if c["kind"] == "place":
            s["rope"] = wd.Rope(c["head_dim"], c["rotary"], theta=500000.0, sections=_sections(c) if c["axes"] > 1 else (), neighbours=c["neighbours"])
        kv.begin(ids, before)
        if sum(before):
            kv.append(0, old[0].data_ptr(), old[1].data_ptr(), _type(c))
        kv.begin(ids, [n] * len(ids))
        if c["kind"] == "tree":
            kv.append(0, new[0].data_ptr(), new[1].data_ptr(), _type(c))
        torch.cuda.synchronize()
        return s
    layer = []
    for i, x in enumerate(old):
        x, mask = _into_pages(x, [0] * len(before), before, page, n_pages)
        zero = torch.zeros(x.shape[0], c["kv_heads"], device="cuda")
        v, scale = _put(torch.zeros_like(x, dtype=torch.int8), zero, x.float(), mask, c["codes"])
        if c["kind"] == "tree":
            x, mask = _into_pages(new[i], before, [n] * len(lengths), page, n_pages)
            v, scale = _put(v, scale, x.float(), mask, c["codes"])
        layer += [_held(v, c["codes"]), scale]
        del x, mask, v
    # the pages lie in any order, as those of a cache that has been in use
    order = torch.randperm(len(lengths) * n_pages, device="cuda", generator=gen)
    s["table"] = torch.argsort(order).reshape(len(lengths), n_pages)
    s["k"], s["ks"], s["v"], s["vs"] = (x.view(torch.uint8)[order].view(x.dtype) if x.element_size() == 1 else x[order] for x in layer)
    return s


def _prepare_verify(c, seed):
    """Logits of a target and of a draft model that is like it, the drafted tokens, as they come out of the draft, and random numbers."""
    gen, rng, vocab, n = _gen(seed), random.Random(seed), c["vocab"], c["count"]
    parents = [list(range(-1, n - 1)) if c["chain"] else _parents(n, rng) for _ in range(c["seqs"])]
    rows = n * c["seqs"]
    target = torch.randn(rows, vocab, device="cuda", generator=gen)
    draft = 0.8 * target + 0.6 * torch.randn(rows, vocab, device="cuda", generator=gen)
    # a few tokens stand out in both
    likely = torch.randint(0, vocab - vocab // 200, (rows, 8), device="cuda", generator=gen)
    high = math.log(vocab) - 1.0 + 5.0 * torch.rand(rows, 8, device="cuda", generator=gen)
    target.scatter_(1, likely, high)
    draft.scatter_(1, likely, high + 0.7 * torch.randn(rows, 8, device="cuda", generator=gen))
    for x in (target, draft):
        x[:, -(vocab // 200):] = -math.inf  # rows of the head that stand for no token
    target, draft = target.to(TYPES[c["dtype"]]), draft.to(TYPES[c["dtype"]])
    heat = 0.6 + 0.5 * torch.rand(c["seqs"], device="cuda", generator=gen)
    heat[7::8] = 0.0  # greedy
    p = torch.tensor(parents, device="cuda")
    at = (p.clamp(min=0) + n * torch.arange(c["seqs"], device="cuda")[:, None]).reshape(-1)
    if c["draft"]:
        z = draft.float() / torch.where(heat > 0, heat, torch.full_like(heat, 0.05)).repeat_interleave(n)[:, None]
        z = torch.softmax(z, dim=1).cumsum(dim=1)
        u = torch.rand(rows, device="cuda", generator=gen) * z[at, -1]
        tokens = torch.stack([torch.searchsorted(z[a], v) for a, v in zip(at.tolist(), u)]).clamp_(max=vocab - vocab // 200 - 1)
        del z
    else:
        best = draft.float().topk(8, dim=1).indices
        place = torch.tensor([[sum(q == p for q in ps[:i]) for i, p in enumerate(ps)] for ps in parents], device="cuda").reshape(-1)
        tokens = best[at, place]
    s = dict(case=c, target=target, draft=draft if c["draft"] else None, tokens=tokens.to(torch.int32).contiguous(), parents=p.to(torch.int32).reshape(-1).contiguous(),
             uniforms=torch.rand(rows, device="cuda", generator=gen), heat=heat)
    s["levels"] = 1 + max(max(_depths(ps)) for ps in parents)
    s["branches"] = max([max(ps.count(v) for v in ps) for ps in parents if n > 1] or [0])
    s["path"], s["count"], s["next"] = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (rows, c["seqs"], c["seqs"]))
    return s


def prepare(case, seed):
    state = _prepare_verify(case, seed) if case["kind"] == "verify" else _prepare_steps(case, seed)
    torch.cuda.synchronize()
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def _angles(s):
    """[rows, pairs] in 64 bits."""
    c = s["case"]
    pairs = c["rotary"] // 2
    freq = torch.exp(torch.arange(pairs, device="cuda", dtype=torch.float64) * (-2.0 * math.log(500000.0) / c["rotary"]))
    axis = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), torch.tensor(_sections(c), device="cuda"))
    return s["positions"].double()[:, axis] * freq


def _rotated(x, norm, angles, c, kind):
    """Norm and rotation of heads [rows, heads, dim]."""
    x = x.to(kind)
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(dim=2, keepdim=True) + EPS) * norm.to(kind)
    cos, sin = torch.cos(angles).to(kind)[:, None], torch.sin(angles).to(kind)[:, None]
    r, rest = x[:, :, : c["rotary"]], x[:, :, c["rotary"]:]
    a, b = (r[:, :, 0::2], r[:, :, 1::2]) if c["neighbours"] else (r[:, :, : c["rotary"] // 2], r[:, :, c["rotary"] // 2:])
    y0, y1 = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([y0, y1], dim=3).flatten(2) if c["neighbours"] else torch.cat([y0, y1], dim=2)
    return torch.cat([y, rest], dim=2)


def _placed(s):
    """q as rotated, and the tokens of the pages that the step's rows lie in as numbers; the pages of the state stay as they are."""
    c = s["case"]
    page, n, lengths = c["page"], c["count"], s["lengths"]
    norms = s["norms"] or (None, None)
    angles = _angles(s)
    q = _rotated(s["q"], norms[0], angles, c, torch.float32)
    # (a key becomes a code: its rounding to F32 has to be the right one)
    k = _rotated(s["new"][0], norms[1], angles, c, torch.float64).float()
    dev = k.device
    counts, firsts = torch.tensor(s["counts"], device=dev), torch.tensor(s["firsts"], device=dev)
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=dev), counts)
    at = seq * s["n_pages"] * page + firsts[seq] + torch.arange(seq.shape[0], device=dev) - (torch.cumsum(counts, 0) - counts)[seq]
    touched = torch.unique_consecutive(at // page)
    rows = s["table"].reshape(-1)[touched]
    place = torch.searchsorted(touched, at // page) * page + at % page

    def put(x, codes, scale):
        x, mask = _into_pages(x, [v - n for v in lengths], [n] * len(lengths), page, s["n_pages"])
        v, new = _put(codes.view(torch.uint8)[rows].view(codes.dtype).float(), scale[rows], x[touched].float(), mask[touched], c["codes"])
        return (v.float() * new[:, None, :, None]).reshape(-1, c["kv_heads"], c["head_dim"])[place]

    return [q, put(k, s["k"], s["ks"]), put(s["new"][1], s["v"], s["vs"])]


def _ancestors(parents, levels):
    """[.., n, n]: whether a node is another's ancestor, or itself; and the nodes' depths."""
    n = parents.shape[-1]
    node = torch.arange(n, device=parents.device)
    seen = (node[:, None] == node).expand(*parents.shape, n).clone()
    at = parents.long()
    for _ in range(levels - 1):
        seen |= (at[..., None] == node) & (at >= 0)[..., None]
        at = torch.where(at >= 0, parents.long().gather(-1, at.clamp(min=0)), at)
    return seen, seen.sum(dim=-1) - 1


def _attention(s):
    c, dev, kind = s["case"], s["q"].device, torch.float32
    n, kvh, hd, m = c["seqs"], c["kv_heads"], c["head_dim"], c["count"]
    g = c["heads"] // kvh

    def dense(codes, scale):
        x = codes.view(torch.uint8)[s["table"]].view(codes.dtype).to(kind) * scale[s["table"]].to(kind)[:, :, :][:, :, None, :, None]
        return x.reshape(n, -1, kvh, hd).permute(0, 2, 1, 3)

    q = s["q"].to(kind).reshape(n, m, kvh, g, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, g * m, hd)
    x = torch.matmul(q, dense(s["k"], s["ks"]).transpose(2, 3)) * (1.0 / math.sqrt(hd))
    tree, depth = _ancestors(s["parents"].reshape(n, m), s["levels"])
    start = (torch.tensor(s["lengths"], device=dev) - m)[:, None, None]
    token = torch.arange(x.shape[3], device=dev)[None, None]
    node = (token - start).clamp(0, m - 1).expand(n, m, -1)
    position = start + torch.where(token < start, token - start, depth[:, None].gather(2, node[:, :1]))
    seen = torch.where(token < start, torch.ones_like(node, dtype=torch.bool), tree.gather(2, node) & (token < start + m))
    if c["window"]:
        seen &= position > start + depth[:, :, None] - c["window"]
    x = x.reshape(n, kvh, g, m, -1).masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(dim=4, keepdim=True))
    total = x.sum(dim=4, keepdim=True)
    o = torch.matmul(x.reshape(n, kvh, g * m, -1), dense(s["v"], s["vs"])).reshape(n, kvh, g, m, hd) / total
    return o.permute(0, 3, 1, 2, 4).reshape(n * m, c["heads"], hd)


def _verified(s):
    """All sequences go down their trees together, a level a turn; a node's children are judged in order. In 64 bits: draws are made next to borders."""
    c, dev = s["case"], s["target"].device
    n, m, vocab = c["seqs"], c["count"], c["vocab"]
    first = m * torch.arange(n, device=dev)
    tokens, parents, uniforms = s["tokens"].long().reshape(n, m), s["parents"].long().reshape(n, m), s["uniforms"].double().reshape(n, m)
    heat = s["heat"].double()[:, None]
    greedy = heat <= 0
    node = torch.arange(m, device=dev).expand(n, m)
    at, alive = torch.zeros(n, dtype=torch.long, device=dev), torch.ones(n, dtype=torch.bool, device=dev)
    path = torch.full((n, m), -1, dtype=torch.int32, device=dev)
    count, following = torch.zeros(n, dtype=torch.int32, device=dev), torch.full((n,), -1, dtype=torch.int32, device=dev)

    def probabilities(logits):
        z = logits[first + at].double()
        z = (z - z.amax(dim=1, keepdim=True)) / torch.where(greedy, torch.ones_like(heat), heat)
        z = torch.exp(z)
        return z / z.sum(dim=1, keepdim=True)

    for level in range(s["levels"]):
        path[:, level] = torch.where(alive, at, torch.full_like(at, -1)).int()
        count += alive.int()
        p = probabilities(s["target"])
        best = s["target"][first + at].float().argmax(dim=1, keepdim=True)
        p = torch.where(greedy, torch.zeros_like(p).scatter_(1, best, 1.0), p)
        drawn = ~greedy if s["draft"] is not None else torch.zeros_like(greedy)
        q = probabilities(s["draft"]) if s["draft"] is not None else None
        r, total, times = p, p.sum(dim=1, keepdim=True), torch.zeros_like(heat)
        children = torch.sort(torch.where(parents == at[:, None], node, torch.full_like(node, m)), dim=1).values
        chosen = torch.full_like(at, -1)
        for j in range(s["branches"]):
            child = children[:, j: j + 1]
            there = (child < m) & (chosen < 0)[:, None] & alive[:, None]
            child = child.clamp(max=m - 1)
            x, u = tokens.gather(1, child), uniforms.gather(1, child)
            proposed = torch.where(drawn, q.gather(1, x), torch.ones_like(u)) if q is not None else torch.ones_like(u)
            taken = there & (u * total * proposed < r.gather(1, x))
            chosen = torch.where(taken[:, 0], child[:, 0], chosen)
            left = there & ~taken
            without = r.scatter(1, x, 0.0)
            if q is not None:
                times = torch.where(left & drawn, times + total, times)
                without = torch.where(drawn, torch.clamp(p - times * q, min=0), without)
            r = torch.where(left, without, r)
            total = r.sum(dim=1, keepdim=True)
        # those that go no further draw the token behind
        sums = torch.cumsum(r, dim=1)
        behind = torch.searchsorted(sums, uniforms[:, :1] * sums[:, -1:], right=True)[:, 0].clamp(max=vocab - 1)
        ends = alive & (chosen < 0)
        following = torch.where(ends, behind.int(), following)
        alive = alive & (chosen >= 0)
        at = torch.where(alive, chosen, at)
    return [path.reshape(-1), count, following]


def _run_own(s):
    c = s["case"]
    if c["kind"] == "tree":
        s["kv"].attend_tree(0, s["q"].data_ptr(), s["out"].data_ptr(), s["parents"].data_ptr(), _type(c), window=c["window"])
        return s["out"]
    if c["kind"] == "place":
        norms = [x.data_ptr() for x in s["norms"]] if s["norms"] else (None, None)
        s["kv"].append_rope(0, s["rope"], s["new"][0].data_ptr(), s["new"][1].data_ptr(), s["q"].data_ptr(), s["out"].data_ptr(), s["positions"].data_ptr(), q_norm_ptr=norms[0],
                            k_norm_ptr=norms[1], eps=EPS, type=_type(c))
        s["kv"].read(0, s["ids"], s["firsts"], s["counts"], s["back"][0].data_ptr(), s["back"][1].data_ptr(), _type(c))
        return [s["out"]] + s["back"]
    import warpdecode_b200 as wd

    wd.verify_drafts(s["target"].data_ptr(), c["seqs"] * c["count"], c["vocab"], s["tokens"].data_ptr(), s["uniforms"].data_ptr(), s["path"].data_ptr(), s["count"].data_ptr(),
                     s["next"].data_ptr(), n_seqs=c["seqs"], draft_ptr=s["draft"].data_ptr() if c["draft"] else None, parents_ptr=None if c["chain"] else s["parents"].data_ptr(),
                     temperature_ptr=s["heat"].data_ptr(), type=_type(c))
    return [s["path"], s["count"], s["next"]]


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["kind"] == "verify":
        return _verified(state)
    if c["kind"] == "tree":
        return _attention(state).to(TYPES[c["dtype"]])
    return [x.to(TYPES[c["dtype"]]) for x in _placed(state)]


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------------
def _exact_place(c, s):
    """Row by row as complex numbers; the pages one by one."""
    pairs = c["rotary"] // 2
    axis = [a for a, k in enumerate(_sections(c)) for _ in range(k)]
    freq = torch.tensor([500000.0 ** (-2.0 * i / c["rotary"]) for i in range(pairs)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), torch.stack([s["positions"][:, axis[i]].double() * freq[i] for i in range(pairs)], dim=1))

    def rotated(x, w):
        y = x.double().clone()
        if w is not None:
            y = y * torch.rsqrt(y.square().sum(dim=2, keepdim=True) / c["head_dim"] + EPS) * w.double()
        first = torch.arange(0, c["rotary"], 2, device="cuda") if c["neighbours"] else torch.arange(pairs, device="cuda")
        second = first + (1 if c["neighbours"] else pairs)
        z = torch.complex(y[:, :, first], y[:, :, second]) * turn[:, None]
        y[:, :, first], y[:, :, second] = z.real, z.imag
        return y

    w = s["norms"] or (None, None)
    outs = [rotated(s["q"], w[0])]
    rows = [rotated(s["new"][0], w[1]).float().double(), s["new"][1].double()]
    for x, codes, scale in ((rows[0], s["k"], s["ks"]), (rows[1], s["v"], s["vs"])):
        parts = []
        for i, n in enumerate(s["lengths"]):
            begin = n - c["count"]
            for p in range(s["firsts"][i] // c["page"], -(-n // c["page"])):
                lo, hi = max(begin, p * c["page"]), min(n, (p + 1) * c["page"])
                old, at = lo - p * c["page"], s["table"][i, p]
                now = x[i * c["count"] + lo - begin:i * c["count"] + hi - begin]
                s0 = scale[at].double()
                s1 = torch.maximum(s0, (now.abs().amax(dim=(0, 2)) / LIMIT[c["codes"]]).float().double())
                z = torch.cat([codes.view(torch.uint8)[at, :old].view(codes.dtype).double() * s0[None, :, None], now]) / s1[None, :, None]
                if c["codes"] == "int8":
                    z = torch.round(z)
                else:
                    _, e = torch.frexp(z)  # z = m 2^e with m in [1/2, 1): 4 bits from 2^(e - 1) on down to 2^-9
                    u = torch.ldexp(torch.ones_like(z), torch.clamp(e - 4, min=-9))
                    z = torch.round(z / u) * u
                parts.append(z * s1[None, :, None])
        outs.append(torch.cat(parts))
    return outs


def _exact_tree(c, s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    m, g, all_parents = c["count"], c["heads"] // c["kv_heads"], s["parents"].tolist()
    for i, n in enumerate(s["lengths"]):
        parents, start = all_parents[i * m:(i + 1) * m], n - m
        depth = _depths(parents)
        hidden = torch.ones(m, n, dtype=torch.bool)
        for r in range(m):
            hidden[r, max(0, start + depth[r] - c["window"] + 1) if c["window"] else 0:start] = False
            a = r
            while a >= 0 and not (c["window"] and depth[r] - depth[a] >= c["window"]):
                hidden[r, start + a] = False
                a = parents[a]
        hidden = hidden.cuda()
        pages = s["table"][i, : -(-n // c["page"])]
        for h in range(c["kv_heads"]):
            k = (s["k"].view(torch.uint8)[pages][:, :, h].view(s["k"].dtype).double() * s["ks"][pages, h].double()[:, None, None]).reshape(-1, c["head_dim"])[:n]
            v = (s["v"].view(torch.uint8)[pages][:, :, h].view(s["v"].dtype).double() * s["vs"][pages, h].double()[:, None, None]).reshape(-1, c["head_dim"])[:n]
            for a in range(h * g, (h + 1) * g):
                z = (s["q"][i * m:(i + 1) * m, a].double() @ k.T / math.sqrt(c["head_dim"])).masked_fill(hidden, -math.inf)
                out[i * m:(i + 1) * m, a] = torch.softmax(z, dim=1) @ v
    return out


def _exact_verify(c, s):
    """Sequence by sequence; the residual of each rejection made from the one before it."""
    m = c["count"]
    path, counts, following = [], [], []
    for i in range(c["seqs"]):
        tokens, parents = s["tokens"][i * m:(i + 1) * m].tolist(), s["parents"][i * m:(i + 1) * m].tolist()
        u, t = s["uniforms"][i * m:(i + 1) * m].tolist(), s["heat"][i].item()
        at, went = 0, [0]
        while True:
            z = s["target"][i * m + at].double()
            if t > 0:
                r = torch.softmax(z / t, dim=0)
            else:
                r = torch.zeros_like(z)
                r[int(torch.nonzero(z == z.max())[0])] = 1.0
            q = torch.softmax(s["draft"][i * m + at].double() / t, dim=0) if c["draft"] and t > 0 else None
            to = -1
            for child in [v for v in range(m) if parents[v] == at]:
                x = tokens[child]
                if u[child] * (q[x].item() if q is not None else 1.0) < r[x].item():
                    to = child
                    break
                r = r.clone()
                if q is not None:
                    r = torch.clamp(r - q, min=0)
                else:
                    r[x] = 0.0
                r = r / r.sum()
            if to < 0:
                sums = torch.cumsum(r.cpu(), dim=0)
                following.append(int(torch.nonzero(sums > u[0] * sums[-1].item())[0]))
                break
            at = to
            went.append(at)
        counts.append(len(went))
        path += went + [-1] * (m - len(went))
    return [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (path, counts, following)]


def exact(case, seed):
    """The operators' definitions in 64 bits, on the inputs of prepare()."""
    global own
    held, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = held
    if case["kind"] == "tree":
        return _exact_tree(case, s)
    if case["kind"] == "verify":
        return _exact_verify(case, s)
    if case["seqs"] * -(-case["count"] // case["page"]) > 1500:
        return None
    return _exact_place(case, s)
