"""The operators of a step that checks drafted tokens, by which their kernels' speed is judged.

A draft proposes a tree of next tokens for every request (a node's parent is the token that it would follow; node 0 is the token
sampled last, which is not cached yet).  One step of the model looks at all of them: the layout of the step is made on the device
from the requests' lengths and the nodes' parents, every layer's attention lets a node see the cached tokens and its own
ancestors, the nodes' logits pass the penalties, biases and grammar masks that sampling asks for, and the longest path of
drafted tokens that the model would have chosen itself is kept: its keys and values go from the step's buffers to the cache.

Sizes are the benchmark's: the heads, layers and vocabularies of Llama-3-8B, Llama-3.2-1B and Llama-2-13B, pages of 16 tokens.
How many tokens a request has cached and drafted is spread between two bounds by a fixed rule, so that a case names its work.
"""
import math

import torch

own = False

PAGE = 16
# query heads, kv heads, head size, layers, vocabulary
SHAPES = {"8b": (32, 8, 128, 32, 128256), "1b": (32, 8, 64, 16, 128256), "13b": (40, 40, 128, 40, 32000)}
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
DEVICE = "cuda"


def _spread(lo, hi, n):
    """n whole numbers between lo and hi, the largest of them hi, in no order."""
    return [hi if i == 0 else lo + int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(n)]


def _layout(name, requests, nodes, cached):
    return dict(name=name, op="layout", requests=requests, nodes_lo=nodes[0], nodes_hi=nodes[1], cached_lo=cached[0], cached_hi=cached[1])


def _attention(name, shape, requests, nodes, cached, dtype="bfloat16", window=0):
    return dict(name=name, op="attention", shape=shape, dtype=dtype, requests=requests, nodes_lo=nodes[0], nodes_hi=nodes[1],
                cached_lo=cached[0], cached_hi=cached[1], window=window)


def _logits(name, vocab, requests, nodes, cached, biases):
    return dict(name=name, op="logits", vocab=vocab, requests=requests, nodes_lo=nodes[0], nodes_hi=nodes[1], cached_lo=cached[0],
                cached_hi=cached[1], biases=biases)


def _accept(name, shape, requests, nodes, cached, dtype="bfloat16"):
    return dict(name=name, op="accept", shape=shape, dtype=dtype, requests=requests, nodes_lo=nodes[0], nodes_hi=nodes[1],
                cached_lo=cached[0], cached_hi=cached[1])


def listed():
    return [
        # one user early in an answer with a short draft: what a launch costs
        _layout("layout 1x8", 1, (8, 8), (97, 97)),
        # a full batch with trees of every size
        _layout("layout 64x64", 64, (1, 64), (130, 8000)),
        # one user's short draft behind a short context: the least attention there is
        _attention("tree 8b 1x8", "8b", 1, (8, 8), (97, 97)),
        # the benchmark's eight requests of 2,048 tokens with trees of a usual size
        _attention("tree 8b 8x32", "8b", 8, (32, 32), (2047, 2047)),
        # a server between its busy hours, a small model: an odd number of requests, all lengths different
        _attention("tree 1b 27 ragged", "1b", 27, (1, 64), (130, 2300)),
        # a full batch with large trees: the most work
        _attention("tree 8b 64x64", "8b", 64, (33, 64), (2048, 4096)),
        # two long documents: the keys of one request have to be shared out over the device
        _attention("tree 8b 2 long", "8b", 2, (48, 48), (24000, 32000)),
        # 32-bit throughout, as a model is checked, with a sliding window
        _attention("tree 1b float32", "1b", 3, (13, 48), (515, 1500), dtype="float32", window=1024),
        # eight requests that decode one token each, every option on
        _logits("logits 8x1", 128256, 8, (1, 1), (2047, 2047), 300),
        # the nodes of sixteen trees: each has the tokens on its own path beside its request's
        _logits("logits 16x32", 128256, 16, (17, 32), (130, 2300), 64),
        # one user's short draft, a small model
        _accept("accept 1b 1x8", "1b", 1, (8, 8), (97, 97)),
        # a full batch of large trees, all layers of the cache
        _accept("accept 8b 64x64", "8b", 64, (33, 64), (60, 200)),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _unnamed(make, *args):
    case = make("", *args)
    del case["name"]
    return case


def draw(rng):
    op = rng.choice(["layout", "attention", "attention", "attention", "logits", "accept"])
    requests, nodes = _log(rng, 1, 64), _log(rng, 1, 64)
    lo = rng.randint(1, nodes)
    if op == "layout":
        cached = _log(rng, 1, 8000)
        return _unnamed(_layout, requests, (lo, nodes), (rng.randint(0, cached), cached))
    if op == "attention":
        shape = rng.choice(sorted(SHAPES))
        dtype = "float32" if rng.random() < 0.25 else "bfloat16"
        # no more keys and values than the largest listed case has, in 32 bits a sixteenth of its products
        kvh = SHAPES[shape][1]
        cached = _log(rng, 16, max(16, min(32000, 64 * 3500 * 8 // (requests * kvh), (64 * 64 * 3500 // 16 // (requests * nodes)) if dtype == "float32" else 32000)))
        window = rng.choice([0, 0, 0, rng.randint(100, 4096)])
        return _unnamed(_attention, shape, requests, (lo, nodes), (rng.randint(0, cached), cached), dtype, window)
    if op == "logits":
        vocab = rng.choice([128256, 32000, rng.randint(1000, 130000)])
        requests = max(1, min(requests, 400 * 128256 // (nodes * vocab)))
        cached = _log(rng, 1, 4000)
        return _unnamed(_logits, vocab, requests, (lo, nodes), (rng.randint(0, cached), cached), rng.choice([0, rng.randint(1, 300)]))
    shape = rng.choice(sorted(SHAPES))
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    requests = max(1, min(requests, 64 * 8 // SHAPES[shape][1] // (2 if dtype == "float32" else 1)))
    cached = _log(rng, 1, 200)
    return _unnamed(_accept, shape, requests, (lo, nodes), (rng.randint(0, cached), cached), dtype)


def _lengths(case):
    """Nodes and cached tokens of every request."""
    r = case["requests"]
    return _spread(case["nodes_lo"], case["nodes_hi"], r), _spread(case["cached_lo"], case["cached_hi"], r)[::-1]


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32).to(dtype)


def _parents(rng, lens):
    """Trees in which a node mostly follows one of the eight nodes before it: some deep, some wide."""
    out = []
    for n in lens:
        reach = int(torch.randint(1, 9, (1,), generator=rng))
        back = torch.randint(0, reach, (n,), generator=rng).tolist()
        out += [max(0, i - 1 - back[i]) if i else -1 for i in range(n)]
    return out


def _ancestors(parents, lens):
    """Bit j of row i: node j is node i or one of its ancestors, as signed 32-bit words."""
    words = (max(lens) + 31) // 32
    rows, at = [], 0
    for n in lens:
        mine = []
        for i in range(n):
            p = parents[at + i]
            mine.append((mine[p] if p >= 0 else 0) | (1 << i))
        rows += mine
        at += n
    split = [[(m >> (32 * w)) & 0xffffffff for w in range(words)] for m in rows]
    return torch.tensor(split, dtype=torch.int64).to(torch.int32).to(DEVICE)


def _pages(rng, blocks_of):
    """A block table in which the requests' pages lie in no order, -1 behind each request's own, and the number of pages."""
    total = sum(blocks_of)
    order = torch.randperm(total, generator=rng).tolist()
    table, at = [], 0
    for b in blocks_of:
        table.append(order[at:at + b] + [-1] * (max(blocks_of) - b))
        at += b
    return _int(table), total


def prepare(case, seed):
    rng = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    lens, cached = _lengths(case)
    n, r = sum(lens), len(lens)
    parents = _parents(rng, lens)
    st = dict(op=case["op"], parents=_int(parents), tree_len=_int(lens), prefix_len=_int(cached), cu_q=_int(_starts(lens)), n=n,
              words=(max(lens) + 31) // 32, most=max(lens),
              seq=torch.repeat_interleave(torch.arange(r, dtype=torch.int32), torch.tensor(lens)).to(DEVICE))
    if case["op"] == "layout":
        st["table"], _ = _pages(rng, [(c + m + PAGE - 1) // PAGE for c, m in zip(cached, lens)])
        st["out"] = dict(cu_q=torch.zeros(r + 1, dtype=torch.int32, device=DEVICE), token_seq=torch.zeros(n, dtype=torch.int32, device=DEVICE),
                         positions=torch.zeros(n, dtype=torch.int32, device=DEVICE), slots=torch.zeros(n, dtype=torch.int64, device=DEVICE),
                         mask=torch.zeros((n, st["words"]), dtype=torch.int32, device=DEVICE))
    elif case["op"] == "attention":
        heads, kvh, hd, _, _ = SHAPES[case["shape"]]
        dtype = TYPES[case["dtype"]]
        st.update(heads=heads, kvh=kvh, hd=hd, scale=hd ** -0.5, window=case["window"], mask=_ancestors(parents, lens))
        st["table"], pages = _pages(rng, [max(1, (c + PAGE - 1) // PAGE) for c in cached])
        # what the merged projection leaves: queries, then the drafted tokens' keys, then their values
        qkv = _normal(g, (n, (heads + 2 * kvh) * hd), dtype)
        st["q"], st["k"], st["v"] = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kvh) * hd], qkv[:, (heads + kvh) * hd:]
        st["cache"] = _normal(g, (pages, 2, kvh, PAGE, hd), dtype)
        depth = [0] * n
        at = _starts(lens)
        for s in range(r):
            for i in range(1, lens[s]):
                depth[at[s] + i] = depth[at[s] + parents[at[s] + i]] + 1
        st["positions"] = _int([cached[s] + depth[at[s] + i] for s in range(r) for i in range(lens[s])])
        st["out"] = torch.empty((n, heads * hd), dtype=dtype, device=DEVICE)
    elif case["op"] == "logits":
        vocab = case["vocab"]
        st.update(vocab=vocab, mask=_ancestors(parents, lens))
        st["logits"] = _normal(g, (n, vocab), torch.float32) * 3.0
        # words of a text: few are frequent, most are rare
        zipf = lambda shape: (vocab * torch.rand(shape, generator=g, device=DEVICE) ** 4).to(torch.int32).clamp_(max=vocab - 1)  # noqa: E731
        st["history"], st["history_len"] = zipf((r, max(max(cached), 1))), _int(cached)
        st["prompt_len"] = _int([c // 2 for c in cached])
        st["tokens"] = zipf((n,))
        st["presence"] = torch.rand(r, generator=g, device=DEVICE) * 1.5
        st["frequency"] = torch.rand(r, generator=g, device=DEVICE)
        st["repetition"] = 1.0 + torch.rand(r, generator=g, device=DEVICE) * 0.5
        st["bias_start"] = _int([case["biases"] * i for i in range(r + 1)])
        st["bias_token"] = torch.randint(0, vocab, (case["biases"] * r,), generator=g, device=DEVICE, dtype=torch.int32)
        st["bias_value"] = _normal(g, (case["biases"] * r,), torch.float32) * 5.0
        # grammars of four kinds, from almost everything to a few tokens; every fifth row is free
        words = (vocab + 31) // 32
        some = torch.randint(-2 ** 31, 2 ** 31, (4, words), generator=g, device=DEVICE, dtype=torch.int64).to(torch.int32)
        more = torch.randint(-2 ** 31, 2 ** 31, (4, words), generator=g, device=DEVICE, dtype=torch.int64).to(torch.int32)
        few = torch.where(torch.rand((words,), generator=g, device=DEVICE) < 0.02, some[3] & more[3], 0)
        st["allowed"] = torch.stack([some[0] | more[0], some[1], some[2] & more[2], few.to(torch.int32)])
        st["allowed_row"] = _int([-1 if i % 5 == 4 else i % 4 for i in range(n)])
        st["out"] = torch.empty((n, vocab), dtype=torch.float32, device=DEVICE)
    else:
        heads, kvh, hd, layers, vocab = SHAPES[case["shape"]]
        dtype = TYPES[case["dtype"]]
        st.update(kvh=kvh, hd=hd)
        table, pages = _pages(rng, [(c + m + PAGE - 1) // PAGE for c, m in zip(cached, lens)])
        st["cache"] = torch.zeros((layers, pages, 2, kvh, PAGE, hd), dtype=dtype, device=DEVICE)
        kv = _normal(g, (layers, n, 2 * kvh * hd), dtype)
        st["k"], st["v"] = kv[:, :, :kvh * hd], kv[:, :, kvh * hd:]
        at = _starts(lens)
        st["slots"] = torch.cat([table[s].long()[torch.arange(cached[s], cached[s] + lens[s], device=DEVICE) // PAGE] * PAGE
                                 + torch.arange(cached[s], cached[s] + lens[s], device=DEVICE) % PAGE for s in range(r)])
        # a draft is right in about seven of ten places; a tree may offer a token twice behind the same node
        tokens = torch.randint(0, vocab, (n,), generator=rng).tolist()
        target = torch.randint(0, vocab, (n,), generator=rng).tolist()
        lucky = torch.rand(n, generator=rng).tolist()
        for s in range(r):
            for i in range(1, lens[s]):
                p = at[s] + parents[at[s] + i]
                if lucky[p] < 0.7:
                    target[p] = tokens[at[s] + i]
                elif lucky[p] < 0.75:
                    tokens[at[s] + i] = target[p]
        st["tokens"], st["target"] = _int(tokens), _int(target)
        st["longest"] = min(32, max(lens))
        st["out"] = dict(n_kept=torch.zeros(r, dtype=torch.int32, device=DEVICE),
                         path=torch.zeros((r, st["longest"]), dtype=torch.int32, device=DEVICE),
                         next_token=torch.zeros(r, dtype=torch.int32, device=DEVICE), new_len=torch.zeros(r, dtype=torch.int32, device=DEVICE))
    return st


def run(st):
    if own:
        from lmsf_b200 import kernels
        o = st["out"]
        if st["op"] == "layout":
            kernels.tree_layout(o["cu_q"], o["token_seq"], o["positions"], o["slots"], o["mask"], st["parents"], st["tree_len"], st["prefix_len"],
                                st["table"], PAGE)
            return o
        if st["op"] == "attention":
            kernels.attention_tree(o, st["q"], st["k"], st["v"], st["cache"], st["table"], PAGE, st["cu_q"], st["prefix_len"], st["mask"], st["scale"],
                                   st["heads"], st["kvh"], st["hd"], positions=st["positions"], window=st["window"])
            return o
        if st["op"] == "logits":
            kernels.adjust_logits(o, st["logits"], row_req=st["seq"], history=(st["history"], st["history_len"], st["prompt_len"]),
                                  penalties=(st["presence"], st["frequency"], st["repetition"]), tree=(st["tokens"], st["mask"], st["cu_q"]),
                                  bias=(st["bias_start"], st["bias_token"], st["bias_value"]), allowed=(st["allowed"], st["allowed_row"]))
            return o
        kernels.tree_accept(o["n_kept"], o["path"], o["next_token"], o["new_len"], st["target"], st["tokens"], st["parents"], st["cu_q"],
                            st["prefix_len"], slots=st["slots"], k=st["k"], v=st["v"], cache=st["cache"])
        return dict(o, cache=st["cache"])
    return {"layout": _plain_layout, "attention": _plain_attention, "logits": _plain_logits, "accept": _plain_accept}[st["op"]](st)


def _bits(words, width):
    """Rows of 32-bit words -> truth values [rows, width]."""
    b = (words.unsqueeze(-1) >> torch.arange(32, device=DEVICE, dtype=torch.int32)) & 1
    return b.flatten(1)[:, :width] != 0


def _padded(st, flat, fill):
    """[n, ...] -> [requests, most nodes, ...]."""
    out = torch.full((st["tree_len"].shape[0], st["most"], *flat.shape[1:]), fill, dtype=flat.dtype, device=DEVICE)
    out[st["seq"].long(), _place(st)] = flat
    return out


def _place(st):
    """Every node's place in its own tree."""
    return torch.arange(st["n"], device=DEVICE) - st["cu_q"].long()[st["seq"].long()]


def _closure(st):
    """[requests, node, node]: whether the second is the first or an ancestor of it."""
    parents = _padded(st, st["parents"], -1).long()
    one = torch.eye(st["most"], device=DEVICE)
    step = one + (parents.unsqueeze(-1) == torch.arange(st["most"], device=DEVICE)).float()
    for _ in range(max(1, (st["most"] - 1).bit_length())):
        step = (step @ step).clamp(max=1.0)
    return step > 0


def _plain_layout(st):
    lens, cached = st["tree_len"].long(), st["prefix_len"].long()
    starts = torch.cat([lens.new_zeros(1), lens.cumsum(0)])
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEVICE), lens, output_size=st["n"])
    place = torch.arange(st["n"], device=DEVICE) - starts[seq]
    up = _closure(st)[seq, place]
    positions = cached[seq] + up.sum(-1) - 1
    where = cached[seq] + place
    slots = st["table"].long()[seq, where // PAGE] * PAGE + where % PAGE
    wide = torch.nn.functional.pad(up, (0, 32 * st["words"] - st["most"])).view(st["n"], st["words"], 32)
    words = (wide.long() << torch.arange(32, device=DEVICE)).sum(-1)
    return dict(cu_q=starts.to(torch.int32), token_seq=seq.to(torch.int32), positions=positions.to(torch.int32), slots=slots, mask=words.to(torch.int32))


def _plain_attention(st):
    kvh, hd, group = st["kvh"], st["hd"], st["heads"] // st["kvh"]
    r, most = st["tree_len"].shape[0], st["most"]
    seq, place = st["seq"].long(), _place(st)
    paged = st["cache"][st["table"].long().clamp(min=0)]                       # [requests, blocks, 2, kv heads, page, head size]
    paged = paged.permute(2, 0, 3, 1, 4, 5).flatten(3, 4).float()             # [2, requests, kv heads, keys, head size]
    new = [_padded(st, t.reshape(st["n"], kvh, hd), 0).transpose(1, 2).float() for t in (st["k"], st["v"])]
    keys, values = torch.cat([paged[0], new[0]], 2), torch.cat([paged[1], new[1]], 2)
    q = _padded(st, st["q"].reshape(st["n"], kvh, group, hd), 0).permute(0, 2, 3, 1, 4).flatten(2, 3).float()
    at = torch.arange(paged.shape[3], device=DEVICE)
    seen = (at < st["prefix_len"].long()[seq].unsqueeze(1))
    if st["window"]:
        seen &= at > (st["positions"].long() - st["window"]).unsqueeze(1)
    seen = _padded(st, torch.cat([seen, _bits(st["mask"], most)], 1), False)   # [requests, most, keys + most]
    scores = (q @ keys.transpose(2, 3)) * st["scale"]
    scores = scores.view(r, kvh, group, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = weights.sum(-1, keepdim=True)
    mixed = (weights.flatten(2, 3) @ values).view(r, kvh, group, most, hd) / torch.where(total == 0, 1.0, total)
    return mixed.permute(0, 3, 1, 2, 4).flatten(2)[seq, place].to(st["q"].dtype)


def _plain_logits(st):
    n, vocab, seq = st["n"], st["vocab"], st["seq"].long()
    requests, longest = st["history"].shape
    at = torch.arange(longest, device=DEVICE)
    inside = at < st["history_len"].long().unsqueeze(1)
    said = inside & (at >= st["prompt_len"].long().unsqueeze(1))
    where = st["history"].long()
    occurs = torch.zeros((requests, vocab), device=DEVICE).scatter_add_(1, where, inside.float())
    counts = torch.zeros((requests, vocab), device=DEVICE).scatter_add_(1, where, said.float())
    on_path = _bits(st["mask"], st["most"])                                   # [nodes, place in the tree]
    offered = _padded(st, st["tokens"], 0).long()[seq]
    path = torch.zeros((n, vocab), device=DEVICE).scatter_add_(1, offered, on_path.float())
    counts = counts[seq] + path
    occurs = occurs[seq] + path
    x = st["logits"]
    rep = st["repetition"][seq].unsqueeze(1)
    x = torch.where(occurs > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - st["frequency"][seq].unsqueeze(1) * counts
    x = x - st["presence"][seq].unsqueeze(1) * (counts > 0)
    owner = torch.repeat_interleave(torch.arange(requests, device=DEVICE), (st["bias_start"][1:] - st["bias_start"][:-1]).long(),
                                    output_size=st["bias_token"].shape[0])
    bias = torch.zeros((requests, vocab), device=DEVICE).index_put_((owner, st["bias_token"].long()), st["bias_value"], accumulate=True)
    x = x + bias[seq]
    free = st["allowed_row"] < 0
    allowed = _bits(st["allowed"], vocab)[st["allowed_row"].long().clamp(min=0)] | free.unsqueeze(1)
    return x.masked_fill_(~allowed, -math.inf)


def _plain_accept(st):
    r, most = st["tree_len"].shape[0], st["most"]
    cached = st["prefix_len"]
    nodes = torch.arange(most, device=DEVICE)
    parents, tokens, target = (_padded(st, st[name], -1).long() for name in ("parents", "tokens", "target"))
    right = (parents >= 0) & (tokens == target.gather(1, parents.clamp(min=0)))
    # of the children that offer the chosen token, the first
    behind = torch.where(right, parents, most)
    first = torch.full((r, most + 1), most, device=DEVICE).scatter_reduce_(1, behind, nodes.expand(r, most), "amin")
    good = (right & (first.gather(1, behind) == nodes)) | (nodes == 0)
    alive = ~(_closure(st) & ~good.unsqueeze(1)).any(-1) & (nodes < st["tree_len"].long().unsqueeze(1))
    longest = st["longest"]
    n_kept = alive.sum(1).clamp(max=longest)
    rank = torch.where(alive, alive.long().cumsum(1) - 1, longest).clamp(max=longest)
    path = torch.full((r, longest + 1), -1, device=DEVICE, dtype=torch.long).scatter_(1, rank, nodes.expand(r, most))[:, :longest]
    step = torch.arange(longest, device=DEVICE)
    path = torch.where(step < n_kept.unsqueeze(1), path, -1)
    last = path.gather(1, (n_kept - 1).clamp(min=0).unsqueeze(1))
    next_token = torch.where(n_kept > 0, target.gather(1, last.clamp(min=0)).squeeze(1), -1)
    # the kept nodes' keys and values to the places behind the cached tokens
    which, nth = (path >= 0).nonzero(as_tuple=True)
    begin = st["cu_q"].long()[which]
    source, slot = begin + path[which, nth], st["slots"][begin + nth]
    layers, kvh, hd = st["cache"].shape[0], st["kvh"], st["hd"]
    for plane, t in ((0, st["k"]), (1, st["v"])):
        st["cache"][:, slot // PAGE, plane, :, slot % PAGE] = t[:, source].reshape(layers, -1, kvh, hd).transpose(0, 1)
    return dict(n_kept=n_kept.to(torch.int32), path=path.to(torch.int32), next_token=next_token.to(torch.int32),
                new_len=cached + n_kept.to(torch.int32), cache=st["cache"])


def work(case):
    lens, cached = _lengths(case)
    n, r = sum(lens), len(lens)
    words = (max(lens) + 31) // 32
    if case["op"] == "layout":
        return {"bytes": 4 * n + 12 * r + n * (4 + 4 + 8 + 4 * words) + 4 * sum((m + PAGE - 1) // PAGE for m in lens), "flops": n}
    if case["op"] == "attention":
        heads, kvh, hd, _, _ = SHAPES[case["shape"]]
        size = 4 if case["dtype"] == "float32" else 2
        keys = [min(c, case["window"] or c) for c in cached]
        return {"bytes": size * (2 * n * heads * hd + 2 * kvh * hd * (sum(keys) + n)) + 4 * n * words,
                "flops": 4 * heads * hd * sum(m * (k + 1) for m, k in zip(lens, keys))}
    if case["op"] == "logits":
        v = case["vocab"]
        return {"bytes": 8 * n * v + 4 * sum(cached) + 8 * r * case["biases"] + 4 * 4 * ((v + 31) // 32) + 4 * n * (2 + words), "flops": 4 * n * v}
    heads, kvh, hd, layers, _ = SHAPES[case["shape"]]
    size = 4 if case["dtype"] == "float32" else 2
    # a request keeps its first node at the least, and drafts keep about as many more as half of their nodes' logarithm
    kept = sum(min(m, 1 + m.bit_length() // 2) for m in lens)
    return {"bytes": 12 * n + 20 * r + 2 * kept * layers * 2 * kvh * hd * size, "flops": n}


def exact(case, seed):
    st = prepare(case, seed)
    lens, cached = _lengths(case)
    at = _starts(lens)
    parents = st["parents"].tolist()
    if case["op"] == "layout":
        table, seqs, pos, slots, masks = st["table"].tolist(), [], [], [], []
        for s, m in enumerate(lens):
            chain = []
            for i in range(m):
                p = parents[at[s] + i]
                chain.append(([] if p < 0 else chain[p]) + [i])
                seqs.append(s)
                pos.append(cached[s] + len(chain[i]) - 1)
                slots.append(table[s][(cached[s] + i) // PAGE] * PAGE + (cached[s] + i) % PAGE)
                bits = sum(1 << j for j in chain[i])
                masks.append([(bits >> (32 * w)) & 0xffffffff for w in range(st["words"])])
        return dict(cu_q=_int(at), token_seq=_int(seqs), positions=_int(pos), slots=torch.tensor(slots, device=DEVICE),
                    mask=torch.tensor(masks, dtype=torch.int64).to(torch.int32).to(DEVICE))
    if case["op"] == "attention":
        if sum(m * c for m, c in zip(lens, cached)) * SHAPES[case["shape"]][0] * st["hd"] > 2e11:
            return None
        heads, kvh, hd, window = st["heads"], st["kvh"], st["hd"], st["window"]
        out = torch.zeros((at[-1], heads * hd), dtype=torch.float64, device=DEVICE)
        for s, m in enumerate(lens):
            pages = st["table"][s, :(cached[s] + PAGE - 1) // PAGE].long()
            rows = slice(at[s], at[s + 1])
            visible = torch.ones((m, cached[s] + m), dtype=torch.bool, device=DEVICE)
            for i in range(m):
                p = int(st["positions"][at[s] + i])
                if window:
                    visible[i, :max(0, min(cached[s], p - window + 1))] = False
                word = st["mask"][at[s] + i].tolist()
                visible[i, cached[s]:] = torch.tensor([(word[j // 32] >> (j % 32)) & 1 for j in range(m)], dtype=torch.bool)
            for h in range(kvh):
                side = []
                for plane, t in ((0, st["k"]), (1, st["v"])):
                    old = st["cache"][pages, plane, h].double().reshape(-1, hd)[:cached[s]]
                    side.append(torch.cat([old, t[rows, h * hd:(h + 1) * hd].double()]))
                for e in range(h * (heads // kvh), (h + 1) * (heads // kvh)):
                    z = torch.einsum("id,jd->ij", st["q"][rows, e * hd:(e + 1) * hd].double(), side[0]) * st["scale"]
                    w = torch.softmax(z.masked_fill(~visible, -math.inf), -1).nan_to_num(0.0)
                    out[rows, e * hd:(e + 1) * hd] = torch.einsum("ij,jd->id", w, side[1])
        return out
    if case["op"] == "logits":
        vocab, words = st["vocab"], st["mask"].tolist()
        history, tokens = st["history"].long(), st["tokens"].long()
        out = st["logits"].double()
        for s, m in enumerate(lens):
            half = cached[s] // 2
            prompt, said = history[s, :half], history[s, half:cached[s]]
            start, end = st["bias_start"][s], st["bias_start"][s + 1]
            bias = torch.zeros(vocab, dtype=torch.float64, device=DEVICE)
            bias.index_add_(0, st["bias_token"][start:end].long(), st["bias_value"][start:end].double())
            for i in range(m):
                row = at[s] + i
                path = tokens[[at[s] + j for j in range(m) if (words[row][j // 32] >> (j % 32)) & 1]]
                count = torch.bincount(torch.cat([said, path]), minlength=vocab).double()
                there = torch.bincount(prompt, minlength=vocab) + count > 0
                rep = st["repetition"][s].double()
                z = out[row]
                z = torch.where(there & (z > 0), z / rep, torch.where(there, z * rep, z))
                z = z - st["frequency"][s].double() * count - st["presence"][s].double() * (count > 0).double() + bias
                kind = int(st["allowed_row"][row])
                if kind >= 0:
                    v = torch.arange(vocab, device=DEVICE)
                    z = torch.where((st["allowed"][kind][v // 32] >> (v % 32)) & 1 == 1, z, -math.inf)
                out[row] = z
        return out
    tokens, target, slots, longest = st["tokens"].tolist(), st["target"].tolist(), st["slots"].tolist(), st["longest"]
    n_kept, paths, nexts, cache = [], [], [], st["cache"].double()
    for s, m in enumerate(lens):
        path = [0] if m else []
        while path and len(path) < longest:
            node = [i for i in range(m) if parents[at[s] + i] == path[-1] and tokens[at[s] + i] == target[at[s] + path[-1]]]
            if not node:
                break
            path.append(node[0])
        for nth, node in enumerate(path):
            slot = slots[at[s] + nth]
            for plane, t in ((0, st["k"]), (1, st["v"])):
                cache[:, slot // PAGE, plane, :, slot % PAGE] = t[:, at[s] + node].double().reshape(cache.shape[0], st["kvh"], st["hd"])
        n_kept.append(len(path))
        paths.append(path + [-1] * (longest - len(path)))
        nexts.append(target[at[s] + path[-1]] if path else -1)
    return dict(n_kept=_int(n_kept), path=_int(paths), next_token=_int(nexts), new_len=_int([c + k for c, k in zip(cached, n_kept)]), cache=cache)
