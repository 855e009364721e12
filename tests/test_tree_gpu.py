"""The operators on drafted trees (csrc/tree.cu, attention_tree*.cu, adjust_logits.cu) against plain loops in 64 bits."""
import math
import random

import pytest
import torch

import plain_tree as P

pytestmark = pytest.mark.gpu
D = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=D)


def flag():
    return torch.zeros(1, dtype=torch.int32, device=D)


def make_table(rng, prefix, lens, bs, spare=1):
    """Pages in no order, -1 behind a request's own."""
    need = [(p + n + bs - 1) // bs for p, n in zip(prefix, lens)]
    order = list(range(sum(need) + spare))
    rng.shuffle(order)
    width, table = max(need + [1]) + 1, []
    for b in need:
        table.append(order[:b] + [-1] * (width - b))
        order = order[b:]
    return table, sum(need) + spare


# ----------------------------------------------------------------------------- layout

@pytest.mark.parametrize("lens,prefix,words,bs", [([1], [0], 1, 16), ([8], [97], 1, 16), ([0, 5, 0, 33, 64], [3, 0, 9, 250, 31], 2, 16), ([256, 255], [1, 100000], 8, 32),
                                                  ([7] * 70, list(range(70)), 3, 1), ([31, 32, 1], [8, 7, 6], 1, 24), ([], [], 1, 16)])
@pytest.mark.parametrize("window", [0, 1, 3])
@pytest.mark.parametrize("shape", ["tree", "forest", "chain", "deep"])
def test_layout(lens, prefix, words, bs, window, shape):
    """Whole numbers: equal.  Nine rows behind the last request's stay as they were."""
    from lmsf_b200 import kernels
    rng = random.Random(len(lens) + sum(lens) + window)
    trees = [list(range(-1, n - 1)) if shape in ("chain", "deep") else P.random_parents(rng, n, roots=0.2 if shape == "forest" else 0.0) for n in lens]
    table, _ = make_table(rng, prefix, lens, bs)
    if table:
        table[-1][-2] = -1                                        # the last request's last page was not reserved
    n, spare = sum(lens), 9
    cu, seq, pos, slots, mask = P.layout(trees, prefix, table, bs, words, window)
    o = [torch.full((len(lens) + 1,), -7, dtype=torch.int32, device=D)] + [torch.full((n + spare,), -7, dtype=torch.int32, device=D) for _ in range(2)]
    o += [torch.full((n + spare,), -7, dtype=torch.int64, device=D), torch.full((n + spare, words), -7, dtype=torch.int32, device=D)]
    parents = None if shape == "chain" else ints([p for t in trees for p in t] + [0] * spare)
    f = flag()
    kernels.tree_layout(*o, parents, ints(lens), ints(prefix), ints(table).reshape(len(lens), len(table[0]) if table else 1), bs, window=window, error_flag=f)
    assert o[0].tolist() == cu
    for got, want in zip(o[1:4], (seq, pos, slots)):
        assert got.tolist() == want + [-7] * spare
    assert o[4][:n].cpu().equal(mask) and (o[4][n:] == -7).all()
    assert f.item() == 0


def test_layout_of_ordinary_portions():
    """No parents and no mask: portions of any length."""
    from lmsf_b200 import kernels
    lens, prefix, bs = [1, 1900, 0, 777], [40, 3, 5, 16000], 16
    table, _ = make_table(random.Random(1), prefix, lens, bs)
    n = sum(lens)
    cu, seq, pos, slots, _ = P.layout([list(range(-1, m - 1)) for m in lens], prefix, table, bs, 1)
    o = [torch.empty(5, dtype=torch.int32, device=D), torch.empty(n, dtype=torch.int32, device=D), torch.empty(n, dtype=torch.int32, device=D),
         torch.empty(n, dtype=torch.int64, device=D)]
    kernels.tree_layout(*o, None, None, ints(lens), ints(prefix), ints(table), bs)
    for got, want in zip(o, (cu, seq, pos, slots)):
        assert got.tolist() == want


def test_layout_of_what_is_no_tree():
    """A parent that is not before its node leaves it alone; trees and rows beyond the buffers are cut off; the error word says so."""
    from lmsf_b200 import kernels
    z = lambda n, d=torch.int32: torch.full((n,), -7, dtype=d, device=D)  # noqa: E731
    table = ints([[0, 1, 2], [3, 4, 5]])
    for parents, lens, n, want_cu, want_mask in (([-1, 1, 5, -2, 0], [5, 0], 5, [0, 5, 5], [1, 2, 4, 8, 17]),
                                                 ([-1, 0, 1, -1, 0], [3, 4], 5, [0, 3, 5], [1, 3, 7, 1, 3]),
                                                 ([-1, 0, 1, -1, 0], [-2, 5], 5, [0, 0, 5], [1, 3, 7, 8, 17]),
                                                 ([-1] + [0] * 39, [40, 1], 40, [0, 32, 33], [1] + [1 + (1 << i) for i in range(1, 32)])):
        o, f = [z(3), z(n), z(n), z(n, torch.int64), torch.full((n, 1), -7, dtype=torch.int32, device=D)], flag()
        kernels.tree_layout(*o, ints(parents), ints(lens), ints([4, 9]), table, 16, error_flag=f)
        assert o[0].tolist() == want_cu and f.item() == 5
        got = [x & 0xffffffff for x in o[4].flatten().tolist()]
        assert got[:len(want_mask)] == want_mask
        assert (o[4][want_cu[-1]:] == -7).all() and (o[1][want_cu[-1]:] == -7).all()


# ----------------------------------------------------------------------------- attention

def attention_case(seed, lens, prefix, heads, kvh, hd, bs, dtype, window=0, masks="tree", words=None, spare_rows=0, poison=True):
    """Inputs on the device, with NaN wherever nobody looks: in pages behind the cached keys, in the spare page, in rows behind the last request's."""
    rng = random.Random(seed)
    g = torch.Generator(device=D).manual_seed(seed)
    dt = DTYPES[dtype]
    n = sum(lens) + spare_rows
    table, pages = make_table(rng, prefix, [0] * len(lens), bs)
    cache = torch.full((pages, 2, kvh, bs, hd), math.nan if poison else 0.0, dtype=dt, device=D)
    for s, p in enumerate(prefix):
        for b in range((p + bs - 1) // bs):
            m = min(bs, p - b * bs)
            cache[table[s][b], :, :, :m] = torch.randn((2, kvh, m, hd), generator=g, device=D).to(dt)
    rows = torch.randn((n, (heads + 2 * kvh) * hd + 8), generator=g, device=D).to(dt)
    if spare_rows and poison:
        rows[sum(lens):] = math.nan
    cu = [0]
    for m in lens:
        cu.append(cu[-1] + m)
    words = words or max(1, (max(lens + [1]) + 31) // 32)
    trees = [P.random_parents(rng, m) for m in lens]
    _, _, pos, _, mask = P.layout(trees, prefix, table, bs, words)
    if masks == "any":                                            # bits of nodes after the row, bits behind the tree, rows that see no node
        mask = torch.randint(-2 ** 31, 2 ** 31, mask.shape, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        mask[::3] = 0
    mask = torch.cat([mask, torch.full((spare_rows, words), -1, dtype=torch.int32)])
    q, k, v = rows[:, :heads * hd], rows[:, heads * hd:(heads + kvh) * hd], rows[:, (heads + kvh) * hd:(heads + 2 * kvh) * hd]
    return dict(q=q, k=k, v=v, cache=cache, table=table, bs=bs, cu=cu, prefix=prefix, mask=mask, scale=hd ** -0.5, heads=heads, kvh=kvh, hd=hd,
                positions=pos + [0] * spare_rows, window=window, dtype=dt, n=sum(lens))


def call_attention(c, out=None):
    from lmsf_b200 import kernels
    if out is None:
        out = torch.full((c["q"].shape[0], c["heads"] * c["hd"]), 7.0, dtype=c["dtype"], device=D)
    S, f = len(c["prefix"]), flag()
    kernels.attention_tree(out, c["q"], c["k"], c["v"], c["cache"], ints(c["table"]).reshape(S, -1), c["bs"], ints(c["cu"]), ints(c["prefix"]),
                           c["mask"].to(D), c["scale"], c["heads"], c["kvh"], c["hd"], positions=ints(c["positions"]), window=c["window"], error_flag=f)
    assert f.item() == 0
    return out


def check_attention(c, out):
    ref = P.attention(c["q"], c["k"], c["v"], c["cache"], c["table"], c["bs"], c["cu"], c["prefix"], c["mask"], c["scale"], c["heads"], c["kvh"], c["hd"],
                      c["positions"], c["window"])
    n = c["n"]
    bound = P.attention_bound(*ref, c["scale"], c["hd"], max(c["prefix"] + [0]) + 64, c["dtype"])[:n]
    off = (out[:n].cpu().double() - ref[0][:n]).abs()
    assert torch.isfinite(off).all()
    assert (off <= bound).all(), float((off / bound).max())
    assert (out[n:] == 7.0).all()


SHAPES = [  # lens, prefix, heads, kv heads, head size, page
    ([1], [0], 2, 1, 64, 16), ([1], [1], 4, 2, 64, 16), ([8], [97], 8, 2, 128, 16), ([5, 0, 13], [0, 50, 129], 6, 2, 64, 16),
    ([33, 64, 1, 17], [128, 300, 77, 515], 8, 2, 128, 16), ([64], [255], 16, 2, 64, 32), ([70, 3], [40, 200], 4, 4, 128, 64), ([9, 20], [130, 66], 3, 3, 80, 16),
    ([40], [200], 5, 1, 96, 16), ([12], [300], 7, 1, 128, 8), ([30, 2], [31, 400], 4, 2, 48, 128), ([6], [60], 2, 1, 16, 4), ([11], [77], 4, 2, 40, 16),
    ([7], [50], 2, 2, 33, 16), ([10, 4], [100, 9], 4, 2, 256, 16), ([21], [90], 3, 1, 192, 24), ([200], [130], 4, 2, 64, 16), ([3] * 40, list(range(0, 200, 5)), 4, 2, 64, 16),
    ([2, 2], [700, 1], 40, 1, 64, 16), ([37], [1500], 2, 1, 64, 256), ([64, 65], [64, 63], 8, 2, 112, 16), ([4], [33], 8, 8, 32, 16)]


@pytest.mark.parametrize("lens,prefix,heads,kvh,hd,bs", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "bf16 on the CUDA cores"])
@pytest.mark.parametrize("masks,window", [("tree", 0), ("any", 0), ("tree", 37), ("any", 150)])
def test_attention(lens, prefix, heads, kvh, hd, bs, dtype, masks, window, monkeypatch):
    """Lengths of none and one, pages that end inside a tile, odd sizes and groups, rows that see no drafted token or nothing at all (no cached
    tokens and an empty mask), NaN everywhere that nobody looks."""
    from lmsf_b200 import kernels
    if dtype.startswith("bf16 "):
        monkeypatch.setattr(kernels, "USE_TC_TREE", False)
        dtype = "bf16"
    c = attention_case(sum(lens) + hd, lens, prefix, heads, kvh, hd, bs, dtype, window, masks, spare_rows=3)
    check_attention(c, call_attention(c))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_leaves_hidden_infinities_alone(dtype):
    """NaN and infinities in keys and values of nodes that a row does not see, of cached keys behind a row's window and of pages that the cache does not have;
    rows that do see a value of infinity get it."""
    c = attention_case(5, [20, 9], [100, 70], 4, 2, 64, 16, dtype, window=60)
    sets = [{i, 0} for i in range(20)] + [{i} for i in range(9)]
    c["mask"] = torch.cat([P.words_of(sets[:20], 1), P.words_of(sets[20:], 1), ])
    c["positions"] = [100 + i for i in range(20)] + [70] * 9      # row i of the first sees cached keys behind 40 + i
    c["k"][7], c["v"][7] = math.nan, math.nan
    c["k"][25], c["v"][25] = math.inf, -math.inf
    c["v"][3, 10], c["v"][4, 11] = math.inf, -math.inf
    page = c["table"][0][45 // 16]
    c["cache"][page, 0, :, 45 % 16], c["cache"][page, 1, :, 45 % 16] = math.nan, math.inf      # seen by rows 0 .. 4 of the first
    out = call_attention(c)
    dead = [0, 1, 2, 3, 4, 7, 25]
    alive = [t for t in range(29) if t not in dead]
    ref = P.attention(c["q"], c["k"], c["v"], c["cache"], c["table"], c["bs"], c["cu"], c["prefix"], c["mask"], c["scale"], 4, 2, 64, c["positions"], 60)
    bound = P.attention_bound(*ref, c["scale"], 64, 200, c["dtype"])
    assert ((out.cpu().double() - ref[0]).abs() <= bound)[alive].all()
    assert not torch.isfinite(out[dead]).all(1).any()
    # with the cached key mended the two rows have one infinite column of each of kv head 0's two heads
    c["cache"][page, :, :, 45 % 16] = 0.5
    out = call_attention(c)
    for row, col, sign in ((3, 10, 1), (4, 11, -1)):
        inf = torch.isinf(out[row]).nonzero().flatten().tolist()
        assert inf == [col, 64 + col] and (out[row, inf] * sign > 0).all() and not torch.isnan(out[row]).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_without_some_pages(dtype):
    """Pages of -1 and beyond the cache inside the cached tokens hide their keys; so does the end of the block table."""
    c = attention_case(8, [9, 6, 5], [200, 130, 90], 8, 2, 64, 16, dtype)
    c["table"][0][3], c["table"][0][12], c["table"][1][0], c["table"][1][8] = -1, -1, c["cache"].shape[0] + 5, -9
    c["table"] = [row[:10] for row in c["table"]]
    check_attention(c, call_attention(c))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_one_long_request(dtype, hd):
    """A unit that many blocks share, and the joining of its parts; the same bits in every run."""
    c = attention_case(2, [6], [9000], 4, 2, hd, 16, dtype)
    c["positions"] = c["positions"]
    out = call_attention(c)
    check_attention(c, out)
    for _ in range(3):
        assert call_attention(c).equal(out)


def test_attention_behind_32_bits():
    """A cache whose last pages lie behind 2^32 elements: offsets in 64 bits."""
    from lmsf_b200 import kernels
    pages, kvh, bs, hd = 2 ** 32 // (2 * 8 * 16 * 128) + 40, 8, 16, 128
    small = attention_case(4, [7], [150], 16, kvh, hd, bs, "bf16")
    cache = torch.empty((pages, 2, kvh, bs, hd), dtype=torch.bfloat16, device=D)
    far = [pages - 1 - i for i in range(10)]
    cache[far] = small["cache"][small["table"][0][:10]]
    want = call_attention(small)
    got = torch.empty_like(want)
    kernels.attention_tree(got, small["q"], small["k"], small["v"], cache, ints([far]), bs, ints(small["cu"]), ints([150]), small["mask"].to(D), small["scale"], 16, kvh, hd)
    assert got.equal(want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_captured_with_other_lengths(dtype):
    """One captured call serves other lengths, tables and masks of the same sizes, also on another stream; eager calls between replays do not
    disturb it."""
    from lmsf_b200 import kernels
    a = attention_case(1, [5, 20, 7], [40, 300, 0], 8, 2, 64, 16, dtype, spare_rows=8, poison=False)
    b = attention_case(2, [12, 1, 27], [290, 17, 200], 8, 2, 64, 16, dtype, poison=False)
    width = 24
    dev = {}
    def fill(c):
        table = [(row + [-1] * width)[:width] for row in c["table"]]
        new = dict(q=c["q"].clone(), k=c["k"].clone(), v=c["v"].clone(), table=ints(table), cu=ints(c["cu"]), prefix=ints(c["prefix"]), mask=c["mask"].to(D))
        cache = torch.zeros((64, 2, 2, 16, 64), dtype=c["dtype"], device=D)
        cache[:c["cache"].shape[0]] = c["cache"]
        new["cache"] = cache
        for name, t in new.items():
            dev[name] = dev[name].copy_(t) if name in dev else t
    out = torch.full((40, 512), 7.0, dtype=DTYPES[dtype], device=D)
    run = lambda o: kernels.attention_tree(o, dev["q"], dev["k"], dev["v"], dev["cache"], dev["table"], 16, dev["cu"], dev["prefix"], dev["mask"], a["scale"], 8, 2, 64)  # noqa: E731
    fill(a)
    run(out)                                                      # builds and loads
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(out)
    for c in (b, a, b):
        out.fill_(7.0)
        fill(c)
        graph.replay()
        check_attention(c, out[:c["q"].shape[0]])
        other = torch.empty_like(out)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(other)
        torch.cuda.current_stream().wait_stream(side)
        assert other[:c["n"]].equal(out[:c["n"]])


# ----------------------------------------------------------------------------- logits

def adjust_case(seed, vocab, lens, width=50, biases=6, n_masks=3, listed_twice=True):
    rng = random.Random(seed)
    g = torch.Generator(device=D).manual_seed(seed)
    R, rows = len(lens), sum(lens)
    seq = [s for s, n in enumerate(lens) for _ in range(n)]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    logits = torch.randn((rows, vocab), generator=g, device=D) * 3
    ids = lambda n: [rng.choice([rng.randrange(vocab), rng.randrange(min(vocab, 9)), -1, vocab, 2 ** 31 - 1, -2 ** 31]) if rng.random() < 0.2 else rng.randrange(vocab)  # noqa: E731
                     for _ in range(n)]
    history = [ids(width) for _ in range(R)]
    length = [rng.randrange(0, width + 1) for _ in range(R)]
    prompt = [rng.randrange(0, n + 1) for n in length]
    pen = [torch.tensor([rng.uniform(*lim) for _ in range(R)], dtype=torch.float32) for lim in ((-2, 2), (-2, 2), (0.3, 2))]
    words = (max(lens) + 31) // 32
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tokens = ids(rows)
    start, btok, bval = [0], [], []
    for _ in range(R):
        n = rng.randrange(0, biases + 1)
        mine = ids(n)
        if n > 1 and listed_twice:
            mine[-1] = mine[0]
        btok += mine
        bval += [rng.uniform(-9, 9) if rng.random() < 0.9 else -math.inf for _ in range(n)]
        start.append(len(btok))
    bits = torch.randint(-2 ** 31, 2 ** 31, (n_masks, (vocab + 31) // 32), generator=torch.Generator().manual_seed(seed + 1)).to(torch.int32)
    bits[0] = 0
    which = [rng.randrange(-1, n_masks) for _ in range(rows)]
    bval = torch.tensor(bval, dtype=torch.float32)
    host = dict(row_req=seq, history=(torch.tensor(history, dtype=torch.int32).reshape(R, width), length, prompt), penalties=tuple(pen), tree=(tokens, mask, cu),
                bias=(start, btok, bval.tolist()), allowed=(bits, which))
    dev = dict(row_req=ints(seq), history=(ints(history).reshape(R, width), ints(length), ints(prompt)), penalties=tuple(p.to(D) for p in pen),
               tree=(ints(tokens), mask.to(D), ints(cu)), bias=(ints(start), ints(btok), bval.to(D)), allowed=(bits.to(D), ints(which)))
    return logits, host, dev


def check_adjusted(got, logits, host):
    """At most seven roundings of 2^-24 of what went in (a division or product, a product and two subtractions, the biases' sum and its addition)."""
    ref, size = P.adjust(logits, **host)
    got = got.cpu().double()
    fine = torch.isfinite(ref)
    assert torch.equal(fine, torch.isfinite(got)) and torch.equal(got[~fine], ref[~fine])
    assert ((got - ref).abs()[fine] <= (7 * 2.0 ** -24 * (size + logits.cpu().double().abs() * 4))[fine] + 1e-38).all()


@pytest.mark.parametrize("vocab,lens", [(1, [1]), (31, [2, 1]), (33, [1, 0, 3]), (4096, [2, 2]), (4097, [5]), (1000, [40, 33]), (8195, [1, 1, 1]), (20011, [3])])
@pytest.mark.parametrize("parts", ["all", "penalties", "history", "tree", "bias", "allowed", "nothing"])
@pytest.mark.parametrize("place", ["apart", "self", "strided"])
def test_adjust(vocab, lens, parts, place):
    from lmsf_b200 import kernels
    logits, host, dev = adjust_case(vocab + len(lens), vocab, lens)
    keep = {"all": ["history", "penalties", "tree", "bias", "allowed"], "penalties": ["penalties"], "history": ["history", "penalties"],
            "tree": ["tree", "penalties"], "bias": ["bias"], "allowed": ["allowed"], "nothing": []}[parts]
    host = {k: v for k, v in host.items() if k in keep or k == "row_req"}
    dev = {k: v for k, v in dev.items() if k in keep or k == "row_req"}
    x, out = logits.clone(), torch.full_like(logits, 7.0)
    if place == "self":
        out = x
    elif place == "strided":
        x = torch.full((logits.shape[0], vocab + 5), 3.0, device=D)
        x[:, 2:vocab + 2] = logits
        x = x[:, 2:vocab + 2]
        wide = torch.full((logits.shape[0], vocab + 3), 7.0, device=D)
        out = wide[:, 1:vocab + 1]
    f = flag()
    kernels.adjust_logits(out, x, error_flag=f, **dev)
    check_adjusted(out, logits, host)
    assert f.item() == 0
    if place == "strided":
        assert (wide[:, 0] == 7.0).all() and (wide[:, vocab + 1:] == 7.0).all()


@pytest.mark.parametrize("vocab,width", [(128256, 3000), (50257, 9000)])
def test_adjust_of_a_vocabulary(vocab, width):
    """Real sizes, a long history with many repetitions."""
    from lmsf_b200 import kernels
    logits, host, dev = adjust_case(3, vocab, [2, 1], width=width, biases=300)
    out = torch.empty_like(logits)
    kernels.adjust_logits(out, logits, **dev)
    check_adjusted(out, logits, host)


def test_adjust_counts_every_occurrence():
    """One token a thousand times, a bias listed forty times (added in the order of the list: the sum is the sequential one, bit for bit)."""
    from lmsf_b200 import kernels
    vocab = 5000
    x = torch.zeros((1, vocab), device=D)
    value = [1.0, 2.0 ** -24, -0.3] + [2.0 ** -25 * i for i in range(37)]
    out = torch.empty_like(x)
    kernels.adjust_logits(out, x, history=(ints([[77] * 1000 + [9]]), ints([1000]), ints([400])),
                          penalties=tuple(torch.tensor([p], device=D) for p in (0.5, 0.25, 1.5)),
                          bias=(ints([0, 40]), ints([4999] * 40), torch.tensor(value, device=D)))
    total = torch.zeros(())
    for b in value:
        total = total + torch.tensor(b)
    want = torch.zeros(vocab)
    want[77], want[4999] = -(600 * 0.25) - 0.5, total
    assert out[0].cpu().equal(want)


def test_adjust_hides_what_is_no_number():
    """NaN and infinities that a mask hides are -inf; a mask that allows nothing leaves -inf alone; requests and masks that do not exist are reported."""
    from lmsf_b200 import kernels
    x = torch.randn((3, 100), device=D)
    x[0, 5], x[0, 6], x[1, 7] = math.nan, math.inf, math.nan
    bits = torch.zeros((2, 4), dtype=torch.int32, device=D)
    bits[1] = -1
    out, f = torch.empty_like(x), flag()
    kernels.adjust_logits(out, x, allowed=(bits, ints([0, 1, -1])), error_flag=f)
    assert (out[0] == -math.inf).all() and torch.isnan(out[1, 7]) and out[2].equal(x[2]) and f.item() == 0
    kernels.adjust_logits(out, x, allowed=(bits, ints([0, 2, -1])), error_flag=f)
    assert f.item() == 5 and (out[0] == -math.inf).all() and out[2].equal(x[2])
    f.zero_()
    pen = tuple(torch.full((2,), p, device=D) for p in (1.0, 1.0, 1.5))
    kernels.adjust_logits(out, x, row_req=ints([2, 0, -1]), penalties=pen, history=(ints([[1], [2]]), ints([1, 1]), ints([0, 0])), error_flag=f)
    assert f.item() == 5 and out[2].equal(x[2]) and float(out[1, 1]) != float(x[1, 1])


def test_adjust_is_what_the_sampler_applies():
    """The same bits as apply_penalties for tokens of prompt and output."""
    from lmsf_b200 import kernels
    vocab, R = 3001, 4
    g = torch.Generator(device=D).manual_seed(2)
    x = torch.randn((R, vocab), generator=g, device=D) * 4
    hist = torch.randint(0, vocab, (R, 700), generator=g, device=D, dtype=torch.int32)
    length, prompt = [700, 650, 1, 0], [300, 650, 0, 0]
    pen = tuple(torch.rand(R, generator=g, device=D) + 0.5 for _ in range(3))
    rows, toks, counts = [], [], []
    for r in range(R):
        h = hist[r].tolist()[:length[r]]
        for t in sorted(set(h)):
            rows.append(r)
            toks.append(t)
            counts.append(h[prompt[r]:].count(t))
    want = x.clone()
    kernels.apply_penalties(want, ints(rows), ints(toks), ints(counts), *pen)
    got = torch.empty_like(x)
    kernels.adjust_logits(got, x, history=(hist, ints(length), ints(prompt)), penalties=pen)
    assert got.equal(want)


# ----------------------------------------------------------------------------- acceptance

def accept_case(seed, lens, vocab=40, right=0.8):
    rng = random.Random(seed)
    parents, tokens, target, cu = [], [], [], [0]
    for n in lens:
        p = P.random_parents(rng, n)
        tok = [rng.randrange(vocab) for _ in range(n)]
        tgt = [rng.randrange(vocab) for _ in range(n)]
        for i in range(1, n):
            if rng.random() < right:
                if rng.random() < 0.5:
                    tgt[p[i]] = tok[i]
                else:
                    tok[i] = tgt[p[i]]
        parents += p
        tokens += tok
        target += tgt
        cu.append(cu[-1] + n)
    return parents, tokens, target, cu


def call_accept(parents, tokens, target, cu, prefix, longest, **kw):
    from lmsf_b200 import kernels
    S = len(cu) - 1
    o = [torch.full((S,), -9, dtype=torch.int32, device=D), torch.full((S, longest), -9, dtype=torch.int32, device=D)]
    o += [torch.full((S,), -9, dtype=torch.int32, device=D) for _ in range(2)]
    kernels.tree_accept(*o, ints(target), ints(tokens), ints(parents), ints(cu), ints(prefix), **kw)
    return o


def check_accept(o, paths, nexts, prefix, longest):
    assert o[0].tolist() == [len(p) for p in paths]
    assert o[1].tolist() == [p + [-1] * (longest - len(p)) for p in paths]
    assert o[2].tolist() == nexts
    assert o[3].tolist() == [a + len(p) for a, p in zip(prefix, paths)]


@pytest.mark.parametrize("lens,longest", [([1], 1), ([8], 8), ([0, 5, 0, 64, 33], 32), ([256, 255, 1], 256), ([256], 3), ([40] * 70, 16), ([], 4)])
@pytest.mark.parametrize("right", [0.0, 0.7, 1.0])
def test_accept(lens, longest, right):
    parents, tokens, target, cu = accept_case(sum(lens) + longest, lens, right=right)
    prefix = [7 * s for s in range(len(lens))]
    paths, nexts = P.accept(target, tokens, parents, cu, longest)
    check_accept(call_accept(parents, tokens, target, cu, prefix, longest), paths, nexts, prefix, longest)


def test_accept_chain_and_twins():
    """A chain of 256 that is right throughout; of two children with one token the first is taken, though only the second leads on."""
    n = 256
    chain = (list(range(-1, n - 1)), list(range(n)), list(range(1, n + 1)), [0, n])
    check_accept(call_accept(*chain, [5], 256), [list(range(n))], [n], [5], 256)
    check_accept(call_accept([-1, 0, 0, 2], [1, 4, 4, 6], [4, 9, 6, 8], [0, 4], [0], 8), [[0, 1]], [9], [0], 8)


def test_accept_of_what_is_no_tree():
    """Parents in a ring, or behind their nodes, end the walk; more than 256 rows are reported."""
    f = flag()
    o = call_accept([2, 0, 1], [5, 5, 5], [5, 5, 5], [0, 3], [0], 9, error_flag=f)
    check_accept(o, [[0, 1, 2]], [5], [0], 9)
    o = call_accept([1, 2, 0], [5, 5, 5], [5, 5, 5], [0, 3], [0], 9, error_flag=f)
    check_accept(o, [[0, 2]], [5], [0], 9)
    assert f.item() == 0
    n = 300
    o = call_accept(list(range(-1, n - 1)), list(range(n)), list(range(1, n + 1)), [0, n], [5], 256, error_flag=f)
    check_accept(o, [list(range(256))], [256], [5], 256)
    assert f.item() == 5


@pytest.mark.parametrize("lens", [[1], [8, 0, 30], [64] * 9])
@pytest.mark.parametrize("calls,kvh,hd,bs,dtype", [(1, 1, 64, 16, "bf16"), (3, 2, 128, 16, "bf16"), (2, 8, 64, 32, "f32"), (5, 3, 5, 16, "bf16"), (2, 2, 6, 8, "bf16"),
                                                   (2, 1, 33, 4, "f32"), (4, 2, 20, 24, "bf16")])
def test_accept_writes_the_cache(lens, calls, kvh, hd, bs, dtype):
    """Kept rows' keys and values in their slots, bit for bit; nothing else of the cache is touched; rows of any alignment."""
    parents, tokens, target, cu = accept_case(sum(lens) + hd, lens, right=0.9)
    rng = random.Random(hd)
    prefix = [rng.randrange(0, 70) for _ in lens]
    table, pages = make_table(rng, prefix, lens, bs)
    n, longest = sum(lens), 32
    _, _, _, slots, _ = P.layout([parents[cu[s]:cu[s + 1]] for s in range(len(lens))], prefix, table, bs, 8)
    g = torch.Generator(device=D).manual_seed(hd)
    cache = torch.randn((calls, pages, 2, kvh, bs, hd), generator=g, device=D).to(DTYPES[dtype])
    kv = torch.randn((calls, n, 2 * kvh * hd + 3), generator=g, device=D).to(DTYPES[dtype])
    k, v = kv[..., :kvh * hd], kv[..., kvh * hd:2 * kvh * hd]
    paths, nexts = P.accept(target, tokens, parents, cu, longest)
    want = cache.clone()
    for s, path in enumerate(paths):
        for i, t in enumerate(path):
            page, off = divmod(slots[cu[s] + i], bs)
            want[:, page, 0, :, off] = k[:, cu[s] + t].reshape(calls, kvh, hd)
            want[:, page, 1, :, off] = v[:, cu[s] + t].reshape(calls, kvh, hd)
    f = flag()
    o = call_accept(parents, tokens, target, cu, prefix, longest, slots=ints(slots, torch.int64), k=k, v=v, cache=cache, error_flag=f)
    check_accept(o, paths, nexts, prefix, longest)
    assert cache.equal(want) and f.item() == 0


def test_accept_without_a_slot():
    """Slots of -1 and beyond the cache are not written, and reported."""
    cache, f = torch.zeros((2, 3, 2, 1, 4, 8), device=D), flag()
    k = torch.ones((2, 4, 8), device=D)
    for bad in (-1, 12, 2 ** 40):
        f.zero_()
        cache.zero_()
        call_accept([-1, 0, 1, 2], [0, 1, 2, 3], [1, 2, 3, 4], [0, 4], [1], 4, slots=ints([1, bad, 3, 4], torch.int64), k=k, v=k, cache=cache, error_flag=f)
        assert f.item() == 2
        assert cache.sum() == 3 * 2 * 2 * 8 and (cache[:, 0, :, 0, [1, 3]] == 1).all() and (cache[:, 1, :, 0, 0] == 1).all()


# ----------------------------------------------------------------------------- a run of them

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_step_of_trees_is_what_single_steps_give(dtype):
    """Layout, rotation, attention, logits, choice and acceptance of drafted trees; then the kept tokens one at a time through the framework's
    own decode kernels.  The cache holds the same keys and values bit for bit, and the kept rows' attention outputs agree with the single steps'
    to the sum of both kernels' roundings (`attention_bound` each)."""
    from lmsf_b200 import kernels
    dt = DTYPES[dtype]
    heads, kvh, hd, bs, vocab, width = 8, 2, 64, 16, 211, 8 * 64
    rng, g = random.Random(4), torch.Generator(device=D).manual_seed(4)
    lens, prefix = [9, 1, 24], [37, 0, 90]
    table, pages = make_table(rng, prefix, lens, bs)
    S, n = 3, sum(lens)
    bt, plen, tlen = ints(table), ints(prefix), ints(lens)
    cache = torch.randn((1, pages, 2, kvh, bs, hd), generator=g, device=D).to(dt)
    single = cache.clone()
    emb = torch.randn((vocab, (heads + 2 * kvh) * hd), generator=g, device=D).to(dt)
    head_w = torch.randn((width, vocab), generator=g, device=D)
    inv_freq = 10000.0 ** (-torch.arange(0, hd, 2, device=D, dtype=torch.float32) / hd)
    parents = [p for m in lens for p in P.random_parents(rng, m, reach=3)]
    tokens = ints([rng.randrange(vocab) for _ in range(n)])
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, device=D)  # noqa: E731
    cu, seq, pos, slots, mask = i32(S + 1), i32(n), i32(n), torch.empty(n, dtype=torch.int64, device=D), i32(n, 1)
    hist = ints([[rng.randrange(vocab) for _ in range(100)] for _ in range(S)])
    pen = tuple(torch.full((S,), p, device=D) for p in (0.4, 0.3, 1.2))
    allowed = torch.randint(-2 ** 31, 2 ** 31, (1, (vocab + 31) // 32), generator=torch.Generator().manual_seed(1)).to(torch.int32).to(D)

    def run():
        kernels.tree_layout(cu, seq, pos, slots, mask, ints(parents), tlen, plen, bt, bs)
        qkv = emb[tokens.long()].clone()
        # queries and keys are rotated in place, as one matrix of heads + kv heads
        kernels.rope_cache_write(qkv[:, :(heads + kvh) * hd], None, None, pos, None, None, bs, None, inv_freq, hd, True, heads + kvh, 0, hd)
        q, k, v = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kvh) * hd], qkv[:, (heads + kvh) * hd:]
        out = torch.empty((n, heads * hd), dtype=dt, device=D)
        kernels.attention_tree(out, q, k, v, cache[0], bt, bs, cu, plen, mask, hd ** -0.5, heads, kvh, hd)
        logits = out.float() @ head_w
        kernels.adjust_logits(logits, logits, row_req=seq, history=(hist, plen, ints([10, 0, 50])), penalties=pen, tree=(tokens, mask, cu),
                              allowed=(allowed, ints([0] * n)))
        target = i32(n)
        kernels.sample(target, logits)
        o = [i32(S), i32(S, 16), i32(S), i32(S)]
        return qkv, k, v, out, target, o

    # the draft is made to be right along some paths: what the model would choose behind a node is put into its last child
    for _ in range(6):
        *_, target, _ = run()
        chosen, new = target.tolist(), tokens.tolist()
        for s in range(S):
            first = sum(lens[:s])
            mine = parents[first:first + lens[s]]
            for i in range(1, lens[s]):
                if mine[i] not in mine[i + 1:]:
                    new[first + i] = chosen[first + mine[i]]
        tokens = ints(new)
    qkv, k, v, out, target, o = run()
    kernels.tree_accept(*o, target, tokens, ints(parents), cu, plen, slots=slots, k=k[None], v=v[None], cache=cache)
    paths, nexts = P.accept(target.tolist(), tokens.tolist(), parents, cu.tolist(), 16)
    check_accept(o, paths, nexts, prefix, 16)
    assert max(len(p) for p in paths) >= 3
    ref = P.attention(qkv[:, :heads * hd], k, v, torch.cat([cache[0]]), table, bs, cu.tolist(), prefix, mask.cpu(), hd ** -0.5, heads, kvh, hd)
    bound = P.attention_bound(*ref, hd ** -0.5, hd, 200, dt)
    for s in range(S):
        for i, t in enumerate(paths[s]):
            row = cu.tolist()[s] + t
            x = emb[tokens[row:row + 1].long()].clone()
            q1, k1, v1 = x[:, :heads * hd], x[:, heads * hd:(heads + kvh) * hd], x[:, (heads + kvh) * hd:]
            at, zero = ints([prefix[s] + i]), ints([0])
            kernels.rope_cache_write(q1, k1, v1, at, zero, bt[s:s + 1], bs, single[0], inv_freq, hd, True, heads, kvh, hd)
            one = torch.empty_like(q1)
            kernels.attention_generic(one, q1, single[0], bt[s:s + 1], bs, zero, at, hd ** -0.5, 0, heads, kvh, hd)
            assert ((one.cpu().double() - out[row:row + 1].cpu().double()).abs() <= 2 * bound[row:row + 1]).all()
    assert single.equal(cache)


# ----------------------------------------------------------------------------- calls at the edge of what is allowed

@pytest.mark.parametrize("shape", ["tree", "chain"])
@pytest.mark.parametrize("prefix", [2 ** 31 - 1, 2 ** 31 - 4])
def test_layout_behind_the_last_position(shape, prefix):
    """Positions that 32 bits do not hold: the request is laid out where its last one still is, has no slots and is reported."""
    from lmsf_b200 import kernels
    n, f = 7, flag()
    o = [torch.empty(2, dtype=torch.int32, device=D), ints([0] * n), ints([0] * n), torch.zeros(n, dtype=torch.int64, device=D), torch.zeros((n, 1), dtype=torch.int32, device=D)]
    parents = None if shape == "chain" else ints([-1, 0, 0, 1, 2, 3, 3])
    kernels.tree_layout(*o, parents, ints([n]), ints([prefix]), ints([[0, 1, 2]]), 16, error_flag=f)
    first = 2 ** 31 - 1 - n
    depth = list(range(n)) if shape == "chain" else [0, 1, 1, 2, 2, 3, 3]
    assert o[0].tolist() == [0, n] and o[2].tolist() == [first + d for d in depth]
    assert o[3].tolist() == [-1] * n and f.item() == 5


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_a_row_without_a_stride(dtype, hd):
    """One row: what its tensors say of the distance to the next means nothing."""
    c = attention_case(6, [1], [70], 4, 2, hd, 16, dtype)
    want = call_attention(c)
    check_attention(c, want)
    for name in ("q", "k", "v"):
        t = c[name].clone()
        for stride in (0, 1, 8):
            assert call_attention({**c, name: t.as_strided(t.shape, (stride, 1))}).equal(want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_nodes_that_share_keys(dtype, hd):
    """Rows of k and v that are one row in memory."""
    c = attention_case(7, [19], [70], 4, 2, hd, 16, dtype)
    c["k"], c["v"] = c["k"][3:4].expand(19, -1), c["v"][5:6].expand(19, -1)
    check_attention(c, call_attention(c))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_without_a_cache(dtype):
    """No page at all: a node sees its ancestors only."""
    c = attention_case(9, [40, 3], [0, 0], 4, 2, 64, 16, dtype)
    want = call_attention(c)
    check_attention(c, want)
    bare = {**c, "cache": c["cache"][:0], "prefix": [100, 5]}         # pages of the table that are none: nobody sees their keys
    out = call_attention(bare)
    check_attention(bare, out)


def test_adjust_of_many_biases():
    """More entries than are looked at at once, tokens listed many times far apart: every one counts once, in float32 and the list's order."""
    from lmsf_b200 import kernels
    rng = random.Random(3)
    vocab, rows, n = 5000, 2, [1700, 513]
    token = [rng.choice([7, 4095, 4096, rng.randrange(vocab)]) for _ in range(sum(n))]
    value = [rng.uniform(-2, 2) for _ in token]
    logits = torch.randn((rows, vocab), device=D)
    v32 = torch.tensor(value, dtype=torch.float32)
    out = torch.empty_like(logits)
    kernels.adjust_logits(out, logits, bias=(ints([0, n[0], sum(n)]), ints(token), v32.to(D)))
    add = torch.zeros((rows, vocab), dtype=torch.float32)
    for i, t in enumerate(token):
        add[0 if i < n[0] else 1, t] += v32[i]
    assert (out.cpu() == logits.cpu() + add).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_as_many_requests_as_a_launch_takes(dtype):
    from lmsf_b200 import kernels
    rng = random.Random(12)
    lens, prefix = [rng.choice([0, 1, 1, 2, 5]) for _ in range(1024)], [rng.choice([0, 1, 17, 40, 130]) for _ in range(1024)]
    c = attention_case(12, lens, prefix, 4, 2, 64, 16, dtype, spare_rows=3)
    check_attention(c, call_attention(c))
    more = {**c, "prefix": prefix + [0], "cu": c["cu"] + [c["cu"][-1]], "table": c["table"] + [[-1] * len(c["table"][0])]}
    with pytest.raises(kernels.KernelError, match="1024"):
        call_attention(more)


@pytest.mark.parametrize("rows,vocab", [(70000, 3), (66000, 64)])
def test_adjust_of_very_many_rows(rows, vocab):
    """More rows than a grid has in one dimension."""
    from lmsf_b200 import kernels
    g = torch.Generator(device=D).manual_seed(2)
    logits = torch.randn((rows, vocab), generator=g, device=D)
    req = torch.randint(0, 2, (rows,), generator=g, device=D, dtype=torch.int32)
    which = torch.randint(-1, 2, (rows,), generator=g, device=D, dtype=torch.int32)
    bits = ints([[0b101] + [0] * ((vocab + 31) // 32 - 1), [0b010] + [-1] * ((vocab + 31) // 32 - 1)])
    f = flag()
    out = torch.empty_like(logits)
    kernels.adjust_logits(out, logits, row_req=req, bias=(ints([0, 1, 2]), ints([0, 1]), torch.tensor([0.5, -2.0], device=D)), allowed=(bits, which), error_flag=f)
    want = logits.clone()
    want[:, 0] += torch.where(req == 0, 0.5, 0.0)
    want[:, 1] += torch.where(req == 1, -2.0, 0.0)
    for m in range(2):
        hidden = [v for v in range(vocab) if not ((bits[m, v // 32].item() >> (v % 32)) & 1)]
        rows_of = (which == m).nonzero().flatten()
        want[rows_of[:, None], torch.tensor(hidden, device=D)] = -math.inf
    assert out.equal(want) and f.item() == 0


def test_two_streams_at_once():
    """Calls side by side keep workspaces of their own: the same bits as one after the other."""
    cases = [attention_case(20 + i, lens, prefix, 8, 2, 128, 16, "bf16") for i, (lens, prefix) in enumerate([([33, 64, 1], [700, 300, 2000]), ([48], [5000])])]
    args = []
    for c in cases:
        S = len(c["prefix"])
        args.append((c["q"], c["k"], c["v"], c["cache"], ints(c["table"]).reshape(S, -1), c["bs"], ints(c["cu"]), ints(c["prefix"]), c["mask"].to(D), c["scale"], 8, 2, 128))
    from lmsf_b200 import kernels
    want = [torch.empty_like(c["q"].contiguous()) for c in cases]
    for w, a in zip(want, args):
        kernels.attention_tree(w, *a)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[torch.empty_like(w) for _ in range(10)] for w in want]
    torch.cuda.synchronize()
    for i in range(10):
        for st, outs, a in zip(streams, got, args):
            with torch.cuda.stream(st):
                kernels.attention_tree(outs[i], *a)
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(o.equal(w) for o in outs)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_captured_step_of_all_four(dtype):
    """Layout, attention, logits and acceptance captured as one graph: replayed on other lengths, trees and tokens it gives the bits of eager calls."""
    from lmsf_b200 import kernels
    dt, S, N, H, KV, hd, bs, pages, vocab, calls = DTYPES[dtype], 3, 24, 8, 2, 64, 16, 80, 700, 2
    g = torch.Generator(device=D).manual_seed(5)
    rnd = lambda *shape: torch.randn(shape, generator=g, device=D).to(dt)  # noqa: E731
    tokens, parents = torch.zeros(N, dtype=torch.int32, device=D), torch.zeros(N, dtype=torch.int32, device=D)
    lens, prefix = torch.zeros(S, dtype=torch.int32, device=D), torch.zeros(S, dtype=torch.int32, device=D)
    table = torch.randperm(pages, generator=g, device=D)[:S * 26].view(S, 26).to(torch.int32)
    q, k, v = rnd(N, H * hd), rnd(calls, N, KV * hd), rnd(calls, N, KV * hd)
    w = torch.randn((H * hd, vocab), generator=g, device=D) * 0.05
    history = torch.randint(0, vocab, (S, 400), generator=g, device=D, dtype=torch.int32)
    penalties = tuple(torch.rand(S, generator=g, device=D) + 0.5 for _ in range(3))
    bits = torch.randint(-2 ** 31, 2 ** 31, (2, (vocab + 31) // 32), generator=g, device=D).to(torch.int32)
    which = torch.randint(-1, 2, (N,), generator=g, device=D, dtype=torch.int32)
    cache0 = rnd(calls, pages, 2, KV, bs, hd)
    kernels.error_word(torch.device(D)).zero_()

    def buffers():
        i = lambda *shape: torch.full(shape, -9, dtype=torch.int32, device=D)  # noqa: E731
        return dict(cu=i(S + 1), seq=torch.zeros(N, dtype=torch.int32, device=D), pos=i(N), slots=torch.full((N,), -9, dtype=torch.int64, device=D), mask=torch.zeros((N, 1), dtype=torch.int32, device=D),
                    out=torch.zeros((N, H * hd), dtype=dt, device=D), logits=torch.zeros((N, vocab), device=D), kept=i(S), path=i(S, 8), nxt=i(S), new=i(S), cache=cache0.clone())

    def step(b):
        kernels.tree_layout(b["cu"], b["seq"], b["pos"], b["slots"], b["mask"], parents, lens, prefix, table, bs)
        kernels.attention_tree(b["out"], q, k[0], v[0], b["cache"][0], table, bs, b["cu"], prefix, b["mask"], hd ** -0.5, H, KV, hd)
        torch.mm(b["out"].float(), w, out=b["logits"])
        kernels.adjust_logits(b["logits"], b["logits"], row_req=b["seq"], history=(history, prefix, prefix), penalties=penalties, tree=(tokens, b["mask"], b["cu"]), allowed=(bits, which))
        target = b["logits"].argmax(1).to(torch.int32)
        kernels.tree_accept(b["kept"], b["path"], b["nxt"], b["new"], target, tokens, parents, b["cu"], prefix, b["slots"], k, v, b["cache"])

    def inputs(seed):
        rng = random.Random(seed)
        n = [rng.randrange(0, 9) for _ in range(S)]
        trees = [P.random_parents(rng, m) for m in n]
        flat = [p for t in trees for p in t]
        parents.copy_(ints(flat + [0] * (N - len(flat))))
        tokens.copy_(torch.randint(0, vocab, (N,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32))
        lens.copy_(ints(n))
        prefix.copy_(ints([rng.randrange(0, 390) for _ in range(S)]))

    captured = buffers()
    inputs(0)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(captured)                                               # (libraries are loaded and workspaces made before the capture)
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step(captured)
    torch.cuda.synchronize()
    for seed in range(1, 7):
        inputs(seed)
        eager = buffers()
        for name, t in buffers().items():
            captured[name].copy_(t)
        torch.cuda.synchronize()
        step(eager)
        graph.replay()
        torch.cuda.synchronize()
        for name in eager:
            assert captured[name].equal(eager[name]), (seed, name)
    assert kernels.error_word(torch.device(D)).item() == 0
    del graph


# ----------------------------------------------------------------------------- what one thread leaves for another

@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("prefix", [0, 100, 128, 300])
def test_attention_whose_halves_add_up(hd, prefix):
    """Units of one item, whose tiles the two halves of a block take in turn and whose outputs they read from each other: one tile (a half without any), two,
    three and four; the same bits in every run."""
    c = attention_case(hd + prefix, [3, 1, 9] * 30, [prefix] * 90, 4, 2, hd, 16, "bf16")
    out = call_attention(c)
    check_attention(c, out)
    for _ in range(10):
        assert call_attention(c).equal(out)


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("heads,kvh", [(8, 2), (3, 1), (7, 1)])
@pytest.mark.parametrize("prefix", [[0, 0, 0], [700, 0, 300]])
def test_attention_of_warps_with_a_few_rows(hd, heads, kvh, prefix):
    """Units of two items of which the second ends inside a warp: each finished by one block (one tile, as many blocks as units), and cut."""
    per = 128 // (heads // kvh)
    lens = [per + 1, 2 * per - 1, per + per // 2]
    c = attention_case(hd + heads, lens, prefix, heads, kvh, hd, 16, "bf16", spare_rows=2)
    out = call_attention(c)
    check_attention(c, out)
    for _ in range(3):
        assert call_attention(c).equal(out)


# ----------------------------------------------------------------------------- windows of rows that lie anywhere behind the cached tokens

def on_cores(monkeypatch, dtype):
    """"bf16 on the CUDA cores" -> "bf16", with the tensor cores left out."""
    from lmsf_b200 import kernels
    if dtype.startswith("bf16 "):
        monkeypatch.setattr(kernels, "USE_TC_TREE", False)
        return "bf16"
    return dtype


@pytest.mark.parametrize("dtype", ["f32", "bf16", "bf16 on the CUDA cores"])
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 16), (96, 128)])
@pytest.mark.parametrize("far", [0, 1, 130, 276, 599, 5000])
def test_attention_of_positions_far_behind_the_cache(dtype, hd, bs, far, monkeypatch):
    """A row's window follows its position wherever that lies: `far` and more behind the last cached token and the tree.  Every other request's cached
    keys that no row sees are NaN, and so are their values."""
    dtype, window = on_cores(monkeypatch, dtype), 600
    prefix, lens = [1024, 1000, 385, 700], [1, 7, 40, 2]
    c = attention_case(far + hd, lens, prefix, 4, 2, hd, bs, dtype, window)
    rng = random.Random(far)
    for s in range(4):
        for t in range(c["cu"][s], c["cu"][s + 1]):
            c["positions"][t] = prefix[s] + far + (rng.randrange(0, 2 * window) if t % 3 else 0)
        least = min(c["positions"][c["cu"][s]:c["cu"][s + 1]])
        for i in range(min(prefix[s], least - window + 1) if s % 2 == 0 else 0):
            c["cache"][c["table"][s][i // bs], :, :, i % bs] = math.nan
    check_attention(c, call_attention(c))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "bf16 on the CUDA cores"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_with_a_window_over_a_table_that_ends(dtype, hd, monkeypatch):
    """Cached tokens behind the table's last block are seen by nobody, and move nobody's window."""
    c = attention_case(hd, [5, 1, 30], [1000, 900, 650], 4, 2, hd, 16, on_cores(monkeypatch, dtype), window=600)
    c["table"] = [row[:40] for row in c["table"]]
    check_attention(c, call_attention(c))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_hides_infinities_behind_a_far_window(dtype):
    """A value of infinity in a cached place reaches the rows whose window holds it, and no other."""
    prefix, window = 512, 300
    c = attention_case(3, [6], [prefix], 4, 2, 64, 16, dtype, window=window)
    c["positions"] = [512, 640, 700, 730, 900, 513]
    place, col = 390, 9                                           # seen by positions up to 689
    c["cache"][c["table"][0][place // 16], 1, :, place % 16, col] = math.inf
    out = call_attention(c)
    for t, p in enumerate(c["positions"]):
        inf = torch.isinf(out[t]).nonzero().flatten().tolist()
        assert inf == ([col + 64 * h for h in range(4)] if p - window < place else []) and not torch.isnan(out[t]).any()
    c["cache"][c["table"][0][place // 16], 1, :, place % 16, col] = 0.25
    check_attention(c, call_attention(c))


# ----------------------------------------------------------------------------- options that are there for nobody

@pytest.mark.parametrize("option", ["penalties", "bias", "masks"])
def test_adjust_reports_options_of_no_request(option):
    """Penalties or biases of no request, masks of which there is none: a row that asks for one is reported and passes, one that asks for no mask is not."""
    from lmsf_b200 import kernels
    none = torch.zeros(0, device=D)
    kw = dict(penalties=dict(penalties=(none, none, none)), bias=dict(bias=(ints([0]), ints([]), none)), masks=dict(allowed=(ints([]).reshape(0, 4), ints([-1, 0, -1]))))[option]
    x, f = torch.randn((3, 100), device=D), flag()
    out = torch.empty_like(x)
    kernels.adjust_logits(out, x, row_req=ints([0, 0, 0]), error_flag=f, **kw)
    assert f.item() == 5 and out.equal(x)
    f.zero_()
    kernels.adjust_logits(out, x, row_req=ints([5, -1, 0]), allowed=(ints([]).reshape(0, 4), ints([-1, -1, -1])), error_flag=f)
    assert f.item() == 0 and out.equal(x)


# ----------------------------------------------------------------------------- forms of a call that large steps and views of buffers take

@pytest.mark.parametrize("vocab,requests,nodes,width", [(210, 310, 31, 12), (40, 3900, 9, 6), (2100, 160, 31, 12)])
@pytest.mark.parametrize("order", ["in order", "shuffled", "strangers"])
def test_adjust_of_several_rows_a_block(vocab, requests, nodes, width, order):
    """So many rows that a block takes two (4,736 chunks and more) or eight (18,944) in turn, with every option: what is marked for a request is kept over its rows, and
    made anew where the next row is another's, in the middle of a block too.  Strangers: rows between those of one request that ask for one beyond the tensors; they pass with their mask alone."""
    from lmsf_b200 import kernels
    rng = random.Random(vocab)
    lens = [rng.choice([nodes, nodes - 1, nodes // 2, 1, nodes]) for _ in range(requests)]
    short = {210: 4736, 40: 18944, 2100: 2368}[vocab] - sum(lens)
    lens += [nodes] * max(0, -(-short // nodes))
    logits, host, dev = adjust_case(vocab, vocab, lens, width=width)
    rows, seq = sum(lens), list(host["row_req"])
    host["allowed"][1][:] = [w if r % 6 == 0 else -1 for r, w in enumerate(host["allowed"][1])]
    if order == "shuffled":                                       # (bits of a row's mask are places in its request's tree, whichever that is)
        for at in range(0, rows, 5):
            part = seq[at:at + 5]
            rng.shuffle(part)
            seq[at:at + 5] = part
    host["row_req"], asked, strange = seq, list(seq), []
    if order == "strangers":
        strange = list(range(3, rows, 7))
        for r in strange:
            asked[r] = len(lens) + r % 3 if r % 2 else -1 - r % 3
    dev["row_req"], dev["allowed"] = ints(asked), (dev["allowed"][0], ints(host["allowed"][1]))
    f, out = flag(), torch.full_like(logits, 7.0)
    kernels.adjust_logits(out, logits, error_flag=f, **dev)
    assert f.item() == (5 if strange else 0)
    plain = [r for r in range(rows) if r not in set(strange)]
    some = [r for r in plain if vocab != 40 or r % 3 == 0]       # (the plain loops are slow: of the most rows every third)
    tokens, mask, cu = host["tree"]
    want_host = dict(host, row_req=[seq[r] for r in some], tree=(tokens, mask[some], cu), allowed=(host["allowed"][0], [host["allowed"][1][r] for r in some]))
    check_adjusted(out[some], logits[some], want_host)
    if strange:
        want, _ = P.adjust(logits[strange], [0] * len(strange), allowed=(host["allowed"][0], [host["allowed"][1][r] for r in strange]))
        assert out[strange].cpu().double().equal(want)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "bf16 on the CUDA cores"])
@pytest.mark.parametrize("hd,heads,kvh", [(64, 8, 2), (128, 4, 2), (112, 6, 6), (33, 4, 2)])
@pytest.mark.parametrize("lens,prefix", [([37, 5, 64], [0, 0, 0]), ([40, 3], [900, 130])])
@pytest.mark.parametrize("first,more", [(3, 7), (1, 16), (8, 16), (0, 9)])
def test_attention_into_columns_of_a_buffer(dtype, hd, heads, kvh, lens, prefix, first, more, monkeypatch):
    """The output as columns of wider rows, at every alignment, of units that one block finishes and of those that are joined; what lies around it is left alone."""
    c = attention_case(hd + first, lens, prefix, heads, kvh, hd, 16, on_cores(monkeypatch, dtype), spare_rows=2)
    n, w = c["q"].shape[0], heads * hd
    wide = torch.full((n, w + more), 7.0, dtype=c["dtype"], device=D)
    out = wide[:, first:first + w]
    call_attention(c, out)
    check_attention(c, out)
    assert (wide[:, :first] == 7.0).all() and (wide[:, first + w:] == 7.0).all()


@pytest.mark.parametrize("what", ["q", "k", "v", "rows of k", "cache", "negative", "zero", "group"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_that_the_tensor_cores_do_not_take(what, hd):
    """bfloat16 of their head sizes, but rows off 16 bytes, a scale that is not positive, more than 128 heads a group."""
    heads, kvh = (129, 1) if what == "group" else (8, 2)
    c = attention_case(hd, [20, 3], [200, 70], heads, kvh, hd, 16, "bf16")
    if what in ("q", "k", "v"):
        wide = torch.zeros((c[what].shape[0], c[what].shape[1] + 8), dtype=torch.bfloat16, device=D)
        wide[:, 1:-7] = c[what]
        c[what] = wide[:, 1:-7]
    elif what == "rows of k":
        wide = torch.zeros((c["k"].shape[0], c["k"].shape[1] + 3), dtype=torch.bfloat16, device=D)
        wide[:, :-3] = c["k"]
        c["k"] = wide[:, :-3]
    elif what == "cache":
        line = torch.zeros(c["cache"].numel() + 1, dtype=torch.bfloat16, device=D)
        line[1:] = c["cache"].flatten()
        c["cache"] = line[1:].view(c["cache"].shape)
    elif what != "group":
        c["scale"] = -0.07 if what == "negative" else 0.0
    check_attention(c, call_attention(c))
