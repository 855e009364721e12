"""Plain implementations of the operators on drafted trees: loops and 64-bit floats, one request and one row at a time."""
import math

import torch


def random_parents(rng, n, reach=6, roots=0.0):
    """A tree of n nodes; a node follows one of the `reach` nodes before it, or with probability `roots` the cached tokens."""
    return [-1 if i == 0 or rng.random() < roots else max(0, i - 1 - rng.randrange(reach)) for i in range(n)]


def ancestors(parents):
    """For every node the set of its ancestors and itself."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else frozenset()) | {i})
    return out


def words_of(sets, words):
    """Sets of nodes -> int32 [rows, words]."""
    rows = []
    for s in sets:
        bits = sum(1 << j for j in s)
        rows.append([(bits >> (32 * w)) & 0xffffffff for w in range(words)])
    return torch.tensor(rows, dtype=torch.int64).reshape(len(sets), words).to(torch.int32)


def layout(trees, prefix, table, block_size, words, window=0):
    """trees: a list of parents per request.  -> the five outputs as lists and tensors."""
    cu, seq, pos, slots, sets = [0], [], [], [], []
    for s, parents in enumerate(trees):
        own = ancestors(parents)
        for i in range(len(parents)):
            depth = len(own[i]) - 1
            place = prefix[s] + i
            blk = place // block_size
            page = table[s][blk] if blk < len(table[s]) else -1
            seq.append(s)
            pos.append(prefix[s] + depth)
            slots.append(page * block_size + place % block_size if page >= 0 else -1)
            sets.append({j for j in own[i] if not window or len(own[j]) - 1 > depth - window})
        cu.append(cu[-1] + len(parents))
    return cu, seq, pos, slots, words_of(sets, words)


def bit(row, j):
    return j // 32 < len(row) and (row[j // 32] >> (j % 32)) & 1


def attention(q, k, v, cache, table, block_size, cu, prefix, mask, scale, heads, kvh, hd, positions=None, window=0):
    """-> out [N, heads * hd] in 64 bits, and how far a kernel may be from it: a row's and column's sum of weight * |v|, and the largest sum over
    the head of |q k| that a row meets.  Everything on the CPU."""
    q, k, v, cache = (t.detach().cpu().double() for t in (q, k, v, cache))
    n, group, pages = q.shape[0], heads // kvh, cache.shape[0]
    out, absolute, largest = (torch.zeros((n, heads, hd), dtype=torch.float64) for _ in range(3))
    for s in range(len(prefix)):
        for t in range(cu[s], cu[s + 1]):
            row = mask[t].tolist()
            for g in range(kvh):
                ks, vs = [], []
                for i in range(prefix[s]):
                    blk = i // block_size
                    page = table[s][blk] if blk < len(table[s]) else -1
                    if 0 <= page < pages and (not window or i > positions[t] - window):
                        ks.append(cache[page, 0, g, i % block_size])
                        vs.append(cache[page, 1, g, i % block_size])
                for j in range(cu[s + 1] - cu[s]):
                    if bit(row, j):
                        ks.append(k[cu[s] + j, g * hd:(g + 1) * hd])
                        vs.append(v[cu[s] + j, g * hd:(g + 1) * hd])
                if not ks:
                    continue
                K, V = torch.stack(ks), torch.stack(vs)
                for h in range(g * group, (g + 1) * group):
                    x = q[t, h * hd:(h + 1) * hd]
                    w = torch.softmax(K @ x * scale, 0)
                    out[t, h] = w @ V
                    absolute[t, h] = w @ V.abs()
                    largest[t, h] = float((K.abs() @ x.abs()).max())
    return out.flatten(1), absolute.flatten(1), largest.flatten(1)


def attention_bound(out, absolute, largest, scale, hd, keys, dtype):
    """How far a kernel may be from `attention`.  A score is a sum of hd products times scale, rounded hd + 4 times by 2^-24 (2^-23 where
    sums are cut off), each of at most `largest`; its error e moves its weight by a factor 1 + e, and so numerator and denominator: 2 e of the
    sum of weight * |v|.  The sums over the keys and their rescaling round keys + 16 times more.  In bfloat16 the weights are rounded (2^-8
    of each) and the result is (2^-8); 1.1 covers the products of these."""
    e = 2 * (hd + 8) * 2.0 ** -23 * abs(scale) * largest + (keys + 16) * 2.0 ** -23
    bound = e * absolute
    if dtype == torch.bfloat16:
        bound = 1.1 * (bound + 2.0 ** -8 * absolute + 2.0 ** -8 * out.abs())
    else:
        bound = bound + 2.0 ** -24 * out.abs()
    return bound + 1e-30


def adjust(logits, row_req, history=None, penalties=None, tree=None, bias=None, allowed=None):
    """-> 64-bit result and the sum of the absolute values that went into each."""
    x = logits.detach().cpu().double().clone()
    rows, vocab = x.shape
    size = x.abs().clone()
    for r in range(rows):
        req = row_req[r]
        if penalties is not None:
            presence, frequency, repetition = (p[req].item() for p in penalties)
            prompt, said = set(), {}
            if history is not None:
                tokens, length, n_prompt = history
                for i, t in enumerate(tokens[req].tolist()[:length[req]]):
                    if not 0 <= t < vocab:
                        continue
                    if i < n_prompt[req]:
                        prompt.add(t)
                    else:
                        said[t] = said.get(t, 0) + 1
            if tree is not None:
                tokens, mask, cu = tree
                row = mask[r].tolist()
                for j in range(cu[req + 1] - cu[req]):
                    t = int(tokens[cu[req] + j])
                    if bit(row, j) and 0 <= t < vocab:
                        said[t] = said.get(t, 0) + 1
            for t in prompt | set(said):
                z = float(x[r, t])
                z = z / repetition if z > 0 else z * repetition
                c = said.get(t, 0)
                size[r, t] = abs(z) + abs(frequency * c) + abs(presence)
                x[r, t] = z - frequency * c - (presence if c else 0.0)
        if bias is not None:
            start, token, value = bias
            for e in range(start[req], start[req + 1]):
                if 0 <= token[e] < vocab:
                    x[r, token[e]] += value[e]
                    size[r, token[e]] += abs(value[e])
        if allowed is not None and allowed[1][r] >= 0:
            row = allowed[0][allowed[1][r]].tolist()
            for t in range(vocab):
                if not bit(row, t):
                    x[r, t] = -math.inf
    return x, size


def accept(target, tokens, parents, cu, longest):
    """-> paths (lists of places) and next tokens."""
    paths, nexts = [], []
    for s in range(len(cu) - 1):
        n = cu[s + 1] - cu[s]
        path = [0] if n else []
        while path and len(path) < longest:
            last = path[-1]
            child = [i for i in range(last + 1, n) if parents[cu[s] + i] == last and tokens[cu[s] + i] == target[cu[s] + last]]
            if not child:
                break
            path.append(child[0])
        paths.append(path)
        nexts.append(target[cu[s] + path[-1]] if path else -1)
    return paths, nexts
