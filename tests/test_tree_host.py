"""The refusals of the operators on drafted trees that need no device, and their plain implementations by themselves."""
import math
import random

import pytest
import torch

import plain_tree as P
from lmsf_b200 import kernels
from lmsf_b200.kernels import KernelError

I = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
L = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
F = lambda *s: torch.zeros(s, dtype=torch.float32)  # noqa: E731


def layout_args(**kw):
    a = dict(cu_q=I(3), token_seq=I(9), positions=I(9), slots=L(9), mask=I(9, 2), parents=I(9), tree_len=I(2), prefix_len=I(2),
             block_table=I(2, 4), block_size=16)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [dict(cu_q=I(2)), dict(token_seq=L(9)), dict(positions=I(8)), dict(slots=I(9)), dict(slots=L(18)[::2]), dict(mask=I(8, 2)),
                                dict(mask=I(9, 9)), dict(mask=I(9, 0)), dict(mask=I(9)), dict(parents=I(4)), dict(tree_len=I(3)), dict(prefix_len=I(1)),
                                dict(block_table=I(3, 4)), dict(block_table=I(4)), dict(block_size=0), dict(window=-1), dict(mask=None, window=4),
                                dict()])
def test_layout_refuses(kw):
    """Shapes, types and options; with nothing else wrong, tensors that are on no device."""
    with pytest.raises(KernelError):
        kernels.tree_layout(**layout_args(**kw))


def attention_args(**kw):
    a = dict(out=F(9, 64), q=F(9, 64), k=F(9, 32), v=F(9, 32), cache=F(5, 2, 2, 16, 16), block_table=I(2, 4), block_size=16, cu_q=I(3), prefix_len=I(2),
             mask=I(9, 1), scale=0.25, n_q_heads=4, n_kv_heads=2, head_dim=16)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [dict(out=F(9, 48)), dict(out=F(64, 9).t()), dict(k=F(9, 64)), dict(v=F(8, 32)), dict(cache=F(5, 2, 2, 16, 32)),
                                dict(cache=F(5, 1, 2, 16, 16)), dict(cache=F(5, 2, 2, 16, 16).transpose(2, 3)), dict(block_size=8), dict(block_table=I(3, 4)),
                                dict(cu_q=I(2)), dict(cu_q=L(3)), dict(mask=I(9)), dict(mask=I(9, 0)), dict(mask=I(8, 1)), dict(n_q_heads=3),
                                dict(n_kv_heads=3), dict(window=5), dict(window=-1), dict(window=5, positions=I(8)), dict(scale=math.nan),
                                dict(q=F(9, 64).half()), dict(v=F(9, 32).bfloat16()), dict(q=F(9, 128)[:, ::2]), dict()])
def test_attention_refuses(kw):
    with pytest.raises(KernelError):
        kernels.attention_tree(**attention_args(**kw))


def adjust_args(**kw):
    a = dict(out=F(6, 40), logits=F(6, 40), row_req=I(6), history=(I(2, 7), I(2), I(2)), penalties=(F(2), F(2), F(2)), tree=(I(6), I(6, 1), I(3)),
             bias=(I(3), I(5), F(5)), allowed=(I(3, 2), I(6)))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [dict(out=F(6, 41)), dict(logits=F(6, 40).bfloat16()), dict(logits=F(40, 6).t()), dict(logits=F(1, 40).expand(6, 40)), dict(row_req=I(5)),
                                dict(row_req=None), dict(history=(I(3, 7), I(2), I(2))), dict(history=(L(2, 7), I(2), I(2))), dict(history=(I(2, 7), I(3), I(2))),
                                dict(penalties=None), dict(penalties=(F(2), F(3), F(2))), dict(tree=(I(5), I(6, 1), I(3))), dict(tree=(I(6), I(6), I(3))),
                                dict(tree=(I(6), I(6, 1), I(4))), dict(bias=(I(4), I(5), F(5))), dict(bias=(I(3), I(5), F(4))), dict(allowed=(I(3, 1), I(6))),
                                dict(allowed=(I(2), I(6))), dict(allowed=(I(3, 2), I(3))), dict()])
def test_adjust_refuses(kw):
    with pytest.raises(KernelError):
        kernels.adjust_logits(**adjust_args(**kw))


def test_adjust_refuses_a_shifted_self():
    x = F(13, 40)
    with pytest.raises(KernelError, match="apart"):
        kernels.adjust_logits(x[::2][:6], x[:6])


def accept_args(**kw):
    a = dict(n_kept=I(2), path=I(2, 4), next_token=I(2), new_len=I(2), target=I(9), tokens=I(9), parents=I(9), cu_q=I(3), prefix_len=I(2), slots=L(9),
             k=F(3, 9, 32), v=F(3, 9, 32), cache=F(3, 5, 2, 2, 16, 16))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [dict(n_kept=I(3)), dict(path=I(2)), dict(path=I(2, 0)), dict(path=I(2, 257)), dict(path=I(3, 4)), dict(next_token=L(2)), dict(tokens=I(8)),
                                dict(parents=I(10)), dict(cu_q=I(2)), dict(slots=None), dict(k=None), dict(cache=None), dict(slots=I(9)),
                                dict(cache=F(3, 5, 1, 2, 16, 16)), dict(cache=F(5, 2, 2, 16, 16)), dict(k=F(3, 9, 16)), dict(k=F(3, 9, 32).bfloat16()),
                                dict(v=F(3, 32, 9).transpose(1, 2)), dict(cache=F(3, 5, 2, 2, 16, 16).half(), k=F(3, 9, 32).half(), v=F(3, 9, 32).half()), dict()])
def test_accept_refuses(kw):
    with pytest.raises(KernelError):
        kernels.tree_accept(**accept_args(**kw))


def test_plain_tree_and_a_chain():
    """A chain's ancestors are the nodes before it; a walk down a tree that was built to be right takes all of it."""
    rng = random.Random(3)
    assert P.ancestors([-1, 0, 1]) == [{0}, {0, 1}, {0, 1, 2}]
    cu, seq, pos, slots, mask = P.layout([[-1, 0, 0, 2]], [15], [[7, 3]], 16, 1)
    assert (cu, seq, pos, slots) == ([0, 4], [0] * 4, [15, 16, 16, 17], [7 * 16 + 15, 48, 49, 50])
    assert mask.flatten().tolist() == [1, 3, 5, 13]
    assert P.layout([[-1, 0, 0, 2]], [15], [[7, 3]], 16, 1, window=2)[4].flatten().tolist() == [1, 3, 5, 12]
    tokens = [rng.randrange(50) for _ in range(20)]
    assert P.accept(tokens[1:] + [99], tokens, list(range(-1, 19)), [0, 20], 32) == ([list(range(20))], [99])
    assert P.accept(tokens[1:] + [99], tokens, list(range(-1, 19)), [0, 20], 6) == ([list(range(6))], [tokens[6]])


# ----------------------------------------------------------------------------- calls that would read what is not there

@pytest.mark.parametrize("kw", [dict(history=(I(2, 7), None, I(2))), dict(history=(I(2, 7), I(2), None)), dict(history=(None, I(2), I(2))), dict(penalties=(F(2), None, F(2))),
                                dict(penalties=(F(2), F(2), None)), dict(tree=(I(6), I(6, 1), None)), dict(tree=(I(6), None, I(3))), dict(tree=(None, I(6, 1), I(3))),
                                dict(bias=(I(3), None, F(5))), dict(bias=(I(3), I(5), None)), dict(bias=(None, I(5), F(5))), dict(allowed=(I(3, 2), None)),
                                dict(allowed=(None, I(6)))])
def test_adjust_refuses_half_an_option(kw):
    with pytest.raises(KernelError, match="belong together"):
        kernels.adjust_logits(**adjust_args(**kw))


@pytest.mark.parametrize("kw", [dict(history=(I(2, 7), I(2))), dict(penalties=(F(2),)), dict(tree=(I(6), I(6, 1), I(3), I(3))), dict(bias=()), dict(allowed=(I(3, 2), I(6), I(6)))])
def test_adjust_refuses_an_option_of_other_parts(kw):
    with pytest.raises(KernelError, match="tensors"):
        kernels.adjust_logits(**adjust_args(**kw))


def test_adjust_apart_or_itself():
    both, line = F(6, 96), F(6 * 40 + 20)
    bad = [(line[:240].view(6, 40), line[20:].view(6, 40)), (both[:, :40], both[:, 30:70]), (both[:, 40:80], both[:, :48][:, 8:])]
    for out, logits in bad:
        with pytest.raises(KernelError, match="apart"):
            kernels.adjust_logits(out, logits)
    for out, logits in [(both[:, :40], both[:, 40:80]), (both[:, 56:], both[:, :40]), (both, both), (line[:40].view(1, 40), line[40:80].view(1, 40))]:
        with pytest.raises(KernelError, match="CUDA tensors"):       # nothing else is wrong with them
            kernels.adjust_logits(out, logits)


def test_attention_refuses_an_output_over_its_inputs():
    rows = F(9, 64 + 2 * 32)
    q, k, v = rows[:, :64], rows[:, 64:96], rows[:, 96:]
    for out in (q, rows[:, 32:96], rows[:, 64:]):
        with pytest.raises(KernelError, match="shares memory"):
            kernels.attention_tree(**attention_args(out=out, q=q, k=k, v=v))
    wide = F(9, 2 * 64 + 2 * 32)
    with pytest.raises(KernelError, match="CUDA tensors"):            # columns of one buffer
        kernels.attention_tree(**attention_args(out=wide[:, 64:128], q=wide[:, :64], k=wide[:, 128:160], v=wide[:, 160:]))


@pytest.mark.parametrize("kw", [dict(scale=1e300), dict(scale=-1e39), dict(scale=math.inf)])
def test_attention_refuses_a_scale_beyond_float32(kw):
    with pytest.raises(KernelError, match="scale"):
        kernels.attention_tree(**attention_args(**kw))


def test_attention_refuses_what_32_bits_do_not_count():
    none = dict(out=F(0, 64), q=F(0, 64), k=F(0, 32), v=F(0, 32), cu_q=I(1), prefix_len=I(0))
    with pytest.raises(KernelError, match="32 bits"):
        kernels.attention_tree(**attention_args(**none, mask=I(0, 2 ** 25 + 1), block_table=I(0, 4)))
    with pytest.raises(KernelError, match="32 bits"):
        kernels.attention_tree(**attention_args(**none, mask=I(0, 1), block_table=I(0, 2 ** 26 + 1)))
    with pytest.raises(KernelError, match="CUDA tensors"):
        kernels.attention_tree(**attention_args(**none, mask=I(0, 2 ** 25), block_table=I(0, 2 ** 26)))


# ----------------------------------------------------------------------------- memory that is written to and read or written again in one call

def test_attention_refuses_rows_of_out_over_one_another():
    for out in (F(1, 64).expand(9, 64), F(9 * 64).as_strided((9, 64), (63, 1)), F(9 * 64).as_strided((9, 64), (8, 1))):
        with pytest.raises(KernelError, match="rows of out"):
            kernels.attention_tree(**attention_args(out=out))
    one = dict(out=F(1, 64).as_strided((1, 64), (0, 1)), q=F(1, 64), k=F(1, 32), v=F(1, 32), mask=I(1, 1))
    with pytest.raises(KernelError, match="CUDA tensors"):            # a single row's stride says nothing
        kernels.attention_tree(**attention_args(**one))
    with pytest.raises(KernelError, match="CUDA tensors"):
        kernels.attention_tree(**attention_args(out=F(9, 80)[:, 3:67]))


def test_attention_refuses_an_output_in_the_cache():
    size = 5 * 2 * 2 * 16 * 16                                        # of the cache; 9 rows of 64 are 576
    line = F(size + 2000)
    cache = line[1000:1000 + size].view(5, 2, 2, 16, 16)
    spread = F(9 * 3000)                                              # rows 3,000 apart, the cache after the first, its last value on the second or not
    for out in (line[1000:1576].view(9, 64), line[425:1001].view(9, 64), line[1000 + size - 1:][:576].view(9, 64), line[500:].as_strided((9, 64), (600, 1))):
        with pytest.raises(KernelError, match="the cache"):
            kernels.attention_tree(**attention_args(out=out, cache=cache))
    for out in (line[424:1000].view(9, 64), line[1000 + size:][:576].view(9, 64)):
        with pytest.raises(KernelError, match="CUDA tensors"):        # right before and behind it
            kernels.attention_tree(**attention_args(out=out, cache=cache))
    small = dict(cache=spread[64:64 + 2560].view(1, 2, 2, 40, 16), block_size=40)
    with pytest.raises(KernelError, match="CUDA tensors"):            # between two rows
        kernels.attention_tree(**attention_args(out=spread.as_strided((9, 64), (2624, 1)), **small))
    with pytest.raises(KernelError, match="the cache"):
        kernels.attention_tree(**attention_args(out=spread.as_strided((9, 64), (2623, 1)), **small))
    with pytest.raises(KernelError, match="CUDA tensors"):            # a cache of no pages
        kernels.attention_tree(**attention_args(cache=F(0, 2, 2, 16, 16)))


def test_accept_refuses_keys_in_the_cache():
    """Rows are copied in no order: one that lies in the cache may have been written over before it is read."""
    size = 3 * 5 * 2 * 2 * 16 * 16
    line = F(size + 4000)
    cache = line[2000:2000 + size].view(3, 5, 2, 2, 16, 16)
    inside, first, last = (line[at:at + 864].view(3, 9, 32) for at in (5000, 2000 - 863, 2000 + size - 1))
    third = line[1000:].as_strided((3, 9, 32), (600, 40, 1))          # the third layer's rows alone
    for t in (inside, first, last, third):
        for name in ("k", "v"):
            with pytest.raises(KernelError, match="apart from the cache"):
                kernels.tree_accept(**accept_args(cache=cache, **{name: t}))
    for t in (line[2000 - 864:2000].view(3, 9, 32), line[2000 + size:][:864].view(3, 9, 32), F(1, 1, 32).expand(3, 9, 32)):
        with pytest.raises(KernelError, match="CUDA tensors"):        # right before and behind it, and one row for all
            kernels.tree_accept(**accept_args(cache=cache, k=t, v=t))
    with pytest.raises(KernelError, match="CUDA tensors"):            # nothing is written to a cache of no pages
        kernels.tree_accept(**accept_args(cache=cache[:, :0]))
