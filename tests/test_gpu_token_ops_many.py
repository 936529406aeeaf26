"""Attention over many documents: CTAs that take several heads of a document in turn, documents
that are found by more than one round of search, long ones among very many short ones."""
import functools
import math

import pytest

from test_gpu_token_ops import HALVES, Problem, binding, kernel  # noqa: F401

pytestmark = pytest.mark.gpu

try:
    import torch
except ImportError:  # collected without torch: the GPU run has it
    torch = None


def lengths(seed, count, low, high):
    return torch.randint(low, high + 1, (count,), generator=torch.Generator().manual_seed(seed)).tolist()


# About 600 row tiles' places and seven key heads: 4200 tiles, which a CTA takes 4, 3 or 2 heads at a time,
# as two, three or four of them fit on an SM, and the last has fewer. (queries, keys of a document)
HEADS = {
    "one-tile": (300, 1, (64, 64), (64, 64), {}),
    "one-tile-ragged": (330, 1, (40, 64), (40, 64), dict(causal=True)),
    "three-tiles": (300, 1, (64, 64), (130, 192), {}),
    "more-tiles": (300, 1, (64, 64), (100, 400), {}),
    "two-query-heads": (220, 2, (33, 64), (33, 200), dict(causal=True)),
    "two-row-tiles": (200, 1, (65, 128), (65, 128), dict(causal=True, prefixes=True)),
}


@pytest.mark.parametrize("name,dim,axes,cap,dtype", [
    (name, dim, *((0, 0.0), (2, 0.0), (3, 20.0))[(i + j) % 3], HALVES[(i + j) % 2])
    for i, name in enumerate(HEADS) for j, dim in enumerate((32, 64, 128))])
def test_attention_several_heads_a_cta(name, axes, cap, dim, dtype, monkeypatch):
    monkeypatch.setenv("S2S_MASKED_ATTN", "mma")
    count, group, q, kv, more = HEADS[name]
    more = dict(more)
    q_lens = lengths(dim, count, *q)
    kv_lens = q_lens if q == kv else [max(a, b) for a, b in zip(q_lens, lengths(dim + 1, count, *kv))]
    prefix = [n // 2 for n in q_lens] if more.pop("prefixes", False) else None
    P = Problem(dtype, dim, 7 * group, 7, q_lens, kv_lens, axes=axes, cap=cap, prefix=prefix, **more)
    out, lse = P.run()
    P.check(out, lse)
    again, _ = P.run(lse=False)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dim,axes,dtype", [(32, 0, "float16"), (32, 2, "bfloat16"), (64, 2, "float16"), (128, 0, "bfloat16")])
def test_attention_hidden_values_with_several_heads_a_cta(axes, dim, dtype, monkeypatch):
    """NaN in one channel of the last key of every document, infinity in another head's: only the last rows
    of those heads see them. (An infinity gives infinity, or NaN where the weight is nothing in 16 bits: with
    positions 60 apart on two axes it can be e^-78 of the largest.)"""
    monkeypatch.setenv("S2S_MASKED_ATTN", "mma")
    lens = lengths(dim, 330, 40, 64)
    P = Problem(dtype, dim, 7, 7, lens, lens, causal=True, axes=axes)
    want = P.expected()
    last = torch.tensor(lens).cumsum(0) - 1
    P.v[last, 5, 3] = float("nan")
    P.v[last, 0, 1] = float("inf")
    out, lse = P.run()
    got = out.cpu().double()
    seen = torch.zeros(got.shape, dtype=torch.bool)
    seen[last, 5, 3] = seen[last, 0, 1] = True
    infinite = got[last, 0, 1]
    assert got[last, 5, 3].isnan().all() and (infinite[~infinite.isnan()] == math.inf).all()
    assert axes or not infinite.isnan().any()
    assert ((got - want[0]).abs() <= want[2])[~seen].all()
    assert ((lse.cpu().double() - want[1]).abs() <= want[3]).all()


MANY = {
    "unequal": (lengths(1, 2000, 0, 40), None),
    "unequal-keys": (lengths(2, 1500, 0, 20), lengths(3, 1500, 0, 90)),
    "one-long-first": ([1200] + [1] * 700, None),
    "one-long-last": ([1] * 1100 + [0] * 40 + [900], None),
    "long-between": ([3] * 300 + [700] + [0] * 500 + [17] * 200 + [600] + [1] * 90, None),
    "decoding-and-a-prompt": ([1] * 200 + [500, 300], lengths(4, 200, 1, 900) + [500, 2000]),
    "empty": ([0] * 1500 + [5] + [0] * 1500, None),
}


@functools.lru_cache(maxsize=None)
def many(name, dim, axes, causal, dtype):
    """The problem and what the definition says, for both kernels."""
    q_lens, kv_lens = MANY[name]
    P = Problem(dtype, dim, 2, 1, q_lens, kv_lens or q_lens, causal=causal, axes=axes)
    return P, P.expected()


@pytest.mark.parametrize("dim,axes,causal,dtype", [(64, 0, True, "float16"), (128, 1, True, "bfloat16"),
                                                   (32, 2, False, "float16")])
@pytest.mark.parametrize("name", list(MANY))
def test_attention_over_very_many_documents(name, dim, axes, causal, dtype, kernel):
    P, want = many(name, dim, axes, causal, dtype)
    P.check(*P.run(), want=want)
