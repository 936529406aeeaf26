"""The token operators at the ends of their ranges: large scores, small weights, biases that
grow far, tokens near 2^31, against plain 64-bit implementations.

Tolerances count roundings, u = eps / 2 of the tensors' type; each test says which.
"""
import math

import pytest

from test_gpu_token_ops import HALVES, Problem, binding, heads, kernel, unit  # noqa: F401

pytestmark = pytest.mark.gpu

try:
    import torch
except ImportError:  # collected without torch: the GPU run has it
    torch = None


def softmax(P):
    """Outputs and log sums of one-headed keys without a mask, in 64 bits, weights divided by their sum (a
    log sum in 64 bits has no room for that of a few keys beside scores of 2^50)."""
    out, lse, a, b = [], [], 0, 0
    for nq, nk in zip(P.q_lens, P.kv_lens):
        z = P.q[a:a + nq].double() @ P.k[b:b + nk, 0].double().T * P.scale  # [query][head][key]
        if P.cap:
            z = P.cap * torch.tanh(z / P.cap)
        for x in range(P.axes):
            far = (P.q_pos[x, a:a + nq, None].double() - P.kv_pos[x, None, b:b + nk].double()).abs()
            z = z - P.slopes[x].double().abs()[:, None] * far[:, None]
        out.append(torch.softmax(z, 2) @ P.v[b:b + nk, 0].double())
        lse.append(torch.logsumexp(z, 2).T)
        a, b = a + nq, b + nk
    return torch.cat(out), torch.cat(lse, 1)


def check(P):
    """Scores that are exact in 32 bits: what is left are the exponentials' argument and value (2^-20
    with the sums of a few thousand terms), the weights' rounding and the output's."""
    out, lse = P.run()
    o, w = softmax(P)
    u, big = unit(P.dtype), P.v.abs().max().double()
    got, sums = out.cpu().double(), lse.cpu().double()
    assert ((got - o).abs() <= u * o.abs() + (u + 2.0 ** -20) * big).all(), float((got - o).abs().max())
    assert ((sums - w).abs() <= 2.0 ** -20 + 2.0 ** -21 * w.abs()).all(), float((sums - w).abs().max())


@pytest.mark.parametrize("dtype,power", [("float16", e) for e in (8, 20, 23, 26, 30, 33)] +
                         [("bfloat16", e) for e in (8, 20, 30, 40, 100)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [50]), ([1], [5000]), ([300, 40], [300, 700])])
@pytest.mark.parametrize("axes", [0, 1])
def test_attention_scores_of_any_size(q_lens, kv_lens, axes, dtype, power, kernel):
    """Scores up to the types' products, 2^power times 1 to 3 quarters (so exact in 32 bits): the largest
    take everything, and equal ones share it. Of either sign; with a bias, all of it."""
    P = Problem(dtype, 64, 2, 1, q_lens, kv_lens, scale=0.125, axes=axes)
    a, g = (power - 3) // 2, torch.Generator().manual_seed(power)  # 64 products of 2^(power - 3) quarters
    P.q[:] = 2.0 ** a
    P.q[:, 1] = -(2.0 ** a)  # one head has the whole in reverse
    P.k[:] = 2.0 ** (power - 3 - a) / 4 * torch.randint(1, 4, P.k.shape[:2], generator=g)[..., None]
    assert P.q.isfinite().all() and P.k.isfinite().all()
    if axes:
        P.slopes[:] = 0.5
        P.q_pos[:], P.kv_pos[:] = 2 ** 23, 0  # 2^22 off every score (in 32 bits nothing, where they are far larger)
        if power > 23:
            P.q_pos[:] = 0
    check(P)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("far", [2 ** 10, 2 ** 23, 2 ** 29, 2 ** 30 + 5, 2 ** 31 - 1])
def test_attention_distances_of_any_size(far, dtype, kernel):
    """The only keys of a document lie far from its queries, which no softmax notices."""
    P = Problem(dtype, 64, 2, 1, [1, 150], [1, 40], axes=1)
    P.q.zero_()
    P.slopes[:] = 0.75
    P.q_pos[:] = far // 2
    P.kv_pos[:] = far // 2 - far
    check(P)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("low", [12.0, 17.5, 18.5])
@pytest.mark.parametrize("q_lens,keys", [([1], 65536), ([3], 20000), ([130], 65536)])
def test_attention_many_small_weights(q_lens, keys, low, dtype, kernel):
    """One key far above very many that share a part of the sum: small as each weight is (2^-25 of the
    largest and less), together they count. Weights of 16 bits are right to u of themselves, or in fp16
    to 2^-25 where the largest is 2^15 (mma) or 2^7 (tcgen05); those of the keys here err alike. Sums are
    32-bit, off by 2^-24 of themselves for each tile of 64 keys or more and for each key of it that a
    thread has."""
    P = Problem(dtype, 64, 1, 1, q_lens, [keys], scale=0.5)
    P.q.zero_()
    P.k.zero_()
    P.q[..., 0] = 1.0
    P.k[..., 0] = -2 * low  # exact in both types
    P.k[77] = 0.0
    P.v[:] = 1.0
    P.v[77] = 0.0
    out, lse = P.run()
    o, w = P.expected()[:2]
    rest = keys * math.exp(-low)
    tol = 2 * unit(dtype) * o + 2.0 ** -19 * rest
    if dtype == "float16":
        tol += keys * 2.0 ** (-40 if kernel == "mma" else -32)
    got = out.cpu().double()
    assert ((got - o).abs() <= tol).all(), (float(got.min()), float(o.min()))
    assert ((lse.cpu().double() - w).abs() <= 2.0 ** -19 + (keys // 64 + 64) * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim,axes", [(64, 1), (64, 2), (128, 1), (128, 3)])
@pytest.mark.parametrize("span", [40, 700, 2000, 30000])
def test_attention_bias_between_neighbours(span, dim, axes, dtype, kernel):
    """Queries spread over a tile, each with a key at its place or beside it, at slopes whose products
    with the positions have no room in 32 bits: the bias is the distance's, not a difference of such
    products. Scores are zero, so a bias is off by 2^-23 of itself, and those that count are below 4."""
    n, g = 256, torch.Generator().manual_seed(span + dim)
    P = Problem(dtype, dim, 2, 2, [n], [n], axes=axes)
    P.q.zero_()
    P.slopes = 0.7 + 0.1 * torch.rand(axes, 2, generator=g)
    P.q_pos = torch.randint(0, span, (axes, n), generator=g).to(torch.int32)
    P.kv_pos = P.q_pos + torch.randint(0, 2, (axes, n), generator=g).to(torch.int32)
    out, lse = P.run()
    o, w = P.expected()[:2]
    u, big = unit(dtype), P.v.abs().max().double()
    e = 2.0 ** -20  # of a score: the bias, its sum with the others, the exponential
    assert ((lse.cpu().double() - w).abs() <= 2 * e).all(), float((lse.cpu().double() - w).abs().max())
    assert ((out.cpu().double() - o).abs() <= u * o.abs() + (u + 2 * e + n * 2.0 ** -25) * big).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim,axes", [(64, 1), (64, 2), (128, 3)])
@pytest.mark.parametrize("reach", [2 ** 24 + 1, 2 ** 27 + 3, 2 ** 30 + 7])
def test_attention_keys_far_from_queries_that_are_apart(reach, dim, axes, dtype, kernel):
    """Queries anywhere in 2^23, keys up to `reach` from there, some beside a query: distances are right to
    2^-22 of themselves, and the bias with its slope's and its own rounding to 2^-21. Scores are zero."""
    n, g = 200, torch.Generator().manual_seed(reach % 1000 + axes)
    P = Problem(dtype, dim, 2, 2, [n, 1], [n, 1], axes=axes)
    P.q.zero_()
    P.slopes = 2.0 ** 4 / reach * (0.5 + torch.rand(axes, 2, generator=g))
    P.q_pos = torch.randint(0, 2 ** 23, (axes, n + 1), generator=g).to(torch.int32)
    P.q_pos[:, :2] = torch.tensor([0, 2 ** 23 - 1])
    P.kv_pos = torch.randint(-reach, reach + 1, (axes, n + 1), generator=g).to(torch.int32)
    P.kv_pos[:, ::3] = P.q_pos[:, ::3] + 2
    P.kv_pos[:, -1] = reach
    out, lse = P.run()
    o, w = P.expected()[:2]
    u, big = unit(dtype), P.v.abs().max().double()
    e = axes * 24 * 1.5 * 2.0 ** -21 + 2.0 ** -20  # slopes times distances are below 24 times 1.5 an axis
    assert ((lse.cpu().double() - w).abs() <= 2 * e).all(), float((lse.cpu().double() - w).abs().max())
    assert ((out.cpu().double() - o).abs() <= u * o.abs() + (u + 2 * e + n * 2.0 ** -25) * big).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim,axes", [(32, 0), (64, 0), (64, 1), (128, 0), (128, 2)])
def test_attention_a_cap_far_above_the_scores_changes_nothing(dim, axes, dtype, kernel):
    """tanh x / x is 1 in 32 bits below 2^-12, so the outputs have the bits of a call without a cap."""
    more = dict(causal=True, axes=axes)
    plain, sums = Problem(dtype, dim, 4, 2, [300, 40], [300, 700], **more).run()
    out, lse = Problem(dtype, dim, 4, 2, [300, 40], [300, 700], cap=2.0 ** 20, **more).run()
    assert torch.equal(lse, sums) and torch.equal(out, plain)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cap", [2.0 ** 11, 2.0 ** 14, 2.0 ** 25, 2.0 ** 33])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [5000]), ([300, 40], [300, 700])])
def test_attention_large_scores_under_large_caps(q_lens, kv_lens, cap, dim, dtype, kernel):
    """Scores of 1 to 3 quarters of the cap: each of the three capped ones is the same number for all its keys,
    and they lie 2^8 and more apart, so that equal keys share a row as without a cap."""
    P = Problem(dtype, dim, 2, 1, q_lens, kv_lens, scale=8.0 / dim, cap=cap)
    a, g = int(math.log2(cap) - 3) // 2, torch.Generator().manual_seed(dim)
    P.q[:] = 2.0 ** a
    P.q[:, 1] = -(2.0 ** a)
    P.k[:] = cap / 8 / 2.0 ** a / 4 * torch.randint(1, 4, P.k.shape[:2], generator=g)[..., None]
    check(P)
