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
