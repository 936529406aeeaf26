"""The token operators at the largest sizes that they take."""
import math

import pytest

from test_gpu_token_ops import binding, heads

pytestmark = pytest.mark.gpu

try:
    import torch
except ImportError:  # collected without torch: the GPU run has it
    torch = None


def needs(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes * 1e9:
        pytest.skip("needs %d GB of device memory" % gigabytes)


def test_attention_over_the_most_keys():
    """A document of 2^31 - 256 keys whose last one has a fifth of the weight: zero scores but for its own of
    20, one value of 5 in a row of zeros. The sums count whole numbers below 2^24 a lane, so the weights'
    rounding (2^-11), the output's and the score's and sums' 2^-20 (1 + 20) remain."""
    needs(40)
    C, n = binding(), 2 ** 31 - 256
    rows = torch.zeros(n, 1, 8, device="cuda", dtype=torch.float16)  # keys and values
    rows[n - 1, 0, 0] = 5.0
    q = torch.zeros(1, 1, 8, device="cuda", dtype=torch.float16)
    q[..., 0] = 4.0
    out, lse = torch.full_like(q, 7.0), torch.zeros(1, 1, device="cuda")
    C.attention("float16", 8, 1.0, heads(q), heads(rows), heads(rows), heads(out), 1, n, d_lse=lse.data_ptr(),
                stream=torch.cuda.current_stream().cuda_stream)
    total = n - 1 + math.exp(20)
    want = 5 * math.exp(20) / total
    got = out.cpu().double().flatten()
    assert abs(got[0] - want) <= want * (2 * 2.0 ** -11 + 21 * 2.0 ** -20) and (got[1:] == 0).all()
    assert abs(lse.item() - math.log(total)) <= 21 * 2.0 ** -20
    C.device_status(0)


@pytest.mark.parametrize("tokens", [2 ** 31 - 16, 2 ** 31 - 15, 2 ** 31 - 1])
def test_rotary_of_the_most_tokens(tokens):
    """One pair (1, 1) a token, in place: half a turn for all but the last, which turns by pi / 4. Values
    are 2^0.5 at most, so they are off by u 2^0.5 for the output's rounding and 2^-20 for the angle's and
    the products'."""
    needs(30)
    C = binding()
    x = torch.ones(tokens, 1, 2, device="cuda", dtype=torch.float16)
    pos = torch.zeros(tokens, device="cuda", dtype=torch.int32)
    pos[:] = 4
    pos[-1] = 1
    plan = C.rotary_plan([1])
    plan.frequency[0] = math.pi / 4
    C.rotary(plan, "float16", 2, tokens, pos.data_ptr(), tokens, [(heads(x), heads(x))],
             stream=torch.cuda.current_stream().cuda_stream)
    tol = 2.0 ** -11 * math.sqrt(2) + 2.0 ** -20
    last = x[-1, 0].cpu().double()
    assert abs(last[0]) <= tol and abs(last[1] - math.sqrt(2)) <= tol
    x[-1] = -1.0
    for first in range(0, tokens, 2 ** 28):
        part = x[first:first + 2 ** 28]
        assert (part + 1).abs().max().item() <= tol
