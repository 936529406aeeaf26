"""Reports of waits that gave up: attention calls and forwards have their own. The waits here are met by
nobody and end after 20 ms by themselves."""
import numpy as np
import pytest

from s2s_testlib import pkg
from test_gpu_token_ops import Problem, binding, kernel  # noqa: F401

pytestmark = pytest.mark.gpu

try:
    import torch
except ImportError:  # collected without torch: the GPU run has it
    torch = None


@pytest.fixture
def forward():
    """A synchronous forward of a small image."""
    H = binding().Handle(pkg().weights.Weights.seeded("lightweight_sr", 0, True))
    x = np.random.default_rng(0).random((1, 3, 16, 16), np.float32)
    yield lambda: np.asarray(H.forward_batch(x)[0])
    H.close()


def timeout(call):
    C = binding()
    with pytest.raises(C.S2SError) as e:
        call()
    assert e.value.code == C.S2S_ERR_TIMEOUT


def test_a_forward_does_not_report_an_attention_call(forward):
    C = binding()
    want = forward()
    C.debug_wait_gives_up()
    assert np.array_equal(forward(), want)
    timeout(C.device_status)  # once, by whom it is for
    C.device_status()
    assert np.array_equal(forward(), want)


def test_a_look_at_the_device_leaves_a_forward_its_report(forward):
    C = binding()
    want = forward()
    C.debug_wait_gives_up(attention=False)
    timeout(C.device_status)
    timeout(forward)
    C.device_status()
    assert np.array_equal(forward(), want)


@pytest.mark.parametrize("attention", [False, True])
def test_attention_is_right_whatever_gave_up_before(attention, kernel, forward):
    """Enough work that some of its waits are not met at once."""
    C = binding()
    P = Problem("bfloat16", 64, 8, 8, [2000, 500], [2000, 500], causal=True)
    want, sums = P.run()
    C.debug_wait_gives_up(attention=attention)
    out, lse = P.run()
    assert torch.equal(out, want) and torch.equal(lse, sums)
    timeout(C.device_status)
    if not attention:
        timeout(forward)
    C.device_status()


def test_a_captured_call_after_a_report(kernel):
    C = binding()
    P = Problem("float16", 64, 4, 2, [300], [900], axes=1)
    want, _ = P.run()
    s = torch.cuda.Stream()
    out, _ = P.run(stream=s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        P.call(s.cuda_stream)
    C.debug_wait_gives_up()
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    timeout(C.device_status)
    C.device_status()
