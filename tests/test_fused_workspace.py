"""Workspaces of log probabilities that a call could not use, in Python on the CPU."""
import pytest

import hybrid_attention as ha
from test_fused_refusals import Weight, ends_at_the_handle, no_torch  # noqa: F401 (a fixture)
from test_kv_refusals import Fake


def test_tensors_with_bytes_of_their_own(no_torch):  # noqa: F811
    """A tensor is checked whether or not its bytes are said: more than it has would be written behind it."""
    w, a = Weight(100, 64), Fake(3 * 64)

    def call(n, said=None, **kind):
        ws = Fake(n, **kind)
        ws.element_size = lambda: 2
        w.logprobs(3, a, ha.LogProbs(lse=Fake(3, "float32")), ws, said)
    for good in ((1000, None), (1000, 2000), (1000, 16)):
        ends_at_the_handle(lambda: call(*good))
    for n, said, kind in ((1000, 2001, {}), (0, 16, {}), (1000, 16, dict(gpu=1)), (1000, 16, dict(cuda=False)), (1000, 16, dict(contiguous=False))):
        with pytest.raises(TypeError):
            call(n, said, **kind)
    ends_at_the_handle(lambda: w.logprobs(3, a, ha.LogProbs(lse=4096), 8192, 1 << 40))  # (an address is the caller's word)
