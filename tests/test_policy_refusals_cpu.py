"""azg_amd.policy without a GPU: what it refuses by the state of its arguments."""
import pytest
import torch

import azg_amd  # noqa: F401
from azg_amd import policy


def test_tangents_are_refused():
    from torch.autograd import forward_ad as fwd
    x = torch.zeros((3, 5))
    policy._check_tangents("f", x, None, 1.0)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="f has no forward-mode derivative"):
            policy._check_tangents("f", x, d)
        with torch.no_grad(), pytest.raises(RuntimeError):
            policy._check_tangents("f", d)
        with pytest.raises(RuntimeError):
            policy._check_teacher("f", x, d[:, :2], torch.zeros((3, 2), dtype=torch.int64))
        policy._check_tangents("f", x, d.detach(), torch.zeros(3, dtype=torch.int64), None)
    policy._check_tangents("f", x)


def test_too_many_rows_are_refused():
    """As an expanded tensor can have them: refused by what the library says of them, each time."""
    for n, V in ((2 ** 36, 5), (2 ** 35, 2 ** 28)):
        for _ in range(2):
            with pytest.raises(ValueError, match="2\\^35 rows"):
                policy._work(policy._logprobs_work(n, V, 0, 0), torch.device("cpu"))
            with pytest.raises(ValueError, match="2\\^35 rows"):
                policy._work(policy._distill_work(n, V, 0, True), torch.device("cpu"))
    assert policy._work(policy._logprobs_work(4, 65, 0, 5), torch.device("cpu")) is None
