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
