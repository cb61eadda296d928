"""azg_amd.policy over the whole range of its inputs (csrc/azg_policy.hip): logits and teachers' log-probabilities of
any finite size, values that are no numbers beside illegal actions, sums held to bounds that do not grow with the row."""
import math

import policy_oracle as po
import pytest
import torch
from test_gpu_policy import DT, _actions, _check_distill, _check_logprobs, _full, _logits, _mask, _policy, _teacher

pytestmark = pytest.mark.gpu

# a row by a wave, by a block, in registers (blocks of 256, 512 and 1024), in parts
FORMS = [(5, 343, "f32"), (6, 1001, "bf16"), (2100, 3001, "f16"), (130, 5003, "f32"), (130, 20011, "bf16"),
         (128, 40001, "f32"), (128, 70001, "bf16"), (3, 20011, "f32"), (2, 100003, "bf16")]


@pytest.mark.parametrize("low", ["f32", "bf16", -1e38, -1e35, -2000.0])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("n,V,dtype", FORMS)
def test_teacher_of_any_size(n, V, dtype, rest, low):
    """Entries far below the others (a mask's fill that a short list of alternatives brings along) are probability 0."""
    x = _logits(n, V, DT[dtype])
    t, ids = _teacher(x, 20, None)
    t[:, 7:] = torch.finfo(DT[low]).min if isinstance(low, str) else low
    t[0, 1:] = t[0, 7]
    _check_distill(x, None, t, ids, rest, t_dtype=torch.bfloat16 if low == "bf16" else torch.float32)


def test_teacher_of_one_size():
    """Entries that are all the lowest value are equally likely; as probabilities (rest) they are 0."""
    p = _policy()
    x = _logits(4, 343, torch.float32)
    ids = _teacher(x, 9, None)[1].cuda()
    low = torch.full((4, 9), torch.finfo(torch.float32).min, device="cuda")
    for a, b in zip(p.distill_loss_grad(x, low, ids), p.distill_loss_grad(x, low * 0, ids)):
        assert torch.equal(a, b)
    loss, d = p.distill_loss_grad(x, low, ids, rest=True, weight=1.0)
    none, dn = p.distill_loss_grad(x, torch.full_like(low, -1e4), ids, rest=True, weight=1.0)
    assert loss.isfinite() and torch.equal(loss, none) and torch.equal(d, dn)
