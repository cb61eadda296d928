"""azg_amd.policy without a GPU: its refusals, how leading dimensions fold into rows, and the C entries' checks."""
import ctypes
import math
import struct

import pytest
import torch

import azg_amd  # noqa: F401
from azg_amd import _lib, policy


def test_cpu_tensors_are_refused():
    x = torch.zeros((3, 5))
    with pytest.raises(_lib.AzgError, match="no CPU fallback"):
        policy.action_logprobs(x)
    with pytest.raises(_lib.AzgError):
        policy.distill_loss(x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64))
    with pytest.raises(_lib.AzgError):
        policy.distill_loss_grad(x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64))
    for bad in (x.double(), x.long(), [1.0]):
        with pytest.raises(ValueError):
            policy.action_logprobs(bad)


def test_argument_checks():
    x = torch.zeros((3, 5))
    with pytest.raises(ValueError, match="broadcast"):
        policy._check_mask("f", x, torch.ones((3, 4), dtype=torch.bool))
    with pytest.raises(ValueError, match="bool or uint8"):
        policy._check_mask("f", x, torch.ones((3, 5)))
    assert policy._check_mask("f", x, torch.ones(5, dtype=torch.bool)).stride() == (0, 1)
    with pytest.raises(ValueError, match="int64 or int32"):
        policy._check_ints("f", "actions", torch.zeros(3), (3,), x.device)
    with pytest.raises(ValueError, match="expected"):
        policy._check_ints("f", "actions", torch.zeros(4, dtype=torch.int64), (3,), x.device)
    t, i = torch.zeros((3, 2)), torch.zeros((3, 2), dtype=torch.int64)
    policy._check_teacher("f", x, t, i)
    for bt, bi in ((t[:2], i[:2]), (t, i[:, :1]), (t.double(), i), (t, i.float()), (t[:, :0], i[:, :0]),
                   (t.repeat(1, 65), i.repeat(1, 65)), (t.clone().requires_grad_(True), i)):
        with pytest.raises(ValueError):
            policy._check_teacher("f", x, bt, bi)


@pytest.mark.parametrize("make", [
    lambda: torch.zeros(6, 5), lambda: torch.zeros(5), lambda: torch.zeros(2, 3, 5), lambda: torch.zeros(1, 1, 1, 5),
    lambda: torch.zeros(6, 9)[:, 2:7], lambda: torch.zeros(2, 4, 5)[:, :-1], lambda: torch.zeros(2, 3, 4, 5)[:, :, 1:],
    lambda: torch.zeros(1, 5).expand(6, 5), lambda: torch.zeros(3, 1, 5).expand(3, 4, 5),
    lambda: torch.zeros(4, 3, 5).transpose(0, 1), lambda: torch.zeros(3, 4, 2, 5)[:, 1:3, :1],
    lambda: torch.zeros(4, 3, 2, 5).permute(2, 1, 0, 3), lambda: torch.zeros(5, 6).t(), lambda: torch.zeros(0, 5)])
@pytest.mark.parametrize("masked", [0, 1, 2])
def test_rows_reach_every_element(make, masked):
    """Each row's offset by the folded strides is the tensor's own."""
    x = make()
    store = torch.arange(max(1, x.untyped_storage().nbytes() // 4), dtype=torch.float32)
    x = store.as_strided(x.shape, x.stride(), x.storage_offset())
    mask = None
    if masked == 1:
        mask = torch.ones(5, dtype=torch.uint8).expand(x.shape)
    elif masked == 2:
        mask = (torch.rand(x.shape) < 0.5).to(torch.uint8)
    y, m, n, L = policy._rows(x, mask, 1.0)
    _, _, rows, inner, so, si, mo, mi, vocab, dtype, temp = struct.unpack("PPqqqqqqqif", L)
    assert len(L) == 80 and vocab == 5 and rows == n and n * 5 == x.numel() and torch.equal(y, x)
    assert (dtype, temp) == (0, 1.0)
    for t, so, si, size in ((y, so, si, 4), (m, mo, mi, 1)):
        if t is None:
            continue
        base = t.data_ptr()
        for r, row in enumerate(t.reshape(-1, 5) if t.numel() else []):
            off = (r // inner) * so + (r % inner) * si
            got = (ctypes.c_float if size == 4 else ctypes.c_uint8).from_address(base + off * size).value
            assert got == float(row[0])


def test_c_entries_refuse():
    L = _lib.lib()
    x = torch.zeros((2, 5))
    f = torch.zeros(64)

    def logits(**kw):
        d = dict(x=x.data_ptr(), mask=0, rows=2, inner=2, stride_outer=0, stride_inner=5, mask_outer=0, mask_inner=0,
                 vocab=5, dtype=0, temperature=1.0)
        d.update(kw)
        return policy._LOGITS(*d.values())

    p = f.data_ptr()
    bad = [dict(x=0), dict(rows=0), dict(rows=2 ** 40), dict(inner=0), dict(vocab=0), dict(vocab=2 ** 31),
           dict(dtype=3), dict(dtype=-1), dict(temperature=0.0), dict(temperature=math.nan), dict(temperature=math.inf),
           dict(temperature=-1.0), dict(stride_inner=-5), dict(stride_outer=-1), dict(mask_inner=-1),
           dict(rows=2 ** 34, vocab=2 ** 28)]
    t = policy._TEACHER(p, p, 0, 1, 3, 0)
    for kw in bad:
        g = logits(**kw)
        assert L.azg_logprobs_fwd(g, None, 0, 0, None, None, p, p, None, None, None, 0, None) == -1, kw
        assert b"azg_logprobs_fwd" in L.azg_last_error()
        assert L.azg_logprobs_bwd(g, None, 0, p, None, 0, p, 0, None, 0, p, None) == -1
        assert L.azg_distill_fwd(g, t, p, p, None, 0, 1.0, None, p, None, 0, None) == -1
        assert L.azg_distill_bwd(g, t, p, None, 0, 1.0, p, None) == -1
        assert L.azg_logprobs_work(g, 8) == -1 and L.azg_distill_work(g, 1) == -1
    g = logits()
    assert L.azg_logprobs_fwd(None, None, 0, 0, None, None, p, p, None, None, None, 0, None) == -1
    for a in ((None, 0, 0, None, p, p, p, None, None), (p, 0, 0, None, None, p, p, None, None),
              (None, 0, -1, None, None, p, p, p, p), (None, 0, 129, None, None, p, p, p, p),
              (None, 0, 3, None, None, p, p, None, p), (None, 0, 3, None, None, p, p, p, None),
              (None, 0, 0, None, None, None, p, None, None), (None, 0, 0, None, None, p, None, None, None)):
        assert L.azg_logprobs_fwd(g, *a, None, 0, None) == -1, a
    assert L.azg_logprobs_bwd(g, None, 0, p, p, 0, None, 0, None, 0, p, None) == -1  # g_logp without actions
    assert L.azg_logprobs_bwd(g, None, 0, None, None, 0, p, 0, None, 0, p, None) == -1
    for k in (dict(logp=0), dict(ids=0), dict(dtype=3), dict(k=0), dict(k=129)):
        d = dict(logp=p, ids=p, dtype=0, ids64=1, k=3, rest=0)
        d.update(k)
        u = policy._TEACHER(*d.values())
        assert L.azg_distill_fwd(g, u, p, p, None, 0, 1.0, None, p, None, 0, None) == -1
        assert L.azg_distill_bwd(g, u, p, None, 0, 1.0, p, None) == -1
    # rows in parts need their scratch memory
    g = logits(vocab=2 ** 20)
    assert L.azg_logprobs_work(g, 8) > 0 and L.azg_distill_work(g, 1) > 0
    assert L.azg_logprobs_fwd(g, None, 0, 0, None, None, p, p, None, None, None, 0, None) == -1
    assert L.azg_distill_fwd(g, t, p, p, None, 0, 1.0, None, p, p, 16, None) == -1
    assert b"work" in L.azg_last_error()
    # statistics and scratch memory at 16 bytes
    g = logits()
    assert L.azg_logprobs_fwd(g, None, 0, 0, p + 4, None, p, p, None, None, None, 0, None) == -1
    assert L.azg_logprobs_bwd(g, None, 0, p + 8, None, 0, p, 0, None, 0, p, None) == -1
    assert L.azg_distill_fwd(g, t, p + 4, p, None, 0, 1.0, None, p, None, 0, None) == -1
    assert L.azg_distill_fwd(g, t, p, p, None, 0, 1.0, None, p, p + 4, 2 ** 20, None) == -1
    assert L.azg_distill_bwd(g, t, p + 4, None, 0, 1.0, p, None) == -1
