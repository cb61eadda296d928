"""azg_amd.policy on the GPU (csrc/azg_policy.hip) against the definitions in 64 bits (policy_oracle.py):
types, row lengths from one action to a quarter of a million, odd sizes and strides, ties, masks that leave a
row empty, values that are no numbers in masked places, gradients, captured graphs, streams, refusals."""
import math

import policy_oracle as po
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _policy():
    from azg_amd import policy
    return policy


def _logits(n, V, dtype, layout="packed", values="normal", seed=0):
    g = torch.Generator().manual_seed(1000 * seed + 7 * n + V)
    x = torch.randn((n, V), generator=g) * 2.5
    if values == "ties":
        x = torch.round(x)
    elif values == "constant":
        x = torch.full((n, V), 0.75)
    elif values == "rising":
        x = torch.arange(V).float().mul_(20.0 / V).expand(n, V).clone()
    elif values == "falling":
        x = -torch.arange(V).float().mul_(20.0 / V).expand(n, V).clone()
    elif values == "cluster":  # the largest next to each other
        x[:, V // 3:V // 3 + 300] += 30.0
    elif values == "stripes":  # the largest all at one distance
        x[:, 5 % V::256] += 30.0
    elif values == "wide":
        x = x * 40.0
    elif values == "lowest":
        x = torch.where(torch.rand((n, V), generator=g) < 0.5, torch.finfo(dtype).min, x)
        x[0] = torch.finfo(dtype).min
    elif values == "minf":
        x = torch.where(torch.rand((n, V), generator=g) < 0.5, -math.inf, x)
        x[0] = -math.inf
        x[-1, :] = -math.inf
        x[-1, V // 2] = 1.0
    x = x.to(dtype)
    if layout == "packed":
        return x.cuda()
    if layout == "padded":
        buf = torch.full((n, V + 13), math.nan, dtype=dtype, device="cuda")
        buf[:, 3:V + 3] = x.cuda()
        return buf[:, 3:V + 3]
    if layout == "shifted":
        assert n % 2 == 0
        buf = torch.full((2, n // 2 + 1, V), math.nan, dtype=dtype, device="cuda")
        buf[:, :-1] = x.cuda().view(2, n // 2, V)
        return buf[:, :-1]
    if layout == "transposed":
        return x.t().contiguous().cuda().t()
    if layout == "expanded":
        return x[:1].cuda().expand(n, V)
    raise AssertionError(layout)


def _mask(kind, n, V, seed=0):
    if kind == "none":
        return None
    g = torch.Generator().manual_seed(seed + V)
    if kind == "shared":
        m = torch.rand((V,), generator=g) < 0.3
        m[V // 2] = True
        return m.cuda()
    m = torch.rand((n, V), generator=g) < 0.3
    if kind == "empty":  # a row that leaves nothing, a row that leaves one
        m[0] = False
        m[-1] = False
        m[-1, V - 1] = n > 1
    elif kind == "u8":
        return (m.to(torch.uint8) * 3).cuda()
    return m.cuda()


def _actions(n, V, seed=0):
    a = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed + V))
    if n > 2:
        a[1] = -1
        a[2] = V
    return a


def _full(mask, n, V):
    return None if mask is None else mask.expand(n, V) if mask.dim() == 1 else mask


def _check_logprobs(x, mask, actions, top, T=1.0, grads=True, seed=0):
    p = _policy()
    V = x.shape[-1]
    n = x.numel() // V
    lead = x.shape[:-1]
    xm = mask if mask is None or mask.dim() == 1 else mask.view(x.shape)
    act = actions.cuda().view(lead)
    flat = x.reshape(n, V)
    m2 = _full(mask, n, V)
    r = p.action_logprobs(x, act, top=top, temperature=T, mask=xm)
    want = po.logprobs(flat, actions, m2, T, top)
    for k in ("lse", "entropy", "logp"):
        po.check(getattr(r, k), want[k][0], want[k][1], k)
    if top:
        assert torch.equal(r.top_ids.cpu().view(n, top), want["top_ids"].cpu())
        po.check(r.top_logp, *want["top_logp"], "top_logp")
    else:
        assert r.top_ids is None and r.top_logp is None
    if not grads:
        return
    g = torch.Generator().manual_seed(seed + 5)
    g1, g2, g3 = (torch.randn((n,), generator=g) for _ in range(3))
    leaf = x.detach().requires_grad_(True)
    q = p.action_logprobs(leaf, act, top=top, temperature=T, mask=xm)
    d, = torch.autograd.grad((q.logp, q.entropy, q.lse), leaf, [t.cuda().view(lead) for t in (g1, g2, g3)])
    assert d.shape == x.shape and d.dtype == x.dtype
    dw, tol = po.logprobs_grad(flat, actions, m2, T, g1, g2, g3)
    po.check(d, dw, tol, "gradient")


SIZES = [1, 2, 3, 7, 8, 9, 63, 64, 65, 127, 129, 343, 511, 1000, 1025, 2049, 4097, 16391, 65543, 131072, 262147]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", SIZES)
def test_logprobs_sizes(V, dtype):
    n = 5 if V < 20000 else 3
    for top in sorted({0, 1, min(V, 5), min(V, 64), min(V, 128)}):
        _check_logprobs(_logits(n, V, DT[dtype]), None, _actions(n, V), top, grads=top in (0, 5))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind", ["random", "empty", "shared", "u8"])
@pytest.mark.parametrize("V", [1, 65, 343, 3001, 40001])
def test_logprobs_masks(V, kind, dtype):
    for layout in ("packed", "padded"):
        x = _logits(4, V, DT[dtype], layout)
        m = _mask(kind, 4, V)
        x[_full(m, 4, V) == 0] = math.nan  # no number at an illegal action
        _check_logprobs(x, m, _actions(4, V), min(V, 20))
        x[_full(m, 4, V) == 0] = math.inf
        _check_logprobs(x, m, _actions(4, V), min(V, 70), T=0.5)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("values", ["ties", "constant", "rising", "falling", "cluster", "stripes", "wide", "lowest",
                                    "minf"])
@pytest.mark.parametrize("V", [65, 343, 5003, 70001])
def test_logprobs_values(V, values, dtype):
    x = _logits(3, V, DT[dtype], values=values)
    for top in (1, 20, min(V, 128)):
        _check_logprobs(x, None, _actions(3, V), min(V, top), T=1.0 if top > 1 else 3.0, grads=top == 20)


@pytest.mark.parametrize("layout", ["padded", "shifted", "transposed", "expanded"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,V", [(6, 343), (6, 9001), (70, 343), (300, 129)])
def test_logprobs_layouts(n, V, dtype, layout):
    _check_logprobs(_logits(n, V, DT[dtype], layout), _mask("random", n, V), _actions(n, V), 9)


@pytest.mark.parametrize("n", [1, 2, 63, 257, 1025, 5000])
def test_logprobs_rows(n):
    _check_logprobs(_logits(n, 129, torch.float32), _mask("random", n, 129), _actions(n, 129), 3)
    _check_logprobs(_logits(n, 1500, torch.bfloat16), None, _actions(n, 1500), 17, grads=n < 1000)


def test_logprobs_not_a_number():
    """A legal NaN or +inf makes the row's numbers NaN; the order of the alternatives is NaN, +inf, then the rest."""
    p = _policy()
    for V in (64, 343, 20001):
        x = _logits(3, V, torch.float32)
        x[0, V // 2] = math.nan
        x[0, 3] = math.inf
        x[1, 7] = math.inf
        r = p.action_logprobs(x, torch.zeros(3, dtype=torch.int32, device="cuda"), top=3)
        assert r.logp[:2].isnan().all() and r.entropy[:2].isnan().all() and r.lse[:2].isnan().all()
        assert r.top_logp[:2].isnan().all() and r.logp[2].isfinite()
        ids = r.top_ids.cpu()
        assert ids[0, 0] == V // 2 and ids[0, 1] == 3 and ids[1, 0] == 7
        rest = torch.sort(x.cpu()[1], descending=True, stable=True).indices[1:3]
        assert torch.equal(ids[1, 1:], rest)
        leaf = x.clone().requires_grad_(True)
        p.action_logprobs(leaf).entropy.sum().backward()
        assert leaf.grad[:2].isnan().all() and leaf.grad[2].isfinite().all()


def _teacher(x, k, mask, seed=0, noise=0.5):
    """(log-probabilities, ids) of a teacher near the student, with missing, doubled and low entries"""
    n, V = x.shape
    g = torch.Generator().manual_seed(seed + 11 * V + k)
    t = x.detach().float().clamp(-60, 60) + noise * torch.randn((n, V), generator=g).cuda()
    if mask is not None:
        t = t.masked_fill(~mask.cuda().bool(), -math.inf)
    v, i = torch.topk(t, min(k, V), dim=1)
    lse = torch.logsumexp(t, 1, keepdim=True)
    v = torch.where(v == -math.inf, v, v - lse)
    i = torch.where(v == -math.inf, -1, i)
    return v.cpu(), i.cpu()


def _check_distill(x, mask, t, ids, rest, T=1.0, seed=0, t_dtype=torch.float32, i_dtype=torch.int64):
    p = _policy()
    V = x.shape[-1]
    n = x.numel() // V
    lead = x.shape[:-1]
    k = ids.shape[-1]
    flat = x.reshape(n, V)
    m2 = _full(mask, n, V)
    xm = mask if mask is None or mask.dim() == 1 else mask.view(x.shape)
    t = t.to(t_dtype)
    args = (t.cuda().view(*lead, k), ids.to(i_dtype).cuda().view(*lead, k))
    kw = dict(temperature=T, mask=xm, rest=rest)
    loss, tol, d, dd = po.distill(flat, t.float(), ids, m2, T, rest)
    rows = p.distill_loss(x, *args, reduction="none", **kw)
    assert rows.shape == lead and rows.dtype == torch.float32
    po.check(rows, loss, tol, "row loss")
    g = torch.Generator().manual_seed(seed + 3)
    w = torch.randn((n,), generator=g).cuda()
    # the whole and its gradient in one call, weighted by row
    total, dx = p.distill_loss_grad(x, *args, weight=w.view(lead), **kw)
    w64 = w.double()
    if loss.isfinite().all():
        po.check(total, (loss * w64).sum(), (tol * w64.abs()).sum() + po.H * (loss * w64).sum().abs() + 1e-30, "total")
    assert dx.shape == x.shape and dx.dtype == x.dtype
    po.check(dx, d * w64[:, None], po.grad_tol(d, dd, w64[:, None], x.dtype), "gradient")
    # through autograd: rows weighted from outside, and the mean
    leaf = x.detach().requires_grad_(True)
    d1, = torch.autograd.grad(p.distill_loss(leaf, *args, reduction="none", **kw), leaf, w.view(lead))
    po.check(d1, d * w64[:, None], po.grad_tol(d, dd, w64[:, None], x.dtype), "autograd rows")
    mean = p.distill_loss(leaf, *args, **kw)
    d2, = torch.autograd.grad(mean * 3.0, leaf)
    w3 = torch.full((1, 1), 3.0 / n, dtype=torch.float64, device=x.device)
    if loss.isfinite().all():
        po.check(mean, loss.mean(), tol.mean() + po.H * 2 * loss.mean().abs(), "mean")
    po.check(d2, d * w3, po.grad_tol(d, dd, w3, x.dtype), "autograd mean")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", SIZES)
def test_distill_sizes(V, dtype):
    n = 5 if V < 20000 else 3
    x = _logits(n, V, DT[dtype])
    for k in sorted({1, min(V, 5), min(V, 64), min(V, 128)}):
        t, ids = _teacher(x, k, None)
        for rest in (False, True):
            _check_distill(x, None, t, ids, rest)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("kind", ["random", "empty", "shared", "u8"])
@pytest.mark.parametrize("V", [1, 65, 343, 3001, 40001])
def test_distill_masks(V, kind, dtype):
    for layout in ("packed", "padded"):
        x = _logits(4, V, DT[dtype], layout)
        m = _mask(kind, 4, V)
        x[_full(m, 4, V) == 0] = 0.0
        t, ids = _teacher(x, min(V, 25), _full(m, 4, V))
        x[_full(m, 4, V) == 0] = math.nan
        for rest in (False, True):
            _check_distill(x, m, t, ids, rest, T=2.0)


@pytest.mark.parametrize("layout", ["padded", "shifted", "transposed", "expanded"])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,V", [(6, 343), (6, 9001), (70, 343), (300, 129)])
def test_distill_layouts(n, V, dtype, layout):
    x = _logits(n, V, DT[dtype], layout)
    m = _mask("random", n, V)
    t, ids = _teacher(x.reshape(n, V), 9, m)
    _check_distill(x, m, t, ids, True)


@pytest.mark.parametrize("V", [130, 343, 9001])
@pytest.mark.parametrize("rest", [False, True])
def test_distill_entries(V, rest):
    """The same action twice, missing entries in between, rows without any, ids outside the actions, low
    probabilities, entries at illegal actions, 16-bit log-probabilities, 32-bit ids."""
    x = _logits(6, V, torch.float32)
    t, ids = _teacher(x, 40, None)
    ids[0, 5] = ids[0, 2]
    ids[0, 39] = ids[0, 2]
    ids[1, 3:7] = -1
    t[1, 20] = -math.inf
    ids[2] = -1
    ids[3, 0] = V
    ids[3, 1] = 2 ** 31 - 1
    ids[3, 2] = -(2 ** 31)
    t[4, 10:] -= 200.0
    t[5, 0] -= 1e30
    _check_distill(x, None, t, ids, rest)
    _check_distill(x, None, t.clamp_min(-3e4), ids, rest, t_dtype=torch.float16, i_dtype=torch.int32)
    _check_distill(x, None, t, ids, rest, t_dtype=torch.bfloat16)
    # raw logits instead of log-probabilities: any constant per row
    if not rest:
        _check_distill(x, None, t + 17.0, ids, rest)
    m = torch.ones((6, V), dtype=torch.bool)
    m[4, ids[4, 1]] = False
    m[5] = False
    _check_distill(x, m.cuda(), t, ids, rest)
    x[0, ids[0, 4]] = -math.inf
    _check_distill(x, None, t, ids, rest)


@pytest.mark.parametrize("V", [3, 60, 128])
def test_distill_all_actions_given(V):
    """rest with nothing outside the entries: the whole distribution is given."""
    x = _logits(4, V, torch.float32)
    t, ids = _teacher(x, V, None)
    _check_distill(x, None, t, ids, True)
    _check_distill(x, None, t, ids, False)


@pytest.mark.parametrize("V", [343, 9001])
def test_distill_peaked(V):
    """A teacher and a student that are nearly sure: the student's mass outside the entries far below its largest
    probability, and still its own maximum and sum."""
    x = _logits(3, V, torch.float32)
    x[:, 4] += 90.0
    x[1, 4] += 400.0
    t, ids = _teacher(x, 8, None)
    t[:, 1:] = torch.linspace(-3, -9, 7)
    t[:, 0] = math.log(0.9)
    _check_distill(x, None, t, ids, True)


@pytest.mark.parametrize("values", ["wide", "lowest", "minf", "constant"])
@pytest.mark.parametrize("dtype", list(DT))
def test_distill_values(values, dtype):
    for V in (343, 20011):
        x = _logits(4, V, DT[dtype], values=values)
        ok = x.float() > torch.finfo(DT[dtype]).min
        t, ids = _teacher(_logits(4, V, torch.float32, seed=3), 20, ok)
        for rest in (False, True):
            _check_distill(x, None, t, ids, rest)


# enough rows that none is split over blocks: a wave, a block of each size and the rows in registers
MANY = [(2100, 3001, "f32"), (2100, 4096, "f32"), (2100, 8190, "bf16"), (2100, 1500, "f16"), (130, 2050, "f32"),
        (130, 8193, "f32"), (130, 9001, "f16"), (130, 16384, "f32"), (130, 20011, "bf16"), (130, 32768, "f16"),
        (130, 33001, "f32"), (130, 65536, "f32"), (130, 65537, "f32"), (129, 65543, "bf16"), (128, 131072, "f16"),
        (128, 131073, "bf16")]


@pytest.mark.parametrize("n,V,dtype", MANY)
def test_logprobs_many_rows(n, V, dtype):
    for kind, top in (("none", 9), ("empty", 40), ("random", 128), ("shared", 0)):
        if n > 2000 and kind in ("random", "shared"):
            continue
        _check_logprobs(_logits(n, V, DT[dtype]), _mask(kind, n, V), _actions(n, V), top, grads=kind in ("none", "empty"))


@pytest.mark.parametrize("values", ["ties", "constant", "falling", "rising", "cluster", "stripes", "lowest", "minf"])
@pytest.mark.parametrize("n,V,dtype", [(130, 3001, "f32"), (130, 20011, "bf16"), (130, 20011, "f32")])
def test_logprobs_many_rows_values(n, V, dtype, values):
    x = _logits(n, V, DT[dtype], values=values)
    for top in (20, 100):
        _check_logprobs(x, None, _actions(n, V), top, grads=top == 20)


@pytest.mark.parametrize("n,V,dtype", MANY)
def test_distill_many_rows(n, V, dtype):
    for kind, k, rest in (("none", 33, True), ("empty", 100, True), ("shared", 7, False)):
        if n > 2000 and kind == "shared":
            continue
        x = _logits(n, V, DT[dtype])
        m = _mask(kind, n, V)
        t, ids = _teacher(x, k, _full(m, n, V))
        ids[3, k - 1] = ids[3, 0]
        if m is not None:
            x[_full(m, n, V) == 0] = math.nan
        _check_distill(x, m, t, ids, rest)


@pytest.mark.parametrize("values", ["wide", "lowest", "minf", "constant"])
@pytest.mark.parametrize("n,V,dtype", [(130, 700, "f32"), (130, 12001, "f32"), (130, 20011, "bf16"), (130, 70001, "f16")])
def test_distill_many_rows_values(n, V, dtype, values):
    x = _logits(n, V, DT[dtype], values=values)
    t, ids = _teacher(_logits(n, V, torch.float32, seed=3), 20, x.float() > torch.finfo(DT[dtype]).min)
    for rest in (False, True):
        _check_distill(x, None, t, ids, rest)


def test_more_rows_than_one_grid_dimension():
    """2^22 rows of a wave, 2^20 of a block, and a few more."""
    p = _policy()
    n = 2 ** 22 + 5
    x = torch.randn((n, 3), generator=torch.Generator().manual_seed(0)).cuda().requires_grad_(True)
    a = (torch.arange(n) % 3).cuda()
    r = p.action_logprobs(x, a, top=1)
    d, = torch.autograd.grad(r.logp, x, torch.ones(n, device="cuda"))
    loss, e = p.distill_loss_grad(x, torch.zeros((n, 1), device="cuda"), a[:, None], weight=1.0)
    for s in (slice(0, 50), slice(2 ** 22 - 25, n)):
        want = po.logprobs(x[s], a[s], None, 1.0, 1)
        po.check(r.logp[s], *want["logp"], "logp")
        assert torch.equal(r.top_ids[s].cpu(), want["top_ids"].cpu())
        g = torch.ones(x[s].shape[0])
        po.check(d[s], *po.logprobs_grad(x[s], a[s], None, 1.0, g, None, None), "gradient")
        po.check(-e[s], *po.logprobs_grad(x[s], a[s], None, 1.0, g, None, None), "distillation of one action")
    n, V = 2 ** 20 + 3, 8200
    row = _logits(1, V, torch.bfloat16)
    r = p.action_logprobs(row.expand(n, V), torch.full((n,), 7, device="cuda"))
    want = po.logprobs(row, torch.tensor([7]), None, 1.0, 0)
    po.check(r.logp, want["logp"][0].expand(n), want["logp"][1].expand(n), "logp")


def test_masks_that_broadcast():
    p = _policy()
    B, Q, V = 3, 4, 343
    x = _logits(B * Q, V, torch.float32).view(B, Q, V)
    a = _actions(B * Q, V).view(B, Q)
    g = torch.Generator().manual_seed(4)
    for shape in ((V,), (1, V), (Q, V), (B, 1, V), (1, 1, V), (B, Q, V), (B, Q, 1)):
        m = (torch.rand(shape, generator=g) < 0.5).cuda()
        m[..., 0] = True
        full = m.expand(B, Q, V).reshape(B * Q, V)
        r = p.action_logprobs(x, a.cuda(), top=5, mask=m)
        want = po.logprobs(x.view(-1, V), a, full, 1.0, 5)
        po.check(r.entropy, *want["entropy"], "entropy")
        assert torch.equal(r.top_ids.cpu().view(-1, 5), want["top_ids"].cpu())
        t, ids = _teacher(x.view(-1, V), 6, full)
        loss, tol, _, _ = po.distill(x.view(-1, V), t, ids, full, 1.0, True)
        got = p.distill_loss(x, t.view(B, Q, 6).cuda(), ids.view(B, Q, 6).cuda(), mask=m, rest=True, reduction="none")
        po.check(got, loss, tol, "loss")
    y = _logits(2 * 3 * 4, 65, torch.bfloat16).view(2, 3, 4, 65)
    z = y.transpose(0, 2)  # strides of three levels: copied
    r = p.action_logprobs(z, top=3)
    want = po.logprobs(z.reshape(-1, 65), None, None, 1.0, 3)
    assert r.logp is None and r.entropy.shape == (4, 3, 2)
    po.check(r.entropy, *want["entropy"], "entropy")
    assert torch.equal(r.top_ids.cpu().view(-1, 3), want["top_ids"].cpu())


@pytest.mark.parametrize("T", [1e-6, 1e-3, 0.1, 7.0, 1e3, 1e6])
@pytest.mark.parametrize("dtype", list(DT))
def test_temperatures(T, dtype):
    for n, V in ((5, 343), (3, 20011)):
        x = _logits(n, V, DT[dtype])
        _check_logprobs(x, _mask("random", n, V), _actions(n, V), 11, T=T)
        t, ids = _teacher(x, 11, None)
        for rest in (False, True):
            _check_distill(x, None, t, ids, rest, T=T)


def test_weights():
    p = _policy()
    x = _logits(12, 343, torch.float32)
    t, ids = _teacher(x, 9, None)
    t, ids = t.cuda(), ids.cuda()
    loss, tol, d, dd = po.distill(x, t, ids, None, 1.0, True)
    for w in (None, 2.0, 0.0, -1, torch.tensor(0.25), torch.tensor(0.25, dtype=torch.float64),
              torch.arange(12).float() - 3, (torch.arange(12) * 0.5).bfloat16(), torch.arange(24).float()[::2],
              torch.tensor(1.5).expand(12)):
        wt = w.cuda() if isinstance(w, torch.Tensor) else w
        got, g = p.distill_loss_grad(x, t, ids, rest=True, weight=wt)
        full = torch.full((12,), 1 / 12 if w is None else float(w), dtype=torch.float64, device="cuda") \
            if not isinstance(w, torch.Tensor) or w.dim() == 0 else wt.double()
        total = (loss * full).sum()
        po.check(got, total, (tol * full.abs()).sum() + po.H * (3 * loss * full.abs()).sum() + 1e-30, "total")
        po.check(g, d * full[:, None], po.grad_tol(d, dd, full[:, None], x.dtype), "gradient")


def test_strided_small_inputs():
    """Actions, teacher entries and incoming gradients of other strides and types."""
    p = _policy()
    n, V, k = 10, 343, 7
    x = _logits(n, V, torch.bfloat16)
    a = _actions(n, V)
    wide = torch.stack([a, a + 1], 1).cuda()
    want = po.logprobs(x, a, None, 1.0, 0)
    for act in (wide[:, 0], wide[:, 0].int(), torch.stack([a, a]).cuda()[1]):
        po.check(p.action_logprobs(x, act).logp, *want["logp"], "logp")
    t, ids = _teacher(x, k, None)
    tt, ii = t.t().contiguous().cuda().t(), ids.t().contiguous().cuda().t()
    loss, tol, d, dd = po.distill(x, t, ids, None, 1.0, False)
    po.check(p.distill_loss(x, tt, ii, reduction="none"), loss, tol, "loss")
    leaf = x.detach().requires_grad_(True)
    g = torch.randn((n, 2), generator=torch.Generator().manual_seed(1)).cuda()
    got, = torch.autograd.grad(p.distill_loss(leaf, tt, ii, reduction="none"), leaf, g[:, 1])
    w = g[:, 1].double()[:, None]
    po.check(got, d * w, po.grad_tol(d, dd, w, x.dtype), "gradient")
    s = p.distill_loss(leaf, tt, ii, reduction="sum")
    po.check(s, loss.sum(), tol.sum() + po.H * 2 * loss.sum().abs(), "sum")
    got, = torch.autograd.grad(s, leaf)
    one = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    po.check(got, d, po.grad_tol(d, dd, one, x.dtype), "gradient of the sum")
    # only one of the outputs used
    q = p.action_logprobs(leaf, wide[:, 0])
    got, = torch.autograd.grad(q.lse, leaf, g[:, 0])
    dw, tw = po.logprobs_grad(x, a, None, 1.0, None, None, g[:, 0])
    po.check(got, dw, tw, "gradient of lse")


def test_results_may_be_written():
    """The results are the caller's: changed in place, with and without a graph behind them."""
    p = _policy()
    x = _logits(6, 65, torch.float32)
    a = _actions(6, 65)
    keep = torch.tensor([1.0, 0.0, 1.0, 1.0, 0.0, 1.0])
    leaf = x.clone().requires_grad_(True)
    r = p.action_logprobs(leaf, a.cuda(), top=3)
    r.logp.mul_(keep.cuda())
    r.entropy.add_(1.0)
    r.lse.zero_()
    r.top_logp.exp_()
    (r.logp.sum() + r.entropy.sum() + r.lse.sum()).backward()
    dw, tol = po.logprobs_grad(x, a, None, 1.0, keep, torch.ones(6), None)
    po.check(leaf.grad, dw, tol, "gradient")
    with torch.no_grad():
        q = p.action_logprobs(leaf, a.cuda())
        want = po.logprobs(x, a, None, 1.0, 0)
        q.logp.zero_()
        po.check(q.entropy, *want["entropy"], "entropy")
        po.check(q.lse, *want["lse"], "lse")
    t, ids = _teacher(x, 5, None)
    rows = p.distill_loss(leaf, t.cuda(), ids.cuda(), reduction="none")
    rows.mul_(keep.cuda())
    g, = torch.autograd.grad(rows.sum(), leaf)
    _, _, d, dd = po.distill(x, t, ids, None, 1.0, False)
    w = keep.double().cuda()[:, None]
    po.check(g, d * w, po.grad_tol(d, dd, w, x.dtype), "weighted rows")


def test_gradients_against_differences():
    """Central differences of the kernels' own f32 values, V = 9, step s = 2^-6: the third derivatives of these
    functions are under 4 (|logits| < 4, T = 1), so the difference is off by 4 s^2 / 6 < 2e-4, and by the values' own
    error (under 60 h = 4e-6) / s = 3e-4."""
    p = _policy()
    x = torch.randn((4, 9), generator=torch.Generator().manual_seed(2)).cuda()
    a = torch.tensor([0, 8, 3, 5], device="cuda")
    t, ids = _teacher(x, 4, None)
    t, ids = t.cuda(), ids.cuda()
    for f in (lambda z: p.action_logprobs(z, a).logp, lambda z: p.action_logprobs(z, a).entropy,
              lambda z: p.action_logprobs(z, a).lse,
              lambda z: p.distill_loss(z, t, ids, reduction="none"),
              lambda z: p.distill_loss(z, t, ids, rest=True, reduction="none")):
        leaf = x.clone().requires_grad_(True)
        f(leaf).sum().backward()
        s = 2.0 ** -6
        for v in range(9):
            e = torch.zeros_like(x)
            e[:, v] = s
            diff = (f(x + e).double() - f(x - e).double()) / (2 * s)
            assert (diff - leaf.grad[:, v].double()).abs().max() < 5e-4


def test_broadcast_leaf_gets_the_sum():
    p = _policy()
    x = _logits(1, 343, torch.float32).requires_grad_(True)
    a = torch.arange(7, device="cuda")
    g = torch.randn(7, generator=torch.Generator().manual_seed(0))
    d, = torch.autograd.grad(p.action_logprobs(x.expand(7, 343), a).logp, x, g.cuda())
    dw, tol = po.logprobs_grad(x.expand(7, 343), a, None, 1.0, g, None, None)
    # the seven rows are summed by torch in f32: six additions
    po.check(d, dw.sum(0, keepdim=True), (tol + 6 * po.H * dw.abs()).sum(0, keepdim=True), "sum over rows")


def test_scalar_gradients_and_one_row():
    """mean().backward() reaches the kernel as one value for all rows; 1-d logits are one row."""
    p = _policy()
    x = _logits(50, 343, torch.float32).requires_grad_(True)
    p.action_logprobs(x).entropy.mean().backward()
    g = torch.full((50,), 1.0 / 50)
    dw, tol = po.logprobs_grad(x, None, None, 1.0, None, g, None)
    po.check(x.grad, dw, tol, "entropy mean")
    y = _logits(1, 343, torch.float32)[0]
    r = p.action_logprobs(y, torch.tensor(4, device="cuda"), top=2)
    assert r.logp.shape == () and r.top_ids.shape == (2,)
    want = po.logprobs(y[None], torch.tensor([4]), None, 1.0, 2)
    po.check(r.logp, want["logp"][0][0], want["logp"][1][0], "one row")
    t, ids = _teacher(y[None], 5, None)
    assert p.distill_loss(y, t[0].cuda(), ids[0].cuda(), reduction="none").shape == ()


def test_no_rows():
    p = _policy()
    x = torch.empty((0, 343), device="cuda", requires_grad=True)
    a = torch.empty((0,), dtype=torch.int64, device="cuda")
    r = p.action_logprobs(x, a, top=4)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 4)
    r.logp.sum().backward()
    assert x.grad.shape == (0, 343)
    t = torch.empty((0, 4), device="cuda")
    i = torch.empty((0, 4), dtype=torch.int32, device="cuda")
    assert p.distill_loss(x, t, i).item() == 0.0
    loss, d = p.distill_loss_grad(x, t, i)
    assert loss.item() == 0.0 and d.shape == (0, 343)


def test_offsets_past_32_bits():
    """Rows more than 2^32 elements apart, and a gradient of more than 2^32 elements."""
    p = _policy()
    V = 343
    base = torch.empty(2 ** 32 + 2 ** 31 + 4 * V, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((3, V), (2 ** 31 + 2 ** 30 + 5, 1))
    x.copy_(_logits(3, V, torch.bfloat16))
    _check_logprobs(x, None, _actions(3, V), 9)
    t, ids = _teacher(x, 9, None)
    _check_distill(x, None, t, ids, True)
    del base, x
    V, n = 131072, 32800
    row = _logits(1, V, torch.bfloat16)
    t, ids = _teacher(row, 9, None)
    x = row.expand(n, V)
    loss, d = p.distill_loss_grad(x, t.cuda().expand(n, 9), ids.cuda().expand(n, 9), rest=True, weight=1.0)
    lw, tol, dw, dd = po.distill(row, t, ids, None, 1.0, True)
    one = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    for r in (0, 16384, n - 1):
        po.check(d[r:r + 1], dw, po.grad_tol(dw, dd, one, torch.bfloat16), f"row {r}")
    po.check(loss, lw.sum() * n, tol.sum() * n + po.H * n * lw.sum().abs(), "total")
    g = torch.ones(n, device="cuda")
    leaf = x.detach().requires_grad_(True)
    d, = torch.autograd.grad(p.action_logprobs(leaf).entropy, leaf, g)
    dw, tol = po.logprobs_grad(row, None, None, 1.0, None, torch.ones(1), None)
    for r in (0, n - 1):
        po.check(d[r:r + 1], dw, tol, f"entropy row {r}")


def _everything(x, a, t, ids, mask):
    p = _policy()
    r = p.action_logprobs(x, a, top=8, mask=mask)
    leaf = x.detach().requires_grad_(True)
    q = p.action_logprobs(leaf, a, mask=mask)
    d1, = torch.autograd.grad((q.logp.sum() - 0.1 * q.entropy.mean(),), leaf)
    loss, d2 = p.distill_loss_grad(x, t, ids, rest=True, mask=mask)
    lr = p.distill_loss(x, t, ids, reduction="none", mask=mask)
    leaf2 = x.detach().requires_grad_(True)
    d3, = torch.autograd.grad(p.distill_loss(leaf2, t, ids, mask=mask), leaf2)
    return [r.logp, r.entropy, r.lse, r.top_logp, r.top_ids, d1, loss, d2, lr, d3]


@pytest.mark.parametrize("n,V,dtype", [(40, 343, "f32"), (2, 100003, "bf16"), (600, 2500, "f16")])
def test_captured_and_replayed(n, V, dtype):
    """Captured once, replayed with other inputs, eager work and synchronisations between: every replay gives the
    eager result bit for bit, also with a second graph of the same calls replayed in turn."""
    def inputs(seed):
        x = _logits(n, V, DT[dtype], seed=seed)
        t, ids = _teacher(x, 12, None, seed)
        return x, _actions(n, V, seed).cuda(), t.cuda(), ids.cuda()
    mask = _mask("random", n, V)
    mask[:, 0] = True
    bufs = [[b.clone() for b in inputs(0)] for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _everything(*bufs[0], mask)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_everything(*b, mask))
        graphs.append(g)
    for rep in range(4):
        ins = [inputs(10 + 2 * rep + i) for i in range(2)]
        for b, i in zip(bufs, ins):
            for u, v in zip(b, i):
                u.copy_(v)
        for g in graphs:
            g.replay()
        want = [_everything(*i, mask) for i in ins]
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for u, v in zip(o, w):
                assert torch.equal(u, v), rep


def test_two_streams_and_same_bits():
    """Calls on two streams at once do not share scratch memory; a call repeated gives the same bits."""
    sets = []
    for s in range(2):
        n, V = 3, 90001
        x = _logits(n, V, torch.bfloat16, seed=s)
        t, ids = _teacher(x, 30, None, s)
        sets.append((x, _actions(n, V, s).cuda(), t.cuda(), ids.cuda(), None))
    want = [_everything(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = _everything(*sets[i])
        torch.cuda.synchronize()
        for o, w in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(o, w))


def test_inputs_stay():
    x = _logits(5, 9001, torch.bfloat16, "padded")
    whole = x._base.clone()
    t, ids = _teacher(x, 9, None)
    t, ids = t.cuda(), ids.cuda()
    keep = t.clone(), ids.clone()
    _everything(x, _actions(5, 9001).cuda(), t, ids, None)
    assert torch.equal(x._base.view(torch.int16), whole.view(torch.int16))
    assert torch.equal(t, keep[0]) and torch.equal(ids, keep[1])


def test_changed_logits_refused():
    """Autograd's own check: logits changed in place between forward and backward."""
    p = _policy()
    x = _logits(4, 65, torch.float32).requires_grad_(True)
    y = x * 1.0
    r = p.action_logprobs(y)
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.entropy.sum().backward()


def test_refusals():
    from azg_amd._lib import AzgError
    p = _policy()
    x = _logits(4, 65, torch.float32)
    a = torch.zeros(4, dtype=torch.int64, device="cuda")
    t = torch.zeros((4, 3), device="cuda")
    i = torch.zeros((4, 3), dtype=torch.int64, device="cuda")
    for bad in (lambda: p.action_logprobs(x.double(), a), lambda: p.action_logprobs(x, a[:3]),
                lambda: p.action_logprobs(x, a.float()), lambda: p.action_logprobs(x, a.cpu()),
                lambda: p.action_logprobs(x, a, top=-1), lambda: p.action_logprobs(x, a, top=66),
                lambda: p.action_logprobs(x, a, top=True), lambda: p.action_logprobs(x, a, top=2.0),
                lambda: p.action_logprobs(x, a, temperature=0.0),
                lambda: p.action_logprobs(x, a, temperature=math.nan),
                lambda: p.action_logprobs(x, a, temperature=-1.0),
                lambda: p.action_logprobs(x, a, temperature=math.inf),
                lambda: p.action_logprobs(x, a, mask=torch.ones(4, 64, dtype=torch.bool, device="cuda")),
                lambda: p.action_logprobs(x, a, mask=torch.ones(4, 65, device="cuda")),
                lambda: p.action_logprobs(x, a, mask=torch.ones(4, 65, dtype=torch.bool)),
                lambda: p.action_logprobs(torch.empty((4, 0), device="cuda"), a),
                lambda: p.action_logprobs(torch.tensor(1.0, device="cuda")),
                lambda: p.distill_loss(x, t[:3], i[:3]), lambda: p.distill_loss(x, t, i[:, :2]),
                lambda: p.distill_loss(x, t.long(), i), lambda: p.distill_loss(x, t, i.float()),
                lambda: p.distill_loss(x, t, i.cpu()), lambda: p.distill_loss(x, t.cpu(), i),
                lambda: p.distill_loss(x, t[:, :0], i[:, :0]),
                lambda: p.distill_loss(x, t.repeat(1, 50), i.repeat(1, 50)),
                lambda: p.distill_loss(x, t, i, reduction="batchmean"),
                lambda: p.distill_loss(x, t.clone().requires_grad_(True), i),
                lambda: p.distill_loss_grad(x, t, i, weight=math.nan),
                lambda: p.distill_loss_grad(x, t, i, weight=torch.ones(3, device="cuda")),
                lambda: p.distill_loss_grad(x, t, i, weight=torch.ones(4)),
                lambda: p.distill_loss_grad(x, t, i, weight=torch.ones(4, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(AzgError):
        p.action_logprobs(x.cpu(), a.cpu())
    with pytest.raises(RuntimeError):
        y = x.clone().requires_grad_(True)
        d, = torch.autograd.grad(p.action_logprobs(y).entropy.sum(), y, create_graph=True)
        d.sum().backward()


def test_teacher_to_student_run():
    """The operators as they are used together, on the framework's own network: a teacher network's top alternatives
    of legal actions, a student's loss against them with its gradient through fc3 and the trunk; the gradient of the
    whole network against torch's own autograd on the loss written out in f64 over the same logits."""
    from azg_amd.nnet import InflexionNNet
    from azg_amd.optim import FusedAdam
    from azg_amd.wino_train import train_trunk
    p = _policy()
    torch.manual_seed(0)
    teacher, student = InflexionNNet(num_channels=256).cuda().eval(), InflexionNNet(num_channels=256).cuda().train()
    student.dropout = 0.0
    g = torch.Generator(device="cuda").manual_seed(1)
    planes = torch.rand((64, 4, 7, 7), generator=g, device="cuda")
    legal = torch.rand((64, 343), generator=g, device="cuda") < 0.3
    opt = FusedAdam([q for q in student.parameters()])
    for step in range(2):
        with torch.no_grad():
            tops = p.action_logprobs(teacher.fc3(train_trunk(teacher, planes)), top=16, mask=legal)
        logits = student.fc3(train_trunk(student, planes))
        loss, d = p.distill_loss_grad(logits, tops.top_logp, tops.top_ids, mask=legal, rest=True)
        z = logits.detach().double().masked_fill(~legal, -math.inf).requires_grad_(True)
        lp = torch.log_softmax(z, 1)
        q = tops.top_logp.double().exp()
        rest = legal.scatter(1, tops.top_ids, False)
        lr = torch.logsumexp(lp.masked_fill(~rest, -math.inf), 1)
        qr = 1 - q.sum(1)
        ref = ((q * (tops.top_logp.double() - lp.gather(1, tops.top_ids))).sum(1) + qr * (qr.log() - lr)).mean()
        dz, = torch.autograd.grad(ref, z)
        # both sides are f32 sums of 343 terms of at most 1 / 64, nearly equal logits: 40 h of the largest
        assert abs(loss.item() - ref.item()) < 100 * po.H * max(1.0, ref.item())
        assert (d.double() - torch.where(legal, dz, 0.0)).abs().max() < 100 * po.H / 64
        opt.zero_grad()
        student.fc4.weight.grad = torch.zeros_like(student.fc4.weight)
        student.fc4.bias.grad = torch.zeros_like(student.fc4.bias)
        logits.backward(d)
        assert student.conv1.weight.grad.abs().sum() > 0
        opt.step()
    # a policy-gradient step on the same network
    logits = student.fc3(train_trunk(student, planes))
    r = p.action_logprobs(logits, tops.top_ids[:, 0], mask=legal)
    adv = torch.randn(64, generator=g, device="cuda")
    (-(adv * r.logp).mean() - 0.01 * r.entropy.mean()).backward()
    assert student.fc3.weight.grad.isfinite().all() and torch.isfinite(r.logp).all()
