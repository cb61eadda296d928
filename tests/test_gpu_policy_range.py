"""azg_amd.policy over the whole range of its inputs (csrc/azg_policy.hip): logits and teachers' log-probabilities of
any finite size, values that are no numbers beside illegal actions, sums held to bounds that do not grow with the row."""
import math

import policy_oracle as po
import pytest
import torch
from test_gpu_policy import (DT, _actions, _check_distill, _check_logprobs, _everything, _logits, _mask, _policy,
                             _teacher)

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


FAR = [s * v for v in (1e7, 1e9, 3e9, 1e10, 1e11, 1e12, 1e15, 1e20, 1e29) for s in (1, -1)]


@pytest.mark.parametrize("which", ["all", "first", "third"])
@pytest.mark.parametrize("n,V,dtype", [f for f in FORMS if f[2] != "f16"])
def test_student_far_at_the_entries(n, V, dtype, which):
    """The student's logits at all entries, or at one, far above or below all others."""
    x0 = _logits(n, V, DT[dtype])
    t, ids = _teacher(x0, 12, None)
    at = {"all": slice(0, 12), "first": slice(0, 1), "third": slice(2, 3)}[which]
    rows = torch.arange(n)[:, None]
    for i, far in enumerate(FAR):
        x = x0.clone()
        x[rows, ids[:, at]] = far
        _check_distill(x, None, t, ids, True)
        if i % 3 == 0:
            _check_distill(x, None, t, ids, False)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
def test_student_far_by_temperature(dtype, rest):
    for n, V in ((5, 343), (130, 20011), (3, 20011)):
        x = _logits(n, V, DT[dtype])
        t, ids = _teacher(x, 12, None)
        for far in (1e4, -1e4, 6e4, -6e4):
            x[torch.arange(n)[:, None], ids[:, :4]] = far
            _check_distill(x, None, t, ids, rest, T=1e-6)


def test_student_far_at_different_entries():
    """Entries at the lowest value, some 1e10 above and below, some illegal, none outside, masked outside."""
    n, V = 8, 343
    x = _logits(n, V, torch.float32)
    t, ids = _teacher(x, 10, None)
    r = torch.arange(n)[:, None]
    x[r[:4], ids[:4, :5]] = torch.finfo(torch.float32).min
    x[r[2:6], ids[2:6, 5:7]] = -1e10
    x[r[3:7], ids[3:7, 7:8]] = 2e10
    x[7] = -1e10
    x[7, ids[7, 0]] = -2e10
    m = torch.rand((n, V), generator=torch.Generator().manual_seed(0)) < 0.5
    for k in range(10):
        m[torch.arange(n), ids[:, k]] = True
    m[1] = False
    m[1, ids[1]] = True  # nothing outside
    m[5, ids[5, 7]] = False
    for mask in (None, m.cuda()):
        for rest in (False, True):
            _check_distill(x, mask, t, ids, rest)


FILLS = [-1e9, -2e9, -1e10]


@pytest.mark.parametrize("T", [0.05, 0.2, 0.4, 0.6, 1.0, 1.2, 1.5, 4.0, 5.0])
@pytest.mark.parametrize("n,V,dtype", [(4, 343, "f32"), (130, 5003, "f32"), (130, 20011, "bf16"), (3, 20011, "f32"),
                                       (2, 100003, "bf16")])
def test_fills_leave_the_entropy(n, V, dtype, T):
    """Legal logits of a mask's fill beside ordinary ones, in turn, in whole stretches of a row, in its last elements:
    entropy, its gradient and the alternatives."""
    for fill in FILLS:
        x = _logits(n, V, DT[dtype])
        f = torch.tensor(fill).to(x.dtype).item()
        x[0, ::2] = f
        x[1, :V // 2] = f
        x[1, V // 2 + 1:V // 2 + 99] = f
        x[-1, V // 3:] = f
        _check_logprobs(x, None, _actions(n, V), 9, T=T)


@pytest.mark.parametrize("fill", [2.4e8, 1e9, 1.5e9, 1.6e9, -2e9, 2.2e9, -2.5e9, 2.9e9, -5e9, 1e10, -3e20])
@pytest.mark.parametrize("n,V,dtype", [(4, 343, "f32"), (6, 1001, "bf16"), (130, 5003, "f32"), (130, 20011, "f32"),
                                       (3, 20011, "f32"), (2, 100003, "bf16")])
def test_rows_of_one_large_value(n, V, dtype, fill):
    """Rows whose largest logit is far from 0: probabilities, entropy and the gradients with incoming ones of a loss scale."""
    p = _policy()
    x = torch.full((n, V), fill).to(DT[dtype]).cuda()
    x[0, ::3] = torch.finfo(DT[dtype]).min
    x[1, 1::2] = -1e30
    _check_logprobs(x, None, _actions(n, V), 5)
    t, ids = _teacher(_logits(n, V, torch.float32), 6, None)
    ids[0, :3] = torch.tensor([1, 4, 7])
    for rest in (False, True):
        _check_distill(x, None, t, ids, rest)
        loss, tol, d, dd = po.distill(x, t, ids, None, 1.0, rest)
        for w in (2.0 ** 16, 2.0 ** -20):
            _, g = p.distill_loss_grad(x, t.cuda(), ids.cuda(), rest=rest, weight=w)
            one = torch.full((1, 1), w, dtype=torch.float64, device="cuda")
            po.check(g, d * one, po.grad_tol(d, dd, one, x.dtype), f"gradient of {w} times the sum")
    for w in (2.0 ** 16, 2.0 ** -20):
        leaf = x.clone().requires_grad_(True)
        g1 = torch.full((n,), w)
        q = p.action_logprobs(leaf, _actions(n, V).cuda())
        d, = torch.autograd.grad((q.logp, q.entropy), leaf, (g1.cuda(), g1.cuda()))
        po.check(d, *po.logprobs_grad(x, _actions(n, V), None, 1.0, g1, g1, None), f"gradient of {w} logp and entropy")


@pytest.mark.parametrize("T", [0.05, 0.2, 0.6, 1.2, 4.0])
@pytest.mark.parametrize("n,V,dtype", [(4, 343, "f32"), (130, 5003, "f32"), (3, 20011, "f32"), (2, 100003, "bf16")])
def test_large_values_at_temperatures(n, V, dtype, T):
    """Ordinary logits beside stretches of a large value, as the row's largest or its smallest."""
    for fill in (3e8, 1e9, 2e9, 3e9, -2e9):
        x = _logits(n, V, DT[dtype])
        x[0, ::2] = fill
        x[1, :V // 2] = fill
        x[-1, V // 3:] = fill
        _check_logprobs(x, None, _actions(n, V), 9, T=T)
        t, ids = _teacher(_logits(n, V, torch.float32, seed=1), 9, None)
        _check_distill(x, None, t, ids, True, T=T)
        _check_distill(x, None, t, ids, False, T=T)


@pytest.mark.parametrize("n,V,dtype", FORMS)
def test_illegal_actions_get_no_gradient(n, V, dtype):
    """A teacher's NaN, and weights that are no finite numbers, leave 0 at the illegal actions of their rows."""
    p = _policy()
    x = _logits(n, V, DT[dtype])
    m = _mask("random", n, V)
    t, ids = _teacher(x, 12, m)
    t[0, 1] = math.nan
    t, ids = t.cuda(), ids.cuda()
    w = torch.ones(n, device="cuda")
    w[-1] = math.inf
    w[1] = math.nan
    for rest in (False, True):
        _, g = p.distill_loss_grad(x, t, ids, mask=m, rest=rest, weight=w)
        leaf = x.clone().requires_grad_(True)
        rows = p.distill_loss(leaf, t, ids, mask=m, rest=rest, reduction="none")
        d, = torch.autograd.grad(rows, leaf, w)
        for q in (g, d):
            assert (q[~m] == 0).all()
            assert q[1][m[1]].isnan().all()
            if rest:
                assert q[0][m[0]].isnan().all()
            if n > 3:
                assert q[2][m[2]].isfinite().all()


def test_forward_mode_is_refused():
    """No forward-mode derivative: a tangent is refused rather than dropped."""
    from torch.autograd import forward_ad as fwd
    p = _policy()
    x = _logits(4, 65, torch.float32)
    a = _actions(4, 65).cuda()
    t, ids = _teacher(x, 5, None)
    t, ids = t.cuda(), ids.cuda()
    w = torch.ones(4, device="cuda")
    with fwd.dual_level():
        dx, dt, dw = (fwd.make_dual(q, torch.ones_like(q)) for q in (x, t, w))
        for bad in (lambda: p.action_logprobs(dx, a), lambda: p.distill_loss(dx, t, ids),
                    lambda: p.distill_loss(x, dt, ids), lambda: p.distill_loss_grad(dx, t, ids),
                    lambda: p.distill_loss_grad(x, dt, ids), lambda: p.distill_loss_grad(x, t, ids, weight=dw)):
            with pytest.raises(RuntimeError, match="forward"):
                bad()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
            p.action_logprobs(dx, a)
        leaf = x.clone().requires_grad_(True)  # a tangent of what reaches the results
        for y in (p.action_logprobs(leaf, a).entropy, p.distill_loss(leaf, t, ids, reduction="none")):
            with pytest.raises(RuntimeError, match="forward"):
                torch.autograd.grad((y * dw).sum(), leaf)
        want = p.action_logprobs(x, a).logp  # no tangent: as outside
        assert torch.equal(p.action_logprobs(dx.detach(), a).logp, want)
    assert torch.equal(p.action_logprobs(x, a).logp, want)


@pytest.mark.parametrize("given", [False, True])
def test_results_without_a_graph_are_separate(given):
    """Each result is a tensor of its own: written with what requires a gradient, and without touching the others' graph."""
    p = _policy()
    x = _logits(6, 65, torch.float32)
    w = torch.full((6,), 2.0, device="cuda", requires_grad=True)
    r = p.action_logprobs(x, _actions(6, 65).cuda() if given else None)
    plain = [q.clone() for q in r if q is not None]
    assert len(plain) == 2 + given and not any(q._is_view() for q in r if q is not None)
    loss = (w * r.entropy).sum()  # entropy is kept for w's gradient
    r.lse.mul_(w)
    if given:
        r.logp.mul_(w)
    assert r.lse.requires_grad and not r.entropy.requires_grad and r.entropy._version == 0
    g, = torch.autograd.grad(loss, w)
    assert torch.equal(g, r.entropy) and torch.equal(r.entropy, plain[-2])
    g, = torch.autograd.grad(r.lse.sum(), w)
    assert torch.equal(g, plain[-1])
    with torch.no_grad():
        q = p.action_logprobs(x)
    q.entropy.mul_(w)
    assert q.entropy.requires_grad
    for shape in ((65,), (0, 65), (2, 0, 65), (2, 3, 65)):  # one row, none, several leading dimensions
        y = _logits(6, 65, torch.float32).reshape(2, 3, 65)
        y = y[0, 0] if len(shape) == 1 else y if 0 not in shape else y.new_empty(shape)
        a = torch.zeros(shape[:-1], dtype=torch.int64, device="cuda") if given else None
        r = p.action_logprobs(y, a)
        assert all(q.shape == shape[:-1] and q.is_contiguous() for q in r if q is not None)


@pytest.mark.parametrize("n,V,dtype", FORMS)
def test_no_probability_above_one(n, V, dtype):
    """Nearly sure policies: log-probabilities are never above 0, entropies never below."""
    p = _policy()
    for sure in (12.0, 17.0, 20.0, 30.0, 100.0):
        x = _logits(n, V, DT[dtype])
        a = torch.arange(n) % V
        x[torch.arange(n), a] += sure
        r = p.action_logprobs(x, a.cuda(), top=3)
        assert (r.logp <= 0).all() and (r.top_logp <= 0).all() and (r.entropy >= 0).all()
        _check_logprobs(x, None, a, 3)
    # One action: s = 2^u, |u| <= 1/2.  With h = 2^-24 the exponential is off by 2 h of itself, its logarithm by 2 h / ln 2
    # for that and by a step of the instruction (h), u - log2 s is exact, and u s / s adds 3 roundings of at most h / 2: times
    # ln 2 under 4 h.
    x = _logits(n, V, torch.float32)[:, :1]
    r = p.action_logprobs(x, torch.zeros(n, dtype=torch.int64, device="cuda"), top=1)
    for q in (-r.logp, -r.top_logp, r.entropy):
        assert (q >= 0).all() and (q < 4 * po.H).all()


def _tight(kind):
    """policy_oracle.row_slack by what the kernels add, h = 2^-24 an addition.  A term passes at most 16 additions within
    its thread's group of 16 or 32 logits (two chains), 2 more into the thread's sum, one for each further group (V / 4096
    of them in a block that takes a whole row: 32 at 131072), 5 for the last group's vectors and the remainder, 6 and 4 in
    the wave and the block, 12 where parts are joined; the exponential is off by 2 h and 4 h |u|, the logarithm by 2 h of
    itself.  A KL leaves f32 behind the thread's group, and its logarithms are f64: 18 additions, the conversion to
    f32 for the gradient, the exponential."""
    def slack(z, p):
        V = z.shape[1]
        u = (z.max(1, keepdim=True).values - z) / math.log(2.0)
        eu = (p * torch.where(torch.isfinite(u), u, torch.zeros_like(u))).sum(1)
        if kind == "kl":
            return po.H * (22 + 4 * eu), eu
        return po.H * (47 + min(V // 4096, 32) + 4 * eu + 2 * math.log1p(V)), eu
    return slack


ENDS = [(6, 343, "f32"), (6, 343, "bf16"), (6, 1001, "f16"), (2100, 3001, "f32"), (130, 5003, "f32"), (130, 5003, "bf16"),
        (130, 20011, "f16"), (130, 40001, "f32"), (130, 70001, "bf16"), (128, 131071, "f16"), (4, 20011, "f32"),
        (3, 100003, "bf16"), (2, 262147, "f32")]


@pytest.mark.parametrize("n,V,dtype", ENDS)
def test_every_element_counts(n, V, dtype, monkeypatch):
    """A row's mass in the elements behind its last vector, in its last and first vectors, next to the bounds of
    groups and parts, in one element in a thousand; and equal logits, of which none may be left out."""
    g = torch.Generator().manual_seed(V)
    x = _logits(n, V, DT[dtype])
    near = torch.arange(0, V + 1024, 1024)
    near = torch.cat([near - 1, near, near + 1])
    places = [torch.arange(V - V % 8, V), torch.arange(max(0, V - 70), V), torch.arange(min(9, V)), near[(near >= 0) & (near < V)],
              torch.randint(0, V, (max(1, V // 1000),), generator=g), torch.arange(V - V % 4, V)]
    for r in range(n):
        if r % 8 == 7:
            x[r] = 0.5
        else:
            at = places[(r + V) % len(places) if n > 6 else (r + V // 2) % len(places)]
            x[r, at] = (11.0 + torch.randn(len(at), generator=g)).to(x.dtype).cuda()
    if n < 8:
        x = torch.cat([x, torch.full_like(x[:1], 0.5)])
        n += 1
    monkeypatch.setattr(po, "row_slack", _tight("logp"))
    for top in (0, 20):
        _check_logprobs(x, None, _actions(n, V), top, grads=top == 0)
    _check_logprobs(x, _mask("random", n, V), _actions(n, V), 9)
    monkeypatch.setattr(po, "row_slack", _tight("kl"))
    t, ids = _teacher(x, 12, None)
    ids[:, 1::2] = torch.randint(0, V, ids[:, 1::2].shape, generator=g)  # half of the mass outside the entries
    for rest in (False, True):
        _check_distill(x, None, t, ids, rest)
        _check_distill(x, _mask("random", n, V), t, ids, rest)


@pytest.mark.parametrize("n,V,dtype", ENDS)
def test_kl_of_near_distributions(n, V, dtype):
    """Logits whose exponentials are powers of two (the temperature makes log2(e) / T one in f32): 20 entries of 1, all else
    2^-14 to 2^-20.  A thread's sum of 32 is exact in f32 (24 bits hold up to 16 of the ones), a row's in f64 alone: added up in
    f32 it would be off by some 3e-8 of itself, and the KL by as much.  Exponentials and logarithms in f64 are good to 1e-11,
    what remains is the KL's own rounding (0.21 at most)."""
    p = _policy()
    T = math.log2(math.e)
    g = torch.Generator().manual_seed(V)
    x = -torch.randint(14, 21, (n, V), generator=g).float()
    ids = (torch.arange(20) * (V // 20) + torch.arange(n)[:, None] % (V // 20)).contiguous()
    x.scatter_(1, ids, 0.0)
    t = torch.log_softmax(x.double() / T, 1).gather(1, ids).float()
    x = x.to(DT[dtype]).cuda()
    for rest in (False, True):
        loss, _, _, _ = po.distill(x, t, ids, None, T, rest)
        assert loss.abs().max() < 0.21  # ln(1 + 262147 * 1.74e-5 / 20)
        tol = 1e-10 + po.H * loss.abs()
        got = p.distill_loss(x, t.cuda(), ids.cuda(), rest=rest, temperature=T, reduction="none").double()
        assert ((got - loss).abs() <= tol).all()
        one, _ = p.distill_loss_grad(x, t.cuda(), ids.cuda(), rest=rest, temperature=T, weight=1.0)
        assert abs(one.double() - loss.sum()) <= tol.sum() + po.H * loss.sum().abs()
        rows = p.distill_loss(x.clone().requires_grad_(True), t.cuda(), ids.cuda(), rest=rest, temperature=T,
                              reduction="none").double()
        assert ((rows - loss).abs() <= tol).all()


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("n,V,dtype", FORMS)
def test_rows_without_an_entry_get_no_gradient(n, V, dtype, rest):
    """Padding: no entry, and logits that are no numbers.  Loss 0 and gradient 0, the other rows' as without them."""
    p = _policy()
    x = _logits(n, V, DT[dtype])
    t, ids = _teacher(x, 12, None)
    m = _mask("random", n, V)
    t, ids, pad = t.cuda(), ids.cuda(), slice(n - 1, n) if n < 3 else slice(1, n, 3)
    ids[pad] = -1
    t[n - 1] = -math.inf
    y = x.clone()
    y[pad] = math.nan
    y[n - 1, V // 2:] = math.inf
    for mask in (None, m):
        want, dwant = p.distill_loss_grad(x, t, ids, mask=mask, rest=rest, weight=1.0)
        for z in (x, y):
            loss, d = p.distill_loss_grad(z, t, ids, mask=mask, rest=rest, weight=1.0)
            assert torch.equal(loss, want) and torch.equal(d, dwant) and (d[pad] == 0).all() and (d[n - 1] == 0).all()
            leaf = z.clone().requires_grad_(True)
            rows = p.distill_loss(leaf, t, ids, mask=mask, rest=rest, reduction="none")
            e, = torch.autograd.grad(rows.sum(), leaf)
            assert (rows[pad] == 0).all() and rows[n - 1] == 0 and (e[pad] == 0).all() and (e[n - 1] == 0).all()


@pytest.mark.parametrize("n,V,dtype", FORMS)
def test_actions_outside_get_no_gradient(n, V, dtype):
    """Padding: an action outside 0..V-1 beside logits that are no numbers has log-probability 0 and no gradient."""
    p = _policy()
    x = _logits(n, V, DT[dtype])
    a = _actions(n, V).clamp(0, V - 1)
    a[n - 1] = -1
    x[n - 1, V // 2:] = math.nan
    x[n - 1, 0] = math.inf
    for mask in (None, _mask("random", n, V)):
        leaf = x.clone().requires_grad_(True)
        r = p.action_logprobs(leaf, a.cuda(), mask=mask)
        g, = torch.autograd.grad(r.logp.sum(), leaf, retain_graph=True)
        assert r.logp[n - 1] == 0 and (g[n - 1] == 0).all() and g[:n - 1].isfinite().all()
        g, = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), leaf)
        assert g[n - 1][slice(None) if mask is None else mask[n - 1]].isnan().all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_largest_vocabulary(dtype):
    """2^29 actions, in thousands of parts: sums, alternatives, gradients up to the last element."""
    p = _policy()
    V = p.VOCAB_MAX
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty((1, V), dtype=DT[dtype], device="cuda")
    for part in x[0].split(2 ** 27):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    ids = torch.tensor([[0, V - 1, V // 2, 12345, V - 131073]], device="cuda")
    x[0, ids[0]] = torch.tensor([20.0, 19.5, 19.0, 18.5, 18.0], device="cuda").to(x.dtype)
    z = x[0].split(2 ** 27)
    total = sum(q.double().sub(20).exp().sum() for q in z)
    lse = 20 + total.log()
    # 16 additions in a group, 2^20 / 4096 groups, 45 joining the threads and parts, exp and its argument: h each
    tol = po.H * (16 + 256 + 45 + 40)
    leaf = x.requires_grad_(True)
    r = p.action_logprobs(leaf, ids[:, 1], top=5)
    assert torch.equal(r.top_ids, ids)
    assert abs(r.lse.item() - lse.item()) < tol + 3 * po.H * lse.item()
    assert abs(r.logp.item() - (19.5 - lse.item())) < tol
    none = p.action_logprobs(leaf.detach(), ids[:, 1])
    assert abs(none.logp.item() - (19.5 - lse.item())) < tol
    d, = torch.autograd.grad(r.logp, leaf)
    t = torch.log(torch.tensor([[0.4, 0.3, 0.1, 0.1, 0.1]], device="cuda"))
    loss, e = p.distill_loss_grad(leaf, t, ids, weight=1.0)
    xe = torch.tensor([20.0, 19.5, 19.0, 18.5, 18.0], dtype=torch.float64, device="cuda")
    want = (t.double().exp() * (t.double() - xe + lse)).sum()
    assert abs(loss.item() - want.item()) < 40 * po.H + 2 * po.H * abs(want.item())
    f, = torch.autograd.grad(p.distill_loss(leaf, t, ids), leaf)
    eps = torch.finfo(x.dtype).eps / 2
    q = t.double().exp() / t.double().exp().sum()
    for i, part in enumerate(z):
        lo = i * 2 ** 27
        prob = (part.detach().double() - lse).exp()
        # the exponential's argument is off by 4 h of its size in log2, 40 here
        off = prob * (2 * tol + 200 * po.H + eps) + po.TINY[x.dtype]
        for got, hot in ((-d, torch.tensor([[0.0, 1, 0, 0, 0]], dtype=torch.float64, device="cuda")), (e, q), (f, q)):
            exact = prob.clone()
            here = (ids[0] >= lo) & (ids[0] < lo + 2 ** 27)
            exact[ids[0, here] - lo] -= hot[0, here]
            most = off.clone()
            most[ids[0, here] - lo] += hot[0, here] * (eps + 16 * po.H)
            assert ((got[0, lo:lo + 2 ** 27].double() - exact).abs() <= most).all()


@pytest.mark.parametrize("n,V,dtype", [(40, 343, "f32"), (2, 100003, "bf16"), (130, 20011, "f32")])
def test_large_values_captured(n, V, dtype):
    """The second pass within a graph, replayed with other inputs, with and without rows that take it."""
    def inputs(seed):
        x = _logits(n, V, DT[dtype], seed=seed)
        t, ids = _teacher(x, 12, None, seed)
        if seed % 2:
            x[0] = -1e10
            x[1, V // 3:] = 3e9
            x[1, ids[1, :6]] = 7e11
        return x, _actions(n, V, seed).cuda(), t.cuda(), ids.cuda()
    bufs = [b.clone() for b in inputs(0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _everything(*bufs, None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _everything(*bufs, None)
    for seed in (1, 2, 3, 4, 3):
        new = inputs(seed)
        for b, v in zip(bufs, new):
            b.copy_(v)
        graph.replay()
        want = _everything(*new, None)
        torch.cuda.synchronize()
        for o, w in zip(out, want):
            assert not o.isnan().any() and torch.equal(o, w), seed
