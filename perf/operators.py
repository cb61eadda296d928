"""What is measured of the policy operators: the log-probabilities of given actions with their entropy and
top alternatives (azg_amd.policy.action_logprobs), and the distillation loss from a teacher's top
alternatives (azg_amd.policy.distill_loss, distill_loss_grad), over the sizes they are used at: one game
state, batches of 7x7 Inflexion (343 actions) and 8x8 Othello (65) positions, and vocabularies of 10^4 to
10^5 entries in 16-bit types.

own = False computes the operators in elementary torch operations in f32; own = True calls the framework."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOSS_SCALE = {"f32": 1.0, "bf16": 1.0, "f16": 1024.0}  # gradients of a mean over thousands of rows leave f16's range
DEV = "cuda"

# op:     score    action_logprobs, forward
#         train    action_logprobs with the gradient of a policy-gradient loss (logp and entropy)
#         loss     distill_loss per row, forward
#         autograd distill_loss (mean) and its gradient through autograd
#         step     distill_loss_grad: loss and gradient in one call
# layout: packed   rows one after the other
#         padded   rows of a wider buffer (a head stacked with others, or padded to a tile)
#         shifted  [B, T + 1, V][:, :-1]: every sequence but its last position
# legal:  the share of legal actions per row; 0 = no mask


def listed():
    return [
        # one position, as a move is chosen: 343 actions, most of them illegal late in a game
        dict(name="score_one_position", op="score", rows=1, vocab=343, dtype="f32", top=8, legal=0.3, layout="packed"),
        # all positions of 4096 concurrent games
        dict(name="score_games", op="score", rows=4096, vocab=343, dtype="f32", top=16, legal=0.3, layout="packed"),
        # the next token of one sequence
        dict(name="score_one_token", op="score", rows=1, vocab=131072, dtype="bf16", top=20, legal=0, layout="packed"),
        # the next token of a small batch, an odd vocabulary in a padded buffer
        dict(name="score_small_batch", op="score", rows=61, vocab=100003, dtype="f16", top=64, legal=0,
             layout="padded"),
        # given sequences scored, a few alternatives each
        dict(name="score_sequences", op="score", rows=8192, vocab=32768, dtype="bf16", top=8, legal=0,
             layout="packed"),
        # a trainer's batch of 512 Othello positions
        dict(name="train_othello", op="train", rows=512, vocab=65, dtype="f32", top=0, legal=0.3, layout="packed"),
        # a policy-gradient step on four sequences of 1024 positions, the last of each left out; odd vocabulary
        dict(name="train_sequences", op="train", rows=4092, vocab=50001, dtype="bf16", top=0, legal=0,
             layout="shifted"),
        # a trainer's batch of 512 positions against the at most 25 actions that 25 simulations visit
        dict(name="step_visits", op="step", rows=512, vocab=343, dtype="f32", top=25, legal=0.3, rest=False,
             layout="packed"),
        # few rows of a large vocabulary: a micro-batch
        dict(name="step_micro_batch", op="step", rows=16, vocab=131072, dtype="bf16", top=64, legal=0, rest=True,
             layout="packed"),
        # a training step on 8192 positions
        dict(name="step_sequences", op="step", rows=8192, vocab=32768, dtype="bf16", top=32, legal=0, rest=True,
             layout="packed"),
        # the same through autograd: f32 logits, odd vocabulary, a long teacher's list
        dict(name="autograd_sequences", op="autograd", rows=2048, vocab=100003, dtype="f32", top=128, legal=0,
             rest=True, layout="packed"),
        # held-out positions: the loss of each row alone
        dict(name="loss_heldout", op="loss", rows=4096, vocab=65536, dtype="f16", top=16, legal=0, rest=False,
             layout="packed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "score", "train", "loss", "autograd", "step", "step"])
    vocab = _log_int(rng, 20, 131072)
    rows = _log_int(rng, 1, min(65536, max(1, 160_000_000 // vocab)))
    case = dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16", "f16"]),
                legal=rng.choice([0, 0, 0.3]), layout=rng.choice(["packed", "packed", "padded", "shifted"]))
    if op == "score":
        case["top"] = rng.choice([0, _log_int(rng, 1, min(128, vocab))])
    elif op == "train":
        case["top"] = 0
    else:
        case["top"] = _log_int(rng, 1, min(128, vocab))
        case["rest"] = rng.random() < 0.5
    return case


def _inputs(case, seed):
    """logits (the student's), actions, mask, and for the distillation the teacher's entries."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, vocab, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    if case["layout"] == "shifted":
        b = next(b for b in (4, 2, 1) if rows % b == 0)
        buf = torch.empty((b, rows // b + 1, vocab), dtype=dt, device=DEV)
        logits = buf[:, :-1]
    elif case["layout"] == "padded":
        logits = torch.empty((rows, vocab + 13), dtype=dt, device=DEV)[:, :vocab]
    else:
        logits = torch.empty((rows, vocab), dtype=dt, device=DEV)
    mask = None
    if case["legal"]:
        mask = torch.rand((rows, vocab), generator=g, device=DEV) < case["legal"]
        mask[:, 0] |= ~mask.any(1)  # a position has a legal action
    lead = logits.shape[:-1]
    k = case["top"]
    distil = case["op"] in ("loss", "autograd", "step")
    t_logp = t_ids = None
    if distil:
        t_logp = torch.empty((*lead, k), dtype=torch.float32, device=DEV)
        t_ids = torch.empty((*lead, k), dtype=torch.int64, device=DEV)
    actions = torch.empty(lead, dtype=torch.int64, device=DEV)
    # rows in slices, so that the making takes little memory beside the inputs
    flat = [t.view(-1, t.shape[-1]) if t is not None else None for t in (t_logp, t_ids)]
    scale = 2.5  # logits of a trained head: most of the mass on tens of entries
    step = max(1, (1 << 26) // vocab)
    outer = logits if logits.dim() == 3 else logits.unsqueeze(0)
    per = outer.shape[1]
    for o in range(outer.shape[0]):
        for r0 in range(0, per, step):
            n = min(step, per - r0)
            f0 = o * per + r0
            x = torch.randn((n, vocab), generator=g, device=DEV) * scale
            outer[o, r0:r0 + n] = x
            m = None if mask is None else mask[f0:f0 + n]
            if distil:
                t = x + 0.5 * torch.randn((n, vocab), generator=g, device=DEV)
                if m is not None:
                    t = t.masked_fill(~m, -math.inf)
                v, i = torch.topk(t, k, dim=1)
                flat[0][f0:f0 + n] = v - torch.logsumexp(t, 1, keepdim=True)
                flat[1][f0:f0 + n] = torch.where(torch.isfinite(v), i, -1)
            else:
                w = torch.rand((n, vocab), generator=g, device=DEV)
                if m is not None:
                    w = w.masked_fill(~m, -1.0)
                actions.view(-1)[f0:f0 + n] = w.argmax(1)
    if mask is not None:
        mask = mask.view(logits.shape)
    return dict(logits=logits, mask=mask, actions=actions, t_logp=t_logp, t_ids=t_ids, gen=g)


def prepare(case, seed):
    s = _inputs(case, seed)
    g = s.pop("gen")
    s["case"] = dict(case)
    lead = s["logits"].shape[:-1]
    if case["op"] == "train":
        # loss = -mean(advantage * logp) - 0.01 mean(entropy): what reaches logp and entropy
        n = case["rows"]
        scale = LOSS_SCALE[case["dtype"]]
        s["g_logp"] = torch.randn(lead, generator=g, device=DEV) * (-scale / n)
        s["g_entropy"] = torch.full(lead, -0.01 * scale / n, device=DEV)
    if case["op"] == "autograd":
        s["g_loss"] = torch.full((), LOSS_SCALE[case["dtype"]], device=DEV)
    if case["op"] in ("train", "autograd"):
        s["logits"].requires_grad_(True)
    return s


# ---- the plain form -------------------------------------------------------------------------

def _masked(s, dtype):
    x = s["logits"].detach().to(dtype)
    return x if s["mask"] is None else x.masked_fill(~s["mask"], -math.inf)


def _plain_logp(x):
    m = x.amax(-1, keepdim=True)
    z = x - m
    return z - z.exp().sum(-1, keepdim=True).log()


def _plain_top(x, k):
    """ids of the k largest, ties to the lowest index: one 64-bit key of value and index."""
    b = (x + 0.0).view(torch.int32).to(torch.int64)
    key = torch.where(b < 0, -(b & 0x7FFFFFFF), b)
    low = torch.arange(x.shape[-1] - 1, -1, -1, device=x.device)
    top = torch.topk(key * (1 << 24) + low, k, dim=-1).values
    return x.shape[-1] - 1 - (top & ((1 << 24) - 1))


def _plain_score(s, x, logp):
    k = s["case"]["top"]
    out = {"logp": logp.gather(-1, s["actions"].unsqueeze(-1)).squeeze(-1)}
    p = logp.exp()
    out["entropy"] = -(p * logp.clamp_min(-1e30)).sum(-1)
    out["lse"] = x.amax(-1) + (x - x.amax(-1, keepdim=True)).exp().sum(-1).log()
    if k:
        ids = _plain_top(x, k)
        vals = logp.gather(-1, ids)
        out["top_logp"] = vals
        out["top_ids"] = torch.where(torch.isfinite(vals), ids, -1)
    return out, p


def _plain_distill(s, x, dtype):
    """per-row loss and the gradient of their sum; the loss is a difference of near values, so what a
    row sums to and the logarithms of its few entries are in f64"""
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    t = s["t_logp"].double()
    there = (s["t_ids"] >= 0) & torch.isfinite(t)
    ids = s["t_ids"].clamp_min(0)
    q = torch.where(there, t.exp(), 0.0)
    if not s["case"]["rest"]:
        q = q / q.sum(-1, keepdim=True)
    lq = torch.where(there, q, 1.0).log()
    lp = torch.where(there, x.gather(-1, ids).double() - m.double() - total.log(), 0.0)
    loss = (q * (lq - lp)).sum(-1)
    p = e / total.to(dtype)
    top = torch.zeros_like(x).scatter_add_(-1, ids, q.to(dtype))
    if not s["case"]["rest"]:
        return loss, p - top
    inside = torch.zeros(x.shape, dtype=torch.int8, device=x.device)
    inside.scatter_add_(-1, ids, there.to(torch.int8))
    xr = torch.where(inside > 0, -math.inf, x)
    mr = xr.amax(-1, keepdim=True)
    er = (xr - torch.where(torch.isfinite(mr), mr, 0.0)).exp()
    lpr = (mr.double() - m.double() + er.sum(-1, keepdim=True, dtype=torch.float64).log() - total.log()).squeeze(-1)
    qr = (1.0 - q.sum(-1)).clamp_min(0.0)
    has = (qr > 0) & torch.isfinite(lpr)
    qr = torch.where(has, qr, 0.0)
    loss = loss + qr * (torch.where(has, qr, 1.0).log() - torch.where(has, lpr, 0.0))
    mass = (q.sum(-1) + qr).unsqueeze(-1).to(dtype)
    ratio = torch.where(has, qr / torch.where(has, lpr, 0.0).exp(), 0.0).unsqueeze(-1).to(dtype)
    return loss, p * mass - torch.where(inside > 0, top, ratio * p)


def _plain(s):
    op, dt = s["case"]["op"], s["logits"].dtype
    x = _masked(s, torch.float32)
    if op in ("score", "train"):
        logp = _plain_logp(x)
        out, p = _plain_score(s, x, logp)
        if op == "train":
            h = out["entropy"].unsqueeze(-1)
            ga, ge = s["g_logp"].unsqueeze(-1), s["g_entropy"].unsqueeze(-1)
            d = -ga * p - ge * p * (logp.clamp_min(-1e30) + h)
            d.scatter_add_(-1, s["actions"].unsqueeze(-1), ga)
            out["grad"] = d.to(dt)
        return out
    loss, d = _plain_distill(s, x, torch.float32)
    if op == "loss":
        return {"loss": loss.float()}
    w = LOSS_SCALE[s["case"]["dtype"]] / loss.numel()
    # distill_loss_grad weighs the loss it returns, autograd scales what reaches the mean
    return {"loss": (loss.sum() * (w if op == "step" else 1.0 / loss.numel())).float(), "grad": (d * w).to(dt)}


# ---- the framework's calls ------------------------------------------------------------------

def _own(s):
    from azg_amd import policy
    op, c = s["case"]["op"], s["case"]
    mask = s["mask"]
    if op == "score":
        r = policy.action_logprobs(s["logits"], s["actions"], top=c["top"], mask=mask)
        out = {"logp": r.logp, "entropy": r.entropy, "lse": r.lse}
        if c["top"]:
            out["top_logp"], out["top_ids"] = r.top_logp, r.top_ids
        return out
    if op == "train":
        r = policy.action_logprobs(s["logits"], s["actions"], mask=mask)
        d, = torch.autograd.grad((r.logp, r.entropy), s["logits"], (s["g_logp"], s["g_entropy"]))
        return {"logp": r.logp.detach(), "entropy": r.entropy.detach(), "lse": r.lse.detach(), "grad": d}
    if op == "loss":
        return {"loss": policy.distill_loss(s["logits"], s["t_logp"], s["t_ids"], mask=mask, rest=c["rest"],
                                            reduction="none")}
    if op == "autograd":
        loss = policy.distill_loss(s["logits"], s["t_logp"], s["t_ids"], mask=mask, rest=c["rest"])
        d, = torch.autograd.grad(loss, s["logits"], s["g_loss"])
        return {"loss": loss.detach(), "grad": d}
    loss, d = policy.distill_loss_grad(s["logits"], s["t_logp"], s["t_ids"], mask=mask, rest=c["rest"],
                                       weight=LOSS_SCALE[c["dtype"]] / c["rows"])
    return {"loss": loss, "grad": d}


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits, row slices --------------------------------------------------

def _exact_rows(c, x, m, a, ga, ge, tl, ti):
    """x [n, V] f64 with the illegal entries in `m` (or None)"""
    ok = torch.ones_like(x, dtype=torch.bool) if m is None else m
    z = torch.where(ok, x, torch.full_like(x, -math.inf))
    lse = torch.logsumexp(z, 1)
    lp = z - lse[:, None]
    p = lp.exp()
    if c["op"] in ("score", "train"):
        h = -torch.special.xlogy(p, p).sum(1)
        r = {"logp": lp[torch.arange(len(x), device=x.device), a], "entropy": h, "lse": lse}
        if c["op"] == "train":
            d = ge[:, None] * (-p * (torch.where(ok, lp, 0.0) + h[:, None])) - ga[:, None] * p
            d[torch.arange(len(x), device=x.device), a] += ga
            r["grad"] = d
        elif c["top"]:
            v, i = torch.sort(z, dim=1, descending=True, stable=True)
            v, i = v[:, :c["top"]], i[:, :c["top"]]
            r["top_logp"] = v - lse[:, None]
            r["top_ids"] = torch.where(v == -math.inf, torch.full_like(i, -1), i)
        return r
    there = (ti >= 0) & (tl > -math.inf)
    q = torch.where(there, tl.exp(), 0.0)
    if not c["rest"]:
        q = q / q.sum(1, keepdim=True)
    tgt = torch.zeros_like(x)
    rest = ok.clone()
    rows = torch.arange(len(x), device=x.device)
    for j in range(ti.shape[1]):
        i = ti[:, j].clamp_min(0)
        tgt[rows, i] += q[:, j]
        rest[rows, i] &= ~there[:, j]
    loss = torch.special.xlogy(q, q).sum(1)
    loss -= torch.where(tgt > 0, tgt * lp, 0.0).sum(1)
    if c["rest"]:
        qr = (1.0 - q.sum(1)).clamp_min(0.0)
        pr = torch.where(rest, p, 0.0).sum(1)
        lpr = torch.logsumexp(torch.where(rest, lp, -math.inf), 1)
        has = (qr > 0) & (lpr > -math.inf)
        qr = torch.where(has, qr, 0.0)
        loss += torch.where(has, torch.special.xlogy(qr, qr) - qr * torch.where(has, lpr, 0.0), 0.0)
        tgt = tgt + torch.where(rest, p * (qr / torch.where(pr > 0, pr, 1.0))[:, None], 0.0)
        return {"loss": loss, "grad": p * (q.sum(1) + qr)[:, None] - tgt}
    return {"loss": loss, "grad": p - tgt}


def exact(case, seed):
    s = prepare(case, seed)
    x = s["logits"].detach()
    lead, n, vocab = x.shape[:-1], case["rows"], case["vocab"]
    step = max(1, (1 << 25) // vocab)
    at = [(i, j) for i in range(lead[0]) for j in range(lead[1])] if len(lead) == 2 else None
    acc = {}
    want_grad = case["op"] in ("train", "autograd", "step")

    def rows_of(t, r0, r1):
        return None if t is None else t.reshape(n, *t.shape[len(lead):])[r0:r1]

    for r0 in range(0, n, step):
        r1 = min(n, r0 + step)
        if at is None:
            xs = x[r0:r1].double()
        else:
            sel = torch.tensor(at[r0:r1], device=DEV)
            xs = x[sel[:, 0], sel[:, 1]].double()
        f64 = [None if t is None else rows_of(t, r0, r1).double() for t in
               (s.get("g_logp"), s.get("g_entropy"), s["t_logp"])]
        r = _exact_rows(case, xs, rows_of(s["mask"], r0, r1), rows_of(s["actions"], r0, r1), f64[0], f64[1], f64[2],
                        rows_of(s["t_ids"], r0, r1))
        if not want_grad:
            r.pop("grad", None)
        for k, v in r.items():
            acc.setdefault(k, []).append(v)
    out = {k: torch.cat(v).reshape(*lead, *v[0].shape[1:]) for k, v in acc.items()}
    if case["op"] in ("autograd", "step"):
        w = LOSS_SCALE[case["dtype"]] / n
        out = {"loss": out["loss"].sum() * (w if case["op"] == "step" else 1.0 / n), "grad": out["grad"] * w}
    return out


def work(case):
    n, v, k = case["rows"], case["vocab"], case["top"]
    e = 4 if case["dtype"] == "f32" else 2
    read = n * v * e + (n * v if case["legal"] else 0)
    op = case["op"]
    if op == "score":  # actions in; logp, entropy, lse and the alternatives out
        return {"bytes": read + n * (8 + 12) + n * k * 12, "flops": 7 * n * v}
    if op == "train":  # the same, what reaches logp and entropy, and the gradient
        return {"bytes": read + n * (8 + 12 + 8) + n * v * e, "flops": 13 * n * v}
    if op == "loss":
        return {"bytes": read + n * k * 12 + 4 * n, "flops": 4 * n * v}
    return {"bytes": read + n * k * 12 + 4 + n * v * e, "flops": 8 * n * v}


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(i)) for i in range(4)]:
        print(c, work(c))
