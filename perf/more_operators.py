"""The operators on rows of logits as workloads: what is timed, on which sizes, and their plain forms.

Four operators on what an lm_head answers with, rows of V logits:

  sample       ops.sample: a token a row from a given uniform number, with temperature, top-k, top-p, min-p
  topk         ops.topk: the k largest logits of a row with their ids, and the row's log-sum-exp
  speculative  ops.speculative_sample: which drafted tokens stand, and the token after them
  distill      ops.distill_loss / ops.distill_loss_and_grad: divergence from a teacher's top logits, gradient

sample.  w_i = exp((l_i - max l) / T); the tokens in the order of (logit descending, id ascending); kept are
the first top_k of them; of these, as long as the mass before a token is below top_p times theirs; and those
with w_i >= min_p.  The answer is the first id, in the order of ids, at which the kept weights add up to more
than u times their sum.  T = 0 is the lowest id of the largest logit.  An infinite negative logit is a masked
token and never drawn.

speculative.  With p = softmax(logits / T) and q = softmax(draft_logits / T_d) position by position, drafted
token d_i stands while u_i q_i(d_i) < p_i(d_i).  At the first that does not, a token is drawn (as above, from
the last uniform number) from max(p - q, 0); where the draft ends (an id below zero, or no further column),
from p.

distill.  p are the teacher's top entries, renormalised, or with the teacher's log-sum-exp taken as they are
and the rest of its mass as one more class; q = softmax(logits / t); the loss is KL(p || q) of a row.

With ``own`` false, ``run`` computes the plain form in elementary torch operations; with ``own`` true it calls
the package.  ``exact`` computes the definition in 64 bits.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one decoded token with a usual setting of all filters: latency counts
        {"name": "sample_decode", "op": "sample", "rows": 1, "v": 248320, "dtype": "bf16", "t": 0.6, "top_k": 20,
         "top_p": 0.95, "min_p": 0.0, "per_row": False},
        # requests of one serving batch, each with its own setting, over an odd vocabulary
        {"name": "sample_mixed", "op": "sample", "rows": 65, "v": 50021, "dtype": "f16", "t": 0.8, "top_k": 50,
         "top_p": 0.9, "min_p": 0.02, "per_row": True},
        # a batch with nucleus sampling alone
        {"name": "sample_nucleus", "op": "sample", "rows": 128, "v": 248320, "dtype": "bf16", "t": 1.0, "top_k": 0,
         "top_p": 0.95, "min_p": 0.0, "per_row": False},
        # a large batch of rollouts from the whole distribution, logits in 32 bits
        {"name": "sample_rollout", "op": "sample", "rows": 512, "v": 248320, "dtype": "f32", "t": 1.0, "top_k": 0,
         "top_p": 1.0, "min_p": 0.0, "per_row": False},
        # candidates of a verify window's five positions
        {"name": "topk_verify", "op": "topk", "rows": 5, "v": 248320, "k": 20, "dtype": "bf16", "lse": False},
        # a teacher's lists for distillation, a chunk of a long prompt
        {"name": "topk_teacher", "op": "topk", "rows": 2011, "v": 248320, "k": 64, "dtype": "bf16", "lse": True},
        # one sequence with four drafted tokens: latency counts
        {"name": "speculative_one", "op": "speculative", "seqs": 1, "n": 4, "v": 248320, "dtype": "bf16", "t": 0.7},
        # a serving batch, drafts of up to three tokens
        {"name": "speculative_batch", "op": "speculative", "seqs": 48, "n": 3, "v": 248320, "dtype": "bf16", "t": 1.0},
        # a quantised model's divergence from its teacher, a short evaluation text: no gradient
        {"name": "distill_measure", "op": "distill", "rows": 333, "v": 248320, "k": 64, "dtype": "bf16", "lse": True,
         "mode": "loss"},
        # a small training step in 32 bits, through autograd
        {"name": "distill_small", "op": "distill", "rows": 127, "v": 32001, "k": 20, "dtype": "f32", "lse": False,
         "mode": "autograd"},
        # a training step of a draft head through autograd
        {"name": "distill_train", "op": "distill", "rows": 1024, "v": 248320, "k": 64, "dtype": "bf16", "lse": False,
         "mode": "autograd"},
        # the same in chunks of rows, loss and gradient in one call, the rest of the teacher's mass counted
        {"name": "distill_chunk", "op": "distill", "rows": 2048, "v": 248320, "k": 128, "dtype": "bf16", "lse": True,
         "mode": "fused"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "topk", "speculative", "distill", "distill"])
    v = rng.choice([248320, _log(rng, 1000, 248320)])
    case = {"op": op, "v": v, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "sample":
        return {**case, "rows": min(_log(rng, 1, 2048), (512 * 248320) // (2 * v)),
                "t": rng.choice([0.0, rng.uniform(0.3, 1.3), rng.uniform(0.3, 1.3)]),
                "top_k": rng.choice([0, 1, _log(rng, 2, 1000), _log(rng, 2, v)]),
                "top_p": rng.choice([1.0, rng.uniform(0.5, 0.99)]),
                "min_p": rng.choice([0.0, 0.0, rng.uniform(0.01, 0.3)]), "per_row": rng.random() < 0.5}
    if op == "topk":
        return {**case, "rows": min(_log(rng, 1, 4096), (1024 * 248320) // v), "k": _log(rng, 1, 256),
                "lse": rng.random() < 0.5}
    if op == "speculative":
        n = rng.randint(1, 8)
        return {**case, "seqs": min(_log(rng, 1, 128), max(1, (360 * 248320) // ((2 * n + 1) * v))), "n": n,
                "t": rng.uniform(0.5, 1.2)}
    return {**case, "rows": min(_log(rng, 1, 4096), (1024 * 248320) // v), "k": _log(rng, 1, 256),
            "lse": rng.random() < 0.5, "mode": rng.choice(["loss", "autograd", "fused"])}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _logits(gen, rows, v):
    """fp32 logits [rows, v]: a bulk of unlikely tokens and some dozens that stand out, by how much differs
    from row to row (certain answers, open ones)."""
    x = torch.randn((rows, v), generator=gen, device="cuda") * 1.8
    n = min(32, v)
    at = torch.randint(0, v, (rows, n), generator=gen, device="cuda")
    height = 15.0 - 7.0 * torch.rand((rows, 1), generator=gen, device="cuda") ** 2
    x.scatter_(1, at, height + 2.5 * torch.randn((rows, n), generator=gen, device="cuda"))
    return x


def _filled(rows, v, dt, make):
    """[rows, v] of type dt, made in parts of rows so that the 32-bit form is never whole."""
    out = torch.empty((rows, v), dtype=dt, device="cuda")
    for r in range(0, rows, 256):
        out[r:r + 256] = make(min(256, rows - r), r)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, op, v = _DT[case["dtype"]], case["op"], case["v"]
    s = {"case": case, "dtype": dt}
    if op == "sample":
        rows = case["rows"]
        s["logits"] = _filled(rows, v, dt, lambda n, r: _logits(gen, n, v))
        s["u"] = torch.rand(rows, generator=gen, device="cuda")
        s["kw"] = {"temperature": case["t"], "top_k": case["top_k"], "top_p": case["top_p"], "min_p": case["min_p"]}
        if case["per_row"]:
            # every request brings its own numbers; some have a filter switched off
            f = torch.rand((4, rows), generator=gen, device="cuda")
            s["kw"] = {
                "temperature": case["t"] * (0.8 + 0.4 * f[0]),
                "top_k": torch.where(f[1] < 0.2, 0.0, case["top_k"] * 2 * f[1]).to(torch.int32),
                "top_p": (case["top_p"] + (1 - case["top_p"]) * 2 * f[2]).clamp_max(1.0),
                "min_p": case["min_p"] * 2 * f[3],
            }
        return s
    if op == "topk":
        s["logits"] = _filled(case["rows"], v, dt, lambda n, r: _logits(gen, n, v))
        return s
    if op == "speculative":
        B, n = case["seqs"], case["n"]
        s["logits"] = torch.empty((B, n + 1, v), dtype=dt, device="cuda")
        s["draft_logits"] = torch.empty((B, n, v), dtype=dt, device="cuda")
        s["draft_ids"] = torch.empty((B, n), dtype=torch.int64, device="cuda")
        for b in range(B):
            x = _logits(gen, n + 1, v)
            s["logits"][b] = x
            y = (0.95 * x[:n] + 0.7 * torch.randn((n, v), generator=gen, device="cuda")).to(dt)
            s["draft_logits"][b] = y
            noise = torch.rand((n, v), generator=gen, device="cuda").clamp(1e-20, 1 - 1e-7)
            s["draft_ids"][b] = (y.float() / case["t"] - torch.log(-torch.log(noise))).argmax(-1)
        if B > 1:  # some drafts are shorter
            keep = torch.randint(0, n + 1, (B,), generator=gen, device="cuda")
            keep = torch.where(torch.rand(B, generator=gen, device="cuda") < 0.75, n, keep)
            s["draft_ids"][torch.arange(n, device="cuda") >= keep[:, None]] = -1
        s["u"] = torch.rand((B, n + 1), generator=gen, device="cuda")
        return s
    rows, k = case["rows"], case["k"]
    s["tv"] = torch.empty((rows, k), dtype=dt, device="cuda")
    s["ti"] = torch.empty((rows, k), dtype=torch.int64, device="cuda")
    s["lse"] = torch.empty(rows, device="cuda") if case["lse"] else None

    def student(n, r):
        x = _logits(gen, n, v).to(dt).float()  # the teacher's
        t, i = x.topk(k, dim=-1)
        s["tv"][r:r + n], s["ti"][r:r + n] = t, i
        if case["lse"]:
            s["lse"][r:r + n] = torch.logsumexp(x, -1)
        return x + 0.5 * torch.randn(x.shape, generator=gen, device="cuda")

    s["logits"] = _filled(rows, v, dt, student)
    s["weight"] = torch.full((rows,), 1.0, device="cuda")
    s["weight"][torch.rand(rows, generator=gen, device="cuda") < 0.1] = 0.0  # rows of a prompt carry no loss
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------

def _first_above(weights, u):
    """The first place along the last axis where the cumulated weights pass u times their sum."""
    cum = weights.cumsum(-1)
    at = (cum > u.double().unsqueeze(-1) * cum[..., -1:]).to(torch.int8).argmax(-1)
    return at


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    l = logits.double()  # a token is drawn where a sum of V weights passes a number: 64 bits
    best, first = l.max(-1)
    col = [x if torch.is_tensor(x) else torch.full_like(u, x, dtype=torch.float64)
           for x in (temperature, top_k, top_p, min_p)]
    T, K, P, M = (x.double().unsqueeze(-1) for x in col)
    w = torch.exp((l - best.unsqueeze(-1)) / torch.where(T > 0, T, 1.0))
    if not (torch.is_tensor(top_k) or torch.is_tensor(top_p)) and top_k == 0 and top_p >= 1:
        keep = w >= M
    else:
        order = l.sort(dim=-1, descending=True, stable=True).indices
        ws = w.gather(-1, order)
        rank = torch.arange(l.shape[-1], device=l.device)
        ks = (K <= 0) | (rank < K)
        ws = torch.where(ks, ws, 0.0)
        cum = ws.cumsum(-1)
        ks &= (P >= 1) | (cum - ws < P * cum[..., -1:])
        ks &= ws >= M
        keep = torch.empty_like(ks).scatter_(-1, order, ks)
    ids = _first_above(torch.where(keep, w, 0.0), u)
    return torch.where(T.squeeze(-1) > 0, ids, first)


def _plain_speculative(s):
    T, ids = s["case"]["t"], s["draft_ids"]
    p = torch.softmax(s["logits"].double() / T, -1)
    q = torch.softmax(s["draft_logits"].double() / T, -1)
    n = ids.shape[1]
    at = ids.clamp_min(0).unsqueeze(-1)
    stands = (ids >= 0) & (s["u"][:, :n].double() * q.gather(-1, at).squeeze(-1)
                           < p[:, :n].gather(-1, at).squeeze(-1))
    accepted = stands.to(torch.int64).cumprod(-1).sum(-1)
    b = torch.arange(ids.shape[0], device=ids.device)
    last = p[b, accepted]
    drafted = (accepted < n) & (ids[b, accepted.clamp_max(n - 1)] >= 0)
    rest = torch.where(drafted.unsqueeze(-1), (last - q[b, accepted.clamp_max(n - 1)]).clamp_min(0), last)
    token = _first_above(rest, s["u"][:, n])
    pos = torch.arange(n + 1, device=ids.device)
    out = torch.where(pos < accepted.unsqueeze(-1), torch.nn.functional.pad(ids, (0, 1), value=-1), -1)
    out[b, accepted] = token
    return {"tokens": out, "accepted": accepted}


def _plain_distill(s, rows, grad):
    """(loss, gradient or None) of a range of rows, in 32 bits; sums over a row's list in 64."""
    x, ti = s["logits"][rows].float(), s["ti"][rows]
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    z = e.sum(-1, keepdim=True)
    logq = (x.gather(-1, ti) - torch.log(z)).double()
    tv = s["tv"][rows].double()
    if s["lse"] is None:
        logp = tv - torch.logsumexp(tv, -1, keepdim=True)
    else:
        logp = tv - s["lse"][rows].double().unsqueeze(-1)
    p = torch.exp(logp)
    loss = (p * (logp - logq)).sum(-1)
    a = None
    if s["lse"] is not None:
        rest = (1 - p.sum(-1)).clamp_min(0)
        # without the listed entries: a difference of sums would lose what is small
        other = (e.scatter(-1, ti, 0.0).sum(-1) / z.squeeze(-1)).double()
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - torch.log(other)), 0.0)
        a = (1 - rest / other).float().unsqueeze(-1)
    if not grad:
        return loss.float(), None
    g = e / z
    top = g.gather(-1, ti) - p.float()
    if a is not None:
        g = g * a
    g = g.scatter(-1, ti, top) * s["weight"][rows].unsqueeze(-1)
    return loss.float(), g.to(s["dtype"])


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "sample":
        return {"ids": _plain_sample(s["logits"], s["u"], **s["kw"])}
    if op == "topk":
        # equal values in the order of ids
        order = s["logits"].float().sort(dim=-1, descending=True, stable=True).indices[:, :case["k"]]
        out = {"values": s["logits"].gather(-1, order), "ids": order}
        if case["lse"]:
            x = s["logits"].float()
            m = x.amax(-1, keepdim=True)
            out["lse"] = m.squeeze(-1) + torch.log(torch.exp(x - m).sum(-1))
        return out
    if op == "speculative":
        return _plain_speculative(s)
    parts = [_plain_distill(s, slice(r, r + 512), case["mode"] != "loss") for r in range(0, case["rows"], 512)]
    out = {"loss": torch.cat([p[0] for p in parts])}
    if case["mode"] != "loss":
        out["grad"] = torch.cat([p[1] for p in parts])
    return out


def _own(s):
    from mlxturbo_b200 import ops

    case, op = s["case"], s["case"]["op"]
    if op == "sample":
        return {"ids": ops.sample(s["logits"], s["u"], **s["kw"])}
    if op == "topk":
        got = ops.topk(s["logits"], case["k"], logsumexp=case["lse"])
        return dict(zip(("values", "ids", "lse"), got))
    if op == "speculative":
        tokens, accepted = ops.speculative_sample(s["logits"], s["draft_logits"], s["draft_ids"], s["u"],
                                                  temperature=case["t"])
        return {"tokens": tokens, "accepted": accepted}
    if case["mode"] == "loss":
        return {"loss": ops.distill_loss(s["logits"], s["tv"], s["ti"], teacher_logsumexp=s["lse"])}
    if case["mode"] == "autograd":
        x = s["logits"].detach().requires_grad_()
        loss = ops.distill_loss(x, s["tv"], s["ti"], teacher_logsumexp=s["lse"])
        return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, x, s["weight"])[0]}
    loss, grad = ops.distill_loss_and_grad(s["logits"], s["tv"], s["ti"], s["weight"], teacher_logsumexp=s["lse"])
    return {"loss": loss, "grad": grad}


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------

def work(case):
    op, v, size = case["op"], case["v"], 4 if case["dtype"] == "f32" else 2
    if op == "sample":  # difference, exponential and sum of a logit
        return {"bytes": case["rows"] * (v * size + 12), "flops": 3 * case["rows"] * v}
    if op == "topk":  # one comparison of a logit, the sum's three operations
        return {"bytes": case["rows"] * (v * size + case["k"] * (size + 8)),
                "flops": case["rows"] * v * (4 if case["lse"] else 1)}
    if op == "speculative":
        rows = case["seqs"] * (2 * case["n"] + 1)
        return {"bytes": rows * v * size + case["seqs"] * (case["n"] + 1) * 24, "flops": 3 * rows * v}
    n = case["rows"] * v
    grad = case["mode"] != "loss"
    return {"bytes": n * size * (2 if grad else 1) + case["rows"] * (case["k"] * (size + 8) + 12),
            "flops": n * (5 if grad else 3)}


# --------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------

def _exact_draw(w, u):
    """The first index whose running sum exceeds u * total; one row on the host."""
    cum = np.cumsum(w)
    return int(np.searchsorted(cum, float(u) * cum[-1], side="right"))


def _exact_sample(s):
    case, rows = s["case"], s["case"]["rows"]
    if rows * case["v"] > 40_000_000:
        return None
    row = {n: (x.double().cpu().numpy() if torch.is_tensor(x) else [x] * rows) for n, x in s["kw"].items()}
    u = s["u"].double().cpu().numpy()
    ids = []
    for r in range(rows):
        l = s["logits"][r].double().cpu().numpy()
        T, k, top_p, min_p = (float(row[n][r]) for n in ("temperature", "top_k", "top_p", "min_p"))
        if T <= 0:
            ids.append(int(l.argmax()))
            continue
        order = np.argsort(-l, kind="stable")
        w = np.exp((l[order] - l[order[0]]) / T)
        n = len(w) if k <= 0 else min(int(k), len(w))
        if top_p < 1:
            before = np.concatenate([[0.0], np.cumsum(w[:n])])
            n = int(np.searchsorted(before[:n], top_p * before[n], side="left"))
        n = min(n, int((w >= min_p).sum()))
        kept = np.zeros_like(l)
        kept[order[:n]] = w[:n]
        ids.append(_exact_draw(kept, u[r]))
    return {"ids": torch.tensor(ids, device="cuda")}


def _exact_speculative(s):
    case = s["case"]
    B, n, T = case["seqs"], case["n"], case["t"]
    if B * (2 * n + 1) * case["v"] > 100_000_000:
        return None
    tokens = torch.full((B, n + 1), -1, dtype=torch.int64)
    accepted = torch.zeros(B, dtype=torch.int64)
    ids, u = s["draft_ids"].tolist(), s["u"].double().tolist()

    def prob(row):
        w = row.double().cpu().numpy() / T
        w = np.exp(w - w.max())
        return w / w.sum()

    for b in range(B):
        j, rest = 0, None
        while j < n and ids[b][j] >= 0:
            p, q, d = prob(s["logits"][b, j]), prob(s["draft_logits"][b, j]), ids[b][j]
            if not u[b][j] < p[d] / q[d]:
                rest = np.maximum(p - q, 0.0)
                break
            tokens[b, j] = d
            j += 1
        if rest is None:
            rest = prob(s["logits"][b, j])
        tokens[b, j] = _exact_draw(rest, u[b][n])
        accepted[b] = j
    return {"tokens": tokens.cuda(), "accepted": accepted.cuda()}


def _exact_distill(s):
    case = s["case"]
    loss, grads = [], []
    for r in range(0, case["rows"], 128):
        rows = slice(r, r + 128)
        logq = torch.log_softmax(s["logits"][rows].double(), -1)
        tv, ti = s["tv"][rows].double(), s["ti"][rows]
        p = torch.softmax(tv, -1) if s["lse"] is None else torch.exp(tv - s["lse"][rows].double()[:, None])
        one = torch.zeros_like(logq).scatter_(-1, ti, 1.0)
        dense = torch.zeros_like(logq).scatter_(-1, ti, p)
        L = torch.special.xlogy(p, p).sum(-1) - (dense * logq).sum(-1)
        q = logq.exp()
        factor = torch.ones_like(L)
        if s["lse"] is not None:
            rest, other = (1 - p.sum(-1)).clamp_min(0), (q * (1 - one)).sum(-1)
            L = L + torch.special.xlogy(rest, rest / other)
            factor = 1 - rest / other
        loss.append(L)
        if case["mode"] != "loss":
            g = torch.where(one > 0, q - dense, q * factor[:, None]) * s["weight"][rows].double()[:, None]
            grads.append(g)
    out = {"loss": torch.cat(loss)}
    if case["mode"] != "loss":
        out["grad"] = torch.cat(grads)
    return out


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "sample":
        return _exact_sample(s)
    if op == "speculative":
        return _exact_speculative(s)
    if op == "distill":
        # two 64-bit gradients of the larger cases would not fit beside the outputs
        return _exact_distill(s) if case["rows"] * case["v"] <= 300_000_000 else None
    x = s["logits"].double()
    ids = torch.empty((case["rows"], case["k"]), dtype=torch.int64, device="cuda")
    for r in range(case["rows"]):
        cut = x[r].topk(case["k"]).values[-1]
        at = (x[r] >= cut).nonzero().squeeze(-1)  # in the order of ids
        ids[r] = at[x[r, at].sort(descending=True, stable=True).indices][:case["k"]]
    out = {"values": x.gather(-1, ids), "ids": ids}
    if case["lse"]:
        out["lse"] = torch.logsumexp(x, -1)
    return out
