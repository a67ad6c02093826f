"""The operators at the vocabulary end of a model, as cases that can be timed and compared.

  top_logits  the k largest logits of every row, their ids and the row's log-sum-exp: what a teacher hands
              to a student (eisen_top_logits)
  distill     the distillation loss against a teacher's top logits, mixed with the cross-entropy of the
              targets, and its gradient (eisen_distill_fwd, eisen_distill_bwd, eisen_distill_fused)
  linear_ce   head projection and cross-entropy in pieces of the vocabulary, with no logits kept, and the
              gradients of the hidden states and of the head (eisen_linear_ce_fwd, eisen_linear_ce_bwd)

With `own` false the operators run in their plain form: elementary torch operations in 32 bits, rounded once.
With `own` true `run` calls the library.
"""
import math

import torch

own = False

IGNORE = -1
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _up8(n):
    return (n + 7) // 8 * 8


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the logits of one generated position, to be looked at: latency
        {"name": "top one position", "op": "top", "rows": 1, "vocab": 32000, "k": 8, "dtype": "f32", "temperature": 1.0},
        # a teacher's micro batch on its way to a student
        {"name": "top teacher batch", "op": "top", "rows": 4096, "vocab": 32000, "k": 64, "dtype": "bf16", "temperature": 2.0},
        # f32 logits over a vocabulary whose rows start anywhere
        {"name": "top odd f32", "op": "top", "rows": 777, "vocab": 50001, "k": 33, "dtype": "f32", "temperature": 1.0},
        # a tiny f32 model's step: latency
        {"name": "distill tiny f32", "op": "distill", "way": "fused", "rows": 63, "vocab": 1000, "k": 5, "dtype": "f32",
         "temperature": 1.0, "ce": 0.0, "full": False},
        # a training step's loss: 8 x 2048 tokens over 32000 words, temperature 2, half hard targets
        {"name": "distill step", "op": "distill", "way": "fused", "rows": 16384, "vocab": 32000, "k": 64, "dtype": "bf16",
         "temperature": 2.0, "ce": 0.5, "full": False},
        # a loss inside a larger graph: forward now, backward when its gradient is known; f32
        {"name": "distill tape f32", "op": "distill", "way": "fwd_bwd", "rows": 2048, "vocab": 32000, "k": 32, "dtype": "f32",
         "temperature": 1.0, "ce": 0.0, "full": True},
        # held-out loss over a large odd vocabulary
        {"name": "distill eval odd", "op": "distill", "way": "fwd", "rows": 1023, "vocab": 100003, "k": 128, "dtype": "bf16",
         "temperature": 3.5, "ce": 0.25, "full": True},
        # a few tokens scored by a small model: latency
        {"name": "linear_ce score few", "op": "linear", "way": "fwd", "rows": 5, "hidden": 384, "vocab": 8192, "tied": False},
        # held-out loss of the 2048-wide model on 8 x 2048 tokens
        {"name": "linear_ce eval", "op": "linear", "way": "fwd", "rows": 16384, "hidden": 2048, "vocab": 32000, "tied": False},
        # one sequence of training
        {"name": "linear_ce step 2048", "op": "linear", "way": "fwd_bwd", "rows": 2048, "hidden": 2048, "vocab": 32000, "tied": False},
        # ragged rows, tied table with an odd number of words
        {"name": "linear_ce odd tied", "op": "linear", "way": "fwd_bwd", "rows": 1021, "hidden": 1000, "vocab": 50001, "tied": True},
        # the whole training batch
        {"name": "linear_ce step 16384", "op": "linear", "way": "fwd_bwd", "rows": 16384, "hidden": 2048, "vocab": 32000, "tied": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["top", "distill", "linear"])
    if op == "linear":
        way = rng.choice(["fwd", "fwd_bwd"])
        hidden = 8 * _log_int(rng, 8, 256)
        vocab = _log_int(rng, 1000, 64000)
        rows = min(_log_int(rng, 1, 16384), 16384 * 2048 * 32000 // (hidden * vocab))
        return {"op": op, "way": way, "rows": rows, "hidden": hidden, "vocab": vocab, "tied": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "f32"])
    vocab = _log_int(rng, 1000, 131072)
    most = 4096 * 32000 if op == "top" else 16384 * 32000 // (2 if dtype == "f32" else 1)
    rows = min(_log_int(rng, 1, 16384), most // vocab)
    k = _log_int(rng, 1, 128)
    temperature = rng.choice([1.0, 1.5, 2.0, 3.5])
    if op == "top":
        return {"op": op, "rows": rows, "vocab": vocab, "k": k, "dtype": dtype, "temperature": temperature}
    return {"op": op, "way": rng.choice(["fwd", "fwd_bwd", "fused"]), "rows": rows, "vocab": vocab, "k": k, "dtype": dtype,
            "temperature": temperature, "ce": rng.choice([0.0, 0.25, 0.5]), "full": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------ inputs
def _targets(g, rows, vocab, dev):
    """Random targets; about one row in twenty is ignored."""
    t = torch.randint(0, vocab, (rows,), generator=g, device=dev, dtype=torch.int32)
    drop = torch.rand(rows, generator=g, device=dev) < 0.05
    drop[0] = False
    return torch.where(drop, torch.full_like(t, IGNORE), t), int(rows - drop.sum())


def prepare(case, seed):
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(seed)
    c, rows, vocab = case, case["rows"], case["vocab"]
    f32 = dict(dtype=torch.float32, device=dev)
    if c["op"] == "linear":
        d = c["hidden"]
        h = torch.randn(rows, d, generator=g, device=dev).to(torch.bfloat16)
        ld = d if c["tied"] else _up8(vocab)
        w = (torch.randn(vocab if c["tied"] else d, ld, generator=g, device=dev) * (2.0 / math.sqrt(d))).to(torch.bfloat16)
        targets, valid = _targets(g, rows, vocab, dev)
        s = dict(c, h=h, w=w, ldw=ld, targets=targets, norm=1.0 / valid, row_loss=torch.empty(rows, **f32),
                 lse=torch.empty(rows, **f32), loss=torch.empty((), **f32), status=torch.zeros(2, dtype=torch.int32, device=dev))
        if c["way"] != "fwd":
            s.update(dh=torch.empty_like(h), dw=torch.empty_like(w), grad=torch.full((), 0.5, **f32))
        return s
    dtype = DTYPES[c["dtype"]]
    base = torch.randn(rows, vocab, generator=g, device=dev) * 2.0
    logits = base.to(dtype)
    if c["op"] == "top":
        return dict(c, logits=logits, values=torch.empty(rows, c["k"], **f32), ids=torch.empty(rows, c["k"], dtype=torch.int32, device=dev),
                    lse=torch.empty(rows, **f32))
    # a teacher that mostly agrees with the student and is surer of itself
    k = c["k"]
    base = (base * 1.25).add_(torch.randn(rows, vocab, generator=g, device=dev))  # not in place: f32 logits are `base`
    t_lse = torch.logsumexp(base / c["temperature"], 1) if c["full"] else None
    t_values, t_ids = base.topk(k, 1)
    t_ids = t_ids.to(torch.int32)
    del base
    # some rows of the teacher are shorter than k, a few are empty
    have = torch.full((rows, 1), k, device=dev)
    u = torch.rand(rows, 1, generator=g, device=dev)
    have = torch.where(u < 0.2, (have * torch.rand(rows, 1, generator=g, device=dev)).ceil().long(), have)
    have = torch.where(u < 0.02, torch.zeros_like(have), have)
    have[0] = k
    t_ids = torch.where(torch.arange(k, device=dev) < have, t_ids, torch.full_like(t_ids, -1))
    targets, valid = _targets(g, rows, vocab, dev)
    s = dict(c, logits=logits, t_values=t_values.contiguous(), t_ids=t_ids.contiguous(), t_lse=t_lse, targets=targets,
             kd_weight=(1.0 - c["ce"]) / valid, ce_weight=c["ce"] / valid, row_loss=torch.empty(rows, **f32),
             lse=torch.empty(2, rows, **f32), loss=torch.empty((), **f32), status=torch.zeros(1, dtype=torch.int32, device=dev))
    if c["way"] != "fwd":
        s.update(dlogits=torch.empty_like(logits))
    if c["way"] == "fwd_bwd":
        s.update(grad=torch.full((), 0.5, **f32))
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _plain_lse(x):
    m = x.amax(1, keepdim=True)
    return (m + (x - m).exp_().sum(1, keepdim=True).log()).squeeze(1)


def _plain_top(s):
    x = s["logits"].float()
    values, ids = torch.sort(x, dim=1, descending=True, stable=True)  # equal values: the lowest index first
    return {"values": values[:, : s["k"]], "ids": ids[:, : s["k"]].to(torch.int32), "lse": _plain_lse(x * (1.0 / s["temperature"]))}


def _plain_distill(s):
    T, kd, ce = s["temperature"], s["kd_weight"], s["ce_weight"]
    x = s["logits"].float()
    targets = s["targets"].long()
    valid = targets != IGNORE
    at = targets.clamp(min=0)
    # the teacher's probabilities over the entries it gives
    here = s["t_ids"] >= 0
    ids = s["t_ids"].long().clamp(min=0)
    t = torch.where(here, s["t_values"] * (1.0 / T), -math.inf)
    if s["t_lse"] is not None:
        log_q = t - s["t_lse"][:, None]
    else:
        m = t.amax(1, keepdim=True)
        m = torch.where(m > -math.inf, m, 0.0)
        log_q = t - m - (t - m).exp().sum(1, keepdim=True).clamp(min=1e-30).log()
    q = log_q.exp()
    # the student
    lse1 = _plain_lse(x)
    lse_t = lse1 if T == 1.0 else _plain_lse(x * (1.0 / T))
    log_p = x.gather(1, ids) * (1.0 / T) - lse_t[:, None]
    kl = torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1)
    p_at = (x.gather(1, at[:, None])[:, 0] - lse1).exp()
    row_loss = torch.where(valid, kd * T * T * kl - ce * (p_at + 1e-8).log(), 0.0)
    keep = valid.float()
    out = {"loss": row_loss.sum(), "row_loss": row_loss}
    if s["way"] == "fwd":
        return dict(out, lse=torch.stack((lse_t, lse1)) * keep)
    g = s["grad"] if s["way"] == "fwd_bwd" else 1.0
    d = (x * (1.0 / T)).sub_(lse_t[:, None]).exp_().mul_((kd * T * q.sum(1) * keep)[:, None])
    d.scatter_add_(1, ids, -kd * T * q * keep[:, None])
    if ce:
        d.add_((x - lse1[:, None]).exp_().mul_((ce * keep)[:, None]))
        d.scatter_add_(1, at[:, None], -ce * keep[:, None])
    return dict(out, dlogits=d.mul_(g).to(s["logits"].dtype))


def _plain_linear(s):
    h, vocab = s["h"].float(), s["vocab"]
    w = s["w"].float().t() if s["tied"] else s["w"][:, :vocab].float()
    targets = s["targets"].long()
    valid = targets != IGNORE
    at = targets.clamp(min=0)[:, None]
    x = h @ w
    lse = _plain_lse(x)
    p_at = (x.gather(1, at)[:, 0] - lse).exp()
    row_loss = torch.where(valid, -s["norm"] * (p_at + 1e-8).log(), 0.0)
    out = {"loss": row_loss.sum(), "row_loss": row_loss, "lse": lse * valid}
    if s["way"] == "fwd":
        return out
    keep = valid.float()[:, None]
    d = x.sub_(lse[:, None]).exp_().scatter_add_(1, at, -torch.ones_like(keep)).mul_(keep).mul_(s["norm"] * s["grad"])
    dh, dw = d @ w.t(), h.t() @ d
    return dict(out, dh=dh.to(torch.bfloat16), dw=(dw.t() if s["tied"] else dw).to(torch.bfloat16))


# ------------------------------------------------------------------------------------------ the library
def _stream():
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return t.data_ptr() if t is not None else None


def _own_top(s):
    import eisen_b200 as eb

    x = s["logits"]
    eb.call("eisen_top_logits", _stream(), x.data_ptr(), s["vocab"], s["values"].data_ptr(), s["ids"].data_ptr(), s["lse"].data_ptr(),
            s["rows"], s["vocab"], s["k"], s["temperature"], eb.F32 if x.dtype == torch.float32 else eb.BF16)
    return {"values": s["values"], "ids": s["ids"], "lse": s["lse"]}


def _own_distill(s):
    import eisen_b200 as eb

    x, rows, vocab, k = s["logits"], s["rows"], s["vocab"], s["k"]
    dt = eb.F32 if x.dtype == torch.float32 else eb.BF16
    teacher = (s["t_ids"].data_ptr(), s["t_values"].data_ptr(), _p(s["t_lse"]), s["targets"].data_ptr())
    how = (IGNORE, s["temperature"], s["kd_weight"], s["ce_weight"])
    out = {"loss": s["loss"], "row_loss": s["row_loss"]}
    if s["way"] == "fused":
        eb.call("eisen_distill_fused", _stream(), x.data_ptr(), vocab, *teacher, s["dlogits"].data_ptr(), vocab, s["loss"].data_ptr(),
                s["row_loss"].data_ptr(), s["lse"].data_ptr(), rows, vocab, k, *how, 1.0, dt, s["status"].data_ptr())
        return dict(out, dlogits=s["dlogits"])
    eb.call("eisen_distill_fwd", _stream(), x.data_ptr(), vocab, *teacher, s["loss"].data_ptr(), s["row_loss"].data_ptr(),
            s["lse"].data_ptr(), rows, vocab, k, *how, dt, s["status"].data_ptr())
    if s["way"] == "fwd":
        return dict(out, lse=s["lse"])
    eb.call("eisen_distill_bwd", _stream(), x.data_ptr(), vocab, *teacher, s["lse"].data_ptr(), s["dlogits"].data_ptr(), vocab,
            s["grad"].data_ptr(), rows, vocab, k, *how, dt, 0)
    return dict(out, dlogits=s["dlogits"])


def _own_linear(s):
    import eisen_b200 as eb

    rows, d, vocab, tied = s["rows"], s["hidden"], s["vocab"], 1 if s["tied"] else 0
    if "ws" not in s:  # a workspace is kept from call to call
        s["ws"] = torch.empty(eb.lib().eisen_linear_ce_workspace_bytes(rows, d, vocab, 0, 1 if "dh" in s else 0),
                              dtype=torch.uint8, device=s["h"].device)
    ops = (s["h"].data_ptr(), d, s["w"].data_ptr(), s["ldw"], tied, s["targets"].data_ptr())
    eb.call("eisen_linear_ce_fwd", _stream(), *ops, s["loss"].data_ptr(), s["row_loss"].data_ptr(), s["lse"].data_ptr(),
            s["ws"].data_ptr(), rows, d, vocab, IGNORE, s["norm"], s["status"].data_ptr() + 4, s["status"].data_ptr())
    out = {"loss": s["loss"], "row_loss": s["row_loss"], "lse": s["lse"]}
    if s["way"] == "fwd":
        return out
    eb.call("eisen_linear_ce_bwd", _stream(), *ops, s["lse"].data_ptr(), s["grad"].data_ptr(), s["dh"].data_ptr(), 0, s["dw"].data_ptr(),
            s["ldw"], eb.BF16, 0, s["ws"].data_ptr(), rows, d, vocab, 0, IGNORE, s["norm"], s["status"].data_ptr())
    return dict(out, dh=s["dh"], dw=s["dw"] if tied else s["dw"][:, :vocab])


def run(state):
    if own:
        return {"top": _own_top, "distill": _own_distill, "linear": _own_linear}[state["op"]](state)
    return {"top": _plain_top, "distill": _plain_distill, "linear": _plain_linear}[state["op"]](state)


# ------------------------------------------------------------------------------------------ work and exact values
def work(case):
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "linear":
        d, back = case["hidden"], case["way"] != "fwd"
        bytes_ = 2 * (rows * d + d * vocab) * (2 if back else 1) + 12 * rows
        return {"bytes": bytes_, "flops": (6 if back else 2) * rows * d * vocab}
    size, k = 2 if case["dtype"] == "bf16" else 4, case["k"]
    if case["op"] == "top":
        return {"bytes": rows * (vocab * size + 8 * k + 4), "flops": 4 * rows * vocab}
    passes = 1 if case["way"] == "fwd" else 2
    return {"bytes": rows * (passes * vocab * size + 8 * k + 16), "flops": rows * vocab * (4 + 4 * (passes - 1))}


def _no_pad(dw, s):
    return dw if s["tied"] else dw[:, : s["vocab"]]


def exact(case, seed):
    s = prepare(case, seed)
    T = s.get("temperature", 1.0)
    if s["op"] == "top":
        x = s["logits"].double()
        order = torch.argsort(-x, dim=1, stable=True)[:, : s["k"]]
        return {"values": torch.gather(x, 1, order), "ids": order.to(torch.int32), "lse": torch.logsumexp(x / T, 1)}
    counted = s["targets"] >= 0
    rows = torch.arange(s["rows"], device=counted.device)[counted]
    label = s["targets"][counted].long()
    if s["op"] == "linear":
        back = s["way"] != "fwd"
        h, w = s["h"].double().requires_grad_(back), s["w"].double().requires_grad_(back)
        logits = h[counted] @ (w.T if s["tied"] else w[:, : s["vocab"]])
        lse = torch.logsumexp(logits, 1)
        log_p = logits[torch.arange(len(label), device=label.device), label] - lse
        got = {"loss": None, "row_loss": torch.zeros(s["rows"], dtype=torch.float64, device=h.device), "lse": None}
        got["row_loss"][rows] = -s["norm"] * torch.log(log_p.detach().exp() + 1e-8)
        got["lse"] = torch.zeros_like(got["row_loss"]).index_copy_(0, rows, lse.detach())
        got["loss"] = got["row_loss"].sum()
        if back:  # the 1e-8 takes no part in the gradient
            dh, dw = torch.autograd.grad(-s["norm"] * 0.5 * log_p.sum(), (h, w))
            got.update(dh=dh, dw=_no_pad(dw, s))
        return got
    back = s["way"] != "fwd"
    x = s["logits"].double().requires_grad_(back)
    soft, hard = torch.log_softmax(x[counted] / T, 1), None
    teacher = s["t_values"][counted].double() / T
    there = s["t_ids"][counted] >= 0
    teacher = teacher.masked_fill(~there, -math.inf)
    total = s["t_lse"][counted].double() if s["full"] else torch.logsumexp(teacher, 1)
    q = torch.exp(teacher - total[:, None]).masked_fill(~there, 0.0)
    log_q = torch.where(there, teacher - total[:, None], 0.0)
    log_p = torch.gather(soft, 1, s["t_ids"][counted].long() * there)
    kd = T * T * (q * (log_q - log_p) * there).sum(1)
    hard = torch.log_softmax(x[counted], 1) if s["ce"] else soft
    log_at = hard[torch.arange(len(label), device=label.device), label]
    value = torch.zeros(s["rows"], dtype=torch.float64, device=x.device)
    value[rows] = s["kd_weight"] * kd.detach() - s["ce_weight"] * torch.log(log_at.detach().exp() + 1e-8)
    got = {"loss": value.sum(), "row_loss": value}
    if not back:
        lse = torch.stack((torch.logsumexp(x / T, 1), torch.logsumexp(x, 1)))
        return dict(got, lse=lse * counted)
    scalar = (s["kd_weight"] * kd).sum() - (s["ce_weight"] * log_at.sum() if s["ce"] else 0.0)
    (dx,) = torch.autograd.grad(scalar * (0.5 if s["way"] == "fwd_bwd" else 1.0), x)
    return dict(got, dlogits=dx)
