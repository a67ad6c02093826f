"""The operators at the vocabulary end (top logits, distillation, cross-entropy without logits) against plain
64-bit evaluations of their formulas.

Error bounds are per element and follow the arithmetic.  A sum of n terms of one sign, added in 32 bits in chains of
at most c, is off by at most c * 2^-24 of itself; an exponential by 2^-21 plus 2^-24 of its argument's size; a bf16
result by 2^-8 of itself (half a step).
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import eisen_b200 as eb  # noqa: E402

DT = {torch.float32: eb.F32, torch.bfloat16: eb.BF16}
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
EPS_P = 2.0 ** -15  # relative error of a probability: a log-sum-exp over chains of up to 256 sums, and its own exponential


def dev():
    return torch.device("cuda:0")


def stream():
    return torch.cuda.current_stream().cuda_stream


def P(t):
    return t.data_ptr() if t is not None else None


def rows_at(x, ld, shift=0):
    """`x` in a buffer with row stride ld, starting `shift` elements behind an aligned address."""
    rows, n = x.shape
    buf = torch.zeros(rows * ld + shift + 16, dtype=x.dtype, device=x.device)
    view = buf[shift:shift + rows * ld].view(rows, ld)[:, :n] if rows else buf[:0].view(0, n)
    view.copy_(x)
    return view


def gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


# ------------------------------------------------------------------------------------------ top logits
def top(x, k, temperature=1.0, lse=True):
    rows, vocab = x.shape
    v = torch.full((rows, k), -7.0, device=dev())
    i = torch.full((rows, k), -7, dtype=torch.int32, device=dev())
    s = torch.full((rows,), -7.0, device=dev()) if lse else None
    eb.call("eisen_top_logits", stream(), P(x), x.stride(0), P(v), P(i), P(s), rows, vocab, k, temperature, DT[x.dtype])
    return v, i, s


def check_top(x, k, temperature=1.0):
    v, i, s = top(x, k, temperature)
    d = x.double()
    key = torch.where(torch.isnan(d), torch.full_like(d, math.inf), d) + 0.0
    nan_first = torch.argsort(torch.isnan(d).to(torch.int8), dim=1, descending=True, stable=True)
    order = nan_first.gather(1, torch.argsort(key.gather(1, nan_first), dim=1, descending=True, stable=True))[:, :k]
    # NaN above +inf: both have the key +inf and NaN comes first in the stable order
    assert torch.equal(i.long(), order)
    want = d.gather(1, order)
    assert torch.equal(torch.nan_to_num(v.double(), nan=1e300), torch.nan_to_num(want, nan=1e300))
    lse = torch.logsumexp(d / temperature, 1)
    assert (torch.isnan(lse) == torch.isnan(s)).all() and ((lse == math.inf) == (s == math.inf)).all()
    ok = torch.isfinite(lse)
    assert ((s.double() - lse)[ok].abs() <= EPS_P + 4 * 2.0 ** -24 * lse[ok].abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 255, 255), (9, 1000, 1), (4, 1001, 256),
                                          (33, 8192, 50), (2, 32000, 64), (1, 65536, 8), (3, 100003, 129), (2, 262144, 256)])
def test_top_logits(dtype, rows, vocab, k):
    x = torch.randn(rows, vocab, generator=gen(rows * 31 + vocab + k), device=dev()).to(dtype)
    check_top(x, k, 1.0 + (k % 3))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["constant", "two values", "ascending", "descending", "zeros of both signs", "one column block",
                                  "mostly -inf", "all -inf", "nan and inf", "lowest"])
def test_top_logits_orders(dtype, kind):
    rows, vocab, k = 3, 5003, 67
    at = torch.arange(vocab, device=dev(), dtype=torch.float32)
    x = torch.randn(rows, vocab, generator=gen(5), device=dev())
    if kind == "constant":
        x = torch.full((rows, vocab), 1.5, device=dev())
    elif kind == "two values":
        x = (x > 1.0).float()
    elif kind == "ascending":
        x = (at / 64).floor().expand(rows, -1).clone()
    elif kind == "descending":
        x = -at.expand(rows, -1).clone()
    elif kind == "zeros of both signs":
        x = torch.where(x > 0, torch.tensor(0.0, device=dev()), torch.tensor(-0.0, device=dev())) - 0.0 * at
        x[:, 4000:4010] = 1.0
    elif kind == "one column block":  # all large values with one thread's neighbourhood
        x = torch.where((at >= 1024) & (at < 1104), x + 50.0, x)
    elif kind == "mostly -inf":
        x[:, 20:] = -math.inf
    elif kind == "all -inf":
        x[:] = -math.inf
        v, i, s = top(x.to(dtype), k)
        assert torch.equal(i, torch.arange(k, device=dev(), dtype=torch.int32).expand(rows, -1)) and (v == -math.inf).all()
        assert (s == -math.inf).all()
        return
    elif kind == "nan and inf":
        x[0, 17], x[0, 4999], x[1, 3], x[1, 4], x[2, 100] = math.nan, math.nan, math.inf, math.inf, -math.inf
        x[0, 5] = math.inf
    elif kind == "lowest":
        x[:, 10:] = torch.finfo(dtype).min
    check_top(x.to(dtype), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ld,shift", [(1003, 0), (1008, 1), (1005, 3), (1016, 8)])
def test_top_logits_strides(dtype, ld, shift):
    x = torch.randn(6, 1003, generator=gen(ld), device=dev()).to(dtype)
    check_top(rows_at(x, ld, shift), 17, 2.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,k", [(1500, 700, 5), (1200, 1001, 32), (900, 2000, 200), (700, 8200, 64), (601, 5003, 256), (500, 32000, 64),
                                          (400, 32000, 256), (333, 100003, 20), (310, 300, 300 - 44)])
def test_top_logits_many_rows(dtype, rows, vocab, k):
    """Several rows per CTA; every third row constant, every fifth ascending."""
    x = torch.randn(rows, vocab, generator=gen(rows + vocab + k), device=dev()) * 2
    x[::3] = x[::3, :1]
    x[::5] = (torch.arange(vocab, device=dev()) // 3).float()
    check_top(x.to(dtype), k, 1.5)


@pytest.mark.parametrize("dtype,vocab", [(torch.bfloat16, 131056), (torch.bfloat16, 131065), (torch.bfloat16, 131072), (torch.bfloat16, 131073),
                                         (torch.float32, 65528), (torch.float32, 65533), (torch.float32, 65537), (torch.float32, 99999)])
@pytest.mark.parametrize("shift", [0, 1])
def test_top_logits_around_the_longest_noted_row(dtype, vocab, shift):
    """Rows in numbers, with as many vectors as are noted one by one, and a few more or less."""
    x = torch.randn(300, vocab, generator=gen(vocab), device=dev()).to(dtype)
    check_top(rows_at(x, vocab, shift), 9)


def test_top_logits_longer_than_shared_memory():
    x = torch.randn(2, 700001, generator=gen(2), device=dev())
    x[1, 5000:6000] = 9.0
    check_top(x, 100, 2.0)
    check_top(x.to(torch.bfloat16), 256)


def test_top_logits_no_rows_no_lse():
    x = torch.randn(0, 100, device=dev())
    top(x, 5)
    y = torch.randn(3, 100, generator=gen(1), device=dev())
    v, i, _ = top(y, 5, lse=False)
    assert torch.equal(v, y.topk(5, 1).values)


# ------------------------------------------------------------------------------------------ distillation
class Case:
    """Inputs of a distillation and what the formula gives for them in 64 bits."""

    def __init__(self, dtype, rows, vocab, k, temperature=1.0, kd=0.7, ce=0.3, full=False, ignored=0.2, absent=0.3, seed=0, scale=3.0):
        g = gen(seed * 977 + rows + vocab * 3 + k)
        self.x = (torch.randn(rows, vocab, generator=g, device=dev()) * scale).to(dtype)
        t = torch.randn(rows, vocab, generator=g, device=dev()) * scale
        self.ids = torch.randint(0, vocab, (rows, k), generator=g, device=dev(), dtype=torch.int32)  # they may repeat
        self.tv = t.gather(1, self.ids.long())
        gone = torch.rand(rows, k, generator=g, device=dev()) < absent
        gone |= torch.rand(rows, 1, generator=g, device=dev()) < absent / 3  # whole rows
        self.ids[gone] = -1
        self.tv[gone] = math.nan  # what stands in absent entries is not read
        self.tlse = torch.logsumexp(t.double() / temperature, 1).float() if full else None
        self.y = torch.randint(0, vocab, (rows,), generator=g, device=dev(), dtype=torch.int32)
        self.y[torch.rand(rows, generator=g, device=dev()) < ignored] = -1
        self.T, self.kd, self.ce = temperature, kd, ce

    def expected(self, grad=1.0, targets=True):
        x, T = self.x.double(), float(torch.tensor(self.T, dtype=torch.float32))
        rows, vocab = x.shape
        counts = (self.y >= 0) & (self.y < vocab) if targets else torch.ones_like(self.y, dtype=torch.bool)
        x = torch.where(counts[:, None], x, torch.zeros_like(x))
        y = torch.where(counts, self.y, torch.zeros_like(self.y)).long() if targets else torch.zeros_like(self.y).long()
        here = (self.ids >= 0) & (self.ids < vocab)
        ids = torch.where(here, self.ids, torch.zeros_like(self.ids)).long()
        t = torch.where(here, self.tv.double(), torch.full_like(self.tv, -math.inf).double()) / T
        l = self.tlse.double() if self.tlse is not None else torch.logsumexp(t, 1)
        log_q = t - torch.where(torch.isfinite(l), l, torch.zeros_like(l))[:, None]
        q = torch.exp(log_q)
        self.q, self.at = q, ids
        lt, l1 = torch.logsumexp(x / T, 1), torch.logsumexp(x, 1)
        log_p = x.gather(1, ids) / T - lt[:, None]
        term = torch.where(q > 0, q * (log_q - log_p), torch.zeros_like(q))
        size = torch.where(q > 0, q * (log_q.abs() + log_p.abs() + (t.abs() + lt.abs()[:, None])), torch.zeros_like(q)).sum(1)
        p_at = torch.exp(x.gather(1, y[:, None])[:, 0] - l1)
        self.row = torch.where(counts, self.kd * T * T * term.sum(1) - self.ce * torch.log(p_at + 1e-8), 0.0)
        # logarithms of sums that are off by EPS_P of themselves; the terms' own roundings on top
        self.row_tol = self.kd * T * T * (size * 2.0 ** -20 + 2 * EPS_P * q.sum(1)) + self.ce * (EPS_P + 2.0 ** -20 * (1 + l1.abs()))
        w = counts.double()[:, None] * grad
        p, p1 = torch.exp(x / T - lt[:, None]), torch.exp(x - l1[:, None])
        soft = torch.zeros_like(x).scatter_add_(1, ids, q)
        hard = torch.zeros_like(x).scatter_(1, y[:, None], 1.0)
        Q = q.sum(1, keepdim=True)
        self.d = w * (self.kd * T * (Q * p - soft) + self.ce * (p1 - hard))
        self.d_tol = w.abs() * (self.kd * T * (Q * p + soft) + self.ce * (p1 + hard)) * EPS_P
        # the fused form of bf16 rows holds h = exp((x - max) / 2T) in fp16 between its two passes: off by 2^-11 of
        # itself (half a step of 10 stored bits), and p ~ h^2, softmax(x) ~ h^2T by 2 and 2T times that, to first order (2^-7 of it covers
        # the rest); below fp16's normal range by at most 2^-48 of the row's largest probability, which is at most 1
        power = 2.0 ** -11 * (1 + 2.0 ** -7)
        self.kept_tol = w.abs() * (self.kd * T * Q * (p * 2 * power + 2.0 ** -48) + self.ce * (p1 * max(2.0, 2 * T) * power + 2.0 ** -48))
        self.lse = torch.stack((lt, l1)) * counts
        return self

    def args(self, targets=True):
        return (P(self.ids), P(self.tv), P(self.tlse), P(self.y) if targets else None)

    def fwd(self, flag=None, targets=True, lse=True):
        rows, vocab = self.x.shape
        loss, row, s = torch.full((), 9.0, device=dev()), torch.full((rows,), 9.0, device=dev()), torch.full((2, rows), 9.0, device=dev())
        eb.call("eisen_distill_fwd", stream(), P(self.x), self.x.stride(0), *self.args(targets), P(loss), P(row), P(s) if lse else None,
                rows, vocab, self.ids.shape[1], -1, self.T, self.kd, self.ce, DT[self.x.dtype], P(flag))
        return loss, row, s

    def bwd(self, lse, d, grad=None, accumulate=0, targets=True):
        rows, vocab = self.x.shape
        eb.call("eisen_distill_bwd", stream(), P(self.x), self.x.stride(0), *self.args(targets), P(lse), P(d), d.stride(0), P(grad),
                rows, vocab, self.ids.shape[1], -1, self.T, self.kd, self.ce, DT[self.x.dtype], accumulate)

    def fused(self, d, grad_scale=1.0, flag=None, targets=True, lse=True, x=None):
        x = self.x if x is None else x
        rows, vocab = self.x.shape
        loss, row, s = torch.full((), 9.0, device=dev()), torch.full((rows,), 9.0, device=dev()), torch.full((2, rows), 9.0, device=dev())
        eb.call("eisen_distill_fused", stream(), P(x), x.stride(0), *self.args(targets), P(d), d.stride(0), P(loss), P(row),
                P(s) if lse else None, rows, vocab, self.ids.shape[1], -1, self.T, self.kd, self.ce, grad_scale, DT[x.dtype], P(flag))
        return loss, row, s

    def check_loss(self, loss, row, lse=None):
        err = (row.double() - self.row).abs()
        assert (err <= self.row_tol + 2.0 ** -23 * self.row.abs()).all(), float((err - self.row_tol).max())
        assert abs(float(loss.double() - self.row.sum())) <= float(self.row_tol.sum() + 2.0 ** -20 * self.row.abs().sum())
        if lse is not None:
            assert ((lse.double() - self.lse).abs() <= EPS_P + 4 * 2.0 ** -24 * self.lse.abs()).all()

    def check_grad(self, d, fused=False):
        err = (d.double() - self.d).abs()
        tol = self.d_tol + (self.kept_tol if fused and d.dtype == torch.bfloat16 else 0)
        tol = tol + STEP[d.dtype] * (self.d.abs() + tol)
        tol = tol + torch.finfo(torch.float32).tiny  # results below the normal range
        assert (err <= tol).all(), (float((err - tol).max()), int((err > tol).sum()))


SHAPES = [(1, 1, 1), (2, 3, 2), (3, 8, 5), (5, 1000, 7), (4, 1001, 1), (17, 4099, 64), (3, 32000, 64), (2, 65536, 33), (2, 100003, 128),
          (2, 2000, 1024), (150, 2048, 16)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,k", SHAPES)
@pytest.mark.parametrize("temperature,kd,ce,full", [(1.0, 1.0, 0.0, False), (2.0, 0.5, 0.5, False), (3.5, 0.75, 0.25, True), (1.0, 0.0, 1.0, True),
                                                    (0.5, 0.3, 0.7, False)])
def test_distill(dtype, rows, vocab, k, temperature, kd, ce, full):
    c = Case(dtype, rows, vocab, k, temperature, kd, ce, full).expected()
    flag = torch.zeros(1, dtype=torch.int32, device=dev())
    loss, row, lse = c.fwd(flag)
    c.check_loss(loss, row, lse)
    d = torch.full_like(c.x, 5.0)
    c.bwd(lse, d)
    c.check_grad(d)
    d2 = torch.full_like(c.x, 5.0)
    loss2, row2, lse2 = c.fused(d2, flag=flag)
    c.check_loss(loss2, row2, lse2)
    c.check_grad(d2, fused=True)
    assert int(flag) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_gradient_is_the_loss_differentiated(dtype):
    """The gradient against central differences of the 64-bit loss, at entries of every kind."""
    c = Case(dtype, 4, 300, 9, 2.0, 0.6, 0.4, absent=0.0, ignored=0.0).expected()
    d = torch.empty_like(c.x)
    c.fused(d)
    x0 = c.x.double()
    step = 1e-4
    for r in range(4):
        for i in [int(c.ids[r, 0]), int(c.ids[r, 8]), int(c.y[r]), 0, 299]:
            vals = []
            for sign in (1, -1):
                c.x = x0.clone()
                c.x[r, i] += sign * step
                vals.append(float(c.expected().row[r]))
            c.x = x0
            # the 1e-8 of the loss takes no part in the gradient: at p of 1e-3 and more it changes 1e-5 of it
            p = float(torch.softmax(x0[r], 0)[c.y[r].long()])
            tol = 0.4 * 1e-8 / (p + 1e-8) + 1e-6 + 2 * STEP[dtype] * abs(float(d[r, i])) + EPS_P + float(c.kept_tol[r, i])
            assert abs((vals[0] - vals[1]) / (2 * step) - float(d[r, i].double())) <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(3, 1003), (2, 40001)])
def test_distill_same_id_many_times(dtype, rows, vocab):
    c = Case(dtype, rows, vocab, 40, 1.5, 0.5, 0.5, absent=0.0, ignored=0.0)
    c.ids[:, ::2] = c.y[:, None]  # every second entry is the target
    c.ids[:, 1::4] = 7
    c.expected()
    d = torch.empty_like(c.x)
    c.check_loss(*c.fused(d))
    c.check_grad(d, fused=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ld,shift,ld_d,shift_d", [(1003, 0, 1003, 0), (1008, 1, 1003, 5), (1005, 3, 1010, 3), (1016, 8, 1016, 8)])
def test_distill_strides_and_neighbours(dtype, ld, shift, ld_d, shift_d):
    c = Case(dtype, 6, 1003, 11, 2.0, 0.5, 0.5).expected()
    c.x = rows_at(c.x, ld, shift)
    buf = torch.full((6 * ld_d + 40,), 3.0, dtype=dtype, device=dev())
    view = buf[shift_d:shift_d + 6 * ld_d].view(6, ld_d)[:, :1003]
    loss, row, lse = c.fused(view)
    c.check_loss(loss, row, lse)
    c.check_grad(view, fused=True)
    before = view.clone()
    view.fill_(3.0)
    assert (buf == 3.0).all()  # nothing beside the rows was written
    c.bwd(lse, view)
    c.check_grad(view)
    view.fill_(3.0)
    assert (buf == 3.0).all()
    del before


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1000, 1001, 32000, 40007])
def test_distill_in_place_accumulate_and_upstream_gradient(dtype, vocab):
    c = Case(dtype, 7, vocab, 13, 2.0, 0.5, 0.5).expected(grad=0.37)
    x = c.x.clone()
    loss, row, lse = c.fused(x, grad_scale=0.37, x=x)  # dlogits over the logits
    c.check_loss(loss, row, lse)
    c.check_grad(x, fused=True)
    g = torch.full((), 0.37, device=dev())
    x2 = c.x.clone()
    keep, c.x = c.x, x2
    c.bwd(lse, x2, g)
    c.check_grad(x2)
    c.x = keep
    base = torch.randn(7, vocab, generator=gen(3), device=dev()).to(dtype)
    acc = base.clone()
    c.bwd(lse, acc, g, accumulate=1)
    want = base.double() + c.d
    assert ((acc.double() - want).abs() <= c.d_tol + STEP[dtype] * (want.abs() + c.d_tol)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,k,ignored", [(1500, 700, 5, 0.5), (3000, 1001, 100, 0.05), (1111, 8200, 64, 0.6), (900, 5003, 3, 0.0),
                                                  (700, 32000, 64, 0.4), (601, 24001, 700, 0.1), (400, 100003, 20, 0.3), (333, 50, 1024, 0.3)])
def test_distill_many_rows(dtype, rows, vocab, k, ignored):
    """Several rows per CTA, with rows in between that do not count."""
    c = Case(dtype, rows, vocab, k, 2.0, 0.5, 0.5, ignored=ignored).expected()
    d = torch.full_like(c.x, 5.0)
    loss, row, lse = c.fused(d)
    c.check_loss(loss, row, lse)
    c.check_grad(d, fused=True)
    loss, row, lse = c.fwd()
    c.check_loss(loss, row, lse)
    d.fill_(5.0)
    c.bwd(lse, d)
    c.check_grad(d)


@pytest.mark.parametrize("rows", [3, 400])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0, 1e-3])
def test_distill_large_logits(rows, temperature):
    """bf16 logits of 2e4 and more: the row's largest, over T, is far beyond what a product with it would keep of a
    difference.  One step of these logits is 128, so all probabilities but the largest ones' are 0."""
    c = Case(torch.bfloat16, rows, 3000, 6, temperature, 0.5, 0.5, ignored=0.0, absent=0.0)
    c.x = (c.x.float() * 10 + 20000).to(torch.bfloat16)
    c.ids[:, 0] = c.x.float().argmax(1).int()
    c.tv[:] = -math.inf
    c.tv[:, 0] = 1.0  # the teacher is sure of the student's first choice, whose loss is that of the ties
    c.expected()
    d = torch.full_like(c.x, 5.0)
    loss, row, lse = c.fused(d)
    assert torch.isfinite(loss)
    assert ((lse.double() - c.lse).abs() <= EPS_P + 8 * 2.0 ** -24 * c.lse.abs()).all()
    c.check_grad(d, fused=True)
    d.fill_(5.0)
    c.bwd(lse, d)
    # the log-sum-exps themselves are rounded to 32 bits: 2^-24 of 2e4 / T is the relative error of every probability
    c.d_tol = c.d_tol * (1 + c.lse.abs().max(0).values[:, None] * 2.0 ** -23 / EPS_P)
    c.check_grad(d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distill_row_longer_than_shared_memory(dtype):
    c = Case(dtype, 2, 1000003, 70, 2.0, 0.5, 0.5, ignored=0.0).expected()
    d = torch.full_like(c.x, 5.0)
    loss, row, lse = c.fused(d)
    c.check_loss(loss, row, lse)
    c.check_grad(d, fused=True)
    d.fill_(5.0)
    c.bwd(lse, d)
    c.check_grad(d)


def test_distill_without_targets_and_without_lse():
    c = Case(torch.float32, 5, 777, 6, 2.0, 0.8, 0.0).expected(targets=False)
    d = torch.empty_like(c.x)
    loss, row, _ = c.fused(d, targets=False, lse=False)
    c.check_loss(loss, row)
    c.check_grad(d)
    loss, row, lse = c.fwd(targets=False)
    c.check_loss(loss, row, lse)
    c.bwd(lse, d, targets=False)
    c.check_grad(d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1003, 32000])
def test_distill_ignored_rows_hold_anything(dtype, vocab):
    c = Case(dtype, 6, vocab, 5, 2.0, 0.5, 0.5, ignored=0.0, absent=0.0)
    c.y[1], c.y[4] = -1, -1
    c.x[1] = math.nan
    c.x[4] = math.inf
    c.tv[1] = math.nan
    c.expected()
    c.tv[1] = math.nan
    d = torch.full_like(c.x, 5.0)
    out = c.fused(d)
    keep = torch.tensor([0, 2, 3, 5], device=dev())
    assert (d[1] == 0).all() and (d[4] == 0).all() and float(out[1][1]) == 0.0 and float(out[1][4]) == 0.0
    assert torch.isfinite(out[0])
    err = (d[keep].double() - c.d[keep]).abs()
    tol = c.d_tol[keep] + (c.kept_tol[keep] if dtype == torch.bfloat16 else 0)
    assert (err <= tol + STEP[dtype] * (c.d[keep].abs() + tol) + 1e-30).all()
    d.fill_(5.0)
    c.bwd(out[2], d)
    assert (d[1] == 0).all() and (d[4] == 0).all()
    d.fill_(5.0)
    c.bwd(out[2], d, accumulate=1)
    assert (d[1] == 5).all() and (d[4] == 5).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low", ["-inf", "lowest"])
@pytest.mark.parametrize("vocab", [1003, 32000])
def test_distill_masked_vocabulary(dtype, low, vocab):
    """Most of the vocabulary masked out; the teacher's entries and the targets are among the rest."""
    c = Case(dtype, 4, vocab, 5, 1.0, 0.5, 0.5, ignored=0.0, absent=0.2)
    c.x[:, 50:] = -math.inf if low == "-inf" else torch.finfo(dtype).min
    c.ids = torch.where(c.ids >= 0, c.ids % 50, c.ids)
    c.y = c.y % 50
    c.x[2, 1:] = -math.inf if low == "-inf" else torch.finfo(dtype).min  # one entry left
    c.ids[2], c.y[2] = 0, 0
    c.tv = torch.where(torch.isnan(c.tv) & (c.ids >= 0), torch.zeros_like(c.tv), c.tv)
    c.expected()
    d = torch.full_like(c.x, 5.0)
    loss, row, lse = c.fused(d)
    assert torch.isfinite(loss) and torch.isfinite(d).all() and (d[:, 50:] == 0).all()
    c.check_loss(loss, row, lse)
    c.check_grad(d, fused=True)
    d2 = torch.full_like(c.x, 5.0)
    c.bwd(lse, d2)
    c.check_grad(d2)


def test_distill_teacher_entries_of_minus_infinity_and_empty_rows():
    c = Case(torch.float32, 4, 500, 6, 1.0, 1.0, 0.0, ignored=0.0, absent=0.0)
    c.tv[0, 2:] = -math.inf  # probability 0
    c.tv[1] = -math.inf      # no entry with any weight
    c.ids[2] = -1            # no entry at all
    c.expected()
    d = torch.full_like(c.x, 5.0)
    loss, row, lse = c.fused(d)
    c.check_loss(loss, row, lse)
    c.check_grad(d, fused=True)
    assert (d[1] == 0).all() and (d[2] == 0).all() and float(row[1]) == 0.0 and float(row[2]) == 0.0


def test_distill_ids_and_targets_out_of_range_are_flagged():
    for what in ("id", "target"):
        c = Case(torch.float32, 3, 100, 4, 1.0, 0.5, 0.5, ignored=0.0, absent=0.0)
        if what == "id":
            c.ids[1, 2] = 100
        else:
            c.y[1] = 100
        c.expected()
        flag = torch.zeros(1, dtype=torch.int32, device=dev())
        d = torch.full_like(c.x, 5.0)
        loss, row, lse = c.fused(d, flag=flag)
        assert int(flag) == 1
        c.check_loss(loss, row, lse)
        c.check_grad(d)
        flag.zero_()
        c.fwd(flag)
        assert int(flag) == 1


def test_distill_no_rows():
    c = Case(torch.float32, 0, 100, 4)
    loss, _, _ = c.fwd()
    assert float(loss) == 0.0
    loss, _, lse = c.fused(torch.empty_like(c.x))
    assert float(loss) == 0.0
    c.bwd(lse, torch.empty_like(c.x))


def test_distill_matches_cross_entropy_kernels():
    """With kd_weight 0 the distillation is the cross-entropy of eisen_ce_fused."""
    c = Case(torch.float32, 32, 4096, 3, 1.0, 0.0, 1.0 / 32, ignored=0.1)
    d = torch.empty_like(c.x)
    loss, row, _ = c.fused(d)
    x = c.x.clone()
    l2, r2 = torch.empty((), device=dev()), torch.empty(32, device=dev())
    eb.call("eisen_ce_fused", stream(), P(x), P(c.y), P(l2), P(r2), None, 32, 4096, -1, 1.0 / 32, 1.0, eb.F32, None)
    assert torch.allclose(row, r2, rtol=2.0 ** -18, atol=2.0 ** -20) and torch.allclose(d, x, rtol=EPS_P, atol=1e-12)


# ------------------------------------------------------------------------------------------ cross-entropy without logits
class Head:
    def __init__(self, rows, k, vocab, tied, seed=0, ignored=0.2, pad_h=0, pad_w=0, scale=2.0):
        g = gen(seed * 131 + rows + 7 * k + vocab)
        self.h = rows_at((torch.randn(rows, k, generator=g, device=dev())).to(torch.bfloat16), k + pad_h)
        w = (torch.randn(vocab, k, generator=g, device=dev()) * scale / math.sqrt(k)).to(torch.bfloat16)
        w = w if tied else w.t().contiguous()
        self.ldw = (w.shape[1] + 7) // 8 * 8 + pad_w
        self.w = rows_at(w, self.ldw)
        self.y = torch.randint(0, vocab, (rows,), generator=g, device=dev(), dtype=torch.int32)
        self.y[torch.rand(rows, generator=g, device=dev()) < ignored] = -1
        self.rows, self.k, self.vocab, self.tied = rows, k, vocab, tied
        self.norm = 1.0 / max(1, int((self.y >= 0).sum()))
        self.status = torch.zeros(2, dtype=torch.int32, device=dev())

    def workspace(self, piece=0, backward=1):
        n = eb.lib().eisen_linear_ce_workspace_bytes(self.rows, self.k, self.vocab, piece, backward)
        return torch.full((n + 256,), 0x7f, dtype=torch.uint8, device=dev())

    def operands(self):
        return (P(self.h), self.h.stride(0), P(self.w), self.ldw, 1 if self.tied else 0, P(self.y))

    def fwd(self, ws=None, loss=True):
        ws = self.workspace(backward=0) if ws is None else ws
        out = [torch.full((), 9.0, device=dev()), torch.full((self.rows,), 9.0, device=dev()), torch.full((self.rows,), 9.0, device=dev())]
        eb.call("eisen_linear_ce_fwd", stream(), *self.operands(), P(out[0]) if loss else None, P(out[1]), P(out[2]), P(ws), self.rows, self.k,
                self.vocab, -1, self.norm, P(self.status[1:]), P(self.status))
        return out

    def bwd(self, lse, piece=0, grad=None, dh=True, dw=True, dw_dtype=torch.bfloat16, acc_h=0, acc_w=0, dh0=None, dw0=None, ws=None):
        ws = self.workspace(piece) if ws is None else ws
        dhv = (torch.full((self.rows, self.k), 9.0, dtype=torch.bfloat16, device=dev()) if dh0 is None else dh0.clone()) if dh else None
        dwv = None
        if dw:
            dwv = rows_at((torch.full(tuple(self.w.shape), 9.0, dtype=dw_dtype, device=dev()) if dw0 is None else dw0), self.ldw)
        eb.call("eisen_linear_ce_bwd", stream(), *self.operands(), P(lse), P(grad), P(dhv), acc_h, P(dwv), self.ldw, DT[dw_dtype], acc_w,
                P(ws), self.rows, self.k, self.vocab, piece, -1, self.norm, P(self.status))
        assert int(self.status[0]) == 0
        return dhv, dwv

    def expected(self, grad=1.0):
        h, w = self.h.double(), self.w.double().t() if self.tied else self.w.double()
        counts = (self.y >= 0) & (self.y < self.vocab)
        y = torch.where(counts, self.y, torch.zeros_like(self.y)).long()
        x = h @ w
        # products of bf16 are exact in 32 bits; the accumulator takes in 16 of them at a time, and each time may
        # drop up to one unit in the last place of the sum's size
        eps_x = (self.k / 16 + 16) * 2.0 ** -23 * float((h.abs() @ w.abs()).max())
        lse = torch.logsumexp(x, 1)
        self.lse = lse * counts
        self.eps = eps_x + EPS_P
        p = torch.exp(x - lse[:, None])
        self.row = torch.where(counts, -self.norm * torch.log(p.gather(1, y[:, None])[:, 0] + 1e-8), 0.0)
        hard = torch.zeros_like(x).scatter_(1, y[:, None], 1.0)
        scale = counts.double()[:, None] * self.norm * grad
        d, size = (p - hard) * scale, (p * 2 * self.eps + (p - hard).abs() * (2.0 ** -8 + 2.0 ** -20)) * scale.abs()
        self.dh, self.dh_tol = d @ w.t(), size @ w.t().abs() + (self.vocab / 16 + 64) * 2.0 ** -23 * (d.abs() @ w.t().abs())
        dw, dw_tol = h.t() @ d, h.t().abs() @ size + (self.rows / 16 + 64) * 2.0 ** -23 * (h.t().abs() @ d.abs())
        self.dw, self.dw_tol = (dw.t(), dw_tol.t()) if self.tied else (dw, dw_tol)
        return self

    def check_loss(self, loss, row, lse):
        tol = self.norm * (2 * self.eps + 2.0 ** -20 * (1 + self.lse.abs()))
        assert ((row.double() - self.row).abs() <= tol).all()
        assert abs(float(loss.double() - self.row.sum())) <= float(tol.sum())
        assert ((lse.double() - self.lse).abs() <= self.eps + 4 * 2.0 ** -24 * self.lse.abs()).all()

    @staticmethod
    def within(got, want, tol, step):
        err = (got.double() - want).abs()
        lim = tol + step * (want.abs() + tol) + 1e-30
        assert (err <= lim).all(), (float((err / lim).max()), int((err > lim).sum()))


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("rows,k,vocab,piece", [(1, 64, 64, 0), (5, 384, 8192, 0), (3, 8, 17, 0), (130, 72, 300, 256), (257, 128, 1000, 512),
                                                (256, 256, 2048, 1024), (700, 1000, 5001, 1024), (512, 2048, 4096, 0), (33, 64, 50001, 8192),
                                                (2, 16, 1, 0)])
def test_linear_ce(rows, k, vocab, piece, tied):
    c = Head(rows, k, vocab, tied).expected()
    loss, row, lse = c.fwd()
    c.check_loss(loss, row, lse)
    dh, dw = c.bwd(lse, piece)
    c.within(dh, c.dh, c.dh_tol, 2.0 ** -8)
    c.within(dw, c.dw, c.dw_tol, 2.0 ** -8)
    _, dw32 = c.bwd(lse, piece, dh=False, dw_dtype=torch.float32)
    c.within(dw32, c.dw, c.dw_tol, 2.0 ** -24)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dw_dtype", [torch.bfloat16, torch.float32])
def test_linear_ce_accumulates_and_takes_an_upstream_gradient(tied, dw_dtype):
    c = Head(300, 136, 1203, tied, pad_h=8, pad_w=16).expected(grad=0.25)
    loss, row, lse = c.fwd()
    c.check_loss(loss, row, lse)
    g = torch.full((), 0.25, device=dev())
    dh0 = (torch.randn(300, 136, generator=gen(1), device=dev()) * 1e-2).to(torch.bfloat16)
    dw0 = (torch.randn(tuple(c.w.shape), generator=gen(2), device=dev()) * 1e-2).to(dw_dtype)
    dh, dw = c.bwd(lse, 512, grad=g, acc_h=1, acc_w=1, dh0=dh0, dw0=dw0, dw_dtype=dw_dtype)
    c.within(dh, c.dh + dh0.double(), c.dh_tol, 2.0 ** -7)  # the one-piece form rounds the product before it is added
    c.within(dw, c.dw + dw0.double(), c.dw_tol + 2.0 ** -8 * c.dw.abs(), STEP[dw_dtype])
    only_h, none = c.bwd(lse, 512, grad=g, dw=False)
    assert none is None
    c.within(only_h, c.dh, c.dh_tol, 2.0 ** -8)


@pytest.mark.parametrize("tied", [False, True])
def test_linear_ce_forward_of_any_width(tied):
    """The loss alone takes widths that are no multiple of 8 (rows still are)."""
    c = Head(70, 60, 333, tied, pad_h=4).expected()
    c.check_loss(*c.fwd())


def test_linear_ce_does_not_touch_what_is_beside_its_outputs():
    c = Head(129, 64, 777, False, pad_w=8).expected()
    loss, row, lse = c.fwd()
    ws = c.workspace(256)
    size = eb.lib().eisen_linear_ce_workspace_bytes(129, 64, 777, 256, 1)
    buf = torch.full((64 * c.ldw + 8,), 3.0, dtype=torch.bfloat16, device=dev())
    eb.call("eisen_linear_ce_bwd", stream(), *c.operands(), P(lse), None, None, 0, P(buf), c.ldw, eb.BF16, 0, P(ws), 129, 64, 777, 256, -1, c.norm,
            P(c.status))
    view = buf[:64 * c.ldw].view(64, c.ldw)
    c.within(view[:, :777], c.dw, c.dw_tol, 2.0 ** -8)
    assert (view[:, 777:] == 3.0).all() and (buf[64 * c.ldw:] == 3.0).all() and (ws[size:] == 0x7f).all()


def test_linear_ce_rows_that_do_not_count():
    c = Head(260, 64, 1000, False, ignored=0.0)
    c.y[3], c.y[100], c.y[259] = -1, 1000, -1
    c.h[3] = 30000.0  # finite, and an overflow of exp without its own log-sum-exp
    c.norm = 1.0 / 257
    c.expected()
    loss, row, lse = c.fwd()
    assert int(c.status[1]) == 1 and float(row[3]) == 0.0 and float(row[100]) == 0.0 and float(lse[3]) == 0.0
    keep = [i for i in range(260) if i not in (3, 100, 259)]
    ref = Head(260, 64, 1000, False, ignored=0.0)
    ref.y[3], ref.y[100], ref.y[259] = -1, -1, -1
    ref.norm = 1.0 / 257
    ref.expected()
    ref.check_loss(loss, row, lse)
    dh, dw = c.bwd(lse, 512)
    assert (dh[3] == 0).all() and (dh[100] == 0).all() and (dh[259] == 0).all()
    ref.within(dh[keep], ref.dh[keep], ref.dh_tol[keep], 2.0 ** -8)
    ref.within(dw, ref.dw, ref.dw_tol, 2.0 ** -8)
    c.y[:] = -1
    loss, row, lse = c.fwd()
    assert float(loss) == 0.0
    dh, dw = c.bwd(lse)
    assert (dh == 0).all() and (dw == 0).all()


def test_linear_ce_fixed_order_repeats_bit_for_bit():
    c = Head(700, 512, 3000, False)
    eb.call("eisen_set_deterministic", 1)
    try:
        _, _, lse = c.fwd()
        a = c.bwd(lse, 1024, dw_dtype=torch.float32)
        b = c.bwd(lse, 1024, dw_dtype=torch.float32)
    finally:
        eb.call("eisen_set_deterministic", 0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_linear_ce_is_closer_than_bf16_logits():
    """Peaked rows: logits rounded to bf16 move the probabilities, the f32 accumulators do not."""
    c = Head(256, 256, 4096, False, ignored=0.0, scale=8.0).expected()
    loss, row, lse = c.fwd()
    c.check_loss(loss, row, lse)
    rounded = torch.logsumexp((c.h.float() @ c.w.float()).to(torch.bfloat16).double(), 1)
    assert float((lse.double() - c.lse).abs().max()) < 0.05 * float((rounded - c.lse).abs().max())


# ------------------------------------------------------------------------------------------ all of them
def test_streams_and_graph_replay():
    """Captured on a side stream, replayed on new inputs, beside an eager run on another stream."""
    side = torch.cuda.Stream()
    c = Case(torch.bfloat16, 9, 8200, 16, 2.0, 0.5, 0.5)
    hd = Head(300, 128, 2000, False)
    d, ws = torch.empty_like(c.x), hd.workspace()
    v, i, s = torch.empty(9, 16, device=dev()), torch.empty(9, 16, dtype=torch.int32, device=dev()), torch.empty(9, device=dev())
    loss, row, lse = torch.empty((), device=dev()), torch.empty(9, device=dev()), torch.empty(2, 9, device=dev())
    h_out = [torch.empty((), device=dev()), torch.empty(300, device=dev()), torch.empty(300, device=dev())]
    dh, dw = torch.empty(300, 128, dtype=torch.bfloat16, device=dev()), torch.empty_like(hd.w)

    def calls():
        st = stream()
        eb.call("eisen_top_logits", st, P(c.x), 8200, P(v), P(i), P(s), 9, 8200, 16, 2.0, eb.BF16)
        eb.call("eisen_distill_fused", st, P(c.x), 8200, *c.args(), P(d), 8200, P(loss), P(row), P(lse), 9, 8200, 16, -1, 2.0, 0.5, 0.5, 1.0,
                eb.BF16, None)
        eb.call("eisen_linear_ce_fwd", st, *hd.operands(), P(h_out[0]), P(h_out[1]), P(h_out[2]), P(ws), 300, 128, 2000, -1, hd.norm, None, None)
        eb.call("eisen_linear_ce_bwd", st, *hd.operands(), P(h_out[2]), None, P(dh), 0, P(dw), hd.ldw, eb.BF16, 0, P(ws), 300, 128, 2000, 512, -1,
                hd.norm, None)

    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        calls()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        calls()
    new, newh = Case(torch.bfloat16, 9, 8200, 16, 2.0, 0.5, 0.5, seed=4), Head(300, 128, 2000, False, seed=5)
    for a, b in ((c.x, new.x), (c.ids, new.ids), (c.tv, new.tv), (c.y, new.y), (hd.h, newh.h), (hd.w, newh.w)):
        a.copy_(b)
    hd.y.copy_(newh.y)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    c.expected()
    c.check_loss(loss, row, lse)
    c.check_grad(d, fused=True)
    assert torch.equal(i.long(), torch.argsort(-c.x.double(), dim=1, stable=True)[:, :16])
    hd.expected()
    hd.check_loss(*h_out)
    hd.within(dh, hd.dh, hd.dh_tol, 2.0 ** -8)
    hd.within(dw, hd.dw, hd.dw_tol, 2.0 ** -8)


def test_teacher_to_student():
    """A teacher's logits -> its top entries and log-sum-exp -> the student's loss and gradient."""
    g = gen(11)
    teacher = (torch.randn(40, 3001, generator=g, device=dev()) * 3).to(torch.bfloat16)
    v, i, s = top(teacher, 3, 2.0)
    c = Case(torch.bfloat16, 40, 3001, 3, 2.0, 1.0, 0.0, absent=0.0)
    c.ids, c.tv, c.tlse = i, v, s
    c.expected()
    d = torch.empty_like(c.x)
    c.check_loss(*c.fused(d))
    c.check_grad(d, fused=True)
    # a student that agrees with its teacher has the loss of the entries left out only, and a gradient to match
    full_q = torch.softmax(teacher.double() / 2.0, 1)
    c.x = teacher.clone()
    c.expected()
    c.fused(d)
    rest = 1 - full_q.gather(1, i.long()).sum(1)
    w = (c.y >= 0).double()
    got = d.double().gather(1, i.long()).sum(1)
    want = -w * 2.0 * (1 - rest) * rest
    tol = (c.d_tol + c.kept_tol).gather(1, i.long()).sum(1)
    assert ((got - want).abs() <= tol + 2.0 ** -8 * (d.double().gather(1, i.long()).abs().sum(1) + tol)).all()


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dw_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_linear_ce_weight_gradient_with_any_row_stride(tied, dw_dtype, accumulate):
    """The weight gradient's rows may start at any element, unlike the weight's."""
    c = Head(300, 136, 1203, tied).expected()
    loss, row, lse = c.fwd()
    start = (torch.randn(tuple(c.w.shape), generator=gen(5), device=dev()) * 1e-2).to(dw_dtype)
    cols = c.w.shape[1]
    buf = torch.full((c.w.shape[0], cols + 3), 3.0, dtype=dw_dtype, device=dev())
    buf[:, :cols] = start
    eb.call("eisen_linear_ce_bwd", stream(), *c.operands(), P(lse), None, None, 0, P(buf), cols + 3, DT[dw_dtype], accumulate,
            P(c.workspace(512)), c.rows, c.k, c.vocab, 512, -1, c.norm, P(c.status))
    assert int(c.status[0]) == 0
    # a bf16 sum may round the product before it is added
    c.within(buf[:, :cols], c.dw + accumulate * start.double(), c.dw_tol + accumulate * 2.0 ** -8 * c.dw.abs(), STEP[dw_dtype])
    assert (buf[:, cols:] == 3.0).all()


def test_linear_ce_no_rows():
    c = Head(0, 64, 100, False)
    loss, _, lse = c.fwd()
    assert float(loss) == 0.0
    _, dw = c.bwd(lse)
    assert (dw == 0).all()
    _, dw = c.bwd(lse, acc_w=1, dw0=torch.full((64, 100), 2.0, dtype=torch.bfloat16, device=dev()))
    assert (dw == 2).all()


@pytest.mark.parametrize("rows", [260, 320])
def test_rows_more_than_two_to_the_31_elements_apart(rows):
    """Element offsets pass 32 bits in both row forms, in reading and in writing."""
    ld = (2 ** 31 + 2 ** 20) // (rows - 1) + 5
    buf = torch.empty(rows * ld, dtype=torch.bfloat16, device=dev())
    c = Case(torch.bfloat16, rows, 1000, 7, temperature=2.0).expected()
    far = buf.view(rows, ld)[:, :1000]
    far.copy_(c.x)
    assert (rows - 1) * ld > 2 ** 31
    check_top(far, 9)
    c.x = far
    loss, row, lse = c.fwd()
    c.check_loss(loss, row, lse)
    d = torch.empty(rows, 1000, dtype=torch.bfloat16, device=dev())
    c.bwd(lse, d)
    c.check_grad(d)
    c.check_loss(*c.fused(far))  # the gradient over the logits
    c.check_grad(far, fused=True)
