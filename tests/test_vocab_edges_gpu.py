"""The vocabulary-end operators on rows and calls at the edge of what their documentation allows: teacher rows without
entries, rows whose logits are all the lowest of their type, every kind of exponential in both row forms, sums in a fixed order,
tensors that take no gradient, refusals."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import eisen_b200 as eb  # noqa: E402
from eisen_b200.graph import BF16_MIXED, FP32  # noqa: E402
from test_vocab_graph_gpu import CFG, data, f64_distill, model, new_graph  # noqa: E402
from test_vocab_ops_gpu import Case, EPS_P, Head, P, STEP, dev, gen, top  # noqa: E402

FORMS = [(4, 500), (3, 40000), (700, 500), (400, 12000)]  # few rows (one CTA, several CTAs each), rows in numbers, and in numbers and long


# ------------------------------------------------------------------------------------------ teacher rows without entries
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", FORMS)
def test_rows_without_teacher_entries_whatever_their_log_sum_exp(dtype, rows, vocab):
    """Entries that are absent or -inf have no weight, and a row of them has no distillation term: its given log-sum-exp
    (-inf for a teacher that masks everything, or nothing that was ever set) is not looked at."""
    c = Case(dtype, rows, vocab, 6, 2.0, 0.6, 0.4, full=True, ignored=0.0, absent=0.0)
    empty = [0, 1, rows - 1]
    c.ids[0] = -1
    c.tv[1] = -math.inf
    c.ids[rows - 1, :3] = -1
    c.tv[rows - 1, 3:] = -math.inf
    c.tlse[0], c.tlse[1], c.tlse[rows - 1] = math.nan, -math.inf, -math.inf
    given, c.tlse = c.tlse, c.tlse.clone()
    c.tlse[empty] = 0.0  # in the formula the term is 0 whatever stands here
    c.expected()
    c.tlse = given
    loss, row, lse = c.fwd()
    c.check_loss(loss, row, lse)
    d = torch.full_like(c.x, 5.0)
    c.bwd(lse, d)
    c.check_grad(d)
    d.fill_(5.0)
    c.check_loss(*c.fused(d))
    c.check_grad(d, fused=True)


@pytest.mark.parametrize("rows", [5, 700])
def test_masked_teacher_row_to_student(rows):
    """A teacher row of nothing but -inf through the top logits into the loss."""
    teacher = torch.randn(rows, 900, generator=gen(3), device=dev())
    teacher[2] = -math.inf
    v, i, s = top(teacher, 4, 2.0)
    assert (v[2] == -math.inf).all() and float(s[2]) == -math.inf
    c = Case(torch.float32, rows, 900, 4, 2.0, 1.0, 0.0, ignored=0.0, absent=0.0)
    c.ids, c.tv = i, v
    c.tlse = torch.where(torch.isfinite(s), s, torch.zeros_like(s))
    c.expected()
    c.tlse = s
    d = torch.full_like(c.x, 5.0)
    loss, row, _ = c.fused(d)
    c.check_loss(loss, row)
    c.check_grad(d)
    assert float(row[2]) == 0.0 and (d[2] == 0).all()


# ------------------------------------------------------------------------------------------ tensors of another type
def test_tensors_of_another_type_are_not_read_as_logits():
    """A kernel reads as many elements of the graph's own type as the tensor has: a bf16 buffer is half of that in f32."""
    x, ids, tv, _ = data(4, 64, 3)
    b, f = new_graph(BF16_MIXED), new_graph(FP32)
    act = b.alloc_pooled([4, 64])
    b.load_tensor_data(act, x)
    with pytest.raises(eb.EisenError, match="copy_from"):
        f.copy_from(b, act)
    again = new_graph(BF16_MIXED)
    same = again.copy_from(b, act)
    v, i, s = again.top_logits(same, 3)
    assert (again.ids_to_cpu(i).reshape(4, 3) == np.argsort(-b.data(act).reshape(4, 64), axis=1, kind="stable")[:, :3]).all()
    for g in (b, f):
        t, lg = g.alloc_ids([4, 64], np.zeros(256)), g.alloc([4, 3], tv)
        for call in (lambda: g.top_logits(t, 3), lambda: g.distill(t, g.alloc_ids([4, 3], ids), lg, 4)):
            with pytest.raises(eb.EisenError, match="ids"):
                call()
    teacher = b.copy_from(f, f.alloc([4, 3], tv))  # f32 values go anywhere ...
    with pytest.raises(eb.EisenError, match="shadow"):
        b.top_logits(teacher, 2)  # ... but are no bf16 logits
    assert np.isfinite(b.data(b.distill(act, b.alloc_ids([4, 3], ids), teacher, 4))[0])


# ------------------------------------------------------------------------------------------ a wait that runs out
@pytest.mark.parametrize("rows", [2, 31, 50, 1000])
def test_rows_are_marked_when_a_wait_runs_out(rows):
    """A group that gives up marks the rows of the groups that were through long before, and the device's word says so."""
    out = torch.zeros(rows, device=dev())
    code = torch.zeros(1, dtype=torch.int32)
    eb.call("eisen_pending_fault", code.data_ptr())
    eb.call("eisen_selftest_row_frame", torch.cuda.current_stream().cuda_stream, P(out), rows, 200000)
    eb.call("eisen_pending_fault", code.data_ptr())
    assert int(code) == 6 and torch.isnan(out).all()
    eb.call("eisen_pending_fault", code.data_ptr())
    assert int(code) == 0


def test_a_graph_reports_the_wait_of_its_own_row_kernel():
    g = new_graph()
    eb.call("eisen_graph_selftest_row_frame", g._h, 200000)
    with pytest.raises(eb.EisenError, match="bounded wait"):
        g.synchronize()
    g.synchronize()
    code = torch.zeros(1, dtype=torch.int32)
    eb.call("eisen_pending_fault", code.data_ptr())
    assert int(code) == 0
    with pytest.raises(eb.EisenError):
        eb.call("eisen_selftest_row_frame", None, None, 5, 200000)


def test_ids_are_not_handed_out_past_a_wait_that_ran_out():
    """Reading ids back looks at the graph's fault word as reading values does."""
    g = new_graph()
    _, i, _ = g.top_logits(g.alloc([2, 50], np.arange(100)), 3)
    assert (g.ids_to_cpu(i).reshape(2, 3) == [49, 48, 47]).all()
    eb.call("eisen_graph_selftest_row_frame", g._h, 200000)
    with pytest.raises(eb.EisenError, match="bounded wait"):
        g.ids_to_cpu(i)
    assert (g.ids_to_cpu(i).reshape(2, 3) == [49, 48, 47]).all()


# ------------------------------------------------------------------------------------------ logits far from 0
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0, 3.5])
def test_rows_of_nothing_but_the_lowest_value(dtype, rows, vocab, temperature):
    """A row masked all over by its type's lowest value has equal logits: probabilities 1 / n, whatever its log-sum-exp rounds
    to.  Differences from the row's largest entry are exact here, so the bounds do not grow with the logits."""
    c = Case(dtype, rows, vocab, 6, temperature, 0.6, 0.4, ignored=0.0, absent=0.0)
    low = [0, rows // 2, rows - 1]
    c.x[low] = 0.0
    c.expected()  # the same for any constant
    c.x[low] = torch.finfo(dtype).min
    loss, row, lse = c.fwd()
    c.check_loss(loss, row)
    d = torch.full_like(c.x, 5.0)
    c.bwd(lse, d)
    c.check_grad(d)
    base = torch.ones_like(c.x)
    c.bwd(lse, base, accumulate=1)
    want = 1.0 + c.d
    assert ((base.double() - want).abs() <= c.d_tol + STEP[dtype] * (want.abs() + c.d_tol)).all()
    d.fill_(5.0)
    loss, row, _ = c.fused(d)
    c.check_loss(loss, row)
    c.check_grad(d, fused=True)
    x = c.x.clone()  # the gradient over the logits, from the log-sum-exps
    keep, c.x = c.x, x
    c.bwd(lse, x)
    c.x = keep
    c.check_grad(x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", FORMS)
@pytest.mark.parametrize("shift", [3000.0, -70000.0])
def test_logits_far_from_zero(dtype, rows, vocab, shift):
    """Loss and gradient depend on differences of logits only: far rows meet the bounds of rows around 0, moved as they
    are rounded."""
    c = Case(dtype, rows, vocab, 6, 2.0, 0.6, 0.4, ignored=0.0, absent=0.0)
    if dtype == torch.bfloat16:  # a few steps of the type apart
        c.x = (c.x.float() / 3).round() * (2.0 ** -7 * abs(shift))
    c.x = (c.x.float() + shift).to(dtype)
    far = c.x
    c.x = (far.double() - far.double().amax(1, keepdim=True)).float()  # exact
    assert torch.equal(c.x.double() + far.double().amax(1, keepdim=True), far.double())
    c.expected()
    c.x = far
    loss, row, lse = c.fwd()
    c.check_loss(loss, row)
    d = torch.full_like(c.x, 5.0)
    c.bwd(lse, d)
    c.check_grad(d)
    d.fill_(5.0)
    loss, row, _ = c.fused(d)
    c.check_loss(loss, row)
    c.check_grad(d, fused=True)


@pytest.mark.parametrize("rows", [3, 400])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 2.0, 1e-3])
def test_losses_of_large_logits(rows, temperature):
    """bf16 logits of 2e4: the row losses, which lie in differences of at most a few hundred."""
    c = Case(torch.bfloat16, rows, 3000, 6, temperature, 0.5, 0.5, ignored=0.0, absent=0.0)
    c.x = (c.x.float() * 10 + 20000).to(torch.bfloat16)
    c.ids[:, 0] = c.x.float().argmax(1).int()
    c.tv[:] = -math.inf
    c.tv[:, 0] = 1.0
    whole, c.x = c.x, c.x.double() - c.x.double().amax(1, keepdim=True)
    c.expected()
    c.x = whole
    loss, row, lse = c.fwd()
    c.check_loss(loss, row)
    loss, row, _ = c.fused(torch.empty_like(c.x))
    c.check_loss(loss, row)


# ------------------------------------------------------------------------------------------ one rounding
@pytest.mark.parametrize("rows,k,vocab", [(2048, 2048, 500), (300, 136, 1203), (1024, 4096, 256)])
@pytest.mark.parametrize("tied", [False, True])
def test_linear_ce_adds_before_it_rounds(rows, k, vocab, tied):
    """What a gradient's bf16 rounding left off comes back when the rounded gradient is taken away from it again: a product that is
    rounded before it is added would leave nothing."""
    c = Head(rows, k, vocab, tied)
    _, _, lse = c.fwd()
    dh, dw = c.bwd(lse)
    rest_h, rest_w = c.bwd(lse, acc_h=1, acc_w=1, dh0=-dh, dw0=-dw)
    for rest, whole in ((rest_h, dh), (rest_w, dw)):
        assert (rest.double().abs() <= 2.0 ** -8 * whole.double().abs() + 1e-30).all()
        counted = rest[whole != 0]  # rows that do not count have no gradient
        assert float((counted != 0).double().mean()) > 0.9


# ------------------------------------------------------------------------------------------ sums in a fixed order
@pytest.mark.parametrize("rows,k,vocab,tied,piece", [(700, 512, 3000, False, 1024), (1021, 1000, 50001, True, 0), (2048, 2048, 32000, False, 0),
                                                     (5, 384, 8192, True, 0), (300, 256, 20000, False, 4096)])
def test_linear_ce_repeats_bit_for_bit(rows, k, vocab, tied, piece):
    """Without the fixed-order switch too: the k slices of dh have a buffer each and are added up in order."""
    c = Head(rows, k, vocab, tied)
    _, _, lse = c.fwd()
    dh, dw = c.bwd(lse, piece)
    for _ in range(3):
        again = c.bwd(lse, piece)
        assert torch.equal(dh, again[0]) and torch.equal(dw, again[1])


@pytest.mark.parametrize("rows,k,vocab,piece", [(1024, 520, 20001, 0), (200, 1032, 9000, 0), (700, 512, 9000, 2048), (64, 64, 40000, 8192)])
@pytest.mark.parametrize("accumulate", [0, 1])
def test_linear_ce_hidden_gradient_in_slices(rows, k, vocab, piece, accumulate):
    """Few output tiles and a long vocabulary: slices, a ragged last one, pieces that add to them; a last piece shorter than the first."""
    c = Head(rows, k, vocab, True).expected()
    _, _, lse = c.fwd()
    ws = c.workspace(piece)
    size = eb.lib().eisen_linear_ce_workspace_bytes(rows, k, vocab, piece, 1)
    dh0 = (torch.randn(rows, k, generator=gen(1), device=dev()) * 1e-2).to(torch.bfloat16)
    dh, _ = c.bwd(lse, piece, dw=False, acc_h=accumulate, dh0=dh0, ws=ws)
    c.within(dh, c.dh + accumulate * dh0.double(), c.dh_tol, 2.0 ** -8)
    assert (ws[size:] == 0x7f).all()


# ------------------------------------------------------------------------------------------ tensors that take no gradient
def frozen(g, H):
    """Hidden states that come from another graph: an activation without a gradient."""
    src = new_graph(BF16_MIXED)
    base = src.alloc_pooled(list(H.shape))
    src.load_tensor_data(base, H)
    out = g.copy_from(src, base)
    g.synchronize()
    return out


@pytest.mark.parametrize("tied", [False, True])
def test_head_trained_on_frozen_hidden_states(tied):
    """linear_cross_entropy and lm_head_distill form the head's gradient alone where the hidden states take none."""
    r = np.random.default_rng(5)
    H, W = r.standard_normal((70, 64)).astype(np.float32), (r.standard_normal((64, 1000)) * 0.2).astype(np.float32)
    _, ids, tv, y = data(70, 1000, 5)
    n = int((y >= 0).sum())
    bf = [torch.tensor(a).to(torch.bfloat16).double() for a in (H, W)]
    for how in ("linear", "distill"):
        g = new_graph(BF16_MIXED)
        w = g.alloc([1000, 64] if tied else [64, 1000], W.T if tied else W)
        g.mark_params()
        tid, h = g.alloc_ids([70], y), frozen(g, H)
        if how == "linear":
            loss = g.linear_cross_entropy(h, w, tid, n, tied, 256)
            kd = 0.0
        else:
            kd = 0.6
            loss = g.lm_head_distill(h, w, g.alloc_ids([70, 5], ids), g.alloc([70, 5], tv), n, target_ids=tid, temperature=2.0, kd_weight=kd,
                                     ce_weight=1.0 - kd, trans_b=tied, chunk_rows=32)
        want, dx = f64_distill((bf[0] @ bf[1]).numpy(), ids, tv, y, 2.0, kd, 1.0 - kd)
        # the distillation's logits are rounded to bf16: at most 2^-8 of a logit of size 8 in its part of a loss of about 7
        assert abs(g.data(loss)[0] - want) < (2e-5 if how == "linear" else 1e-2) * want
        g.backward(loss)
        dw = bf[0].T.numpy() @ dx
        got = g.grad(w).reshape(g.shape(w))
        want_w = dw.T if tied else dw
        assert np.linalg.norm(got - want_w) < (2.0 ** -8 if how == "linear" else 2e-2) * np.linalg.norm(want_w)


def test_nothing_takes_a_gradient():
    """A frozen head over frozen hidden states, and a loss of frozen logits: backward leaves them alone."""
    x, ids, tv, y = data(6, 300, 4)
    g = new_graph(FP32)
    g.mark_params()
    src = new_graph(FP32)
    l = g.copy_from(src, src.alloc([6, 300], x))
    g.synchronize()
    loss = g.distill(l, g.alloc_ids([6, 4], ids), g.alloc([6, 4], tv), int((y >= 0).sum()), target_ids=g.alloc_ids([6], y), temperature=1.5)
    want, _ = f64_distill(x, ids, tv, y, 1.5, 1.0, 0.0)
    assert abs(g.data(loss)[0] - want) < 1e-5 * abs(want) + 1e-6
    g.backward(loss)
    r = np.random.default_rng(1)
    g = new_graph(BF16_MIXED)
    g.mark_params()
    h = frozen(g, r.standard_normal((6, 64)).astype(np.float32))
    w = frozen(g, r.standard_normal((64, 304)).astype(np.float32))
    tid = g.alloc_ids([6], y)
    g.backward(g.linear_cross_entropy(h, w, tid, 6))
    g.backward(g.lm_head_distill(h, w, g.alloc_ids([6, 4], ids), g.alloc([6, 4], tv), 6))
    g.synchronize()


# ------------------------------------------------------------------------------------------ refusals leave nothing behind
def test_gradients_of_another_type_are_refused_at_once():
    """A Bf16Mixed parameter's gradient is f32: as logits, or as hidden states, it cannot take the kernels' bf16."""
    x, ids, tv, y = data(6, 304, 4)
    g = new_graph(BF16_MIXED)
    l = g.alloc([6, 304], x)
    w = g.alloc([304, 64], np.zeros(304 * 64))
    g.mark_params()
    t, v, tid = g.alloc_ids([6, 4], ids), g.alloc([6, 4], tv), g.alloc_ids([6], y)
    n = g.tape_len()
    for f in (lambda: g.distill(l, t, v, 6), lambda: g.linear_cross_entropy(l, w, tid, 6), lambda: g.lm_head_distill(l, w, t, v, 6)):
        with pytest.raises(eb.EisenError, match="gradient"):
            f()
    assert g.tape_len() == n
    g.set_no_grad(True)
    assert np.isfinite(g.data(g.distill(l, t, v, 6))[0])


def teacher_state(g):
    return g.num_tensors(), g.tape_len(), g.pool_stats()["live_bytes"]


@pytest.mark.parametrize("precision", [FP32, BF16_MIXED])
def test_top_logits_refused_before_the_forward_pass(precision):
    g, lm = model(precision, 1)
    ids = np.random.default_rng(0).integers(0, CFG["vocab"], (2, 64)).astype(np.int32)
    x = g.alloc_ids([2, 64], ids)
    h = g.alloc_pooled([128, CFG["hidden"]])
    before, launches = teacher_state(g), eb.lib().eisen_launch_count()
    for k, temperature in ((300, 1.0), (0, 1.0), (5, 0.0), (5, float("nan"))):
        with pytest.raises(eb.EisenError):
            lm.top_logits(x, k, temperature)
        assert teacher_state(g) == before and eb.lib().eisen_launch_count() == launches
        with pytest.raises(eb.EisenError):
            g.lm_head_top_logits(h, lm.params()[-1], k, temperature)
        assert teacher_state(g) == before and eb.lib().eisen_launch_count() == launches
    lm.top_logits(x, 5)


def test_top_logits_leaves_nothing_behind_when_the_forward_pass_fails():
    g, lm = model(FP32, 1)
    bad = g.alloc_ids([128], np.zeros(128, dtype=np.int32))  # no batch axis: the first attention refuses it
    before = teacher_state(g)
    with pytest.raises(eb.EisenError):
        lm.top_logits(bad, 5)
    assert teacher_state(g) == before


@pytest.mark.parametrize("precision,vocab,tie", [(FP32, 1024, False), (BF16_MIXED, 1020, False)])
def test_head_pieces_refused_before_the_blocks_run(precision, vocab, tie):
    """f32 operands, or an untied head whose rows do not start on 16 bytes."""
    g, lm = model(precision, 1, tie, vocab=vocab)
    lm.set_head_pieces(0)
    ids = np.random.default_rng(0).integers(0, vocab, (2, 64)).astype(np.int32)
    x, t = g.alloc_ids([2, 64], ids), g.alloc_ids([128], ids.reshape(-1))
    before, launches = teacher_state(g), eb.lib().eisen_launch_count()
    with pytest.raises(eb.EisenError, match="linear_cross_entropy"):
        lm.train_micro_step_dev(x, t, 128)
    assert teacher_state(g) == before and eb.lib().eisen_launch_count() == launches
    if precision == FP32:  # the other head takes it (no bf16 head takes such rows)
        lm.set_head_pieces(None)
        assert np.isfinite(g.data(lm.train_micro_step_dev(x, t, 128))[0])


# ------------------------------------------------------------------------------------------ kinds of exponentials
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [0.7, 1.0, 1.5, 2.5, 3.0, 3.5, 4.0, 5.0])
@pytest.mark.parametrize("rows,vocab", [(3, 9001), (2, 40000), (1300, 600), (330, 9001)])
def test_every_kind_of_exponential_in_every_row_form(dtype, temperature, rows, vocab):
    c = Case(dtype, rows, vocab, 9, temperature, 0.6, 0.4).expected()
    loss, row, lse = c.fwd()
    c.check_loss(loss, row, lse)
    d = torch.full_like(c.x, 5.0)
    c.bwd(lse, d)
    c.check_grad(d)
    d.fill_(5.0)
    c.check_loss(*c.fused(d))
    c.check_grad(d, fused=True)
    c.ce = 0.0  # one exponential where no log-sum-exps are asked for
    c.expected()
    d.fill_(5.0)
    loss, row, _ = c.fused(d, lse=False)
    c.check_loss(loss, row)
    c.check_grad(d, fused=True)


# ------------------------------------------------------------------------------------------ the steps in a data-parallel run
@pytest.mark.parametrize("how", ["pieces", "distill"])
def test_steps_announce_finished_blocks(how):
    """after_block comes for every block, last one first, when that block's gradients are final: what buckets are reduced by."""
    r = np.random.default_rng(0)
    g, lm = model(BF16_MIXED, 3)
    ids = r.integers(0, CFG["vocab"], (1, 128)).astype(np.int32)
    y = r.integers(0, CFG["vocab"], 128).astype(np.int32)
    x, t = g.alloc_ids([1, 128], ids), g.alloc_ids([128], y)
    teacher = g.alloc_ids([128, 4], r.integers(0, CFG["vocab"], (128, 4)).astype(np.int32)), g.alloc([128, 4], r.standard_normal((128, 4)))
    seen = []

    def announce(layer):
        seen.append((layer, {p: g.grad(p).copy() for p in lm.params()}))

    if how == "pieces":
        lm.set_head_pieces(256)
        lm.train_micro_step_dev(x, t, 128, checkpoint=True, after_block=announce)
    else:
        lm.distill_micro_step_dev(x, *teacher, 128, target_ids_id=t, kd_weight=0.5, ce_weight=0.5, checkpoint=True, after_block=announce)
    final = {p: g.grad(p) for p in lm.params()}
    layers = [l for l, _ in seen]
    assert sorted(l for l in layers if 0 <= l < CFG["layers"]) == list(range(CFG["layers"]))
    assert layers == sorted(layers, reverse=True)
    done = set()  # parameters whose gradient was already as it is in the end
    for layer, grads in seen:
        now = {p for p in grads if np.array_equal(grads[p], final[p]) and np.any(final[p])}
        assert done <= now
        done = now
    assert len(seen[0][1]) == len(lm.params()) and len(done) >= len(lm.params()) - 2
