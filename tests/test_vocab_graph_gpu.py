"""The vocabulary-end operators behind Graph and TransformerLM: values and gradients against 64-bit evaluations, whole
training steps against the steps they stand beside."""
import math

import numpy as np
import pytest

from conftest import rel_l2

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import eisen_b200 as eb  # noqa: E402
from eisen_b200.graph import AdamW, BF16_MIXED, FP32, Graph, TransformerLM  # noqa: E402


def new_graph(precision=FP32):
    torch.cuda.init()
    return Graph(precision, torch.cuda.current_stream().cuda_stream)


def f64_distill(x, ids, tv, y, T, kd, ce, lse=None):
    """(loss, gradient) over the rows whose target counts, mean over them."""
    x = torch.tensor(x, dtype=torch.float64, requires_grad=True)
    ids, tv, y = torch.tensor(ids).long(), torch.tensor(tv).double() / T, torch.tensor(y).long()
    on = y >= 0
    tl = torch.tensor(lse).double() if lse is not None else torch.logsumexp(tv, 1)
    lq = tv - tl[:, None]
    lp = torch.log_softmax(x / T, 1).gather(1, ids)
    kl = (lq.exp() * (lq - lp)).sum(1)
    hard = torch.log_softmax(x, 1).gather(1, y.clamp(min=0)[:, None])[:, 0]
    loss = ((kd * T * T * kl - ce * hard) * on).sum() / on.sum()
    value = ((kd * T * T * kl - ce * torch.log(hard.exp() + 1e-8)) * on).sum() / on.sum()
    loss.backward()
    return float(value.detach()), x.grad.numpy()


def data(rows, vocab, k, seed=0):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((rows, vocab)) * 2).astype(np.float32)
    ids = np.stack([r.permutation(vocab)[:k] for _ in range(rows)]).astype(np.int32)
    tv = (r.standard_normal((rows, k)) * 2).astype(np.float32)
    y = r.integers(0, vocab, rows).astype(np.int32)
    y[1::4] = -1
    return x, ids, tv, y


def test_top_logits_op():
    x = np.random.default_rng(1).standard_normal((2, 3, 77)).astype(np.float32)
    g = new_graph()
    v, i, s = g.top_logits(g.alloc([2, 3, 77], x), 5, 2.0)
    assert g.shape(v) == [2, 3, 5] and g.shape(i) == [2, 3, 5] and g.shape(s) == [2, 3]
    order = np.argsort(-x.reshape(6, 77), axis=1, kind="stable")[:, :5]
    assert (g.ids_to_cpu(i).reshape(6, 5) == order).all()
    assert (g.data(v).reshape(6, 5) == np.take_along_axis(x.reshape(6, 77), order, 1)).all()
    want = torch.logsumexp(torch.tensor(x).double() / 2.0, -1).numpy().reshape(-1)
    assert np.abs(g.data(s) - want).max() < 2.0 ** -15


@pytest.mark.parametrize("full", [False, True])
def test_distill_op_value_and_gradient(full):
    x, ids, tv, y = data(9, 500, 7)
    lse = (np.log(np.exp(tv / 2.0).sum(1)) + 0.3).astype(np.float32) if full else None
    want, grad = f64_distill(x, ids, tv, y, 2.0, 0.6, 0.4, lse)
    g = new_graph()
    l = g.alloc([9, 500], x)
    t, v, tid = g.alloc_ids([9, 7], ids), g.alloc([9, 7], tv), g.alloc_ids([9], y)
    s = g.alloc([9], lse) if full else -1
    loss = g.distill(l, t, v, int((y >= 0).sum()), teacher_lse=s, target_ids=tid, temperature=2.0, kd_weight=0.6, ce_weight=0.4)
    assert abs(g.data(loss)[0] - want) < 1e-5 * abs(want) + 1e-6
    g.backward(loss)
    assert rel_l2(g.grad(l), grad) < 2.0 ** -15
    g.backward(loss)  # a second walk adds
    assert rel_l2(g.grad(l), 2 * grad) < 2.0 ** -15


def test_distill_op_under_a_larger_graph():
    """The loss as a term: its gradient comes in from above (f32: twice the loss)."""
    x, ids, tv, y = data(6, 300, 4)
    _, grad = f64_distill(x, ids, tv, y, 1.5, 1.0, 0.0)
    g = new_graph()
    l = g.alloc([6, 300], x)
    t, v, tid = g.alloc_ids([6, 4], ids), g.alloc([6, 4], tv), g.alloc_ids([6], y)
    loss = g.distill(l, t, v, int((y >= 0).sum()), target_ids=tid, temperature=1.5)
    g.backward(g.add(loss, loss))
    assert rel_l2(g.grad(l), 2 * grad) < 2.0 ** -15


@pytest.mark.parametrize("chunk", [0, 5])
@pytest.mark.parametrize("tied", [False, True])
def test_lm_head_distill_f32(chunk, tied):
    x, ids, tv, y = data(12, 200, 6, seed=3)
    r = np.random.default_rng(4)
    H, W = r.standard_normal((12, 32)).astype(np.float32), (r.standard_normal((32, 200)) * 0.3).astype(np.float32)
    want, dx = f64_distill(H.astype(np.float64) @ W.astype(np.float64), ids, tv, y, 2.0, 0.5, 0.5)
    g = new_graph()
    w = g.alloc([200, 32] if tied else [32, 200], W.T if tied else W)
    g.mark_params()
    h = g.alloc([12, 32], H)
    t, v, tid = g.alloc_ids([12, 6], ids), g.alloc([12, 6], tv), g.alloc_ids([12], y)
    args = dict(target_ids=tid, temperature=2.0, kd_weight=0.5, ce_weight=0.5, trans_b=tied, chunk_rows=chunk)
    g.set_no_grad(True)
    assert abs(g.data(g.lm_head_distill(h, w, t, v, int((y >= 0).sum()), **args))[0] - want) < 1e-5
    g.set_no_grad(False)
    loss = g.lm_head_distill(h, w, t, v, int((y >= 0).sum()), **args)
    assert abs(g.data(loss)[0] - want) < 1e-5
    g.backward(loss)
    assert rel_l2(g.grad(h).reshape(12, 32), dx @ W.T) < 1e-5
    dw = H.T @ dx
    assert rel_l2(g.grad(w).reshape(g.shape(w)), dw.T if tied else dw) < 1e-5
    v2, i2, _ = g.lm_head_top_logits(h, w, 3, 1.0, tied, chunk)
    order = np.argsort(-(H @ W), axis=1, kind="stable")[:, :3]
    assert (g.ids_to_cpu(i2).reshape(12, 3) == order).all()


def bf16(a):
    return torch.tensor(a).to(torch.bfloat16)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("piece", [0, 256])
def test_linear_cross_entropy_op(tied, piece):
    """Value, accumulation into both gradients, no_grad evaluation."""
    r = np.random.default_rng(5)
    H, W = r.standard_normal((70, 64)).astype(np.float32), (r.standard_normal((64, 1000)) * 0.2).astype(np.float32)
    y = r.integers(0, 1000, 70).astype(np.int32)
    y[::6] = -1
    hd = bf16(H).double().requires_grad_(True)
    wd = bf16(W).double().requires_grad_(True)
    on = torch.tensor(y >= 0)
    lp = torch.log_softmax(hd @ wd, 1).gather(1, torch.tensor(y).long().clamp(min=0)[:, None])[:, 0]
    loss = -(lp * on).sum() / on.sum()
    loss.backward()
    g = new_graph(BF16_MIXED)
    w = g.alloc([1000, 64] if tied else [64, 1000], W.T if tied else W)
    eye = g.alloc([64, 64], np.eye(64, dtype=np.float32))
    g.mark_params()
    tid = g.alloc_ids([70], y)
    base = g.alloc_pooled([70, 64])
    g.load_tensor_data(base, H)
    h = g.matmul(base, eye)  # an activation with a bf16 gradient
    out = g.linear_cross_entropy(h, w, tid, int((y >= 0).sum()), tied, piece)
    loss = float(loss.detach())
    assert abs(g.data(out)[0] - loss) < 2e-5 * loss
    g.backward(out)
    g.backward(out)  # a second walk adds
    dw = wd.grad.numpy() * 2
    assert rel_l2(g.grad(h).reshape(70, 64), hd.grad.numpy() * 2) < 2.0 ** -8
    assert rel_l2(g.grad(w).reshape(g.shape(w)), dw.T if tied else dw) < 2.0 ** -8
    n = g.tape_len()
    g.set_no_grad(True)
    assert abs(g.data(g.linear_cross_entropy(h, w, tid, int((y >= 0).sum()), tied, piece))[0] - loss) < 2e-5 * loss
    assert g.tape_len() == n


CFG = dict(vocab=1024, hidden=256, heads=4, kv_heads=2, ffn=512, layers=2)


def model(precision, seed, tie=False, **kw):
    c = dict(CFG, **kw)
    g = new_graph(precision)
    lm = TransformerLM(g, c["vocab"], c["hidden"], c["heads"], c["kv_heads"], c["ffn"], c["layers"], tie)
    g.mark_params()
    r = np.random.default_rng(seed)
    for p in lm.params():
        shp = g.shape(p)
        if len(shp) == 2:
            g.load_tensor_data(p, (r.standard_normal(int(np.prod(shp))) * 0.05).astype(np.float32))
    return g, lm


@pytest.mark.parametrize("tie", [False, True])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_train_step_with_head_pieces(tie, checkpoint):
    """The step whose head never holds logits against the step that does: same loss, same gradients up to bf16 logits."""
    r = np.random.default_rng(0)
    ids = r.integers(0, CFG["vocab"], (2, 128)).astype(np.int32)
    y = r.integers(0, CFG["vocab"], 256).astype(np.int32)
    y[::9] = -1
    res = []
    eb.call("eisen_set_deterministic", 1)
    try:
        for pieces in (None, 256):
            g, lm = model(BF16_MIXED, 3, tie)
            lm.set_head_pieces(pieces)
            opt = AdamW(g, lm.params(), 1e-3)
            opt.zero_grad()
            x, t = g.alloc_ids([2, 128], ids), g.alloc_ids([256], y)
            loss = g.data(lm.train_micro_step_dev(x, t, int((y >= 0).sum()), checkpoint))[0]
            grads = [g.grad(p) for p in lm.params()]
            res.append((loss, grads))
            opt.step()
            g.synchronize()
    finally:
        eb.call("eisen_set_deterministic", 0)
    assert abs(res[0][0] - res[1][0]) < 1e-3 * res[0][0]
    assert max(rel_l2(a, b) for a, b in zip(res[1][1], res[0][1])) < 2e-2


@pytest.mark.parametrize("precision", [FP32, BF16_MIXED])
def test_teacher_to_student_step(precision):
    """teacher forward -> top logits -> other graph -> distillation step, against the same loss on whole logits."""
    r = np.random.default_rng(7)
    ids = r.integers(0, CFG["vocab"], (2, 64)).astype(np.int32)
    y = r.integers(0, CFG["vocab"], 128).astype(np.int32)
    y[::5] = -1
    n = int((y >= 0).sum())
    tg, teacher = model(precision, 1, hidden=128, heads=2, kv_heads=1, ffn=256)
    tx = tg.alloc_ids([2, 64], ids)
    before = tg.num_tensors()
    vals, tid, lse = teacher.top_logits(tx, 16, 2.0, chunk_rows=50)
    assert tg.num_tensors() == before + 3 and tg.tape_len() == 0
    whole = tg.data(teacher.forward(tx)).reshape(128, -1)
    tv = tg.data(vals).reshape(128, 16)
    assert rel_l2(tv, -np.sort(-whole, 1)[:, :16]) < (1e-5 if precision == FP32 else 2e-2)
    out = []
    for fused in (True, False):
        g, lm = model(precision, 2)
        opt = AdamW(g, lm.params(), 1e-3)
        opt.zero_grad()
        x, t = g.alloc_ids([2, 64], ids), g.alloc_ids([128], y)
        a, b, c = g.copy_from(tg, tid), g.copy_from(tg, vals), g.copy_from(tg, lse)
        assert (g.ids_to_cpu(a) == tg.ids_to_cpu(tid)).all()
        how = dict(teacher_lse=c, temperature=2.0, kd_weight=0.7, ce_weight=0.3)
        if fused:
            loss = lm.distill_micro_step_dev(x, a, b, n, target_ids_id=t, checkpoint=True, **how)
        else:
            logits = lm.forward(x)
            g.reinterpret_shape(logits, [128, CFG["vocab"]])
            loss = g.distill(logits, a, b, n, target_ids=t, **how)
            g.backward(loss)
        out.append((g.data(loss)[0], [g.grad(p) for p in lm.params()]))
        opt.step()
        g.synchronize()
    tol = 1e-5 if precision == FP32 else 2e-2
    assert abs(out[0][0] - out[1][0]) < (1e-5 if precision == FP32 else 1e-3) * abs(out[1][0])
    assert max(rel_l2(p, q) for p, q in zip(out[0][1], out[1][1])) < tol


def test_distill_step_captured_and_replayed():
    """A whole distillation step as a CUDA graph: replays on new tokens and teacher entries equal eager steps."""
    r = np.random.default_rng(9)
    torch.cuda.init()
    side = torch.cuda.Stream()
    feeds = [(r.integers(0, CFG["vocab"], (1, 64)).astype(np.int32), r.integers(0, CFG["vocab"], (64, 8)).astype(np.int32),
              r.standard_normal((64, 8)).astype(np.float32), r.integers(0, CFG["vocab"], 64).astype(np.int32)) for _ in range(3)]
    eb.call("eisen_set_deterministic", 1)
    try:
        losses = []
        for captured in (False, True):
            g = Graph(BF16_MIXED, side.cuda_stream)
            lm = TransformerLM(g, *[CFG[k] for k in ("vocab", "hidden", "heads", "kv_heads", "ffn", "layers")])
            bufs = [g.alloc_ids([1, 64], feeds[0][0]), g.alloc_ids([64, 8], feeds[0][1]), g.alloc([64, 8], feeds[0][2]), g.alloc_ids([64], feeds[0][3])]
            g.mark_params()
            w = np.random.default_rng(4)
            for p in lm.params():
                shp = g.shape(p)
                if len(shp) == 2:
                    g.load_tensor_data(p, (w.standard_normal(int(np.prod(shp))) * 0.05).astype(np.float32))
            views = []
            for b, shp, ty in zip(bufs, ((1, 64), (64, 8), (64, 8), (64,)), ("<i4", "<i4", "<f4", "<i4")):
                ptr = g.tensor_ptrs(b)[0]

                class _V:
                    __cuda_array_interface__ = {"shape": shp, "typestr": ty, "data": (ptr, False), "version": 2}

                views.append(torch.as_tensor(_V(), device="cuda:0"))

            def step():
                g.clear_activations()
                g.tape_clear()
                return lm.distill_micro_step_dev(bufs[0], bufs[1], bufs[2], 64, target_ids_id=bufs[3], temperature=2.0, kd_weight=0.5, ce_weight=0.5)

            got, made = [], []
            step()
            g.synchronize()
            rec = g.capture(lambda: made.append(step())) if captured else None
            if captured:  # the loss stays where it was during the capture
                ptr = g.tensor_ptrs(made[0])[0]

                class _L:
                    __cuda_array_interface__ = {"shape": (1,), "typestr": "<f4", "data": (ptr, False), "version": 2}

                lview = torch.as_tensor(_L(), device="cuda:0")
            for f in feeds:
                with torch.cuda.stream(side):
                    for v, a in zip(views, f):
                        v.copy_(torch.tensor(a))
                if captured:
                    rec.replay()
                    g.synchronize()
                    got.append(float(lview))
                else:
                    got.append(float(g.data(step())[0]))
            losses.append(got)
            if rec:
                rec.close()
    finally:
        eb.call("eisen_set_deterministic", 0)
    assert losses[0] == losses[1]


def test_graph_refusals():
    g = new_graph(FP32)
    l, h, w = g.alloc([4, 10], np.zeros(40)), g.alloc([4, 8], np.zeros(32)), g.alloc([8, 10], np.zeros(80))
    ids, tv, y = g.alloc_ids([4, 2], np.zeros(8)), g.alloc([4, 2], np.zeros(8)), g.alloc_ids([4], np.zeros(4))
    n = g.num_tensors()
    for f in (lambda: g.linear_cross_entropy(h, w, y, 4),              # bf16 only
              lambda: g.top_logits(l, 11), lambda: g.top_logits(l, 0),
              lambda: g.lm_head_top_logits(l, w, 2),                    # widths differ
              lambda: g.distill(l, tv, ids, 4),                         # ids and logits exchanged
              lambda: g.distill(l, ids, g.alloc([4, 3], np.zeros(12)), 4),
              lambda: g.distill(l, ids, tv, 4, teacher_lse=l),
              lambda: g.distill(l, ids, tv, 4, target_ids=ids),
              lambda: g.distill(l, ids, tv, 4, ce_weight=0.5),          # no targets
              lambda: g.distill(l, ids, tv, 4, temperature=0.0),
              lambda: g.lm_head_distill(l, w, ids, tv, 4),
              lambda: g.ids_to_cpu(l), lambda: g.distill(999, ids, tv, 4)):
        with pytest.raises(eb.EisenError):
            f()
    assert g.tape_len() == 0 and g.num_tensors() >= n
    assert math.isfinite(float(g.data(g.distill(l, ids, tv, 4))[0]))
