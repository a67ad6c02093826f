"""Refusals of the vocabulary-end operators: every one of them is raised before anything is launched."""
import pytest

import eisen_b200 as eb

A = 1 << 20  # an aligned address that is never read


def top(**kw):
    a = dict(logits=A, ld=100, values=A, ids=A, lse=None, rows=2, vocab=100, k=5, temperature=1.0, dtype=eb.F32)
    a.update(kw)
    eb.call("eisen_top_logits", None, *a.values())


@pytest.mark.parametrize("kw", [dict(k=0), dict(k=257, vocab=1000, ld=1000), dict(k=101), dict(ld=99), dict(temperature=0.0), dict(temperature=-1.0),
                                dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e-42), dict(rows=-1), dict(vocab=0),
                                dict(rows=1 << 31), dict(vocab=1 << 31, ld=1 << 31), dict(logits=None), dict(values=None), dict(ids=None),
                                dict(dtype=3), dict(logits=A + 2)])
def test_top_logits_refuses(kw):
    with pytest.raises(eb.EisenError, match="top_logits"):
        top(**kw)


def distill(which, **kw):
    a = dict(logits=A, ld=100, ids=A, t=A, t_lse=None, targets=A, lse=A, d=A, ld_d=100, loss=None, row_loss=A, grad=None, rows=2, vocab=100, k=5,
             ignore=-1, temperature=1.0, kd=1.0, ce=0.5, scale=1.0, dtype=eb.F32, acc=0)
    a.update(kw)
    head = (None, a["logits"], a["ld"], a["ids"], a["t"], a["t_lse"], a["targets"])
    how = (a["rows"], a["vocab"], a["k"], a["ignore"], a["temperature"], a["kd"], a["ce"])
    if which == "fwd":
        eb.call("eisen_distill_fwd", *head, a["loss"], a["row_loss"], a["lse"], *how, a["dtype"], None)
    elif which == "bwd":
        eb.call("eisen_distill_bwd", *head, a["lse"], a["d"], a["ld_d"], a["grad"], *how, a["dtype"], a["acc"])
    else:
        eb.call("eisen_distill_fused", *head, a["d"], a["ld_d"], a["loss"], a["row_loss"], a["lse"], *how, a["scale"], a["dtype"], None)


@pytest.mark.parametrize("which", ["fwd", "bwd", "fused"])
@pytest.mark.parametrize("kw", [dict(k=0), dict(k=1025), dict(ld=99), dict(temperature=0.0), dict(temperature=float("nan")),
                                dict(temperature=float("inf")), dict(rows=-1), dict(vocab=0), dict(rows=1 << 31), dict(logits=None), dict(ids=None),
                                dict(t=None), dict(targets=None), dict(dtype=2), dict(logits=A + 1)])
def test_distill_refuses(which, kw):
    with pytest.raises(eb.EisenError, match="distill_" + which):
        distill(which, **kw)


@pytest.mark.parametrize("which,kw", [("fwd", dict(row_loss=None)), ("fused", dict(row_loss=None)), ("fused", dict(d=None)), ("bwd", dict(d=None)),
                                      ("bwd", dict(lse=None)), ("bwd", dict(ld_d=99)), ("fused", dict(ld_d=99)), ("bwd", dict(d=A + 2))])
def test_distill_refuses_outputs(which, kw):
    with pytest.raises(eb.EisenError, match="distill_" + which):
        distill(which, **kw)


def linear(which, **kw):
    a = dict(h=A, ldh=64, w=A, ldw=104, tied=0, targets=A, loss=None, row_loss=A, lse=A, grad=None, dh=A, dw=A, lddw=104, dwt=eb.BF16, ws=A, rows=4,
             k=64, vocab=100, piece=0)
    a.update(kw)
    ops = (None, a["h"], a["ldh"], a["w"], a["ldw"], a["tied"], a["targets"])
    if which == "fwd":
        eb.call("eisen_linear_ce_fwd", *ops, a["loss"], a["row_loss"], a["lse"], a["ws"], a["rows"], a["k"], a["vocab"], -1, 1.0, None, None)
    else:
        eb.call("eisen_linear_ce_bwd", *ops, a["lse"], a["grad"], a["dh"], 0, a["dw"], a["lddw"], a["dwt"], 0, a["ws"], a["rows"], a["k"], a["vocab"],
                a["piece"], -1, 1.0, None)


@pytest.mark.parametrize("which", ["fwd", "bwd"])
@pytest.mark.parametrize("kw", [dict(h=None), dict(w=None), dict(targets=None), dict(ws=None), dict(lse=None), dict(ldh=56), dict(ldw=96),
                                dict(tied=1, ldw=56), dict(ldh=66), dict(ldw=108), dict(h=A + 8), dict(w=A + 2), dict(ws=A + 4), dict(rows=-1),
                                dict(k=0), dict(vocab=0), dict(rows=1 << 31), dict(vocab=1 << 31, ldw=1 << 31, lddw=1 << 31)])
def test_linear_ce_refuses(which, kw):
    with pytest.raises(eb.EisenError, match="linear_ce_" + which):
        linear(which, **kw)


@pytest.mark.parametrize("kw", [dict(dh=None, dw=None), dict(lddw=99), dict(dwt=2), dict(dh=A + 2), dict(dw=A + 4), dict(k=60, ldh=64)])
def test_linear_ce_bwd_refuses(kw):
    with pytest.raises(eb.EisenError, match="linear_ce_bwd"):
        linear("bwd", **kw)


def test_linear_ce_workspace():
    need = eb.lib().eisen_linear_ce_workspace_bytes
    assert need(16384, 2048, 32000, 0, 0) < 32 << 20            # 8 bytes per row and 256 columns, no logits
    assert need(16384, 2048, 32000, 0, 1) < (256 + 140) << 20   # one slab, and dh in f32
    assert need(16384, 2048, 32000, 256, 1) < need(16384, 2048, 32000, 0, 1)
    assert need(5, 384, 8192, 0, 1) >= need(5, 384, 8192, 0, 0)
    assert need(0, 64, 100, 0, 1) > 0
