"""Refusals of the vocabulary-end operators that lie at the edge of their documentation."""
import pytest

import eisen_b200 as eb
from test_vocab_ops_cpu import A, distill, linear


@pytest.mark.parametrize("which", ["bwd", "fused"])
@pytest.mark.parametrize("ld,ld_d", [(100, 104), (104, 100), (200, 100)])
def test_gradient_over_the_logits_needs_their_row_stride(which, ld, ld_d):
    """Otherwise a row's gradient would go over the logits of another row."""
    with pytest.raises(eb.EisenError, match="row stride"):
        distill(which, logits=A, d=A, ld=ld, ld_d=ld_d)


@pytest.mark.parametrize("kw", [dict(h=A, dh=A), dict(w=A, dw=A)])
def test_gradients_do_not_go_over_their_operands(kw):
    """The hidden states and the weight are read again for every piece and for the other gradient."""
    other = {"h": 2 * A, "w": 3 * A, "dh": 4 * A, "dw": 5 * A, "ws": 6 * A}
    with pytest.raises(eb.EisenError, match="over"):
        linear("bwd", **{**other, **kw})
