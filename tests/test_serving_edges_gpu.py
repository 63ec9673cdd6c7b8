"""Serving a batch from cached rows: inputs at the edge of what the header allows, on a B200.  Helpers, references and their
bounds are those of test_serving_gpu."""
import pytest

torch = pytest.importorskip("torch")

from tests.test_serving_gpu import (  # noqa: E402
    D, SCALE, attn_args, attn_ref, call_verify, check_attn, ctx, gen, lens_for, M, rn, verify_ref, weights_args, weights_ref)  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------- verification


@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("V", [5, 3000, 70001])
def test_draft_probabilities_that_are_nan_or_negative_count_as_zero(ctx, V, pad):
    """In the acceptance test and in the residual, at the drafted token and elsewhere; those of the target likewise."""
    nan = float("nan")
    #       p                            q                  drafted  u_accept -> accepted, tokens
    rows = [({0: 0.25, 3: 0.75}, {0: nan, 1: 1.0}, 0, 0.5, 1, [0, 2]),        # u * 0 < 0.25
            ({0: 0.25, 3: 0.75}, {0: -0.5, 1: 1.0}, 0, 0.5, 1, [0, 2]),
            ({3: 1.0}, {0: -1.0}, 0, 0.5, 0, [3, -1]),                        # 0 < 0 is refused
            ({0: -0.5, 3: 1.0}, {0: -1.0}, 0, 0.9, 0, [3, -1]),               # so is it where p is negative too
            ({0: nan, 3: 1.0}, {0: -1.0}, 0, 0.9, 0, [3, -1]),
            ({2: 0.6, 4: 0.4}, {1: 1.0, 2: nan}, 1, 0.5, 0, [2, -1]),         # the residual at 2 is p, not nothing
            ({4: 1.0}, {1: 1.0, 2: -0.7}, 1, 0.5, 0, [4, -1]),                # and nothing where p is nothing
            ({2: -1.0, 4: 1.0}, {1: 1.0, 2: -7.0}, 1, 0.5, 0, [4, -1]),
            ({4: 0.5}, {1: 1.0, 4: float("inf")}, 1, 0.5, 0, [4, -1])]        # no residual anywhere: from p
    B = len(rows)
    wide_p, wide_q = torch.zeros(B, 2, V + pad, device="cuda"), torch.zeros(B, 1, V + pad, device="cuda")
    p, q = wide_p[..., :V], wide_q[..., :V]
    x = torch.tensor([[r[2]] for r in rows], device="cuda", dtype=torch.int32)
    ua = torch.tensor([[r[3]] for r in rows], device="cuda")
    p[:, 1, 2] = 1.0
    for b, (pv, qv, *_) in enumerate(rows):
        for v, y in pv.items():
            p[b, 0, v] = y
        for v, y in qv.items():
            q[b, 0, v] = y
    n, tok = call_verify(ctx, p, q, x, None, ua, torch.zeros(B, device="cuda"))
    assert n.tolist() == [r[4] for r in rows]
    assert tok.tolist() == [r[5] for r in rows]
