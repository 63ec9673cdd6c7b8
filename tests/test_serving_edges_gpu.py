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


def test_a_border_on_the_last_bit_is_drawn_once(ctx):
    """Weights whose sums differ in the last bit with the order of the additions, and a uniform that puts the border on that
    bit, between two CTAs' runs of the row: either neighbour is right to rounding, but it is the same one every time."""
    B, V = 64, 8192  # eight runs of 1024 entries
    p = torch.zeros(B, 1, V, device="cuda")
    for at, y in [(0, "0x1.577c720000000p+0"), (1024, "0x1.3d2b6a0000000p-35"), (2048, "0x1.d260f60000000p-30"),
                  (3 * 1024 + 7, "0x1.7a01b20000000p-32"), (5120, "0x1.577c720000000p+0"), (5121, "0x1.1d655c0000000p-29")]:
        p[:, 0, at] = float.fromhex(y)
    x, ua, us = torch.zeros(B, 0, device="cuda", dtype=torch.int32), torch.zeros(B, 0, device="cuda"), torch.full((B,), 0.5, device="cuda")
    seen = set()
    for _ in range(50):
        n, tok = call_verify(ctx, p, None, x, None, ua, us)
        assert not n.any()
        seen |= set(tok.flatten().tolist())
    assert len(seen) == 1 and seen <= {3 * 1024 + 7, 5120}, seen
