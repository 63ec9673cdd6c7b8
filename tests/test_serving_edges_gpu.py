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


# ---------------------------------------------------------------------------------------------------- a context's own rows


def test_rows_of_a_context_s_fp32_cache_are_refused_as_bf16(M):
    """The view of a context that keeps fp32 rows (the default): the attention calls read bf16 and refuse it, eviction takes
    it with its own type only; nothing is launched.  A bf16 context's rows stay open to all of them."""
    g = gen(61)
    q = rn(g, 1, 1, 32, D)
    lens = torch.tensor([3], device="cuda", dtype=torch.int32)
    rows = rn(g, 1, 2, 8, D)
    out, lse = torch.zeros_like(q), torch.zeros(1, 1, 32, device="cuda")
    w, pos = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 2, 64, device="cuda", dtype=torch.int32)
    new = torch.zeros_like(lens)
    for kv_dtype in (M.KV_F32, M.KV_BF16):
        c = M.Ctx(num_layers=4, max_seq=64, n_seqs=2, kv_dtype=kv_dtype)
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        k, v, seq_stride, head_stride, n = c.kv_cache_view(3, 1)
        assert n == 0
        attn = attn_args(q, None, None, None, rows, rows, lens, out, lse)
        prefix = dict(prefix_head_stride=head_stride, prefix_row_stride=D, prefix_len=3)
        own = dict(own_seq_stride=seq_stride, own_head_stride=head_stride, own_row_stride=D, own_cap=8)
        wts = weights_args(q, rows, lens, lse, w)
        ev = dict(n_seqs=1, num_kv_heads=2, cap=8, seq_stride=seq_stride, head_stride=head_stride, row_stride=D, budget=2, lens=lens.data_ptr(),
                  next_pos=lens.data_ptr(), weights=w.data_ptr(), positions=pos.data_ptr(), map_seq_stride=128, map_head_stride=64,
                  weights_out=w.data_ptr(), positions_out=pos.data_ptr(), lens_out=new.data_ptr())
        r = rows.data_ptr()
        calls = [lambda: c.shared_prefix_attn_dev(**attn, prefix_k=k, prefix_v=r, **prefix),
                 lambda: c.shared_prefix_attn_dev(**attn, prefix_k=r, prefix_v=v, **prefix),
                 lambda: c.shared_prefix_attn_dev(**{**attn, "own_k": k, **own}),
                 lambda: c.shared_prefix_attn_dev(**{**attn, "own_v": v + 512, **own}),
                 lambda: c.attn_weights_accumulate_dev(**{**wts, "k": k, "k_head_stride": head_stride, "cap": 8})]
        before = c.launch_count
        for call in calls:
            if kv_dtype == M.KV_F32:
                with pytest.raises(M.MfcError, match="fp32 cache"):
                    call()
            else:
                call()
        other = M.KV_BF16 if kv_dtype == M.KV_F32 else M.KV_F32
        with pytest.raises(M.MfcError, match="kv_dtype"):
            c.kv_evict_dev(**ev, k=k, v=v, kv_dtype=other)
        assert c.launch_count == before + (0 if kv_dtype == M.KV_F32 else 9)
        c.kv_evict_dev(**ev, k=k, v=v, kv_dtype=kv_dtype)
        c.synchronize()
        assert new.tolist() == [2]
        c.close()


# ---------------------------------------------------------------------------------------------------- failures and captures


@pytest.mark.parametrize("call", ["attn", "weights"])
def test_a_call_after_a_lost_load_computes_what_it_should(ctx, M, call):
    """The call that follows a failed one, the same entry point: its results against the 64-bit form."""
    g = gen(62)
    B, T, H, Hkv, P, cap = 3, 2, 32, 2, 700, 300
    q, ok, ov = rn(g, B, T, H, D), rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    pk, pv = rn(g, Hkv, P, D), rn(g, Hkv, P, D)
    lens = torch.tensor([300, 130, 5], device="cuda", dtype=torch.int32)
    ro, rl, bo, bl = attn_ref(q, None, pk, pv, ok, ov, lens)
    out, lse = torch.zeros(B, T, H, D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, T, H, device="cuda")
    given = rl.float().contiguous()
    w = torch.zeros(B, Hkv, cap, device="cuda")
    run = (lambda: ctx.shared_prefix_attn_dev(**attn_args(q, None, pk, pv, ok, ov, lens, out, lse))) if call == "attn" else (
        lambda: ctx.attn_weights_accumulate_dev(**weights_args(q, ok, lens, given, w)))
    ctx.set_tuning("gqa_wait_spins", 2000)
    ctx.set_tuning("gqa_inject_lost_load", 1)
    try:
        run()
        with pytest.raises(M.MfcError, match="did not arrive"):
            ctx.synchronize()
    finally:
        ctx.set_tuning("gqa_inject_lost_load", 0)
        ctx.set_tuning("gqa_wait_spins", 0)
    for t in (out, lse):
        t.fill_(float("nan"))
    w.zero_()
    run()
    ctx.synchronize()
    if call == "attn":
        assert ((out.double() - ro).abs() <= bo).all() and ((lse.double() - rl).abs() <= bl).all()
    else:
        ref, tol = weights_ref(q, ok, lens, given, torch.zeros_like(w), 1.0)
        assert ((w.double() - ref).abs() <= tol).all()


def test_the_lse_of_a_replayed_call_follows_the_lengths(ctx):
    g = gen(63)
    B, T, H, Hkv, P, cap = 20, 3, 32, 2, 0, 300
    q, ok, ov = rn(g, B, T, H, D), rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    lens = lens_for(g, B, T, cap)
    out, lse = torch.zeros_like(q), torch.zeros(B, T, H, device="cuda")
    s, home = torch.cuda.Stream(), torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    ctx.set_stream(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ctx.shared_prefix_attn_dev(**attn_args(q, None, None, None, ok, ov, lens, out, lse))
    ctx.set_stream(home)
    for cut in (0, 5, 130):
        lens.copy_((lens - cut).clamp(min=0))
        graph.replay()
        torch.cuda.synchronize()
        ro, rl, bo, bl = attn_ref(q, None, None, None, ok, ov, lens)
        none = torch.isinf(rl)
        assert torch.equal(torch.isneginf(lse), none) and none.any()
        assert ((lse.double() - rl).abs()[~none] <= bl[~none]).all() and ((out.double() - ro).abs() <= bo).all()


# ---------------------------------------------------------------------------------------------------- limits


def test_limits_beside_the_field_ranges_are_refused(ctx, M):
    """Sizes whose single fields are in range: tiles, partial results and lists of moves of one sequence.  Refused on the host,
    before anything is read."""
    t = torch.zeros(4096, device="cuda", dtype=torch.bfloat16)
    P = t.data_ptr()
    q = dict(softmax_scale=SCALE, q=P, q_seq_stride=256, q_token_stride=256, q_head_stride=256)
    prefix = dict(prefix_k=P, prefix_v=P, prefix_head_stride=256, prefix_row_stride=256, own_lens=P, out=P)
    before = ctx.launch_count
    with pytest.raises(M.MfcError, match="2\\^26"):
        ctx.shared_prefix_attn_dev(**q, **prefix, n_seqs=1, n_tokens=1, num_attn_heads=8, num_kv_heads=8, prefix_len=1 << 30)
    with pytest.raises(M.MfcError, match="scratch"):
        ctx.shared_prefix_attn_dev(**q, **prefix, n_seqs=1, n_tokens=16, num_attn_heads=8192, num_kv_heads=1024, prefix_len=200)
    with pytest.raises(M.MfcError, match="too many rows"):
        ctx.attn_weights_accumulate_dev(**q, n_seqs=128, n_tokens=1, num_attn_heads=1, num_kv_heads=1, decay=1.0, k=P, k_seq_stride=256,
                                        k_head_stride=256, k_row_stride=256, cap=1 << 30, lens=P, lse=P, weights=P)
    with pytest.raises(M.MfcError, match="scratch"):
        ctx.kv_evict_dev(n_seqs=1, num_kv_heads=1024, kv_dtype=M.KV_BF16, cap=262144, k=P, v=P + 512, seq_stride=256, head_stride=256, row_stride=256,
                         budget=131072, lens=P, next_pos=P, weights=P, positions=P, map_seq_stride=1, map_head_stride=1, weights_out=P,
                         positions_out=P, lens_out=P + 512)
    assert ctx.launch_count == before


def test_as_many_kv_heads_as_always_fit(ctx):
    """360 tiles of query rows in one sequence, the number that the header promises."""
    g = gen(64)
    for T, H, Hkv in [(1, 360, 360), (16, 16 * 180, 180)]:
        q = rn(g, 1, T, H, D)
        pk, pv = rn(g, Hkv, 300, D), rn(g, Hkv, 300, D)
        ok, ov = rn(g, 1, Hkv, 40, D), rn(g, 1, Hkv, 40, D)
        check_attn(ctx, q, None, pk, pv, ok, ov, torch.tensor([37], device="cuda", dtype=torch.int32))


def test_large_values_under_a_growing_maximum(ctx):
    """V near 2^62, and scores that pass each row's first maximum by up to 2^32 and by more: nothing overflows."""
    g = gen(65)
    B, T, H, Hkv, P, cap = 5, 2, 32, 2, 1400, 200
    q, pk, pv = rn(g, B, T, H, D, scale=2.0), rn(g, Hkv, P, D), rn(g, Hkv, P, D, scale=2.0 ** 60)
    pk *= torch.linspace(0.2, 4.0, P, device="cuda").view(1, P, 1).to(torch.bfloat16)
    ok, ov = rn(g, B, Hkv, cap, D, scale=5.0), rn(g, B, Hkv, cap, D, scale=2.0 ** 60)
    check_attn(ctx, q, q, pk, pv, ok, ov, lens_for(g, B, T, cap))


def test_calls_from_a_thread_that_has_not_used_the_gpu(ctx):
    """The first thing a host thread does on the GPU is the call itself."""
    import threading

    g = gen(66)
    B, T, H, Hkv, P, cap = 3, 2, 32, 2, 300, 100
    q, pk, pv, ok, ov = rn(g, B, T, H, D), rn(g, Hkv, P, D), rn(g, Hkv, P, D), rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    lens = lens_for(g, B, T, cap)
    out, lse, w = torch.zeros_like(q), torch.zeros(B, T, H, device="cuda"), torch.zeros(B, Hkv, cap, device="cuda")
    torch.cuda.synchronize()
    raised = []

    def work(call):
        try:
            call()
        except Exception as e:  # noqa: BLE001 - handed to the test's thread
            raised.append(e)

    for call in (lambda: ctx.shared_prefix_attn_dev(**attn_args(q, None, pk, pv, ok, ov, lens, out, lse)),
                 lambda: ctx.attn_weights_accumulate_dev(**weights_args(q, ok, lens, lse, w))):
        t = threading.Thread(target=work, args=(call,))
        t.start()
        t.join()
    assert not raised, raised
    ctx.synchronize()
    ro, rl, bo, bl = attn_ref(q, None, pk, pv, ok, ov, lens)
    assert ((out.double() - ro).abs() <= bo).all() and ((lse.double() - rl).abs() <= bl).all()
    ref, tol = weights_ref(q, ok, lens, lse, torch.zeros_like(w), 1.0)
    assert ((w.double() - ref).abs() <= tol).all()


def test_a_capture_joined_from_two_streams(ctx):
    """Inputs written on another stream of the same capture, just before the call and just after a call of the context: each call
    follows both."""
    g = gen(67)
    B, T, H, Hkv, P, cap = 20, 2, 32, 2, 900, 200
    src, pk, pv, ok, ov = rn(g, B, T, H, D), rn(g, Hkv, P, D), rn(g, Hkv, P, D), rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    q, other = torch.zeros_like(src), torch.zeros(1 << 27, device="cuda")
    lens, lens2 = lens_for(g, B, T, cap), torch.zeros(B, device="cuda", dtype=torch.int32)
    out, lse, w = torch.zeros_like(q), torch.zeros(B, T, H, device="cuda"), torch.zeros(B, Hkv, cap, device="cuda")
    main, side, home = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    ctx.set_stream(side.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        other.add_(1)  # (some 0.2 ms, so that a call that does not wait for what follows is seen)
        q.copy_(src)
        side.wait_stream(main)
        ctx.shared_prefix_attn_dev(**attn_args(q, None, pk, pv, ok, ov, lens, out, lse))
        other.add_(1)
        lens2.copy_(lens)
        side.wait_stream(main)
        ctx.attn_weights_accumulate_dev(**weights_args(q, ok, lens2, lse, w))
        main.wait_stream(side)
    ctx.set_stream(home)
    for _ in range(2):
        src.copy_(rn(g, B, T, H, D))
        w.zero_()
        lens2.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ro, rl, bo, bl = attn_ref(src, None, pk, pv, ok, ov, lens)
        assert ((out.double() - ro).abs() <= bo).all() and ((lse.double() - rl).abs() <= bl).all()
        ref, tol = weights_ref(src, ok, lens, lse, torch.zeros_like(w), 1.0)
        assert ((w.double() - ref).abs() <= tol).all() and bool((w > 0).any())


def test_written_arrays_that_sequences_or_heads_would_share_are_refused(ctx, M):
    """A stride of 0 along an axis of more than one place, in what a call writes; along an axis of one it means nothing."""
    k, v = (torch.zeros(2, 2, 8, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    w, pos = torch.zeros(2, 2, 8, device="cuda"), torch.zeros(2, 2, 8, device="cuda", dtype=torch.int32)
    lens, new = torch.zeros(2, device="cuda", dtype=torch.int32), torch.zeros(2, device="cuda", dtype=torch.int32)
    q, lse = torch.zeros(2, 1, 2, D, device="cuda", dtype=torch.bfloat16), torch.zeros(2, 1, 2, device="cuda")
    ev = dict(n_seqs=2, num_kv_heads=2, kv_dtype=M.KV_BF16, cap=8, k=k.data_ptr(), v=v.data_ptr(), seq_stride=k.stride(0), head_stride=k.stride(1),
              row_stride=D, budget=2, lens=lens.data_ptr(), next_pos=lens.data_ptr(), weights=w.data_ptr(), positions=pos.data_ptr(),
              map_seq_stride=16, map_head_stride=8, weights_out=w.data_ptr(), positions_out=pos.data_ptr(), lens_out=new.data_ptr())
    wts = weights_args(q, k, lens, lse, w)
    before = ctx.launch_count
    for fn, base, bad in [(ctx.kv_evict_dev, ev, ["seq_stride", "head_stride", "map_seq_stride", "map_head_stride"]),
                          (ctx.attn_weights_accumulate_dev, wts, ["weights_seq_stride", "weights_head_stride"])]:
        for field in bad:
            with pytest.raises(M.MfcError, match="different places"):
                fn(**{**base, field: 0})
    assert ctx.launch_count == before
    ctx.kv_evict_dev(**{**ev, "n_seqs": 1, "seq_stride": 0, "map_seq_stride": 0})
    ctx.attn_weights_accumulate_dev(**{**wts, "n_seqs": 1, "weights_seq_stride": 0})
    ctx.synchronize()
