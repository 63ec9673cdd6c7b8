"""Serving a batch from cached rows, through the C ABI on a B200, against the operators' definitions in 64 bits:
attention over a shared prefix, accumulation of attention weights, eviction, verification of drafted tokens.

Tolerances.  Scores: 256 products of bf16 pairs (exact in fp32) summed in fp32, each addition off by at most 2^-23 of the
partial sum (the tensor core truncates), so |ds| <= 256 * 2^-23 * scale * sum|q k|, plus 2^-22 (|s| + |m|) for the
exponent's argument.  Probabilities enter P V rounded to bf16 (half a step: 2^-8), outputs are rounded to bf16 once."""
import math

import pytest

torch = pytest.importorskip("torch")

D = 256
SCALE = 1.0 / 16.0
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import moeflux_b200

    return moeflux_b200


@pytest.fixture(scope="module")
def ctx(M):
    c = M.Ctx(num_layers=4, max_seq=512, n_seqs=3, kv_dtype=M.KV_BF16)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.synchronize()
    c.close()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def visible(lens, T, cap):
    """[B, T, cap]: which own rows each query token sees."""
    n = lens.view(-1, 1, 1) - (T - 1 - torch.arange(T, device=lens.device)).view(1, T, 1)
    return torch.arange(cap, device=lens.device).view(1, 1, cap) < n


def attn_args(q, gate, pk, pv, ok, ov, lens, out, lse, scale=SCALE):
    B, T, H, _ = q.shape
    Hkv = (pk if pk is not None else ok).shape[0 if pk is not None else 1]
    a = dict(n_seqs=B, n_tokens=T, num_attn_heads=H, num_kv_heads=Hkv, softmax_scale=scale, q=q.data_ptr(),
             q_seq_stride=q.stride(0), q_token_stride=q.stride(1), q_head_stride=q.stride(2), own_lens=lens.data_ptr(),
             out=out.data_ptr(), lse=lse.data_ptr() if lse is not None else None)
    if gate is not None:
        a.update(gate=gate.data_ptr(), gate_seq_stride=gate.stride(0), gate_token_stride=gate.stride(1),
                 gate_head_stride=gate.stride(2))
    if pk is not None:
        a.update(prefix_k=pk.data_ptr(), prefix_v=pv.data_ptr(), prefix_head_stride=pk.stride(0),
                 prefix_row_stride=pk.stride(1), prefix_len=pk.shape[1])
    if ok is not None:
        a.update(own_k=ok.data_ptr(), own_v=ov.data_ptr(), own_seq_stride=ok.stride(0), own_head_stride=ok.stride(1),
                 own_row_stride=ok.stride(2), own_cap=ok.shape[2])
    return a


def attn_ref(q, gate, pk, pv, ok, ov, lens, scale=SCALE):
    """(out, lse, bound on |d out|, bound on |d lse|) in fp64, one sequence at a time."""
    B, T, H, _ = q.shape
    Hkv = pk.shape[0] if pk is not None else ok.shape[1]
    G = H // Hkv
    outs, lses, bo, bl = [], [], [], []
    zero = torch.zeros(Hkv, 0, D, device="cuda", dtype=torch.float64)
    cap = ok.shape[2] if ok is not None else 0
    P = pk.shape[1] if pk is not None else 0
    vis = visible(lens, T, cap)
    for b in range(B):
        n = max(0, min(int(lens[b]), cap))
        k = torch.cat([pk.double() if P else zero, ok[b, :, :n].double() if n else zero], 1)
        v = torch.cat([pv.double() if P else zero, ov[b, :, :n].double() if n else zero], 1)
        qq = q[b].double().view(T, Hkv, G, D)
        s = torch.einsum("thgd,hjd->thgj", qq, k) * scale
        a = torch.einsum("thgd,hjd->thgj", qq.abs(), k.abs()) * scale
        see = torch.cat([torch.ones(T, P, dtype=torch.bool, device="cuda"), vis[b, :, :n]], 1).view(T, 1, 1, -1)
        s = s.masked_fill(~see, float("-inf"))
        z = torch.logsumexp(s, -1, keepdim=True) if s.shape[-1] else torch.full((T, Hkv, G, 1), float("-inf"), device="cuda", dtype=torch.float64)
        p = torch.nan_to_num(torch.exp(s - z)) * see
        o = torch.einsum("thgj,hjd->thgd", p, v)
        ov_abs = torch.einsum("thgj,hjd->thgd", p, v.abs())
        # error of a score, largest over the rows that matter
        smax = torch.where(see, s.abs(), 0.0).amax(-1, keepdim=True) if s.shape[-1] else torch.zeros_like(z)
        amax = torch.where(see, a, 0.0).amax(-1, keepdim=True) if s.shape[-1] else torch.zeros_like(z)
        ds = 256 * 2.0 ** -23 * amax + 2.0 ** -21 * smax + 2.0 ** -20
        gt = torch.sigmoid(gate[b].double()).view(T, Hkv, G, D) if gate is not None else 1.0
        o = o * gt
        outs.append(o.reshape(T, H, D))
        bo.append((2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * ds + 1e-5) * ov_abs * gt).reshape(T, H, D))
        lses.append(z.reshape(T, H))
        bl.append(ds.reshape(T, H) + 2.0 ** -22 * torch.nan_to_num(z, neginf=0.0).abs().reshape(T, H))
    return torch.stack(outs), torch.stack(lses), torch.stack(bo), torch.stack(bl)


def check_attn(ctx, q, gate, pk, pv, ok, ov, lens, scale=SCALE):
    B, T, H, _ = q.shape
    out = torch.full((B, T, H, D), float("nan"), device="cuda", dtype=torch.bfloat16)
    lse = torch.full((B, T, H), float("nan"), device="cuda")
    ctx.shared_prefix_attn_dev(**attn_args(q, gate, pk, pv, ok, ov, lens, out, lse, scale))
    ctx.synchronize()
    ro, rl, bo, bl = attn_ref(q, gate, pk, pv, ok, ov, lens, scale)
    none = torch.isinf(rl)
    assert torch.equal(torch.isneginf(lse), none)
    assert ((lse.double() - rl).abs()[~none] <= bl[~none]).all()
    assert torch.isfinite(out.float()).all()
    over = (out.double() - ro).abs() - bo
    assert (over <= 0).all(), (float(over.max()), float((out.double() - ro).abs().max()))
    return out, lse


def lens_for(g, B, T, cap):
    lens = torch.randint(min(T, cap), cap + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = cap
    if B > 2:
        lens[1] = 0
        lens[2] = min(1, cap)  # fewer rows than tokens when T > 1
    return lens


@pytest.mark.parametrize("B,T,H,Hkv,P,cap", [
    (1, 1, 32, 2, 1, 1), (1, 1, 32, 2, 0, 1), (1, 1, 32, 2, 300, 0), (2, 1, 32, 2, 127, 5), (2, 1, 32, 2, 128, 128),
    (3, 2, 10, 2, 129, 257), (5, 3, 24, 2, 1000, 300), (9, 1, 7, 1, 515, 130), (4, 16, 16, 1, 200, 64), (3, 9, 16, 1, 0, 300),
    (40, 4, 32, 2, 2000, 640), (17, 5, 8, 8, 640, 200), (300, 1, 16, 1, 130, 140), (1, 1, 32, 2, 40000, 1), (33, 2, 32, 2, 9000, 40)])
def test_shared_prefix_attn(ctx, B, T, H, Hkv, P, cap):
    g = gen(B * 1000 + P + cap)
    q = rn(g, B, T, H, D, scale=1.5)
    gate = rn(g, B, T, H, D) if B % 2 else None
    pk, pv = (rn(g, Hkv, P, D), rn(g, Hkv, P, D)) if P else (None, None)
    ok, ov = (rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)) if cap else (None, None)
    check_attn(ctx, q, gate, pk, pv, ok, ov, lens_for(g, B, T, cap))


@pytest.mark.parametrize("B,T,H,Hkv,P,cap", [(64, 2, 32, 2, 400, 100), (37, 3, 24, 2, 1500, 90), (20, 2, 32, 2, 3000, 200), (4, 1, 32, 2, 20000, 30)])
def test_shared_prefix_attn_with_many_and_few_rows_to_join(ctx, B, T, H, Hkv, P, cap):
    """From 64 to 4096 query rows, from two to some seventy partials a row."""
    g = gen(B + P)
    q, pk, pv = rn(g, B, T, H, D), rn(g, Hkv, P, D), rn(g, Hkv, P, D)
    ok, ov = rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    check_attn(ctx, q, q if B % 2 else None, pk, pv, ok, ov, lens_for(g, B, T, cap))


def test_shared_prefix_attn_without_any_row(ctx):
    g = gen(1)
    q = rn(g, 3, 2, 32, D)
    lens = torch.tensor([0, 5, 1], device="cuda", dtype=torch.int32)
    ok, ov = rn(g, 3, 2, 8, D), rn(g, 3, 2, 8, D)
    out, lse = check_attn(ctx, q, None, None, None, ok, ov, lens)
    assert torch.isneginf(lse[0]).all() and (out[0] == 0).all()
    assert torch.isneginf(lse[2, 0]).all() and (out[2, 0] == 0).all()  # the first of two tokens sees no row yet
    # no rows of either kind anywhere
    out.fill_(float("nan"))
    ctx.shared_prefix_attn_dev(n_seqs=3, n_tokens=2, num_attn_heads=32, num_kv_heads=2, softmax_scale=SCALE, q=q.data_ptr(),
                               q_seq_stride=q.stride(0), q_token_stride=q.stride(1), q_head_stride=D,
                               own_lens=torch.zeros_like(lens).data_ptr(), out=out.data_ptr(), lse=lse.data_ptr())
    ctx.synchronize()
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_shared_prefix_attn_ignores_what_lies_behind_the_lengths(ctx):
    """NaN and infinities in own rows at and beyond a sequence's length, and queries that grow the running maximum by far
    more than the rescaling threshold from tile to tile."""
    g = gen(2)
    B, T, H, Hkv, P, cap = 6, 2, 32, 2, 700, 500
    q = rn(g, B, T, H, D, scale=2.0)
    pk, pv = rn(g, Hkv, P, D), rn(g, Hkv, P, D)
    pk *= torch.linspace(0.1, 8.0, P, device="cuda").view(1, P, 1).to(torch.bfloat16)
    ok, ov = rn(g, B, Hkv, cap, D, scale=3.0), rn(g, B, Hkv, cap, D)
    lens = torch.tensor([0, 1, 127, 128, 129, 499], device="cuda", dtype=torch.int32)
    for b in range(B):
        n = int(lens[b])
        ok[b, :, n:] = float("nan")
        ov[b, :, n:] = float("nan")
        ov[b, :, n : n + 3] = float("inf")
    out, lse = check_attn(ctx, q, None, pk, pv, ok, ov, lens)
    used = torch.arange(cap, device="cuda").view(1, 1, cap, 1) < lens.view(B, 1, 1, 1)
    out0, lse0 = check_attn(ctx, q, None, pk, pv, torch.where(used, ok, 0.0), torch.where(used, ov, 0.0), lens)
    assert torch.equal(out, out0) and torch.equal(lse, lse0)  # not even in the last bit


def test_shared_prefix_attn_strided(ctx):
    """q and gate interleaved per head as a projection emits them, rows of a cache with gaps, heads behind rows, and the
    sequences of a batch that are every other place of a larger cache."""
    g = gen(3)
    B, T, H, Hkv, P, cap = 4, 2, 24, 2, 333, 200
    qg = rn(g, B, T, H, 2 * D)
    q, gate = qg[..., :D], qg[..., D:]
    pk = rn(g, P, Hkv, D + 8)[..., :D].transpose(0, 1)
    pv = rn(g, P, Hkv, D + 8)[..., :D].transpose(0, 1)
    ok = rn(g, 2 * B, cap, Hkv, D).transpose(1, 2)[::2]
    ov = rn(g, 2 * B, cap, Hkv, D).transpose(1, 2)[::2]
    check_attn(ctx, q, gate, pk, pv, ok, ov, lens_for(g, B, T, cap))


@pytest.mark.parametrize("P,cap", [(700, 90), (0, 300), (260, 0)])
def test_shared_prefix_attn_of_a_query_that_is_nan(ctx, P, cap):
    """A NaN among the queries shows in its own output and lse, and in no other."""
    g = gen(6 + P)
    B, T, H, Hkv = 5, 2, 32, 2
    q = rn(g, B, T, H, D)
    pk, pv = (rn(g, Hkv, P, D), rn(g, Hkv, P, D)) if P else (None, None)
    ok, ov = (rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)) if cap else (None, None)
    lens = torch.full((B,), cap, device="cuda", dtype=torch.int32)
    ro, rl, bo, bl = attn_ref(q, None, pk, pv, ok, ov, lens)
    bad = torch.zeros(B, T, H, dtype=torch.bool, device="cuda")
    bad[1, 0, 3] = bad[1, 1, 20] = bad[4, 1, 31] = True
    q[..., 17].masked_fill_(bad, float("nan"))
    out, lse = torch.zeros_like(q), torch.zeros(B, T, H, device="cuda")
    ctx.shared_prefix_attn_dev(**attn_args(q, None, pk, pv, ok, ov, lens, out, lse))
    ctx.synchronize()
    assert out[bad].isnan().all() and lse[bad].isnan().all()
    assert ((out.double() - ro).abs() <= bo)[~bad].all() and ((lse.double() - rl).abs() <= bl)[~bad].all()


def test_shared_prefix_attn_lengths_out_of_range_are_reported(ctx, M):
    g = gen(4)
    q, pk, pv = rn(g, 3, 1, 32, D), rn(g, 2, 200, D), rn(g, 2, 200, D)
    ok, ov = rn(g, 3, 2, 64, D), rn(g, 3, 2, 64, D)
    lens = torch.tensor([64, 65, -1], device="cuda", dtype=torch.int32)
    out, lse = torch.zeros(3, 1, 32, D, device="cuda", dtype=torch.bfloat16), torch.zeros(3, 1, 32, device="cuda")
    ctx.shared_prefix_attn_dev(**attn_args(q, None, pk, pv, ok, ov, lens, out, lse))
    with pytest.raises(M.MfcError, match="range checks"):
        ctx.synchronize()
    ro, rl, bo, _ = attn_ref(q, None, pk, pv, ok, ov, torch.tensor([64, 0, 0], device="cuda", dtype=torch.int32))
    assert ((out.double() - ro).abs() <= bo).all()  # such a sequence counts as empty, the others are right
    check_attn(ctx, q, None, pk, pv, ok, ov, lens.clamp(0, 64))


def test_shared_prefix_attn_repeats_bit_for_bit_and_replays(ctx):
    g = gen(5)
    B, T, H, Hkv, P, cap = 20, 3, 32, 2, 1500, 300
    q, pk, pv = rn(g, B, T, H, D), rn(g, Hkv, P, D), rn(g, Hkv, P, D)
    ok, ov = rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    lens = lens_for(g, B, T, cap)
    out, lse = check_attn(ctx, q, None, pk, pv, ok, ov, lens)
    again, lse2 = torch.zeros_like(out), torch.zeros_like(lse)
    args = attn_args(q, None, pk, pv, ok, ov, lens, again, lse2)
    s = torch.cuda.Stream()
    home = torch.cuda.current_stream().cuda_stream
    s.wait_stream(torch.cuda.current_stream())
    ctx.set_stream(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ctx.shared_prefix_attn_dev(**args)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    lens.copy_((lens - 5).clamp(min=0))  # the lengths are read when the graph runs
    q.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    ctx.set_stream(home)
    ro, rl, bo, bl = attn_ref(q, None, pk, pv, ok, ov, lens)
    assert ((again.double() - ro).abs() <= bo).all()


# ---------------------------------------------------------------------------------------------------- weights


def weights_args(q, k, lens, lse, w, decay=1.0, scale=SCALE):
    B, T, H, _ = q.shape
    return dict(n_seqs=B, n_tokens=T, num_attn_heads=H, num_kv_heads=k.shape[1], softmax_scale=scale, decay=decay,
                q=q.data_ptr(), q_seq_stride=q.stride(0), q_token_stride=q.stride(1), q_head_stride=q.stride(2),
                k=k.data_ptr(), k_seq_stride=k.stride(0), k_head_stride=k.stride(1), k_row_stride=k.stride(2), cap=k.shape[2],
                lens=lens.data_ptr(), lse=lse.data_ptr(), weights=w.data_ptr(), weights_seq_stride=w.stride(0),
                weights_head_stride=w.stride(1))


def weights_ref(q, k, lens, lse, w, decay, scale=SCALE):
    B, T, H, _ = q.shape
    Hkv, cap = k.shape[1], k.shape[2]
    G = H // Hkv
    res, tol = w.double().clone(), torch.zeros_like(w, dtype=torch.float64)
    vis = visible(lens, T, cap)
    for b in range(B):
        n = max(0, min(int(lens[b]), cap))
        if n == 0:
            continue
        qq, kk = q[b].double().view(T, Hkv, G, D), k[b, :, :n].double()
        s = torch.einsum("thgd,hjd->thgj", qq, kk) * scale
        a = torch.einsum("thgd,hjd->thgj", qq.abs(), kk.abs()) * scale
        z = lse[b].double().view(T, Hkv, G, 1)
        p = torch.where(vis[b, :, :n].view(T, 1, 1, n), torch.exp(s - z), 0.0)
        ds = 256 * 2.0 ** -23 * a + 2.0 ** -21 * (s.abs() + z.abs().nan_to_num(posinf=0.0)) + 2.0 ** -20
        res[b, :, :n] = decay * res[b, :, :n] + p.sum((0, 2))
        tol[b, :, :n] = torch.where(p > 0, p * ds, 0.0).sum((0, 2)) + 2.0 ** -22 * T * G * res[b, :, :n].abs()
    return res, tol


@pytest.mark.parametrize("B,T,H,Hkv,cap,decay", [
    (1, 1, 32, 2, 1, 1.0), (1, 1, 32, 2, 1000, 1.0), (3, 1, 7, 1, 65, 0.5), (4, 3, 24, 2, 300, 1.0), (5, 16, 16, 1, 130, 0.96875),
    (40, 2, 8, 8, 257, 1.0), (2, 5, 32, 2, 5000, 0.96875), (200, 1, 10, 2, 64, 1.0)])
def test_attn_weights(ctx, B, T, H, Hkv, cap, decay):
    g = gen(B + cap)
    q, k = rn(g, B, T, H, D, scale=1.5), rn(g, B, Hkv, cap, D)
    lens = lens_for(g, B, T, cap)
    for b in range(B):
        k[b, :, int(lens[b]):] = float("nan")
    w = torch.rand(B, Hkv, cap, generator=g, device="cuda")
    ro, lse, _, _ = attn_ref(q, None, None, None, k, torch.zeros_like(k), lens)
    lse = lse.float().contiguous()
    ref, tol = weights_ref(q, k, lens, lse, w, decay)
    before = w.clone()
    ctx.attn_weights_accumulate_dev(**weights_args(q, k, lens, lse, w, decay))
    ctx.synchronize()
    assert ((w.double() - ref).abs() <= tol).all(), float(((w.double() - ref).abs() - tol).max())
    unused = torch.arange(cap, device="cuda").view(1, 1, cap) >= lens.view(B, 1, 1)
    assert torch.equal(w[unused.expand_as(w)], before[unused.expand_as(w)])


def test_attn_weights_start_afresh(ctx):
    """decay 0: what the sums held, NaN or infinite, is not read."""
    g = gen(8)
    B, T, H, Hkv, cap = 3, 2, 32, 2, 300
    q, k = rn(g, B, T, H, D), rn(g, B, Hkv, cap, D)
    lens = torch.tensor([300, 0, 129], device="cuda", dtype=torch.int32)
    _, lse, _, _ = attn_ref(q, None, None, None, k, torch.zeros_like(k), lens)
    lse = lse.float().contiguous()
    ref, tol = weights_ref(q, k, lens, lse, torch.zeros(B, Hkv, cap, device="cuda"), 0.0)
    w = torch.full((B, Hkv, cap), float("nan"), device="cuda")
    w[..., ::2] = float("inf")
    ctx.attn_weights_accumulate_dev(**weights_args(q, k, lens, lse, w, 0.0))
    ctx.synchronize()
    used = (torch.arange(cap, device="cuda").view(1, 1, cap) < lens.view(B, 1, 1)).expand_as(w)
    assert ((w.double() - ref).abs() <= tol)[used].all()
    assert not torch.isfinite(w[~used]).any()


def test_attn_weights_strided_and_out_of_range(ctx, M):
    g = gen(7)
    B, T, H, Hkv, cap = 3, 2, 32, 2, 150
    q = rn(g, B, T, H, 2 * D)[..., :D]
    k = rn(g, B, cap, Hkv, D + 8)[..., :D].transpose(1, 2)
    wide = torch.rand(B, Hkv, cap + 13, generator=g, device="cuda")
    w, before = wide[..., :cap], wide.clone()
    lens = torch.tensor([150, 151, 60], device="cuda", dtype=torch.int32)
    good = torch.tensor([150, 0, 60], device="cuda", dtype=torch.int32)
    _, lse, _, _ = attn_ref(q, None, None, None, k, torch.zeros_like(k), good)
    lse = lse.float().contiguous()
    ref, tol = weights_ref(q, k, good, lse, w, 1.0)
    ctx.attn_weights_accumulate_dev(**weights_args(q, k, lens, lse, w))
    with pytest.raises(M.MfcError, match="range checks"):
        ctx.synchronize()
    assert ((w.double() - ref).abs() <= tol).all()
    assert torch.equal(wide[..., cap:], before[..., cap:])


# ---------------------------------------------------------------------------------------------------- eviction


def evict_ref(k, v, w, pos, lens, nxt, budget, sink, recent):
    """The rows' new content by the definition, on the host: [(b, h, rows)] of source rows."""
    out = {}
    w, pos = w.cpu().tolist(), pos.cpu().tolist()
    for b in range(k.shape[0]):
        n = int(lens[b])
        for h in range(k.shape[1]):
            def key(j):
                x, ps = w[b][h][j], pos[b][h][j]
                if ps < sink or ps >= int(nxt[b]) - recent:
                    return (0, 0.0, j)
                return (2, 0.0, j) if x != x else (1, -x, j)
            new = min(n, budget)
            kept = set(sorted(range(n), key=key)[:new])
            movers = iter([j for j in range(budget, n) if j in kept])
            out[b, h] = [j if j in kept else next(movers) for j in range(new)]
    return out


@pytest.mark.parametrize("B,Hkv,cap,budget,dtype", [
    (1, 1, 1, 1, "bf16"), (2, 2, 40, 8, "bf16"), (1, 2, 1088, 1024, "bf16"), (3, 1, 700, 699, "f32"), (2, 2, 5000, 77, "bf16"),
    (70, 2, 300, 128, "f32"), (1, 1, 33000, 20001, "bf16"), (5, 3, 64, 100, "bf16"), (160, 2, 1030, 400, "bf16")])
@pytest.mark.parametrize("kind", ["spread", "ties"])
def test_kv_evict(ctx, M, B, Hkv, cap, budget, dtype, kind):
    g = gen(B * 7 + cap)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    k, v = rn(g, B, Hkv, cap, D, dtype=dt), rn(g, B, Hkv, cap, D, dtype=dt)
    w = torch.exp(2 * torch.randn(B, Hkv, cap, generator=g, device="cuda"))
    if kind == "ties":  # few distinct weights, both zeros, infinities and NaN
        w = torch.randint(-1, 3, (B, Hkv, cap), generator=g, device="cuda").float()
        r = torch.rand(B, Hkv, cap, generator=g, device="cuda")
        w[r < 0.1] = -0.0
        w[r > 0.96] = float("nan")
        w[(r > 0.92) & (r < 0.94)] = float("inf")
        w[(r > 0.90) & (r < 0.92)] = float("-inf")
    lens = torch.randint(min(budget, cap), cap + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = cap
    if B > 2:
        lens[1], lens[2] = 0, min(budget, cap)
    pos = torch.rand(B, Hkv, cap, generator=g, device="cuda").argsort(-1).to(torch.int32)
    nxt = lens + 3
    sink, recent = 2, max(3, min(budget, 40) // 4)
    src = evict_ref(k, v, w, pos, lens, nxt, budget, sink, recent)
    k0, v0, w0, p0, l0 = (t.clone() for t in (k, v, w, pos, lens))
    for alias in (False, True):
        k.copy_(k0)
        v.copy_(v0)
        wo, po = (w, pos) if alias else (torch.full_like(w, -7.0), torch.full_like(pos, -7))
        lo = torch.full_like(lens, -7)
        ctx.kv_evict_dev(n_seqs=B, num_kv_heads=Hkv, kv_dtype=M.KV_BF16 if dtype == "bf16" else M.KV_F32, cap=cap, k=k.data_ptr(),
                         v=v.data_ptr(), seq_stride=k.stride(0), head_stride=k.stride(1), row_stride=k.stride(2), budget=budget,
                         n_sink=sink, n_recent=recent, lens=lens.data_ptr(), next_pos=nxt.data_ptr(), weights=w.data_ptr(),
                         positions=pos.data_ptr(), map_seq_stride=w.stride(0), map_head_stride=w.stride(1),
                         weights_out=wo.data_ptr(), positions_out=po.data_ptr(), lens_out=lo.data_ptr())
        ctx.synchronize()
        assert torch.equal(lo, lens.clamp(max=budget)) and torch.equal(lens, l0)
        for (b, h), rows in src.items():
            n = len(rows)
            ix = torch.tensor(rows, device="cuda", dtype=torch.long)
            assert torch.equal(k[b, h, :n], k0[b, h, ix]) and torch.equal(v[b, h, :n], v0[b, h, ix]), (b, h)
            assert torch.equal(k[b, h, n:], k0[b, h, n:]) and torch.equal(v[b, h, n:], v0[b, h, n:])
            assert torch.equal(wo[b, h, :n].nan_to_num(-9.0), w0[b, h, ix].nan_to_num(-9.0)) and torch.equal(po[b, h, :n], p0[b, h, ix])
            rest_w, rest_p = (w0[b, h, n:], p0[b, h, n:]) if alias else (torch.full_like(wo[b, h, n:], -7.0), torch.full_like(po[b, h, n:], -7))
            assert torch.equal(wo[b, h, n:].nan_to_num(-9.0), rest_w.nan_to_num(-9.0)) and torch.equal(po[b, h, n:], rest_p)


@pytest.mark.parametrize("cap,budget", [(200, 90), (5000, 2400), (33000, 9000)])
@pytest.mark.parametrize("crowd", [1, 2, 31, 32, 33, 70])
@pytest.mark.parametrize("values", [1024, 5, 1])
def test_kv_evict_with_a_crowd_at_the_border(ctx, M, cap, budget, crowd, values):
    """`crowd` weights that differ in their last ten bits at most, of `values` different ones, and the border among them."""
    g = gen(cap + crowd)
    w = torch.rand(1, 2, cap, generator=g, device="cuda") + torch.where(torch.arange(cap, device="cuda") < budget - crowd // 2, 3.0, 0.0)
    low = torch.randint(0, values, (2, crowd), generator=g, device="cuda", dtype=torch.int32)
    w[0, :, budget - crowd // 2 : budget - crowd // 2 + crowd] = (low + 0x40000000).view(torch.float32)  # 2.0 and up
    for h in range(2):
        w[0, h] = w[0, h, torch.randperm(cap, generator=g, device="cuda")]
    k, v = rn(g, 1, 2, cap, D), rn(g, 1, 2, cap, D)
    pos = torch.arange(cap, device="cuda", dtype=torch.int32).expand(1, 2, cap).contiguous()
    lens, new = torch.tensor([cap], device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda", dtype=torch.int32)
    src = evict_ref(k, v, w, pos, lens, lens, budget, 0, 0)
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    ctx.kv_evict_dev(n_seqs=1, num_kv_heads=2, kv_dtype=M.KV_BF16, cap=cap, k=k.data_ptr(), v=v.data_ptr(), seq_stride=k.stride(0),
                     head_stride=k.stride(1), row_stride=D, budget=budget, n_sink=0, n_recent=0, lens=lens.data_ptr(),
                     next_pos=lens.data_ptr(), weights=w.data_ptr(), positions=pos.data_ptr(), map_seq_stride=2 * cap, map_head_stride=cap,
                     weights_out=w.data_ptr(), positions_out=pos.data_ptr(), lens_out=new.data_ptr())
    ctx.synchronize()
    assert int(new) == budget
    for (b, h), rows in src.items():
        ix = torch.tensor(rows, device="cuda")
        assert torch.equal(pos[b, h, :budget].long(), ix) and torch.equal(w[b, h, :budget], w0[b, h, ix])
        assert torch.equal(k[b, h, :budget], k0[b, h, ix]) and torch.equal(v[b, h, :budget], v0[b, h, ix])


def test_kv_evict_strided_rows_and_out_of_range(ctx, M):
    g = gen(11)
    B, Hkv, cap, budget = 3, 2, 90, 50
    kw, vw = rn(g, B, cap, Hkv, D + 8), rn(g, B, cap, Hkv, D + 8)
    k0, v0 = kw.clone(), vw.clone()
    w = torch.rand(B, Hkv, cap + 5, generator=g, device="cuda")[..., :cap]
    pos = torch.arange(cap + 5, device="cuda", dtype=torch.int32).expand(B, Hkv, cap + 5).contiguous()[..., :cap]
    lens = torch.tensor([90, 91, -2], device="cuda", dtype=torch.int32)
    nxt, lo = lens.clone(), torch.zeros_like(lens)
    wo, po = torch.zeros(B, Hkv, cap + 5, device="cuda"), torch.zeros(B, Hkv, cap + 5, device="cuda", dtype=torch.int32)
    ctx.kv_evict_dev(n_seqs=B, num_kv_heads=Hkv, kv_dtype=M.KV_BF16, cap=cap, k=kw.data_ptr(), v=vw.data_ptr(),
                     seq_stride=kw.stride(0), head_stride=kw.stride(2), row_stride=kw.stride(1), budget=budget, n_sink=4, n_recent=8,
                     lens=lens.data_ptr(), next_pos=nxt.data_ptr(), weights=w.data_ptr(), positions=pos.data_ptr(),
                     map_seq_stride=w.stride(0), map_head_stride=w.stride(1), weights_out=wo.data_ptr(), positions_out=po.data_ptr(),
                     lens_out=lo.data_ptr())
    with pytest.raises(M.MfcError, match="range checks"):
        ctx.synchronize()
    assert lo.tolist() == [50, 0, 0]
    assert torch.equal(kw[1:], k0[1:]) and torch.equal(vw[1:], v0[1:]) and torch.equal(kw[..., D:], k0[..., D:])
    src = evict_ref(k0[:1].transpose(1, 2), None, w[:1], pos[:1], lens[:1], nxt[:1], budget, 4, 8)
    for (b, h), rows in src.items():
        ix = torch.tensor(rows, device="cuda", dtype=torch.long)
        assert torch.equal(kw[b, :50, h, :D], k0[b, ix, h, :D]) and torch.equal(vw[b, :50, h, :D], v0[b, ix, h, :D])


# ---------------------------------------------------------------------------------------------------- verification


def verify_ref(p, q, x, lens, ua, us):
    p, x, ua, us = p.cpu().double(), x.cpu(), ua.cpu().double(), us.cpu().double()
    q = q.cpu().double() if q is not None else None
    B, K, V = p.shape[0], x.shape[1], p.shape[2]
    ns, toks = [], []
    for b in range(B):
        n_drafts = min(int(lens[b]), K)
        if n_drafts < 0:
            ns.append(0)
            toks.append([-1] * (K + 1))
            continue
        n = 0
        while n < n_drafts:
            t = int(x[b, n])
            if not (0 <= t < V and float(ua[b, n]) * (float(q[b, n, t]) if q is not None else 1.0) < float(p[b, n, t])):
                break
            n += 1
        w = p[b, n].clone()
        if n < n_drafts:
            if q is not None:
                w = w - q[b, n]
            elif 0 <= int(x[b, n]) < V:
                w[int(x[b, n])] = 0.0
        w = torch.where(w > 0, w, 0.0)
        if float(w.sum()) == 0.0:
            w = torch.where(p[b, n] > 0, p[b, n], 0.0)
        c = torch.cumsum(w, 0)
        t = int((c <= float(us[b]) * float(c[-1])).sum()) if float(c[-1]) > 0 else -1
        ns.append(n)
        toks.append([int(y) for y in x[b, :n]] + [t] + [-1] * (K - n))
    return torch.tensor(ns, dtype=torch.int32), torch.tensor(toks, dtype=torch.int32)


def call_verify(ctx, p, q, x, lens, ua, us):
    B, K = x.shape
    n = torch.full((B,), -5, device="cuda", dtype=torch.int32)
    tok = torch.full((B, K + 1), -5, device="cuda", dtype=torch.int32)
    ctx.verify_drafts_dev(n_seqs=B, max_drafts=K, vocab=p.shape[2], target_probs=p.data_ptr(), target_seq_stride=p.stride(0),
                          target_row_stride=p.stride(1), draft_probs=q.data_ptr() if q is not None else None,
                          draft_seq_stride=q.stride(0) if q is not None else 0, draft_row_stride=q.stride(1) if q is not None else 0,
                          draft_tokens=x.data_ptr(), draft_lens=lens.data_ptr() if lens is not None else None, u_accept=ua.data_ptr(),
                          u_sample=us.data_ptr(), n_accepted=n.data_ptr(), tokens=tok.data_ptr())
    ctx.synchronize()
    return n.cpu(), tok.cpu()


@pytest.mark.parametrize("B,K,V,sampled,pad", [
    (1, 1, 1, True, 0), (1, 0, 10, True, 0), (3, 4, 7, True, 0), (2, 4, 1000, False, 0), (9, 8, 4099, True, 1), (64, 3, 1025, True, 3),
    (1, 5, 131072, True, 0), (200, 2, 2048, False, 0), (2, 32, 50001, True, 0), (1, 1, 1200003, True, 0), (24, 4, 40007, False, 0),
    (44, 8, 20011, True, 0), (3, 2, 300, False, 2), (150, 1, 7000, True, 0)])
def test_verify_drafts(ctx, B, K, V, sampled, pad):
    g = gen(B + K + V)
    logits = torch.randn(B, K + 1, V + pad, generator=g, device="cuda") * 2
    p = torch.softmax(logits[..., :V], -1)
    ql = logits[:, :K, :V] + 0.7 * torch.randn(B, K, V, generator=g, device="cuda")
    q = torch.softmax(ql, -1) if sampled else None
    noise = -torch.log(-torch.log(torch.rand(ql.shape, generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
    x = (ql + noise).argmax(-1).to(torch.int32)  # the draft model's samples
    if pad:  # rows that start at no 16-byte boundary
        wide = torch.full((B, K + 1, V + pad), float("nan"), device="cuda")
        wide[..., :V] = p
        p = wide[..., :V]
    lens = torch.randint(0, K + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = K
    if B > 2:
        lens[1] = -1
    ua, us = torch.rand(B, K, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    n, tok = call_verify(ctx, p, q, x, lens, ua, us)
    rn_, rt = verify_ref(p, q, x, lens, ua, us)
    assert torch.equal(n, rn_) and torch.equal(tok, rt)


def test_verify_drafts_edges(ctx):
    V = 3000
    p = torch.zeros(6, 2, V, device="cuda")
    q = torch.zeros(6, 1, V, device="cuda")
    x = torch.zeros(6, 1, device="cuda", dtype=torch.int32)
    ua = torch.full((6, 1), 0.5, device="cuda")
    us = torch.zeros(6, device="cuda")
    p[0, :, 5], q[0, 0, 5], x[0] = 1.0, 1.0, 5                       # equal distributions: accepted, then row 1
    p[1, :, 7], q[1, 0, 7], x[1] = 0.25, 0.5, 7                      # u q = p exactly: refused; the residual is zero: from p
    p[2, 0, 9], q[2, 0, 3], x[2] = 1.0, 1.0, 3                       # p(x) = 0: refused, residual at 9
    x[3] = V                                                         # outside the vocabulary, p all zero: no token
    p[4, 0, 100:200], q[4, 0, 4], x[4], us[4] = 0.01, 1.0, 4, 1.0 - 2.0 ** -24
    p[5, 0, 11], p[5, 0, 12], q[5, 0, 0], x[5] = float("nan"), 0.5, 1.0, 0  # a NaN counts as zero
    n, tok = call_verify(ctx, p, q, x, None, ua, us)
    assert n.tolist() == [1, 0, 0, 0, 0, 0]
    assert tok.tolist() == [[5, 5], [7, -1], [9, -1], [-1, -1], [199, -1], [12, -1]]
    # a uniform outside [0, 1) counts as the nearest end; without draft probabilities the drafted token itself is left out
    us[:] = torch.tensor([1.0, -1.0, float("nan"), 2.0, float("inf"), 0.0], device="cuda")
    p[2, 0, 3], ua[2] = 0.25, 0.9
    n, tok = call_verify(ctx, p, None, x, None, ua, us)
    assert n.tolist() == [1, 0, 0, 0, 0, 0]
    assert tok.tolist() == [[5, 5], [7, -1], [9, -1], [-1, -1], [199, -1], [12, -1]]


# ---------------------------------------------------------------------------------------------------- together


class _Rows:
    """Device memory the context owns, as a torch tensor (for reading cached rows back)."""

    def __init__(self, ptr, shape, strides):
        self.__cuda_array_interface__ = dict(shape=tuple(shape), strides=tuple(2 * s for s in strides), typestr="<i2",
                                             data=(ptr, False), version=3)


def test_a_server_s_steps(M):
    """A prompt is prefilled into a context once; a batch then decodes behind it with drafted tokens: attention over the
    shared rows and each sequence's own, the rows' weights, verification, the lengths cut to what was accepted, and an
    eviction when a sequence passes its budget.  Every call against its 64-bit form on the state the calls before left."""
    g = gen(21)
    layer, P, B, T, H, Hkv, cap, budget, V = 3, 300, 5, 3, 32, 2, 80, 40, 500
    c = M.Ctx(num_layers=4, max_seq=512, n_seqs=2, kv_dtype=M.KV_BF16)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    x = [rn(g, P, n, D) for n in (H, H, Hkv, Hkv)]
    scratch = torch.empty(P, H, D, device="cuda", dtype=torch.bfloat16)
    c.full_attn_prefill_dev(layer, 1, 0, P, x[0].data_ptr(), x[1].data_ptr(), x[2].data_ptr(), x[3].data_ptr(), scratch.data_ptr())
    kp, vp, seq_stride, head_stride, rows = c.kv_cache_view(layer, 1)
    assert rows == P and seq_stride == Hkv * head_stride
    pk, pv = (torch.as_tensor(_Rows(a, (Hkv, P, D), (head_stride, D, 1)), device="cuda").view(torch.bfloat16) for a in (kp, vp))
    c.synchronize()
    assert torch.equal(pv, x[3].transpose(0, 1))  # V goes into the cache as it is

    ok, ov = torch.zeros(B, Hkv, cap, D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, Hkv, cap, D, device="cuda", dtype=torch.bfloat16)
    ok.fill_(float("nan"))
    ov.fill_(float("nan"))
    w = torch.zeros(B, Hkv, cap, device="cuda")
    pos = torch.zeros(B, Hkv, cap, device="cuda", dtype=torch.int32)
    lens = torch.zeros(B, device="cuda", dtype=torch.int32)
    nxt = torch.full((B,), P, device="cuda", dtype=torch.int32)
    out, lse = torch.empty(B, T, H, D, device="cuda", dtype=torch.bfloat16), torch.empty(B, T, H, device="cuda")
    evictions = 0
    for step in range(24):
        # the step's rows: the last accepted token and T - 1 drafts, appended by the caller
        for b in range(B):
            n = int(lens[b])
            ok[b, :, n : n + T], ov[b, :, n : n + T] = rn(g, Hkv, T, D), rn(g, Hkv, T, D)
            w[b, :, n : n + T] = 0.0
            pos[b, :, n : n + T] = nxt[b] + torch.arange(T, device="cuda", dtype=torch.int32)
        lens += T
        q, gate = rn(g, B, T, H, D, scale=1.5), rn(g, B, T, H, D)
        c.shared_prefix_attn_dev(**attn_args(q, gate, pk, pv, ok, ov, lens, out, lse))
        w_before = w.clone()
        c.attn_weights_accumulate_dev(**weights_args(q, ok, lens, lse, w))
        p = torch.softmax(torch.randn(B, T, V, generator=g, device="cuda"), -1)
        qd = torch.softmax(torch.log(p[:, : T - 1]) + 0.3 * torch.randn(B, T - 1, V, generator=g, device="cuda"), -1)
        drafts = torch.multinomial(qd.view(-1, V), 1, generator=g).view(B, T - 1).to(torch.int32)
        ua, us = torch.rand(B, T - 1, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
        n_acc, tok = call_verify(c, p, qd, drafts, None, ua, us)
        ro, rl, bo, bl = attn_ref(q, gate, pk, pv, ok, ov, lens)
        assert ((out.double() - ro).abs() <= bo).all() and ((lse.double() - rl).abs() <= bl).all(), step
        ref, tol = weights_ref(q, ok, lens, lse, w_before, 1.0)
        used = (torch.arange(cap, device="cuda").view(1, 1, cap) < lens.view(B, 1, 1)).expand_as(w)
        assert ((w.double() - ref).abs() <= tol)[used].all(), step
        rn_, rt = verify_ref(p, qd, drafts, torch.full((B,), T - 1), ua, us)
        assert torch.equal(n_acc, rn_) and torch.equal(tok, rt)
        # rows of refused drafts are dropped; the drawn token's row is the next step's first
        lens -= (T - 1 - n_acc.cuda())
        nxt += 1 + n_acc.cuda()
        if int(lens.max()) + T > cap or step % 8 == 7:
            src = evict_ref(ok, ov, w, pos, lens, nxt, budget, P + 2, 6)
            before = [t.clone() for t in (ok, ov, w, pos, lens)]
            new = torch.empty_like(lens)
            c.kv_evict_dev(n_seqs=B, num_kv_heads=Hkv, kv_dtype=M.KV_BF16, cap=cap, k=ok.data_ptr(), v=ov.data_ptr(),
                           seq_stride=ok.stride(0), head_stride=ok.stride(1), row_stride=D, budget=budget, n_sink=P + 2, n_recent=6,
                           lens=lens.data_ptr(), next_pos=nxt.data_ptr(), weights=w.data_ptr(), positions=pos.data_ptr(),
                           map_seq_stride=w.stride(0), map_head_stride=w.stride(1), weights_out=w.data_ptr(),
                           positions_out=pos.data_ptr(), lens_out=new.data_ptr())
            c.synchronize()
            evictions += int((before[4] > budget).sum())
            for (b, h), rows_ in src.items():
                ix = torch.tensor(rows_, device="cuda", dtype=torch.long)
                n = len(rows_)
                for now, was in zip((ok, ov, w, pos), before):
                    assert torch.equal(now[b, h, :n], was[b, h, ix])
                    assert torch.equal(now[b, h, n:].nan_to_num(7), was[b, h, n:].nan_to_num(7))
            assert torch.equal(new, before[4].clamp(max=budget))
            lens = new
    assert evictions > B
    assert torch.equal(pv, x[3].transpose(0, 1)) and c.kv_cache_view(layer, 1)[4] == P  # the shared rows are as they were
    with pytest.raises(M.MfcError):
        c.kv_cache_view(0, 0)  # not a full-attention layer
    with pytest.raises(M.MfcError):
        c.kv_cache_view(layer, 2)
    c.check_guards()
    c.close()


@pytest.mark.parametrize("call", ["attn", "weights"])
def test_a_lost_load_is_reported_and_the_context_survives(ctx, M, call):
    """A barrier armed with no load issued for it: the wait runs out, every role leaves, the status names it, and the next
    call is right."""
    g = gen(31)
    B, T, H, Hkv, cap = 3, 2, 32, 2, 300
    q, ok, ov = rn(g, B, T, H, D), rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    pk, pv = rn(g, Hkv, 700, D), rn(g, Hkv, 700, D)
    lens = torch.tensor([300, 130, 5], device="cuda", dtype=torch.int32)
    out, lse = torch.zeros(B, T, H, D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, T, H, device="cuda")
    w = torch.zeros(B, Hkv, cap, device="cuda")
    run = (lambda: ctx.shared_prefix_attn_dev(**attn_args(q, None, pk, pv, ok, ov, lens, out, lse))) if call == "attn" else (
        lambda: ctx.attn_weights_accumulate_dev(**weights_args(q, ok, lens, lse, w)))
    ctx.set_tuning("gqa_wait_spins", 2000)
    ctx.set_tuning("gqa_inject_lost_load", 1)
    try:
        run()
        with pytest.raises(M.MfcError, match="did not arrive"):
            ctx.synchronize()
    finally:
        ctx.set_tuning("gqa_inject_lost_load", 0)
        ctx.set_tuning("gqa_wait_spins", 0)
    w.zero_()
    run()
    ctx.synchronize()
    check_attn(ctx, q, None, pk, pv, ok, ov, lens)


def test_refusals(ctx, M):
    """One refused call per entry point and check; nothing is launched.  (All checks run without a GPU as well, on the
    host code alone.)"""
    t = torch.zeros(64 * 256, device="cuda", dtype=torch.bfloat16)
    i = torch.zeros(64, device="cuda", dtype=torch.int32)
    f = torch.zeros(64 * 256, device="cuda")
    P, I, F = t.data_ptr(), i.data_ptr(), f.data_ptr()
    attn = dict(n_seqs=1, n_tokens=1, num_attn_heads=2, num_kv_heads=1, softmax_scale=SCALE, q=P, q_seq_stride=512, q_token_stride=512,
                q_head_stride=256, own_k=P, own_v=P, own_seq_stride=1024, own_head_stride=1024, own_row_stride=256, own_cap=4, own_lens=I, out=P)
    wts = dict(n_seqs=1, n_tokens=1, num_attn_heads=2, num_kv_heads=1, softmax_scale=SCALE, decay=1.0, q=P, q_seq_stride=512,
               q_token_stride=512, q_head_stride=256, k=P, k_seq_stride=1024, k_head_stride=1024, k_row_stride=256, cap=4, lens=I, lse=F, weights=F)
    ev = dict(n_seqs=1, num_kv_heads=1, kv_dtype=M.KV_BF16, cap=4, k=P, v=P + 8192, seq_stride=1024, head_stride=1024, row_stride=256, budget=2,
              lens=I, next_pos=I, weights=F, positions=I, map_seq_stride=4, map_head_stride=4, weights_out=F, positions_out=I, lens_out=I + 128)
    vf = dict(n_seqs=1, max_drafts=2, vocab=8, target_probs=F, target_seq_stride=24, target_row_stride=8, draft_tokens=I, u_accept=F,
              u_sample=F, n_accepted=I, tokens=I)
    before = ctx.launch_count
    for fn, base, bad in [
        (ctx.shared_prefix_attn_dev, attn, [dict(n_tokens=0), dict(n_tokens=17), dict(num_attn_heads=17), dict(softmax_scale=0.0), dict(q=None),
                                            dict(out=P + 2), dict(q_head_stride=4), dict(own_row_stride=128), dict(prefix_len=3), dict(n_seqs=4097),
                                            dict(own_head_stride=-1024, num_attn_heads=4, num_kv_heads=2), dict(prefix_len=-1)]),
        (ctx.attn_weights_accumulate_dev, wts, [dict(k=P + 8), dict(k_row_stride=12), dict(lse=None), dict(cap=-1), dict(num_kv_heads=0)]),
        (ctx.kv_evict_dev, ev, [dict(budget=0), dict(kv_dtype=7), dict(v=P), dict(lens_out=I), dict(cap=300000), dict(row_stride=100), dict(weights=None)]),
        (ctx.verify_drafts_dev, vf, [dict(max_drafts=33), dict(vocab=0), dict(tokens=None), dict(u_accept=None), dict(target_probs=F + 2)])]:
        for change in bad:
            with pytest.raises(M.MfcError):
                fn(**{**base, **change})
        with pytest.raises(TypeError):
            fn(**{**base, "no_such_field": 1})
    for fn, base in [(ctx.shared_prefix_attn_dev, attn), (ctx.attn_weights_accumulate_dev, wts), (ctx.kv_evict_dev, ev), (ctx.verify_drafts_dev, vf)]:
        fn(**{**base, "n_seqs": 0})  # an empty batch is no error and no launch
    assert ctx.launch_count == before
    ctx.synchronize()


def test_row_counts_that_pass_32_bits_are_refused(ctx, M):
    t = torch.zeros(4096, device="cuda", dtype=torch.bfloat16)
    P, many = t.data_ptr(), (1 << 30) + 1
    q = dict(n_seqs=1, n_tokens=1, num_attn_heads=1, num_kv_heads=1, softmax_scale=SCALE, q=P, q_seq_stride=256, q_token_stride=256, q_head_stride=256)
    before = ctx.launch_count
    for rows in (many, (1 << 31) - 1):
        with pytest.raises(M.MfcError, match="2\\^30"):
            ctx.shared_prefix_attn_dev(**q, own_k=P, own_v=P, own_seq_stride=256, own_head_stride=256, own_row_stride=256, own_cap=rows, own_lens=P, out=P)
        with pytest.raises(M.MfcError, match="2\\^30"):
            ctx.shared_prefix_attn_dev(**q, prefix_k=P, prefix_v=P, prefix_head_stride=256, prefix_row_stride=256, prefix_len=rows, own_lens=P, out=P)
        with pytest.raises(M.MfcError, match="2\\^30"):
            ctx.attn_weights_accumulate_dev(**q, decay=1.0, k=P, k_seq_stride=256, k_head_stride=256, k_row_stride=256, cap=rows, lens=P, lse=P, weights=P)
    assert ctx.launch_count == before


def test_a_captured_step_of_all_four(ctx, M):
    """One graph of the four calls, replayed on changed inputs, against the same calls made directly."""
    g = gen(41)
    B, T, H, Hkv, P, cap, budget, V = 6, 3, 32, 2, 400, 200, 90, 3001
    q, gate = rn(g, B, T, H, D), rn(g, B, T, H, D)
    pk, pv, ok, ov = rn(g, Hkv, P, D), rn(g, Hkv, P, D), rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    w, pos = torch.rand(B, Hkv, cap, generator=g, device="cuda"), torch.arange(cap, device="cuda", dtype=torch.int32).expand(B, Hkv, cap).contiguous()
    lens = lens_for(g, B, T, cap)
    nxt, new = lens.clone(), torch.zeros_like(lens)
    p = torch.softmax(torch.randn(B, T, V, generator=g, device="cuda"), -1)
    qd = torch.softmax(torch.randn(B, T - 1, V, generator=g, device="cuda"), -1)
    x = torch.randint(0, V, (B, T - 1), generator=g, device="cuda", dtype=torch.int32)
    ua, us = torch.rand(B, T - 1, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    out, lse = torch.zeros(B, T, H, D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, T, H, device="cuda")
    n, tok = torch.zeros(B, device="cuda", dtype=torch.int32), torch.zeros(B, T, device="cuda", dtype=torch.int32)
    state = [ok, ov, w, pos]
    start = [t.clone() for t in state]

    def step():
        ctx.shared_prefix_attn_dev(**attn_args(q, gate, pk, pv, ok, ov, lens, out, lse))
        ctx.attn_weights_accumulate_dev(**weights_args(q, ok, lens, lse, w, 0.9))
        ctx.verify_drafts_dev(n_seqs=B, max_drafts=T - 1, vocab=V, target_probs=p.data_ptr(), target_seq_stride=p.stride(0),
                              target_row_stride=V, draft_probs=qd.data_ptr(), draft_seq_stride=qd.stride(0), draft_row_stride=V,
                              draft_tokens=x.data_ptr(), u_accept=ua.data_ptr(), u_sample=us.data_ptr(), n_accepted=n.data_ptr(),
                              tokens=tok.data_ptr())
        ctx.kv_evict_dev(n_seqs=B, num_kv_heads=Hkv, kv_dtype=M.KV_BF16, cap=cap, k=ok.data_ptr(), v=ov.data_ptr(), seq_stride=ok.stride(0),
                         head_stride=ok.stride(1), row_stride=D, budget=budget, n_sink=2, n_recent=5, lens=lens.data_ptr(),
                         next_pos=nxt.data_ptr(), weights=w.data_ptr(), positions=pos.data_ptr(), map_seq_stride=w.stride(0),
                         map_head_stride=w.stride(1), weights_out=w.data_ptr(), positions_out=pos.data_ptr(), lens_out=new.data_ptr())

    home, side = torch.cuda.current_stream().cuda_stream, torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.set_stream(side.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
        step()  # (the second finds nothing to evict where the lengths still say so: it runs all the same)
    ctx.set_stream(home)
    for turn in range(3):
        q.copy_(rn(g, B, T, H, D))
        us.copy_(torch.rand(B, generator=g, device="cuda"))
        results = []
        for way in ("direct", "graph"):
            for t, s in zip(state, start):
                t.copy_(s)
            torch.cuda.synchronize()
            if way == "direct":
                step()
                step()
                ctx.synchronize()
            else:
                graph.replay()
                torch.cuda.synchronize()
            results.append([t.clone() for t in (*state, out, lse, n, tok, new)])
        for a, b in zip(*results):
            assert torch.equal(a, b), turn


def test_offsets_beyond_32_bits(ctx, M):
    """A cache of more than 2^31 elements, its rows in use in the last place only: every call reaches them."""
    g = gen(43)
    B, Hkv, cap, H, T = 36, 2, 131072, 16, 1
    ok, ov = (torch.zeros(B, Hkv, cap, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    assert ok.numel() > 2 ** 31
    ok[-1], ov[-1] = rn(g, Hkv, cap, D), rn(g, Hkv, cap, D)
    lens = torch.zeros(B, device="cuda", dtype=torch.int32)
    lens[-1], lens[0] = cap, 3
    q = rn(g, B, T, H, D, scale=1.5)
    out, lse = torch.zeros(B, T, H, D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, T, H, device="cuda")
    ctx.shared_prefix_attn_dev(**attn_args(q, None, None, None, ok, ov, lens, out, lse))
    ctx.synchronize()
    ro, rl, bo, bl = attn_ref(q[-1:], None, None, None, ok[-1:], ov[-1:], lens[-1:])
    assert ((out[-1:].double() - ro).abs() <= bo).all() and ((lse[-1:].double() - rl).abs() <= bl).all()
    assert (out[1:-1] == 0).all() and torch.isneginf(lse[1:-1]).all() and (out[0] == 0).all()
    w = torch.zeros(B, Hkv, cap, device="cuda")
    ctx.attn_weights_accumulate_dev(**weights_args(q, ok, lens, lse, w))
    ctx.synchronize()
    ref, tol = weights_ref(q[-1:], ok[-1:], lens[-1:], lse[-1:], torch.zeros_like(w[-1:]), 1.0)
    assert ((w[-1:].double() - ref).abs() <= tol).all() and (w[1:-1] == 0).all()
    pos = torch.arange(cap, device="cuda", dtype=torch.int32).expand(B, Hkv, cap).contiguous()
    budget, new = 60001, torch.zeros_like(lens)
    src = evict_ref(ok[-1:], ov[-1:], w[-1:], pos[-1:], lens[-1:], lens[-1:], budget, 4, 100)
    k0, v0 = ok[-1].clone(), ov[-1].clone()
    ctx.kv_evict_dev(n_seqs=B, num_kv_heads=Hkv, kv_dtype=M.KV_BF16, cap=cap, k=ok.data_ptr(), v=ov.data_ptr(), seq_stride=ok.stride(0),
                     head_stride=ok.stride(1), row_stride=D, budget=budget, n_sink=4, n_recent=100, lens=lens.data_ptr(), next_pos=lens.data_ptr(),
                     weights=w.data_ptr(), positions=pos.data_ptr(), map_seq_stride=w.stride(0), map_head_stride=w.stride(1),
                     weights_out=w.data_ptr(), positions_out=pos.data_ptr(), lens_out=new.data_ptr())
    ctx.synchronize()
    for (_, h), rows in src.items():
        ix = torch.tensor(rows, device="cuda", dtype=torch.long)
        assert torch.equal(ok[-1, h, :budget], k0[h, ix]) and torch.equal(ov[-1, h, :budget], v0[h, ix])
        assert torch.equal(pos[-1, h, :budget].long(), ix)
    assert new.tolist() == [3] + [0] * (B - 2) + [budget]


def test_largest_evicted_cache(ctx, M):
    """262,144 rows, the most a call takes: clusters of sixteen CTAs."""
    g = gen(44)
    cap, budget = 262144, 100001
    k, v = rn(g, 1, 1, cap, D), rn(g, 1, 1, cap, D)
    w = torch.randint(0, 50000, (1, 1, cap), generator=g, device="cuda").float()
    pos = torch.randperm(cap, generator=g, device="cuda").to(torch.int32).view(1, 1, cap)
    lens = torch.tensor([cap], device="cuda", dtype=torch.int32)
    new, k0, v0 = torch.zeros_like(lens), k.clone(), v.clone()
    rows = evict_ref(k, v, w, pos, lens, lens, budget, 4, 1000)[0, 0]
    wo, po = torch.zeros_like(w), torch.zeros_like(pos)
    ctx.kv_evict_dev(n_seqs=1, num_kv_heads=1, kv_dtype=M.KV_BF16, cap=cap, k=k.data_ptr(), v=v.data_ptr(), seq_stride=k.stride(0),
                     head_stride=k.stride(1), row_stride=D, budget=budget, n_sink=4, n_recent=1000, lens=lens.data_ptr(), next_pos=lens.data_ptr(),
                     weights=w.data_ptr(), positions=pos.data_ptr(), map_seq_stride=cap, map_head_stride=cap, weights_out=wo.data_ptr(),
                     positions_out=po.data_ptr(), lens_out=new.data_ptr())
    ctx.synchronize()
    ix = torch.tensor(rows, device="cuda", dtype=torch.long)
    assert torch.equal(k[0, 0, :budget], k0[0, 0, ix]) and torch.equal(v[0, 0, :budget], v0[0, 0, ix])
    assert torch.equal(wo[0, 0, :budget], w[0, 0, ix]) and torch.equal(po[0, 0, :budget], pos[0, 0, ix]) and new.tolist() == [budget]


def test_batches_that_take_several_launches(ctx, M):
    """More query rows, and more moves, than the context's scratch holds at once."""
    g = gen(45)
    B, T, H, Hkv, P, cap = 2400, 2, 32, 2, 150, 20
    q, pk, pv = rn(g, B, T, H, D), rn(g, Hkv, P, D), rn(g, Hkv, P, D)
    ok, ov = rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    lens = lens_for(g, B, T, cap)
    out, lse = torch.zeros(B, T, H, D, device="cuda", dtype=torch.bfloat16), torch.zeros(B, T, H, device="cuda")
    before = ctx.launch_count
    ctx.shared_prefix_attn_dev(**attn_args(q, q, pk, pv, ok, ov, lens, out, lse))
    ctx.synchronize()
    assert ctx.launch_count > before + 2
    some = torch.tensor([0, 1, 2, 599, 600, 601, 1199, 1200, 1201, 1800, B - 1], device="cuda")
    ro, rl, bo, bl = attn_ref(q[some], q[some], pk, pv, ok[some], ov[some], lens[some])
    assert ((out[some].double() - ro).abs() <= bo).all() and ((lse[some].double() - rl).abs() <= bl).all()
    # every sequence differs from its neighbours, so a slip of the offsets would show above; none is left out
    assert torch.isfinite(lse).all() and (out.float().abs().amax((1, 2, 3)) > 0).all()
    B, Hkv, cap, budget = 4000, 4, 60, 30
    k, v = rn(g, B, Hkv, cap, D), rn(g, B, Hkv, cap, D)
    w = torch.rand(B, Hkv, cap, generator=g, device="cuda")
    pos = torch.arange(cap, device="cuda", dtype=torch.int32).expand(B, Hkv, cap).contiguous()
    lens = torch.randint(0, cap + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    new, k0, v0, w0 = torch.zeros_like(lens), k.clone(), v.clone(), w.clone()
    src = evict_ref(k, v, w, pos, lens, lens, budget, 1, 2)
    ctx.kv_evict_dev(n_seqs=B, num_kv_heads=Hkv, kv_dtype=M.KV_BF16, cap=cap, k=k.data_ptr(), v=v.data_ptr(), seq_stride=k.stride(0),
                     head_stride=k.stride(1), row_stride=D, budget=budget, n_sink=1, n_recent=2, lens=lens.data_ptr(), next_pos=lens.data_ptr(),
                     weights=w.data_ptr(), positions=pos.data_ptr(), map_seq_stride=w.stride(0), map_head_stride=w.stride(1),
                     weights_out=w.data_ptr(), positions_out=pos.data_ptr(), lens_out=new.data_ptr())
    ctx.synchronize()
    ix = torch.arange(cap).expand(B, Hkv, cap).clone()
    for (b, h), rows in src.items():
        ix[b, h, : len(rows)] = torch.tensor(rows, dtype=torch.long)
    ix = ix.cuda()
    at = ix.unsqueeze(-1).expand(B, Hkv, cap, D)
    assert torch.equal(k, k0.gather(2, at)) and torch.equal(v, v0.gather(2, at)) and torch.equal(w, w0.gather(2, ix))
    assert torch.equal(pos.long(), ix) and torch.equal(new, lens.clamp(max=budget))


def test_two_contexts_at_once(M):
    """Two servers on one GPU, each with a context, a stream and inputs of its own: the same bits as one after the other."""
    ways = []
    for seed, (B, T, H, Hkv, P, cap) in [(51, (20, 3, 24, 2, 1700, 300)), (52, (7, 1, 32, 2, 900, 500))]:
        g = gen(seed)
        c, s = M.Ctx(num_layers=4, max_seq=64, n_seqs=1, kv_dtype=M.KV_BF16), torch.cuda.Stream()
        c.set_stream(s.cuda_stream)
        V = 20001
        t = dict(q=rn(g, B, T, H, D), pk=rn(g, Hkv, P, D), pv=rn(g, Hkv, P, D), ok=rn(g, B, Hkv, cap, D), ov=rn(g, B, Hkv, cap, D),
                 lens=lens_for(g, B, T, cap), p=torch.softmax(torch.randn(B, 3, V, generator=g, device="cuda"), -1),
                 x=torch.randint(0, V, (B, 2), generator=g, device="cuda", dtype=torch.int32), ua=torch.rand(B, 2, generator=g, device="cuda"),
                 us=torch.rand(B, generator=g, device="cuda"))
        t.update(out=torch.zeros_like(t["q"]), lse=torch.zeros(B, T, H, device="cuda"), w=torch.zeros(B, Hkv, cap, device="cuda"),
                 pos=torch.arange(cap, device="cuda", dtype=torch.int32).expand(B, Hkv, cap).contiguous(), new=torch.zeros_like(t["lens"]),
                 n=torch.zeros(B, device="cuda", dtype=torch.int32), tok=torch.zeros(B, 3, device="cuda", dtype=torch.int32))
        ways.append((c, t, (B, T, H, Hkv, cap, V)))

    def step(c, t, sizes):
        B, T, H, Hkv, cap, V = sizes
        c.shared_prefix_attn_dev(**attn_args(t["q"], t["q"], t["pk"], t["pv"], t["ok"], t["ov"], t["lens"], t["out"], t["lse"]))
        c.attn_weights_accumulate_dev(**weights_args(t["q"], t["ok"], t["lens"], t["lse"], t["w"], 0.5))
        c.kv_evict_dev(n_seqs=B, num_kv_heads=Hkv, kv_dtype=M.KV_BF16, cap=cap, k=t["ok"].data_ptr(), v=t["ov"].data_ptr(),
                       seq_stride=t["ok"].stride(0), head_stride=t["ok"].stride(1), row_stride=D, budget=100, n_sink=2, n_recent=5,
                       lens=t["lens"].data_ptr(), next_pos=t["lens"].data_ptr(), weights=t["w"].data_ptr(), positions=t["pos"].data_ptr(),
                       map_seq_stride=Hkv * cap, map_head_stride=cap, weights_out=t["w"].data_ptr(), positions_out=t["pos"].data_ptr(),
                       lens_out=t["new"].data_ptr())
        c.verify_drafts_dev(n_seqs=B, max_drafts=2, vocab=V, target_probs=t["p"].data_ptr(), target_seq_stride=3 * V, target_row_stride=V,
                            draft_tokens=t["x"].data_ptr(), u_accept=t["ua"].data_ptr(), u_sample=t["us"].data_ptr(),
                            n_accepted=t["n"].data_ptr(), tokens=t["tok"].data_ptr())

    start = [{k: v.clone() for k, v in t.items()} for _, t, _ in ways]
    results = []
    for together in (False, True):
        for (_, t, _), s in zip(ways, start):
            for k, v in s.items():
                t[k].copy_(v)
        torch.cuda.synchronize()
        if together:
            for _ in range(8):
                for way in ways:
                    step(*way)
        else:
            for way in ways:
                for _ in range(8):
                    step(*way)
                way[0].synchronize()
        for c, _, _ in ways:
            c.synchronize()
        results.append([{k: v.clone() for k, v in t.items()} for _, t, _ in ways])
    for a, b in zip(*results):
        for k in a:
            assert torch.equal(a[k], b[k]), k
    for c, _, _ in ways:
        c.close()
