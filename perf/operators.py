"""The serving operators on cached rows: their cases, their plain forms and the calls a user makes.

attention of a batch that shares a long prefix ("prefix"), accumulation of attention weights per cached row ("weights"),
eviction from a cache by those weights ("evict"), verification of drafted tokens ("verify").  Head dim 256 and the
32-query-head / 2-kv-head layout are the library's default configuration; the others are head layouts it accepts.
"""
import math

import torch

own = False

D = 256
SCALE = 1.0 / 16.0


def listed():
    return [
        # two conversations over a short system prompt: launch latency counts
        dict(name="prefix_two", op="prefix", B=2, T=1, H=32, Hkv=2, P=512, cap=128, gate=True),
        # an ordinary decode batch over a document
        dict(name="prefix_batch16", op="prefix", B=16, T=1, H=32, Hkv=2, P=8192, cap=1024, gate=True),
        # odd sizes: a group of 12 heads, three tokens a sequence, lengths that end inside every tile
        dict(name="prefix_odd", op="prefix", B=37, T=3, H=24, Hkv=2, P=10007, cap=777, gate=False),
        # a full batch that verifies three drafted tokens a sequence over a long shared context
        dict(name="prefix_largest", op="prefix", B=64, T=4, H=32, Hkv=2, P=32768, cap=2048, gate=True),
        # one sequence, one token
        dict(name="weights_one", op="weights", B=1, T=1, H=32, Hkv=2, cap=1024, decay=1.0),
        # an ordinary ragged decode batch
        dict(name="weights_ragged", op="weights", B=16, T=1, H=32, Hkv=2, cap=8191, decay=1.0),
        # long caches, four tokens a sequence, old weights fading
        dict(name="weights_largest", op="weights", B=32, T=4, H=32, Hkv=2, cap=32768, decay=0.96875),
        # the steady state of a bounded cache: a few rows over the budget
        dict(name="evict_step", op="evict", B=4, Hkv=2, cap=1088, budget=1024, dtype="bf16"),
        # prompts cut to a budget, fp32 cache, odd length
        dict(name="evict_prompt_f32", op="evict", B=8, Hkv=2, cap=20011, budget=4096, dtype="f32"),
        # a full batch halved
        dict(name="evict_largest", op="evict", B=64, Hkv=2, cap=16384, budget=8192, dtype="bf16"),
        # one sequence with four drafted tokens
        dict(name="verify_one", op="verify", B=1, K=4, V=32768, probs=True),
        # a large batch, eight drafted tokens, a large vocabulary
        dict(name="verify_largest", op="verify", B=128, K=8, V=131072, probs=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_LAYOUTS = [(32, 2), (16, 2), (24, 2), (10, 2), (32, 4), (8, 8), (16, 1), (7, 1)]


def draw(rng):
    op = rng.choice(["prefix", "weights", "evict", "verify"])
    if op == "prefix":
        H, Hkv = rng.choice(_LAYOUTS)
        c = dict(op=op, B=_log(rng, 1, 96), T=rng.choice([1, 1, 2, 3, 4, 5]), H=H, Hkv=Hkv, P=_log(rng, 1, 40000),
                 cap=_log(rng, 8, 2048), gate=rng.random() < 0.5)
        while c["B"] * c["T"] * c["H"] * (c["P"] + c["cap"]) > 64 * 4 * 32 * (32768 + 2048):
            c["P"] = c["P"] * 3 // 4
        return c
    if op == "weights":
        H, Hkv = rng.choice(_LAYOUTS)
        c = dict(op=op, B=_log(rng, 1, 32), T=rng.choice([1, 1, 2, 4, 5]), H=H, Hkv=Hkv, cap=_log(rng, 16, 32768),
                 decay=rng.choice([1.0, 0.96875]))
        while c["B"] * c["Hkv"] * c["cap"] * (512 + 2 * c["T"] * H // Hkv) > 32 * 2 * 32768 * (512 + 128):
            c["cap"] = c["cap"] * 3 // 4
        return c
    if op == "evict":
        cap = _log(rng, 32, 32768)
        c = dict(op=op, B=_log(rng, 1, 64), Hkv=rng.choice([1, 2, 4, 8]), cap=cap, budget=0, dtype=rng.choice(["bf16", "bf16", "f32"]))
        while c["B"] * c["Hkv"] * c["cap"] * (2 if c["dtype"] == "f32" else 1) > 64 * 2 * 16384:
            c["cap"] = c["cap"] * 3 // 4
        c["budget"] = max(1, int(c["cap"] * rng.choice([rng.uniform(0.1, 0.9), rng.uniform(0.9, 1.0)])))
        return c
    return dict(op=op, B=_log(rng, 1, 128), K=rng.choice([1, 2, 3, 4, 5, 8]), V=_log(rng, 1000, 131072), probs=rng.random() < 0.8)


# ---------------------------------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _lens(g, B, lo, cap):
    """Lengths from `lo` to the cache's capacity, one of them full, and in larger batches one empty (an idle place)."""
    n = torch.randint(min(lo, cap), cap + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = cap
    if B >= 8:
        n[B // 2] = 0
    return n


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op = case["op"]
    B = case["B"]
    if op == "prefix":
        T, H, Hkv, P, cap = (case[k] for k in ("T", "H", "Hkv", "P", "cap"))
        s["q"] = _randn(g, B, T, H, D, scale=1.5)
        s["gate_x"] = _randn(g, B, T, H, D) if case["gate"] else None
        s["pk"], s["pv"] = _randn(g, Hkv, P, D), _randn(g, Hkv, P, D)
        s["ok"], s["ov"] = _randn(g, B, Hkv, cap, D), _randn(g, B, Hkv, cap, D)
        s["lens"] = _lens(g, B, T, cap)
        s["out"] = torch.zeros(B, T, H, D, device="cuda", dtype=torch.bfloat16)
        s["lse"] = torch.zeros(B, T, H, device="cuda")
    elif op == "weights":
        T, H, Hkv, cap = (case[k] for k in ("T", "H", "Hkv", "cap"))
        s["q"] = _randn(g, B, T, H, D, scale=1.5)
        s["k"] = _randn(g, B, Hkv, cap, D)
        s["lens"] = _lens(g, B, max(T, cap // 32), cap)
        s["w"] = torch.rand(B, Hkv, cap, generator=g, device="cuda") * 4.0
        # what the attention call of the same step returned: ln sum exp over the rows each query sees
        sc = _own_scores(s["q"], s["k"], s["lens"])
        s["lse"] = torch.logsumexp(sc, -1).view(B, Hkv, T, H // Hkv).transpose(1, 2).reshape(B, T, H).contiguous()
    elif op == "evict":
        Hkv, cap = case["Hkv"], case["cap"]
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        s["k"], s["v"] = _randn(g, B, Hkv, cap, D, dtype=dt), _randn(g, B, Hkv, cap, D, dtype=dt)
        s["lens"] = _lens(g, B, max(1, case["budget"] - case["budget"] // 8), cap)
        # accumulated weights are heavy-tailed; positions are a permutation, as earlier evictions leave them
        s["w"] = torch.exp(2.0 * torch.randn(B, Hkv, cap, generator=g, device="cuda") - 2.0)
        order = torch.arange(cap, device="cuda", dtype=torch.float32)
        order = order + (torch.rand(B, Hkv, cap, generator=g, device="cuda") < 0.3) * torch.randn(B, Hkv, cap, generator=g, device="cuda") * cap / 8
        order.masked_fill_(torch.arange(cap, device="cuda") >= s["lens"].view(B, 1, 1), float("inf"))
        s["pos"] = torch.argsort(torch.argsort(order, -1), -1).to(torch.int32)
        s["next"] = s["lens"].clone()
        s["sink"], s["recent"] = 4, max(1, case["budget"] // 16)
        s["w_out"], s["pos_out"], s["lens_out"] = torch.zeros_like(s["w"]), torch.zeros_like(s["pos"]), torch.zeros_like(s["lens"])
    else:
        K, V = case["K"], case["V"]
        logits = torch.randn(B, K + 1, V, generator=g, device="cuda") * 2.5
        s["p"] = torch.softmax(logits, -1)
        q = logits[:, :K].add_(torch.randn(B, K, V, generator=g, device="cuda") * 0.6)  # the draft model: near the target
        del logits
        gumbel = -torch.log(-torch.log(torch.rand(B, K, V, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)))
        s["x"] = torch.argmax(gumbel.add_(q), -1).to(torch.int32)
        del gumbel
        s["q"] = torch.softmax(q, -1) if case["probs"] else None  # without: drafts that were looked up, not sampled
        s["lens"] = torch.full((B,), K, device="cuda", dtype=torch.int32)
        if B >= 4:
            s["lens"] = torch.randint(0, K + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        s["ua"] = torch.rand(B, K, generator=g, device="cuda")
        s["us"] = torch.rand(B, generator=g, device="cuda")
        s["n"] = torch.zeros(B, device="cuda", dtype=torch.int32)
        s["tok"] = torch.zeros(B, K + 1, device="cuda", dtype=torch.int32)
    return s


# ---------------------------------------------------------------------------------------------------- plain forms


def _seen(lens, T, G, cap):
    """[B, 1, T*G, cap]: whether query (token, head of the group) sees the row."""
    t = torch.arange(T, device=lens.device).repeat_interleave(G)
    n = lens.view(-1, 1, 1, 1) - (T - 1 - t).view(1, 1, -1, 1)
    return torch.arange(cap, device=lens.device).view(1, 1, 1, -1) < n


def _own_scores(q, k, lens):
    """[B, Hkv, T*G, cap] scaled scores against a sequence's own rows, -inf where a query does not see the row."""
    B, T, H, _ = q.shape
    Hkv, cap = k.shape[1], k.shape[2]
    G = H // Hkv
    qq = q.float().view(B, T, Hkv, G, D).transpose(1, 2).reshape(B, Hkv, T * G, D)
    sc = torch.matmul(qq, k.float().transpose(-1, -2)).mul_(SCALE)
    return sc.masked_fill_(~_seen(lens, T, G, cap), float("-inf"))


def _plain_prefix(s):
    B, T, H, Hkv, P = (s[k] for k in ("B", "T", "H", "Hkv", "P"))
    G = H // Hkv
    so = _own_scores(s["q"], s["ok"], s["lens"])
    qp = s["q"].float().view(B * T, Hkv, G, D).transpose(0, 1).reshape(Hkv, B * T * G, D)
    sp = torch.matmul(qp, s["pk"].float().transpose(-1, -2)).mul_(SCALE)
    mp = sp.amax(-1).view(Hkv, B, T * G).transpose(0, 1)
    m = torch.maximum(so.amax(-1), mp)  # [B, Hkv, T*G]
    eo = so.sub_(m.unsqueeze(-1)).exp_()
    ep = sp.sub_(m.transpose(0, 1).reshape(Hkv, B * T * G, 1)).exp_()
    l = eo.sum(-1) + ep.sum(-1).view(Hkv, B, T * G).transpose(0, 1)
    o = torch.matmul(eo, s["ov"].float())
    o = o + torch.matmul(ep, s["pv"].float()).view(Hkv, B, T * G, D).transpose(0, 1)
    o = (o / l.unsqueeze(-1)).view(B, Hkv, T, G, D).transpose(1, 2).reshape(B, T, H, D)
    if s["gate_x"] is not None:
        o = o * torch.sigmoid(s["gate_x"].float())
    lse = (m + torch.log(l)).view(B, Hkv, T, G).transpose(1, 2).reshape(B, T, H)
    return {"out": o.to(torch.bfloat16), "lse": lse}


def _plain_weights(s):
    B, T, H, Hkv, cap = (s[k] for k in ("B", "T", "H", "Hkv", "cap"))
    G = H // Hkv
    sc = _own_scores(s["q"], s["k"], s["lens"])
    lse = s["lse"].view(B, T, Hkv, G).transpose(1, 2).reshape(B, Hkv, T * G, 1)
    p = torch.where(sc == float("-inf"), 0.0, sc.sub_(lse).exp_()).sum(2)
    used = torch.arange(cap, device=p.device) < s["lens"].view(B, 1, 1)
    s["w"].copy_(torch.where(used, s["w"] * s["decay"] + p, s["w"]))
    return {"weights": s["w"]}


def _plain_evict(s):
    B, Hkv, cap, budget = (s[k] for k in ("B", "Hkv", "cap", "budget"))
    dev = s["w"].device
    row = torch.arange(cap, device=dev)
    used = (row < s["lens"].view(B, 1, 1)).expand(B, Hkv, cap)
    safe = (s["pos"] < s["sink"]) | (s["pos"] >= s["next"].view(B, 1, 1) - s["recent"])
    w = torch.where(torch.isnan(s["w"]), float("-inf"), s["w"])
    by_w = torch.sort(w, dim=-1, descending=True, stable=True).indices  # ties: lowest row first
    cls = torch.where(used, torch.where(safe, 0, torch.where(torch.isnan(s["w"]), 2, 1)), 3)
    order = by_w.gather(-1, torch.sort(cls.gather(-1, by_w), dim=-1, stable=True).indices)
    # the protected rows' keys are all alike: among them, too, the lowest row goes first
    tied = torch.where(cls.gather(-1, order) == 0, order, cap + row)
    order = order.gather(-1, torch.sort(tied, dim=-1, stable=True).indices)
    new = s["lens"].clamp(max=budget)
    rank = torch.empty_like(order).scatter_(-1, order, row.expand_as(order))
    kept = rank < new.view(B, 1, 1)
    hole, mover = ~kept & (row < new.view(B, 1, 1)), kept & (row >= budget)
    # the j-th hole takes the j-th kept row behind the budget
    hole_at = torch.sort(torch.where(hole, row, cap), -1).values[..., :budget]
    from_at = torch.sort(torch.where(mover, row, cap), -1).values[..., :budget]
    n = int(budget) if budget < cap else cap
    src = row.expand(B, Hkv, cap).clone()
    pad = torch.zeros(B, Hkv, 1, device=dev, dtype=src.dtype)
    src = torch.cat([src, pad], -1).scatter_(-1, hole_at, from_at.clamp(max=cap - 1))[..., :n]
    live = (row[:n] < new.view(B, 1, 1))
    src = torch.where(live, src, row[:n])
    for t in (s["k"], s["v"]):
        t[:, :, :n] = t.gather(2, src.unsqueeze(-1).expand(B, Hkv, n, D))
    s["w_out"][..., :n] = torch.where(live, s["w"].gather(-1, src), s["w_out"][..., :n])
    s["pos_out"][..., :n] = torch.where(live, s["pos"].gather(-1, src), s["pos_out"][..., :n])
    s["lens_out"].copy_(new)
    return {"k": s["k"], "v": s["v"], "weights": s["w_out"], "positions": s["pos_out"], "lens": s["lens_out"]}


def _plain_verify(s):
    B, K, V = s["B"], s["K"], s["V"]
    x = s["x"].long().unsqueeze(-1)
    px = s["p"][:, :K].gather(-1, x).squeeze(-1).double()
    qx = s["q"].gather(-1, x).squeeze(-1).double() if s["q"] is not None else torch.ones_like(px)
    dev = px.device
    i = torch.arange(K, device=dev)
    fine = (s["ua"].double() * qx < px) & (i < s["lens"].view(B, 1))
    n = torch.cumprod(fine.long(), -1).sum(-1)
    row = n.view(B, 1, 1).expand(B, 1, V)
    p = s["p"].gather(1, row).squeeze(1).double()
    cut = (n < s["lens"]).view(B, 1)
    at = n.clamp(max=K - 1).view(B, 1, 1)
    if s["q"] is not None:
        q = s["q"].gather(1, at.expand(B, 1, V)).squeeze(1).double()
    else:
        q = torch.zeros(B, V, device=dev, dtype=torch.float64).scatter_(1, x.gather(1, at).squeeze(1), float("inf"))
    w = torch.where(cut, p - q, p)
    w = torch.where(w > 0, w, 0.0)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, torch.where(p > 0, p, 0.0))
    c = torch.cumsum(w, -1)
    t = (c <= s["us"].double().view(B, 1) * c[:, -1:]).sum(-1)
    t = torch.where(t < V, t, -1)
    j = torch.arange(K + 1, device=dev)
    x1 = torch.cat([s["x"].long(), torch.full((B, 1), -1, device=dev)], 1)
    tok = torch.where(j < n.view(B, 1), x1, torch.where(j == n.view(B, 1), t.view(B, 1), -1))
    return {"accepted": n.to(torch.int32), "tokens": tok.to(torch.int32)}


# ---------------------------------------------------------------------------------------------------- the calls


_ctxs = {}


def _handle():
    """The context that a user's program keeps open for the current device and stream: its work is ordered by that stream."""
    device = torch.cuda.current_device()
    at = (device, torch._C._cuda_getCurrentRawStream(device))  # (a torch.cuda.Stream object of it takes 3 us to make)
    if at not in _ctxs:
        import moeflux_b200 as M

        _ctxs[at] = M.Ctx(num_layers=4, max_seq=64, kv_dtype=M.KV_BF16, device=device)
        _ctxs[at].set_stream(at[1])
    return _ctxs[at]


def _own_run(s):
    c = _handle()
    op = s["op"]
    if op == "prefix":
        q, gt, pk, ok = s["q"], s["gate_x"], s["pk"], s["ok"]
        c.shared_prefix_attn_dev(
            n_seqs=s["B"], n_tokens=s["T"], num_attn_heads=s["H"], num_kv_heads=s["Hkv"], softmax_scale=SCALE,
            q=q.data_ptr(), q_seq_stride=q.stride(0), q_token_stride=q.stride(1), q_head_stride=q.stride(2),
            gate=gt.data_ptr() if gt is not None else None, gate_seq_stride=q.stride(0), gate_token_stride=q.stride(1),
            gate_head_stride=q.stride(2), prefix_k=pk.data_ptr(), prefix_v=s["pv"].data_ptr(), prefix_head_stride=pk.stride(0),
            prefix_row_stride=pk.stride(1), prefix_len=s["P"], own_k=ok.data_ptr(), own_v=s["ov"].data_ptr(),
            own_seq_stride=ok.stride(0), own_head_stride=ok.stride(1), own_row_stride=ok.stride(2), own_cap=s["cap"],
            own_lens=s["lens"].data_ptr(), out=s["out"].data_ptr(), lse=s["lse"].data_ptr())
        return {"out": s["out"], "lse": s["lse"]}
    if op == "weights":
        q, k, w = s["q"], s["k"], s["w"]
        c.attn_weights_accumulate_dev(
            n_seqs=s["B"], n_tokens=s["T"], num_attn_heads=s["H"], num_kv_heads=s["Hkv"], softmax_scale=SCALE, decay=s["decay"],
            q=q.data_ptr(), q_seq_stride=q.stride(0), q_token_stride=q.stride(1), q_head_stride=q.stride(2), k=k.data_ptr(),
            k_seq_stride=k.stride(0), k_head_stride=k.stride(1), k_row_stride=k.stride(2), cap=s["cap"], lens=s["lens"].data_ptr(),
            lse=s["lse"].data_ptr(), weights=w.data_ptr(), weights_seq_stride=w.stride(0), weights_head_stride=w.stride(1))
        return {"weights": w}
    if op == "evict":
        import moeflux_b200 as M

        k, w = s["k"], s["w"]
        c.kv_evict_dev(
            n_seqs=s["B"], num_kv_heads=s["Hkv"], kv_dtype=M.KV_BF16 if s["dtype"] == "bf16" else M.KV_F32, cap=s["cap"],
            k=k.data_ptr(), v=s["v"].data_ptr(), seq_stride=k.stride(0), head_stride=k.stride(1), row_stride=k.stride(2),
            budget=s["budget"], n_sink=s["sink"], n_recent=s["recent"], lens=s["lens"].data_ptr(), next_pos=s["next"].data_ptr(),
            weights=w.data_ptr(), positions=s["pos"].data_ptr(), map_seq_stride=w.stride(0), map_head_stride=w.stride(1),
            weights_out=s["w_out"].data_ptr(), positions_out=s["pos_out"].data_ptr(), lens_out=s["lens_out"].data_ptr())
        return {"k": k, "v": s["v"], "weights": s["w_out"], "positions": s["pos_out"], "lens": s["lens_out"]}
    p, q = s["p"], s["q"]
    c.verify_drafts_dev(
        n_seqs=s["B"], max_drafts=s["K"], vocab=s["V"], target_probs=p.data_ptr(), target_seq_stride=p.stride(0),
        target_row_stride=p.stride(1), draft_probs=q.data_ptr() if q is not None else None,
        draft_seq_stride=q.stride(0) if q is not None else 0, draft_row_stride=q.stride(1) if q is not None else 0,
        draft_tokens=s["x"].data_ptr(), draft_lens=s["lens"].data_ptr(), u_accept=s["ua"].data_ptr(), u_sample=s["us"].data_ptr(),
        n_accepted=s["n"].data_ptr(), tokens=s["tok"].data_ptr())
    return {"accepted": s["n"], "tokens": s["tok"]}


_PLAIN = {"prefix": _plain_prefix, "weights": _plain_weights, "evict": _plain_evict, "verify": _plain_verify}


def run(state):
    if own:
        return _own_run(state)
    return _PLAIN[state["op"]](state)


# ---------------------------------------------------------------------------------------------------- floors and 64 bits


def work(case):
    B = case["B"]
    if case["op"] == "prefix":
        T, H, Hkv, P = (case[k] for k in ("T", "H", "Hkv", "P"))
        rows = B * (case["cap"] + T) / 2  # lengths are spread evenly
        return {"bytes": 1024.0 * Hkv * (P + rows) + B * T * H * (1028.0 + (512 if case["gate"] else 0)),
                "flops": 4.0 * D * H * T * (B * P + rows)}
    if case["op"] == "weights":
        T, H, Hkv = (case[k] for k in ("T", "H", "Hkv"))
        rows = B * case["cap"] * (33 / 64)
        return {"bytes": rows * Hkv * 520.0 + B * T * H * 516.0, "flops": 2.0 * D * H * T * rows}
    if case["op"] == "evict":
        Hkv, cap, budget = case["Hkv"], case["cap"], case["budget"]
        lo = min(cap, max(1, budget - budget // 8))
        length = (lo + cap) / 2
        moved = max(0.0, budget * (1 - budget / max(length, budget)))
        esize = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": B * Hkv * (8.0 * length + 8.0 * min(length, budget) + moved * 4 * D * esize), "flops": 0}
    return {"bytes": B * case["V"] * 4.0 * (1.5 if case["probs"] else 1.0), "flops": 0}


def exact(case, seed):
    """The attention operators in 64 bits, one kv head and a few sequences at a time; the others return copies and whole numbers."""
    if case["op"] not in ("prefix", "weights"):
        return None
    s = prepare(case, seed)
    B, T, H, Hkv = (case[k] for k in ("B", "T", "H", "Hkv"))
    G = H // Hkv
    dev = s["q"].device
    lens = s["lens"].tolist()
    if case["op"] == "weights":
        w = s["w"].double()
        for b in range(B):
            n = lens[b]
            if n == 0:
                continue
            q = s["q"][b].double().reshape(T, Hkv, G, D)
            sc = torch.einsum("thgd,hjd->thgj", q, s["k"][b, :, :n].double()) / 16.0
            pr = torch.exp(sc - s["lse"][b].double().reshape(T, Hkv, G, 1))
            j, t = torch.arange(n, device=dev), torch.arange(T, device=dev)
            pr = pr * (j.view(1, -1) <= (n - T + t).view(-1, 1)).view(T, 1, 1, n)
            w[b, :, :n] = w[b, :, :n] * case["decay"] + torch.nan_to_num(pr).sum((0, 2))
        return {"weights": w}
    out = torch.empty(B, T, H, D, device=dev, dtype=torch.float64)
    lse = torch.empty(B, T, H, device=dev, dtype=torch.float64)
    for h in range(Hkv):
        heads = slice(h * G, (h + 1) * G)
        pk, pv = s["pk"][h].double(), s["pv"][h].double()
        for b in range(B):
            k = torch.cat([pk, s["ok"][b, h, : lens[b]].double()])
            v = torch.cat([pv, s["ov"][b, h, : lens[b]].double()])
            sc = torch.einsum("tgd,jd->tgj", s["q"][b, :, heads].double(), k) / 16.0
            vis = case["P"] + lens[b] - (T - 1) + torch.arange(T, device=dev)
            vis = torch.clamp(vis, min=case["P"])
            sc = sc.masked_fill(torch.arange(k.shape[0], device=dev).view(1, 1, -1) >= vis.view(T, 1, 1), float("-inf"))
            z = torch.logsumexp(sc, -1)
            out[b, :, heads] = torch.einsum("tgj,jd->tgd", torch.exp(sc - z.unsqueeze(-1)), v)
            lse[b, :, heads] = z
    if s["gate_x"] is not None:
        out = out / (1.0 + torch.exp(-s["gate_x"].double()))
    return {"out": out, "lse": lse}
