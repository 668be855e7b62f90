"""Workloads of the paged cache: block tables and slot maps from request lengths, append through a slot map, per-head
norm with multi-axis rotary positions, attention of ragged batches over pages, cross attention to cached states.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once) or, where `own` is
true, by the calls a user makes of this package."""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a batch of 64: every request gets one token, few need a page (latency of one launch)
        dict(name="plan_step_64", op="plan", requests=64, long_every=0, long=1, past=32768, page=16, spare=1.0),
        # an admission round of a large server: single tokens with chunks among them, fewer free pages than wanted
        dict(name="plan_admit_4096", op="plan", requests=4096, long_every=64, long=1000, past=4096, page=16, spare=0.7),
        # K/V rows of one decode step
        dict(name="append_step_64", op="append", tokens=64, kvh=4, hd=128, page=16, dtype="f16"),
        # K/V rows of a batch of prompt chunks, padded at its end
        dict(name="append_chunk_8191", op="append", tokens=8191, kvh=8, hd=256, page=32, dtype="bf16"),
        # the step in front of a decode step's attention: norm, three axes of positions, rows to their pages
        dict(name="rope_step_64", op="rope", tokens=64, heads=28, kvh=4, hd=128, rot=128, axes=3, inter=False, norm=True,
             page=16, dtype="f16"),
        # the same for packed prompt chunks with images among them
        dict(name="rope_chunk_8192", op="rope", tokens=8192, heads=28, kvh=4, hd=128, rot=128, axes=3, inter=True, norm=True,
             page=64, dtype="bf16"),
        # one short request, one new token: nothing but latency
        dict(name="attend_one_512", op="attend", requests=1, step=1, long_every=0, long=0, keys=512, even=True, heads=14,
             kvh=2, hd=64, window=0, page=16, dtype="f16"),
        # decode of a full batch over long requests: the cache is read once
        dict(name="attend_step_64x32k", op="attend", requests=64, step=1, long_every=0, long=0, keys=32768, even=False,
             heads=28, kvh=4, hd=128, window=0, page=16, dtype="f16"),
        # a prompt chunk deep inside a long request: tensor-core work
        dict(name="attend_chunk_2048_of_32k", op="attend", requests=1, step=2048, long_every=0, long=0, keys=32768,
             even=True, heads=28, kvh=4, hd=128, window=0, page=64, dtype="bf16"),
        # decode steps and prompt chunks in one batch, sliding-window layer
        dict(name="attend_mixed_window", op="attend", requests=64, step=1, long_every=16, long=500, keys=8192, even=False,
             heads=16, kvh=8, hd=256, window=1024, page=32, dtype="f16"),
        # decoder steps against encoder states
        dict(name="cross_step_32x1500", op="cross", requests=32, step=1, long_every=0, long=0, keys=1500, even=False,
             heads=16, kvh=16, hd=64, window=0, page=16, dtype="bf16"),
        # decoder prompts against encoder states
        dict(name="cross_prompt_8x448", op="cross", requests=8, step=448, long_every=0, long=0, keys=4096, even=False,
             heads=28, kvh=4, hd=128, window=0, page=64, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "rope", "attend", "attend", "attend", "cross"])
    page = rng.choice([8, 16, 16, 32, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    if op == "plan":
        return dict(op=op, requests=_log(rng, 1, 4096), long_every=rng.choice([0, 3, 16, 64]), long=_log(rng, 2, 1000),
                    past=_log(rng, 64, 4096), page=page, spare=rng.choice([1.0, 1.0, 0.6]))
    heads, kvh, hd = rng.choice([(28, 4, 128), (14, 2, 64), (32, 32, 96), (16, 8, 256), (32, 8, 128), (16, 16, 64),
                                 (16, 1, 128), (12, 4, 64)])
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 8191), kvh=kvh, hd=hd, page=page, dtype=dtype)
    if op == "rope":
        return dict(op=op, tokens=_log(rng, 1, 4000), heads=heads, kvh=kvh, hd=hd, rot=rng.choice([hd, hd, hd // 2]),
                    axes=rng.choice([1, 2, 3]), inter=rng.random() < 0.5, norm=rng.random() < 0.7, page=page, dtype=dtype)
    keys, step = _log(rng, 32, 16384), rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 1500)])
    step = min(step, keys)
    most = max(1, min(int(3.0e8 / (keys * kvh * hd * 2)), int(4.0e11 / (4.0 * heads * hd * keys * step)), 1 + 12000 // step))
    return dict(op=op, requests=_log(rng, 1, min(256, most)), step=step, long_every=0 if step > 1 else rng.choice([0, 0, 9]),
                long=min(keys, _log(rng, 20, 400)), keys=keys, even=rng.random() < 0.3, heads=heads, kvh=kvh, hd=hd,
                window=0 if op == "cross" else rng.choice([0, 0, 0, 256, 1024]), page=page, dtype=dtype)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _sections(case):
    half, n = case["rot"] // 2, case["axes"]
    if n == 1:
        return [half]
    if case["inter"]:
        rest = [half // n - (1 if half // n > 1 else 0)] * (n - 1)
    else:
        rest = [(half * 3 // 8) if n == 3 else half // 2] * (n - 1)
    return [half - sum(rest)] + rest


def _lengths(case, seed):
    """Host lists (new tokens, keys) of an attention batch: the same numbers of tokens for every seed, in another order."""
    g = torch.Generator().manual_seed(seed)
    new, keys = [], []
    for r in torch.randperm(case["requests"], generator=g).tolist():
        is_long = case["long_every"] and r % case["long_every"] == case["long_every"] - 1
        top = case["long"] if is_long else case["step"]
        new.append(top if case["even"] or top < 3 else top - (r * 7919 + 13) % ((top + 1) // 2))
        k = case["keys"] if case["even"] else int(torch.randint((case["keys"] + 1) // 2, case["keys"] + 1, (1,), generator=g))
        keys.append(max(k, new[-1]) if case["op"] == "attend" else k)
    return new, keys


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, dtype, *shape):
    out = torch.empty(shape, dtype=DTYPES[dtype], device="cuda")
    return out.normal_(generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "plan":
        h = torch.Generator().manual_seed(seed)
        R, P = case["requests"], case["page"]
        past = torch.randint(0, case["past"] + 1, (R,), generator=h)
        new = torch.ones(R, dtype=torch.int64)
        if case["long_every"]:
            at = torch.arange(case["long_every"] - 1, R, case["long_every"])
            new[at] = (at * 7919 + 13) % case["long"] + 1
            new = new[torch.randperm(R, generator=h)]     # the same number of tokens for every seed
        cols = (case["past"] + case["long"] + P) // P + 1
        have, want = (past + P - 1) // P, (past + new + P - 1) // P
        pages = int(have.sum() + (want - have).sum()) + 16
        ids = torch.randperm(pages, generator=h)
        used = int(have.sum())
        table = torch.full((R, cols), -1, dtype=torch.int32)
        table[torch.arange(cols)[None, :] < have[:, None]] = ids[:used].to(torch.int32)
        free = torch.full((pages,), -1, dtype=torch.int32)        # a stack with room for every page
        free[:pages - used] = ids[used:].to(torch.int32)
        count = int((pages - used) * case["spare"])
        tokens = (int(new.sum()) + 15) // 16 * 16
        return dict(past=past.to(torch.int32).cuda(), new=new.to(torch.int32).cuda(), table=table.cuda(), free=free.cuda(),
                    count=_i32([count]), tokens=tokens, pages=pages, cols=cols)
    if op in ("append", "rope"):
        T, P, kvh, hd = case["tokens"], case["page"], case["kvh"], case["hd"]
        pages = (T + P - 1) // P + max(4, T // P // 4)
        slots = torch.randperm(pages * P, generator=g, device="cuda")[:T].to(torch.int32)
        slots[T - T // 32:] = -1                      # a padded batch: the last rows belong to nobody
        d = dict(k=_randn(g, case["dtype"], T, kvh, hd), v=_randn(g, case["dtype"], T, kvh, hd), slots=slots, pages=pages,
                 k_cache=_randn(g, case["dtype"], pages, P, kvh, hd), v_cache=_randn(g, case["dtype"], pages, P, kvh, hd))
        if op == "rope":
            d["q"] = _randn(g, case["dtype"], T, case["heads"], hd)
            d["pos"] = torch.randint(0, 131072, (case["axes"], T), generator=g, device="cuda", dtype=torch.int32)
            if case["norm"]:
                d["qw"] = (1.0 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
                d["kw"] = (1.0 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
        return d
    new, keys = _lengths(case, seed)
    P, kvh, hd = case["page"], case["kvh"], case["hd"]
    need = [(k + P - 1) // P for k in keys]
    cols = max(need)
    pages = sum(need) + 4
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(keys), cols), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(cols, device="cuda")[None, :] < _i32(need)[:, None]] = ids[:sum(need)]
    T = sum(new)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return dict(q=_randn(g, case["dtype"], T, case["heads"], hd), k_cache=_randn(g, case["dtype"], pages, P, kvh, hd),
                v_cache=_randn(g, case["dtype"], pages, P, kvh, hd), table=table, q_start=_i32(start), step=_i32(new),
                keys=_i32(keys), new_host=new, keys_host=keys, start_host=start, pages=pages, cols=cols)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        import importlib
        hkv = importlib.import_module("hector-engine_b200")
        op = case["op"]
        kw = dict(page_size=case["page"], num_pages=state["pages"], dtype={"f16": torch.float16, "bf16": torch.bfloat16}[case.get("dtype", "f16")])
        if op == "plan":
            kw.update(num_heads=1, num_kv_heads=1, head_dim=64, max_requests=case["requests"], max_pages=state["cols"],
                      max_tokens=state["tokens"], flags=hkv.FLAG_APPEND_ONLY)
        elif op in ("append", "rope"):
            kw.update(num_heads=case.get("heads", case["kvh"]), num_kv_heads=case["kvh"], head_dim=case["hd"], max_requests=1,
                      max_pages=1, max_tokens=case["tokens"], flags=hkv.FLAG_APPEND_ONLY)
        else:
            kw.update(num_heads=case["heads"], num_kv_heads=case["kvh"], head_dim=case["hd"], window_size=case["window"],
                      max_requests=case["requests"], max_pages=state["cols"], max_tokens=state["q"].shape[0])
        state["ctx"] = hkv.PagedContext(hkv.PagedGeometry(**kw))
        if op == "plan":
            state["tables"] = state["ctx"].new_step(case["requests"], state["tokens"])
        if op == "rope":
            state["q_out"] = torch.empty_like(state["q"])
        if op in ("attend", "cross"):
            state["out"] = torch.empty_like(state["q"])
    return state


# ---- the operators --------------------------------------------------------------------------------------------------
def run(state):
    return {"plan": _plan, "append": _append, "rope": _rope, "attend": _attend, "cross": _attend}[state["case"]["op"]](state)


def _plan(s):
    if own:
        t = s["tables"]
        s["ctx"].plan(s["past"], s["new"], s["table"], s["free"], s["count"], t)
        return dict(table=s["table"], total=t.total_len, step=t.step_len, q_start=t.q_start, slots=t.slots,
                    positions=t.positions, left=t.free_left)
    P, T = s["case"]["page"], s["tokens"]
    past, new = s["past"].long(), s["new"].long()
    table = s["table"]
    R, cols = table.shape
    incl = torch.cumsum(new, 0)
    start = incl - new
    fits = (past + new <= cols * P) & (incl <= T)
    have, want = (past + P - 1) // P, (past + new + P - 1) // P
    need = torch.where(fits, want - have, 0)
    upto = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (upto <= s["count"]))
    step = torch.where(ok, new, 0)
    total = past + step
    j = torch.arange(cols, device="cuda")[None, :]
    fresh = ok[:, None] & (j >= have[:, None]) & (j < want[:, None])
    take = s["count"] - 1 - (upto - need)[:, None] - (j - have[:, None])
    table = torch.where(fresh, s["free"][take.clamp(0, len(s["free"]) - 1)], table)
    t = torch.arange(T, device="cuda")
    r = torch.searchsorted(incl, t, right=True).clamp(max=R - 1)
    live = (t < incl[-1]) & ok[r]
    pos = past[r] + t - start[r]
    page = table[r, (pos // P).clamp(0, cols - 1)].long()
    i32 = torch.int32
    return dict(table=table, total=total.to(i32), step=step.to(i32),
                q_start=torch.cat([start, incl[-1:]]).to(i32), slots=torch.where(live, page * P + pos % P, -1).to(i32),
                positions=torch.where(live, pos, -1).to(i32), left=(s["count"] - torch.where(ok, need, 0).sum()).to(i32))


def _append(s):
    if own:
        s["ctx"].append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return dict(k=s["k_cache"], v=s["v_cache"])
    _scatter(s, s["k"], s["v"])
    return dict(k=s["k_cache"], v=s["v_cache"])


def _scatter(s, k, v):
    n = s["slots"].shape[0] - s["slots"].shape[0] // 32       # rows behind it belong to nobody
    at = s["slots"][:n].long()
    s["k_cache"].view(-1, *k.shape[1:])[at] = k[:n]
    s["v_cache"].view(-1, *v.shape[1:])[at] = v[:n]


def _axis_of_pair(case):
    """Axis of each rotary pair, on the GPU."""
    half, n, sec = case["rot"] // 2, case["axes"], _sections(case)
    i = torch.arange(half, device="cuda")
    if not case["inter"]:
        ends = torch.cumsum(torch.tensor(sec, device="cuda"), 0)
        return torch.searchsorted(ends, i, right=True).clamp(max=n - 1)
    sec = torch.tensor(sec, device="cuda")
    return torch.where((i % n > 0) & (i // n < sec[i % n]), i % n, 0)


THETA, EPS = 1.0e6, 1.0e-6


def _rope(s):
    c = s["case"]
    if own:
        s["ctx"].norm_rope(s["q"], s["k"], s["v"], s["pos"], slots=s["slots"], k_cache=s["k_cache"], v_cache=s["v_cache"],
                           q_out=s["q_out"], q_norm_w=s.get("qw"), k_norm_w=s.get("kw"), sections=_sections(c),
                           interleaved=c["inter"], rotary_dim=c["rot"], eps=EPS, theta=THETA)
        return dict(q=s["q_out"], k=s["k_cache"], v=s["v_cache"])
    half = c["rot"] // 2
    # far positions: the angle in 64 bits, its cosine and sine in 32
    freq = THETA ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / c["rot"])
    turns = s["pos"].double()[_axis_of_pair(c)].t() * freq / (2 * math.pi)             # [tokens, pairs]
    angle = ((turns - torch.round(turns)) * (2 * math.pi)).float()
    cos, sin = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]

    def turn(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., 2 * half:]], -1).to(x.dtype)

    _scatter(s, turn(s["k"], s.get("kw")), s["v"])
    return dict(q=turn(s["q"], s.get("qw")), k=s["k_cache"], v=s["v_cache"])


MOST_SCORES = 1 << 29


def _groups(new, keys, heads):
    """Consecutive requests whose padded scores fit MOST_SCORES."""
    out, at = [], 0
    while at < len(new):
        end, s, k = at + 1, new[at], keys[at]
        while end < len(new) and max(s, new[end]) * max(k, keys[end]) * heads * (end + 1 - at) <= MOST_SCORES and \
                max(s, new[end]) <= 4 * max(1, min(new[at:end + 1])):
            s, k = max(s, new[end]), max(k, keys[end])
            end += 1
        out.append((at, end, s, k))
        at = end
    return out


def _attend(s):
    c = s["case"]
    causal = c["op"] == "attend"
    scale = 1.0 / math.sqrt(c["hd"])
    if own:
        call = s["ctx"].attention if causal else s["ctx"].cross_attention
        call(s["q"], s["k_cache"], s["v_cache"], s["out"], s["table"], s["q_start"], s["step"], s["keys"],
             max_step=max(s["new_host"]), scale=scale)
        return s["out"]
    H, KVH, HD, P = c["heads"], c["kvh"], c["hd"], c["page"]
    G = H // KVH
    out = torch.empty_like(s["q"])
    q_start, step, keys = s["q_start"].long(), s["step"].long(), s["keys"].long()
    for lo, hi, S, K in _groups(s["new_host"], s["keys_host"], H):
        B, n_pages = hi - lo, (K + P - 1) // P
        ids = s["table"][lo:hi, :n_pages].clamp(min=0).long()
        i = torch.arange(S, device="cuda")
        row = (q_start[lo:hi, None] + i).clamp(max=s["q"].shape[0] - 1)                            # [B, S]
        x = s["q"][row].view(B, S, KVH, G, HD).permute(2, 0, 3, 1, 4)                            # [KVH, B, G, S, HD]
        pos = (keys[lo:hi] - step[lo:hi])[:, None] + i                                             # [B, S]
        j = torch.arange(K, device="cuda")
        live = j < keys[lo:hi, None, None]
        if causal:
            live = live & (j <= pos[..., None])
            if c["window"]:
                live = live & (j > pos[..., None] - c["window"])
        off = torch.zeros(live.shape, device="cuda").masked_fill_(~live, -math.inf)[:, None]     # [B, 1, S, K]
        heads = max(1, min(KVH, MOST_SCORES // (B * G * S * K)))
        parts = []
        for h in range(0, KVH, heads):
            h1 = min(KVH, h + heads)
            k = s["k_cache"][ids, :, h:h1].float().view(B, n_pages * P, h1 - h, HD)[:, :K].permute(2, 0, 3, 1)
            v = s["v_cache"][ids, :, h:h1].float().view(B, n_pages * P, h1 - h, HD)[:, :K].permute(2, 0, 1, 3)
            xq = x[h:h1].float().reshape(h1 - h, B, G * S, HD)
            p = torch.matmul(xq, k).view(h1 - h, B, G, S, K).mul_(scale).add_(off)
            p = p.sub_(p.amax(-1, keepdim=True)).exp_()
            o = torch.matmul(p.view(h1 - h, B, G * S, K), v).view(h1 - h, B, G, S, HD)
            parts.append(o / p.sum(-1, keepdim=True))
        o = torch.cat(parts).permute(1, 3, 0, 2, 4).reshape(B, S, H, HD).to(out.dtype)
        used = i < step[lo:hi, None]
        n = sum(s["new_host"][lo:hi])
        at = s["start_host"][lo]
        out[at:at + n] = o[used] if B > 1 and min(s["new_host"][lo:hi]) < S else o.view(B * S, H, HD)
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "plan":
        R = case["requests"]
        longs = R // case["long_every"] if case["long_every"] else 0
        tokens = R - longs + longs * (1 + case["long"]) / 2
        fresh = tokens / case["page"] * case["spare"]
        return {"bytes": 4.0 * (2 * R + 2 * fresh + 3 * R + 2 + 2 * tokens), "flops": 0}
    if op == "append":
        return {"bytes": case["tokens"] * (8.0 * case["kvh"] * case["hd"] + 4), "flops": 0}
    if op == "rope":
        per = case["heads"] * 2 + case["kvh"] * 4
        return {"bytes": case["tokens"] * (per * case["hd"] * 2.0 + 4 * (case["axes"] + 1)),
                "flops": 10.0 * case["tokens"] * (case["heads"] + case["kvh"]) * case["hd"]}
    rows = pairs = tokens = 0
    new, keys = _lengths(case, 0)
    W = case["window"]
    for n, k in zip(new, keys):
        tokens += n
        if op == "cross":
            rows += k
            pairs += n * k
            continue
        first = k - n + 1                             # keys the first query attends, without a window
        rows += min(k, n - 1 + W) if W else k
        if not W:
            pairs += n * (first + k) / 2
        else:
            full = max(0, min(n, k - W + 1))          # queries that see a whole window: those with W keys or more
            few = n - full
            pairs += full * W + few * (first + first + few - 1) / 2
    return {"bytes": 4.0 * (rows * case["kvh"] * case["hd"] + tokens * case["heads"] * case["hd"]),
            "flops": 4.0 * case["heads"] * case["hd"] * pairs}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None                                   # whole numbers
    x = _inputs(case, seed)
    keep = x["slots"] >= 0 if op in ("append", "rope") else None
    if op == "append":
        planes = {}
        for name, rows, plane in (("k", x["k"], x["k_cache"]), ("v", x["v"], x["v_cache"])):
            planes[name] = plane.double()
            planes[name].view(-1, *rows.shape[1:])[x["slots"][keep].long()] = rows[keep].double()
        return planes
    if op == "rope":
        half, n = case["rot"] // 2, case["axes"]
        sec = _sections(case)
        axis = []
        for i in range(half):
            if case["inter"]:
                a = i % n
                axis.append(a if a and i < n * sec[a] else 0)
            else:
                axis.append(next(a for a in range(n) if i < sum(sec[:a + 1])))
        angle = torch.stack([x["pos"][axis[i]].double() * THETA ** (-2.0 * i / case["rot"]) for i in range(half)], -1)
        e = torch.complex(torch.cos(angle), torch.sin(angle))[:, None]

        def turned(y, w):
            y = y.double()
            if w is not None:
                y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + EPS) * w.double()
            z = torch.complex(y[..., :half], y[..., half:2 * half]) * e
            return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)

        k_plane = x["k_cache"].double()
        k_plane.view(-1, case["kvh"], case["hd"])[x["slots"][keep].long()] = turned(x["k"], x.get("kw"))[keep]
        return dict(q=turned(x["q"], x.get("qw")), k=k_plane, v=None)
    G = case["heads"] // case["kvh"]
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    for r, (n, k) in enumerate(zip(x["new_host"], x["keys_host"])):
        at = torch.arange(k, device="cuda")
        page = x["table"][r].long()[at // case["page"]]
        K, V = x["k_cache"][page, at % case["page"]], x["v_cache"][page, at % case["page"]]
        for t0 in range(0, n, 512):
            t1 = min(n, t0 + 512)
            rows = slice(x["start_host"][r] + t0, x["start_host"][r] + t1)
            for h in range(case["heads"]):
                z = (x["q"][rows, h].double() @ K[:, h // G].double().t()) / math.sqrt(case["hd"])
                if op == "attend":
                    p = torch.arange(k - n + t0, k - n + t1, device="cuda")[:, None]
                    hidden = at[None] > p
                    if case["window"]:
                        hidden |= at[None] <= p - case["window"]
                    z[hidden] = -math.inf
                out[rows, h] = torch.softmax(z, -1) @ V[:, h // G].double()
    return out
