"""GPU tests of the paged cache's operators (hkv_paged_*) against plain 64-bit models; tolerances are derived beside the
models in tests/_paged.py."""
import math

import numpy as np
import pytest

import _paged as P

pytestmark = pytest.mark.gpu

DT = ["float16", "bfloat16"]


def dt(torch, name):
    return getattr(torch, name)


def i32(torch, a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32).cuda()


# ---- plan and release -----------------------------------------------------------------------------------------------
def plan_case(seed, R, page, cols, tokens=None, scarce=False, odd=False):
    rng = np.random.default_rng(seed)
    past = rng.integers(0, cols * page // 2 + 1, R)
    new = rng.choice([0, 1, 1, 1, 2, page, page + 1, 3 * page + 2], R)
    if odd:                                             # what a broken host could send
        past[rng.random(R) < 0.1] = -1
        new[rng.random(R) < 0.1] = -5
        new[rng.random(R) < 0.1] = cols * page + 1
        past[rng.random(R) < 0.1] = 2**31 - 1
    need = int(sum(max(0, -(-(int(p) + int(n)) // page) - -(-int(p) // page)) for p, n in zip(past, new)))
    have = int(sum(-(-max(int(p), 0) // page) for p in past if p < cols * page))
    num_pages = have + need + 3
    ids = rng.permutation(num_pages).astype(np.int32)
    table = np.full((R, cols), -1, np.int32)
    at = 0
    for r in range(R):
        n = -(-int(past[r]) // page) if 0 <= past[r] <= cols * page else 0
        table[r, :n] = ids[at:at + n]
        at += n
    free = np.concatenate([ids[at:], np.full(at, -7, np.int32)])
    count = num_pages - at
    if scarce:
        count = count // 2
    tokens = int(np.maximum(new, 0).sum()) + 5 if tokens is None else tokens
    return past.astype(np.int32), new.astype(np.int32), table, free, count, num_pages, tokens


PLANS = [  # R, page, cols, tokens, scarce, odd
    (1, 16, 8, None, False, False), (2, 1, 40, None, False, False), (31, 7, 9, None, True, False),
    (64, 16, 2048, None, False, False), (257, 128, 3, None, True, True), (1000, 16, 64, 900, True, True),
    (1025, 64, 4, None, False, True), (4096, 8, 32, None, True, False), (3, 16, 8, 0, False, False), (40, 16, 100, 7, False, True),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", PLANS, ids=lambda c: f"R{c[0]}p{c[1]}")
def test_plan_matches_model(hkv, cuda, case, in_place):
    torch = cuda
    R, page, cols, tok, scarce, odd = case
    past, new, table, free, count, num_pages, tokens = plan_case(R * 31 + page, R, page, cols, tok, scarce, odd)
    ref = P.plan_model(past, new, table, free, count, page, tokens)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=2, num_kv_heads=1, head_dim=64, page_size=page, num_pages=num_pages,
                                             max_requests=R, max_pages=cols, max_tokens=max(1, tokens), flags=hkv.FLAG_APPEND_ONLY))
    step = ctx.new_step(R, tokens)
    step.slots.fill_(99)
    step.positions.fill_(99)
    d_past, d_new, d_table, d_free, d_count = (i32(torch, a) for a in (past, new, table, free, [count]))
    if in_place:
        ctx.plan(d_past, d_new, d_table, d_free, d_count, step, total_len=d_past, free_left=d_count)
        got_total, got_left = d_past, d_count
    else:
        for _ in range(2):                              # the same answer again: nothing is kept
            ctx.plan(d_past, d_new, d_table, d_free, d_count, step)
        got_total, got_left = step.total_len, step.free_left
        assert np.array_equal(d_past.cpu().numpy(), past) and int(d_count) == count
    for name, got in (("table", d_table), ("q_start", step.q_start), ("step_len", step.step_len), ("total_len", got_total),
                      ("slots", step.slots), ("positions", step.positions)):
        assert np.array_equal(got.cpu().numpy().astype(np.int64), ref[name].astype(np.int64)), name
    assert int(got_left) == ref["free_left"]
    assert np.array_equal(d_free.cpu().numpy(), free)
    assert ctx.device_status() == 0
    ctx.close()


def test_plan_release_keep_every_page(hkv, cuda):
    """Many steps of joins, growth and leaves: no page is ever held twice or lost; releasing twice changes nothing."""
    torch = cuda
    R, page, cols, num_pages = 37, 8, 24, 300
    rng = np.random.default_rng(5)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=1, head_dim=64, page_size=page, num_pages=num_pages, max_requests=R,
                                             max_pages=cols, max_tokens=2000, flags=hkv.FLAG_APPEND_ONLY))
    step = ctx.new_step(R, 2000)
    lens, table = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.full((R, cols), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(num_pages, dtype=torch.int32, device="cuda"), i32(torch, [num_pages])
    for it in range(40):
        ctx.plan(lens, i32(torch, rng.choice([0, 1, 1, 5, 60], R)), table, free, count, step, total_len=lens, free_left=count)
        if it % 3 == 2:
            gone = i32(torch, rng.random(R) < 0.3)
            for _ in range(2):
                ctx.release(gone, lens, table, free, count)
            assert (lens[gone.bool()] == 0).all()
        n, t, f, c = lens.cpu().numpy(), table.cpu().numpy(), free.cpu().numpy(), int(count)
        held = [t[r, j] for r in range(R) for j in range(-(-int(n[r]) // page))]
        assert sorted(held + list(f[:c])) == list(range(num_pages)), it
    ctx.close()


# ---- append ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape", [(1, 4, 128, 16, 0), (64, 2, 64, 8, 0), (777, 8, 256, 32, 64), (33, 3, 20, 5, 1), (9, 1, 7, 3, 0),
                                   (130, 4, 96, 16, 5)], ids=str)
def test_append_is_exact(hkv, cuda, shape, dtype):
    torch = cuda
    T, KVH, HD, page, extra = shape
    num_pages = -(-T // page) + 3
    gen = torch.Generator().manual_seed(T * HD)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages, max_requests=1,
                                             max_pages=1, max_tokens=T, dtype=dtype, flags=hkv.FLAG_APPEND_ONLY))
    row = KVH * HD
    fused = torch.randn(T, 2 * row + extra, generator=gen).to(dt(torch, dtype)).cuda()   # views into a wider activation
    k, v = fused[:, :row].unflatten(1, (KVH, HD)), \
        fused[:, row + extra:].unflatten(1, (KVH, HD))
    slots = torch.randperm(num_pages * page, generator=gen)[:T].to(torch.int32)
    slots[torch.rand(T, generator=gen) < 0.2] = -1
    kc, vc = (torch.randn(num_pages, page, KVH, HD, generator=gen).to(dt(torch, dtype)).cuda() for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    keep = slots >= 0
    want_k.view(-1, KVH, HD)[slots[keep].long().cuda()] = k[keep.cuda()]
    want_v.view(-1, KVH, HD)[slots[keep].long().cuda()] = v[keep.cuda()]
    ctx.append(k, v, kc, vc, slots.cuda())
    assert torch.equal(kc.view(torch.int16), want_k.view(torch.int16)) and torch.equal(vc.view(torch.int16), want_v.view(torch.int16))
    assert ctx.device_status() == 0
    bad = torch.full((T,), num_pages * page, dtype=torch.int32, device="cuda")    # a slot behind the planes: kept out, reported
    ctx.append(k, v, kc, vc, bad)
    assert ctx.device_status() == 2 and ctx.device_status() == 0
    assert torch.equal(kc.view(torch.int16), want_k.view(torch.int16))
    ctx.close()


# ---- norm + rotary positions ----------------------------------------------------------------------------------------
ROPES = [  # T, H, KVH, HD, rot, axes, sections, interleaved, norm
    (1, 28, 4, 128, 128, 1, None, False, True), (70, 28, 4, 128, 128, 3, [16, 24, 24], False, True),
    (513, 28, 4, 128, 128, 3, [24, 20, 20], True, True), (5, 14, 2, 64, 32, 2, [10, 6], False, False),
    (40, 8, 8, 96, 96, 3, [16, 16, 16], True, True), (333, 16, 8, 256, 128, 4, [16, 16, 16, 16], True, True),
    (19, 4, 2, 512, 512, 2, [0, 256], False, True), (23, 3, 1, 50, 18, 3, [5, 2, 2], True, True), (11, 2, 2, 16, 16, 1, None, False, False),
    (64, 32, 8, 128, 64, 1, None, False, False), (2050, 2, 1, 64, 64, 2, [20, 12], False, True),
    (17, 4, 2, 80, 80, 3, [20, 10, 10], False, True), (9, 2, 1, 32, 16, 2, [4, 4], True, True),
]


def rope_tolerance(torch, dtype, size):
    """Half a step of the type for the result; 32-bit arithmetic in front of it: the norm (sum of squares, division,
    root: under 8 roundings), weight, two products and a sum, and cos/sin of an angle reduced in 64 bits and rounded to
    2^-25 of a turn — 2 pi 2^-25 = 1.9e-7 — together under 24 * 2^-24 of the products' size."""
    return P.unit(torch, dtype) * size + 24 * 2.0 ** -24 * size + 2.0 ** -25


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("layout", ["paged", "dense", "in_place", "fused_view"])
@pytest.mark.parametrize("case", ROPES, ids=lambda c: f"T{c[0]}h{c[1]}x{c[3]}r{c[4]}a{c[5]}")
def test_norm_rope_matches_model(hkv, cuda, case, layout, dtype):
    torch = cuda
    T, H, KVH, HD, rot, axes, sections, inter, norm = case
    D, page = dt(torch, dtype), 16
    num_pages = -(-T // page) + 2
    gen = torch.Generator().manual_seed(T * HD + rot)
    pad = 8 if layout == "fused_view" else 0
    fused = torch.randn(T, (H + 2 * KVH) * HD + pad, generator=gen).to(D).cuda()
    q, k, v = (x.unflatten(1, (-1, HD)) for x in fused[:, pad:].split([H * HD, KVH * HD, KVH * HD], 1))
    if layout != "fused_view":
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pos = torch.randint(-3, 1_000_000, (axes, T), generator=gen, dtype=torch.int32).cuda()
    qw, kw = ((1 + 0.2 * torch.randn(HD, generator=gen)).to(D).cuda() for _ in range(2))
    args = dict(sections=sections, interleaved=inter, rotary_dim=rot, eps=1e-6, theta=1e6, scaling_factor=2.5,
                **(dict(q_norm_w=qw, k_norm_w=kw) if norm else {}))
    model = lambda x, w: P.rope_model(torch, x, pos, w if norm else None, rot, axes, sections, inter, 1e-6, 1e6, 2.5)
    (rq, sq), (rk, sk) = model(q, qw), model(k, kw)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages,
                                             max_requests=1, max_pages=1, max_tokens=T, dtype=dtype, flags=hkv.FLAG_APPEND_ONLY))
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    if layout in ("paged", "fused_view"):
        slots = torch.randperm(num_pages * page, generator=gen)[:T].to(torch.int32)
        slots[torch.rand(T, generator=gen) < 0.1] = -1
        kc, vc = (torch.randn(num_pages, page, KVH, HD, generator=gen).to(D).cuda() for _ in range(2))
        kc0, vc0 = kc.clone(), vc.clone()
        q_out = torch.empty(T, H, HD, dtype=D, device="cuda")
        ctx.norm_rope(q, k, v, pos, slots=slots.cuda(), k_cache=kc, v_cache=vc, q_out=q_out, **args)
        assert torch.equal(q, q0) and torch.equal(k, k0) and torch.equal(v, v0)
        keep = (slots >= 0).cuda()
        at = slots.cuda()[keep].long()
        got_k, rk, sk = kc.view(-1, KVH, HD)[at], rk[keep], sk[keep]
        assert torch.equal(vc.view(-1, KVH, HD)[at], v[keep])
        rest = torch.ones(num_pages * page, dtype=torch.bool, device="cuda")
        rest[at] = False
        assert torch.equal(kc.view(-1, KVH, HD)[rest], kc0.view(-1, KVH, HD)[rest])
        assert torch.equal(vc.view(-1, KVH, HD)[rest], vc0.view(-1, KVH, HD)[rest])
    elif layout == "dense":
        q_out, got_k = torch.empty_like(q), torch.empty_like(k)
        ctx.norm_rope(q, k, None, pos, q_out=q_out, k_out=got_k, **args)
        assert torch.equal(q, q0) and torch.equal(k, k0)
    else:
        ctx.norm_rope(q, k, None, pos, **args)
        q_out, got_k = q, k
    assert ctx.device_status() == 0
    for got, ref, size, what in ((q_out, rq, sq, "q"), (got_k, rk, sk, "k")):
        off = (got.double() - ref).abs() - rope_tolerance(torch, D, size)
        assert off.max() <= 0 if off.numel() else True, f"{what}: {off.max().item():.3e} over"
    ctx.close()


# ---- attention ------------------------------------------------------------------------------------------------------
HEADS = [(28, 4, 128), (14, 2, 64), (8, 8, 96), (16, 8, 256), (32, 2, 128), (16, 16, 64), (24, 1, 64), (4, 4, 256), (40, 1, 128)]
ODD_HEADS = [(3, 1, 7), (6, 2, 80), (2, 2, 512), (4, 2, 33)]


def run_attention(hkv, torch, *, heads, page, steps, keys, window=0, dtype="float16", causal=True, kernel=0, scale=None, seed=0,
                  max_step="max", q_extra=0, pad_rows=3, poison=True, starts=None, check=True, scale_q=1.0):
    H, KVH, HD = heads
    D = dt(torch, dtype)
    gen = torch.Generator().manual_seed(seed + H * HD + page)
    R = len(keys)
    cols = max(1, max(-(-k // page) for k in keys)) + 1
    num_pages = sum(-(-k // page) for k in keys) + 2
    kc, vc, table = P.make_pages(torch, gen, keys, page, num_pages, cols, KVH, HD, D, poison)
    if starts is None:
        starts = np.concatenate([[0], np.cumsum(steps)])
    T = int(max(s + n for s, n in zip(starts, steps))) + pad_rows
    T = max(T, 1)
    q = (scale_q * torch.randn(T, H * HD + q_extra, generator=gen)).to(D).cuda()[:, :H * HD].unflatten(1, (H, HD))
    if q_extra == 0:
        q = q.contiguous()
    out = torch.full((T, H, HD), 123.0, dtype=D, device="cuda")
    most = (max(steps) if steps else 0) if max_step == "max" else max_step
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages,
                                             max_requests=R, max_pages=cols, max_tokens=T, window_size=window, dtype=dtype,
                                             kernel_select=kernel))
    scale = 1 / math.sqrt(HD) if scale is None else scale
    call = ctx.attention if causal else ctx.cross_attention
    args = (q, kc, vc, out, table, i32(torch, starts[:R]), i32(torch, steps), i32(torch, keys))
    call(*args, max_step=most, scale=scale)
    assert ctx.device_status() == 0
    again = torch.full_like(out, 123.0)
    call(args[0], kc, vc, again, *args[4:], max_step=most, scale=scale)
    torch.cuda.synchronize()
    assert torch.equal(out, again), "two calls differ"
    if check:
        ref, tol, live = P.attend_model(torch, q, kc, vc, table, starts, steps, keys, scale, page, window, causal, most)
        assert (out[~live] == 123.0).all(), "a row of no query was written"
        got = out[live].double()
        assert torch.isfinite(got).all()
        off = (got - ref[live]).abs() - tol[live]
        assert off.numel() == 0 or off.max() <= 0, f"{off.max().item():.3e} over a tolerance of {tol[live].max().item():.3e}"
    ctx.close()
    return out


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heads", HEADS + ODD_HEADS, ids=str)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
def test_attention_single_tokens(hkv, cuda, heads, dtype, causal):
    """One query per request, lengths around tile and page borders, empty requests among them."""
    keys = [1, 0, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 777, 1]
    steps = [1, 0, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 0]
    run_attention(hkv, cuda, heads=heads, page=16, steps=steps, keys=keys, dtype=dtype, causal=causal)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 32, 64, 128, 256, 512])
@pytest.mark.parametrize("heads", [(28, 4, 128), (8, 8, 96), (4, 2, 256)], ids=str)
def test_attention_page_sizes(hkv, cuda, heads, page):
    run_attention(hkv, cuda, heads=heads, page=page, steps=[1, 1, 1], keys=[300, 513, 64])
    run_attention(hkv, cuda, heads=heads, page=page, steps=[40, 1, 7, 300], keys=[300, 513, 7, 640], dtype="bfloat16")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("heads", HEADS + ODD_HEADS, ids=str)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
def test_attention_ragged_chunks(hkv, cuda, heads, dtype, causal):
    """Single tokens, chunks of many lengths and whole prompts mixed in one call."""
    steps = [1, 37, 0, 128, 2, 5, 1, 200, 3]
    keys = [90, 37, 50, 600, 2, 400, 700, 201, 129]
    run_attention(hkv, cuda, heads=heads, page=32, steps=steps, keys=keys, dtype=dtype, causal=causal)


@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
@pytest.mark.parametrize("heads", [(28, 4, 128), (16, 8, 256), (8, 8, 64)], ids=str)
def test_attention_window(hkv, cuda, heads, window):
    run_attention(hkv, cuda, heads=heads, page=16, steps=[1, 1, 1, 1], keys=[1, 64, 130, 900], window=window)
    run_attention(hkv, cuda, heads=heads, page=64, steps=[1, 150, 300], keys=[700, 150, 901], window=window, dtype="bfloat16")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
@pytest.mark.parametrize("heads", [(28, 4, 128), (8, 8, 96), (16, 8, 256), (6, 2, 80)], ids=str)
def test_attention_rows_that_attend_nothing(hkv, cuda, heads, causal, dtype):
    """More queries than cached positions (causal: the first ones sit before position 0), and no cached position at all:
    zero rows."""
    torch = cuda
    steps, keys = [5, 200, 1, 40, 2], [2, 150, 0, 0, 1]
    out = run_attention(hkv, torch, heads=heads, page=16, steps=steps, keys=keys, causal=causal, dtype=dtype)
    assert (out[206:246] == 0).all() and (out[205] == 0).all()
    if causal:
        assert (out[:3] == 0).all() and (out[5:55] == 0).all()


@pytest.mark.parametrize("heads", [(28, 4, 128), (16, 8, 256), (8, 8, 64)], ids=str)
def test_attention_bounds_of_a_call(hkv, cuda, heads):
    """max_step cuts longer requests; requests placed apart, and last rows first; q as a view of a wider activation;
    stale lengths beyond the table's columns."""
    torch = cuda
    run_attention(hkv, torch, heads=heads, page=16, steps=[3, 90, 1], keys=[70, 300, 20], max_step=2)
    run_attention(hkv, torch, heads=heads, page=16, steps=[3, 90, 1], keys=[70, 300, 20], max_step=33)
    run_attention(hkv, torch, heads=heads, page=16, steps=[30, 4], keys=[70, 300], starts=[20, 100], q_extra=64)
    run_attention(hkv, torch, heads=heads, page=16, steps=[30, 1], keys=[70, 300], starts=[0, 41], q_extra=1, dtype="bfloat16")


@pytest.mark.parametrize("steps,keys", [([1], [20000]), ([1, 1], [9000, 31]), ([2], [12000]), ([150], [9000]), ([700], [700]), ([1] * 70, [200] * 70),
                                        ([1] * 300, list(range(1, 301))), ([33] * 20, [33 + 50 * i for i in range(20)])],
                         ids=["one_long", "two", "two_tokens", "chunk_long", "prompt", "many", "more_than_sms", "ragged"])
@pytest.mark.parametrize("heads", [(28, 4, 128), (14, 2, 64), (4, 4, 96), (4, 2, 256)], ids=str)
def test_attention_schedules(hkv, cuda, heads, steps, keys):
    """Few long requests (cut over the whole machine), many short ones, and what lies between."""
    run_attention(hkv, cuda, heads=heads, page=16, steps=steps, keys=keys)
    run_attention(hkv, cuda, heads=heads, page=128, steps=steps, keys=keys, dtype="bfloat16", causal=False)


@pytest.mark.parametrize("heads", [(28, 4, 128), (4, 2, 256), (8, 8, 96)], ids=str)
@pytest.mark.parametrize("steps", [[1, 1], [100, 260]], ids=["tokens", "chunks"])
def test_attention_growing_maxima(hkv, cuda, heads, steps):
    """Scores of some hundred, whose running maximum keeps moving."""
    run_attention(hkv, cuda, heads=heads, page=16, steps=steps, keys=[700, 1500], scale=0.5, scale_q=6.0, dtype="bfloat16")
    run_attention(hkv, cuda, heads=heads, page=16, steps=steps, keys=[700, 1500], scale=-0.3, scale_q=4.0)
    run_attention(hkv, cuda, heads=heads, page=16, steps=steps, keys=[700, 1500], scale=0.0)


@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=str)
@pytest.mark.parametrize("heads", [(28, 4, 128), (8, 8, 96), (16, 8, 256), (4, 2, 64), (6, 2, 80)], ids=str)
@pytest.mark.parametrize("steps", [[2, 1, 2], [2, 70, 300]], ids=["tokens", "chunks"])
def test_values_hidden_from_a_query_never_reach_it(hkv, cuda, heads, steps, value):
    """NaN and infinities in the K and V rows of later tokens of a chunk, and in rows that only the window of the first
    queries reaches: the other queries' results are those of clean rows, the ones that look at them are not finite."""
    torch = cuda
    H, KVH, HD = heads
    gen = torch.Generator().manual_seed(11)
    keys, page, window = [40, 333, 700], 16, 150
    kc, vc, table = P.make_pages(torch, gen, keys, page, 70, 50, KVH, HD, torch.float16)
    q = torch.randn(sum(steps), H, HD, generator=gen).half().cuda()
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=70,
                                             max_requests=3, max_pages=50, max_tokens=sum(steps), window_size=window))
    starts = np.concatenate([[0], np.cumsum(steps)])
    args = (table, i32(torch, starts), i32(torch, steps), i32(torch, keys))
    clean, got = torch.empty_like(q), torch.empty_like(q)
    ctx.attention(q, kc, vc, clean, *args, max_step=max(steps))
    for r in range(3):
        for j in {keys[r] - 1, max(0, keys[r] - steps[r] + 1 - window)}:      # the newest row; the first query's oldest
            for plane in (vc, kc):
                pg, row = int(table[r, j // page]), j % page
                old = plane[pg, row].clone()
                plane[pg, row, 0, 3] = value
                ctx.attention(q, kc, vc, got, *args, max_step=max(steps))
                plane[pg, row] = old
                pos = keys[r] - steps[r] + torch.arange(steps[r], device="cuda")
                sees = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
                sees[starts[r]:starts[r] + steps[r]] = (pos >= j) & (pos < j + window)
                assert torch.isfinite(got[~sees]).all()
                assert (got[~sees].double() - clean[~sees].double()).abs().max() < 4e-3     # one more rounding order, no more
                G = H // KVH
                hit = got[sees][:, :G]
                bad = ~torch.isfinite(hit[..., 3] if plane is vc else hit)
                if plane is vc or value != value:
                    assert bad.all()
                assert torch.isfinite(got[:, G:]).all()                         # other KV heads
    ctx.attention(q, kc, vc, got, *args, max_step=max(steps))
    assert torch.equal(got, clean), "a mark was left behind"
    assert ctx.device_status() == 0
    ctx.close()


@pytest.mark.parametrize("heads", [(28, 4, 128), (16, 8, 256), (6, 2, 80)], ids=str)
@pytest.mark.parametrize("steps", [[1, 1], [60, 200]], ids=["tokens", "chunks"])
def test_bad_pages_are_reported_and_never_followed(hkv, cuda, heads, steps):
    """Table entries outside the planes: rows of zeros, bit 2 of the status word, the other request untouched."""
    torch = cuda
    H, KVH, HD = heads
    gen = torch.Generator().manual_seed(3)
    keys, page = [300, 333], 16
    kc, vc, table = P.make_pages(torch, gen, keys, page, 60, 24, KVH, HD, torch.float16)
    q = torch.randn(sum(steps), H, HD, generator=gen).half().cuda()
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=60,
                                             max_requests=2, max_pages=24, max_tokens=sum(steps)))
    starts, d = [0, steps[0]], lambda a: i32(torch, a)
    good, bad = torch.empty_like(q), torch.empty_like(q)
    ctx.attention(q, kc, vc, good, table, d(starts), d(steps), d(keys), max_step=max(steps))
    assert ctx.device_status() == 0
    for value in (-1, 60, 0x7fffffff, -0x80000000):
        t = table.clone()
        t[0, 5] = value
        ctx.attention(q, kc, vc, bad, t, d(starts), d(steps), d(keys), max_step=max(steps))
        assert ctx.device_status() == 2
        assert torch.isfinite(bad).all() and torch.equal(bad[steps[0]:], good[steps[0]:])
        zk, zv = kc.clone(), vc.clone()
        zk[table[0, 5].long()], zv[table[0, 5].long()] = 0, 0
        ref, tol, live = P.attend_model(torch, q, zk, zv, table, starts, steps, keys, ctx.geometry.default_scale, page)
        assert ((bad.double() - ref).abs() <= tol)[:steps[0]].all()
    ctx.close()


def test_refusals(hkv, cuda):
    torch = cuda
    g = dict(num_heads=4, num_kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_requests=3, max_pages=4, max_tokens=20)
    ctx = hkv.PagedContext(hkv.PagedGeometry(**g))
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
    z = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    q, k, v, out, kc, vc = h(5, 4, 64), h(5, 2, 64), h(5, 2, 64), h(5, 4, 64), h(8, 16, 2, 64), h(8, 16, 2, 64)
    table = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    step = ctx.new_step(3, 20)

    def refused(status, fn, *a, **kw):
        with pytest.raises(hkv.HkvError) as e:
            fn(*a, **kw)
        assert e.value.status == status, e.value

    att = lambda **o: ctx.attention(*[o.get(n, d) for n, d in (("q", q), ("kc", kc), ("vc", vc), ("out", out), ("table", table), ("s", z(4)),
                                      ("n", z(3)), ("len", z(3)))], max_step=o.get("m", 1), scale=o.get("scale", 0.1))
    att()
    refused(1, att, q=q.bfloat16())
    refused(1, att, q=q.cpu())
    refused(1, att, q=h(5, 4, 32))
    refused(1, att, out=h(4, 4, 64))
    refused(2, att, out=h(5, 8, 64)[:, :4])
    refused(2, att, q=h(5, 4, 128)[:, :, ::2])
    refused(1, att, kc=h(8, 16, 2, 65)[..., :64])
    refused(1, att, kc=h(7, 16, 2, 64))
    refused(1, att, table=torch.zeros(3, 5, dtype=torch.int32, device="cuda"))
    refused(1, att, table=table.long())
    refused(1, att, n=z(2))
    refused(1, att, m=-1)
    refused(1, att, scale=float("nan"))
    refused(7, att, len=z(4), n=z(4), s=z(5), table=torch.zeros(4, 4, dtype=torch.int32, device="cuda"))
    refused(7, att, q=h(21, 4, 64), out=h(21, 4, 64))
    refused(1, ctx.append, k, v, kc, vc, z(4))
    refused(2, ctx.append, h(5, 4, 64)[:, :2], v, kc, vc, z(5))
    refused(7, ctx.append, h(21, 2, 64), h(21, 2, 64), kc, vc, z(21))
    rope = lambda **o: ctx.norm_rope(o.pop("q", q), o.pop("k", k), o.pop("v", v), o.pop("pos", z(5)), **{**dict(slots=z(5), k_cache=kc, v_cache=vc), **o})
    rope(slots=z(5) - 1)
    refused(1, rope, slots=None)
    refused(1, rope, v_cache=None)
    refused(1, rope, v=None)
    refused(1, rope, q_norm_w=h(64))
    refused(1, rope, q_norm_w=h(32), k_norm_w=h(64))
    refused(2, rope, rotary_dim=33)
    refused(2, rope, rotary_dim=66)
    refused(1, rope, theta=0.0)
    refused(1, rope, theta=float("inf"))
    refused(1, rope, eps=-1.0)
    pos3 = torch.zeros(3, 5, dtype=torch.int32, device="cuda")
    refused(1, rope, pos=pos3)
    refused(1, rope, pos=pos3, sections=[16, 8, 7])
    refused(1, rope, pos=pos3, sections=[40, -4, -4])
    refused(1, rope, pos=pos3, sections=[8, 12, 12], interleaved=True)      # axis 1 would reach pair 34
    refused(1, rope, pos=torch.zeros(5, 5, dtype=torch.int32, device="cuda"), sections=[8, 6, 6, 6, 6])
    refused(1, rope, pos=z(4))
    refused(1, ctx.plan, z(3), z(3), table, z(8), z(1), ctx.new_step(2, 20))
    refused(7, ctx.plan, z(3), z(3), table, z(8), z(1), ctx.new_step(3, 21))
    refused(1, ctx.release, z(3), z(3), table, z(7), z(1))
    ctx.close()
    only = hkv.PagedContext(hkv.PagedGeometry(**g, flags=hkv.FLAG_APPEND_ONLY))
    refused(6, only.attention, q, kc, vc, out, table, z(4), z(3), z(3))
    only.close()


def test_empty_calls_do_nothing(hkv, cuda):
    torch = cuda
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=4, num_kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_requests=3,
                                             max_pages=4, max_tokens=20))
    h = lambda *s: torch.full(s, 7.0, dtype=torch.float16, device="cuda")
    z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")
    kc, vc, out = h(8, 16, 2, 64), h(8, 16, 2, 64), h(5, 4, 64)
    ctx.append(h(0, 2, 64), h(0, 2, 64), kc, vc, z(0))
    ctx.norm_rope(h(0, 4, 64), h(0, 2, 64), h(0, 2, 64), z(0), slots=z(0), k_cache=kc, v_cache=vc)
    ctx.attention(h(5, 4, 64), kc, vc, out, z(0, 4), z(1), z(0), z(0))
    ctx.attention(h(5, 4, 64), kc, vc, out, z(3, 4), z(4), z(3), z(3), max_step=0)
    ctx.attention(h(5, 4, 64), kc, vc, out, z(3, 4), z(4), z(3), z(3) + 9, max_step=4)
    ctx.attention(h(0, 4, 64), kc, vc, h(0, 4, 64), z(3, 4), z(4), z(3), z(3))
    step = ctx.new_step(0, 4)
    ctx.plan(z(0), z(0), z(0, 4), z(8), z(1) + 8, step)
    assert int(step.free_left) == 8 and int(step.q_start) == 0 and (step.slots == -1).all() and (step.positions == -1).all()
    ctx.release(z(0), z(0), z(0, 4), z(8), z(1))
    assert ctx.device_status() == 0
    for t in (kc, vc, out):
        assert (t == 7).all()
    ctx.close()


# ---- the operators together -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,dtype,window", [((28, 4, 128), "float16", 0), ((14, 2, 64), "bfloat16", 40), ((16, 8, 256), "bfloat16", 0),
                                                ((6, 2, 80), "float16", 0)], ids=str)
def test_serving_steps_captured_and_replayed(hkv, cuda, heads, dtype, window):
    """A serving loop of two layers: plan, norm + rotary positions into the pages, attention, all captured once on a side
    stream and replayed with other lengths every step (joins, chunks, single tokens, requests that do not fit), releases
    in between. Every step's tables, cache rows and outputs are held against the models."""
    torch = cuda
    H, KVH, HD = heads
    D = dt(torch, dtype)
    R, page, cols, num_pages, T, layers, most = 11, 16, 20, 90, 160, 2, 64
    rot, sections = HD // 2 // 16 * 32, None
    sections = [rot // 2 - 2 * (rot // 8), rot // 8, rot // 8]
    gen = torch.Generator().manual_seed(HD)
    rng = np.random.default_rng(HD)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages,
                                             max_requests=R, max_pages=cols, max_tokens=T, window_size=window, dtype=dtype))
    step = ctx.new_step(R, T)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    lens, new, gone, pos3 = z(R), z(R), z(R), z(3, T)
    table, free, count = z(R, cols) - 1, torch.arange(num_pages, dtype=torch.int32, device="cuda"), i32(torch, [num_pages])
    qkv = [torch.zeros(T, (H + 2 * KVH) * HD, dtype=D, device="cuda") for _ in range(layers)]
    planes = [[torch.zeros(num_pages, page, KVH, HD, dtype=D, device="cuda") for _ in range(2)] for _ in range(layers)]
    turned = [torch.zeros(T, H, HD, dtype=D, device="cuda") for _ in range(layers)]
    outs = [torch.zeros(T, H, HD, dtype=D, device="cuda") for _ in range(layers)]
    qw, kw = ((1 + 0.2 * torch.randn(HD, generator=gen)).to(D).cuda() for _ in range(2))
    offsets = i32(torch, [[0], [5], [9]])
    rope = dict(q_norm_w=qw, k_norm_w=kw, sections=sections, rotary_dim=rot, theta=1e6)

    def one_step():
        ctx.plan(lens, new, table, free, count, step, total_len=lens, free_left=count)
        torch.add(step.positions, offsets, out=pos3)
        for n in range(layers):
            q, k, v = (x.unflatten(1, (-1, HD)) for x in qkv[n].split([H * HD, KVH * HD, KVH * HD], 1))
            ctx.norm_rope(q, k, v, pos3, slots=step.slots, k_cache=planes[n][0], v_cache=planes[n][1], q_out=turned[n], **rope)
            ctx.attention(turned[n], planes[n][0], planes[n][1], outs[n], table, step.q_start, step.step_len, lens, max_step=most)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one_step()                                       # no tokens yet: nothing happens
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            one_step()
    torch.cuda.current_stream().wait_stream(side)
    for it in range(9):
        fresh = rng.choice([0, 1, 1, 1, 2, 3, 40] if it % 3 else [1, 20, 64], R)
        new.copy_(i32(torch, fresh))
        for x in qkv:
            x.copy_(torch.randn(x.shape, generator=gen))
        before = [[x.clone() for x in pl] for pl in planes]
        n_lens, n_table, n_free, n_count = lens.cpu().numpy(), table.cpu().numpy(), free.cpu().numpy(), int(count)
        ref = P.plan_model(n_lens, fresh, n_table, n_free, n_count, page, T)
        for x in outs:
            x.fill_(77.0)
        graph.replay()
        for name, got in (("table", table), ("q_start", step.q_start), ("step_len", step.step_len), ("total_len", lens),
                          ("slots", step.slots), ("positions", step.positions)):
            assert np.array_equal(got.cpu().numpy(), ref[name]), (it, name)
        assert int(count) == ref["free_left"]
        keep = step.slots >= 0
        at = step.slots[keep].long()
        for n in range(layers):
            q, k, v = (x.unflatten(1, (-1, HD)) for x in qkv[n].split([H * HD, KVH * HD, KVH * HD], 1))
            for x, w, got, pick in ((q, qw, turned[n], slice(None)), (k, kw, planes[n][0].view(-1, KVH, HD)[at], keep)):
                want, size = P.rope_model(torch, x, pos3, w, rot, 3, sections, False, 1e-6, 1e6, 1.0)
                assert ((got.double() - want[pick]).abs() <= rope_tolerance(torch, D, size[pick])).all(), (it, n)
            for plane, old in zip(planes[n], before[n]):
                rest = torch.ones(num_pages * page, dtype=torch.bool, device="cuda")
                rest[at] = False
                assert torch.equal(plane.view(-1, KVH, HD)[rest], old.view(-1, KVH, HD)[rest])
            assert torch.equal(planes[n][1].view(-1, KVH, HD)[at], v[keep])
            want, tol, live = P.attend_model(torch, turned[n], *planes[n], table, ref["q_start"], ref["step_len"], ref["total_len"],
                                             ctx.geometry.default_scale, page, window)
            assert (outs[n][~live] == 77.0).all() and ((outs[n].double() - want).abs() <= tol)[live].all(), (it, n)
        if it % 2:
            gone.copy_(i32(torch, rng.random(R) < 0.4))
            ctx.release(gone, lens, table, free, count)
    assert ctx.device_status() == 0
    del graph
    ctx.close()


@pytest.mark.parametrize("heads", [(16, 8, 256), (28, 4, 128), (14, 2, 64)], ids=str)
def test_attention_many_passes(hkv, cuda, heads):
    """Hundreds of passes over a ragged windowed batch from two contexts in turn: no wait inside the kernels ever runs out
    (the order in which copies land differs from pass to pass), and every pass gives the same bits."""
    torch = cuda
    H, KVH, HD = heads
    gen = torch.Generator().manual_seed(2)
    page, steps = 32, [1, 1, 400, 1, 1, 1, 1, 250] * 4
    keys = [int(x) for x in torch.randint(2000, 6000, (len(steps),), generator=gen)]
    cols = max(-(-k // page) for k in keys)
    num_pages = sum(-(-k // page) for k in keys)
    kc, vc, table = P.make_pages(torch, gen, keys, page, num_pages, cols, KVH, HD, torch.float16)
    T = sum(steps)
    q = torch.randn(T, H, HD, generator=gen).half().cuda()
    starts = np.concatenate([[0], np.cumsum(steps)])
    args = (table, i32(torch, starts), i32(torch, steps), i32(torch, keys))
    ctxs = [hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages,
                                               max_requests=len(steps), max_pages=cols, max_tokens=T, window_size=1024)) for _ in range(2)]
    first, out = torch.empty_like(q), torch.empty_like(q)
    ctxs[0].attention(q, kc, vc, first, *args, max_step=400)
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for it in range(300):
        ctxs[it % 2].attention(q, kc, vc, out, *args, max_step=400)
        if it % 10 == 9:
            differ += (out != first).sum()
    assert [c.device_status() for c in ctxs] == [0, 0]
    assert int(differ) == 0
    for c in ctxs:
        c.close()


def test_planes_beyond_2_to_31_elements(hkv, cuda):
    """Pages at the far end of planes of 2.2e9 elements: append, rotary positions, single tokens and a chunk."""
    torch = cuda
    KVH, HD, H, page = 8, 128, 16, 64
    num_pages = (2_200_000_000 // (KVH * HD * page)) + 1
    kc, vc = (torch.empty(num_pages, page, KVH, HD, dtype=torch.float16, device="cuda") for _ in range(2))
    gen = torch.Generator().manual_seed(4)
    keys, steps = [130, 333], [1, 200]
    need = [3, 6]
    ids = torch.cat([torch.arange(num_pages - 8, num_pages), torch.tensor([0])])[torch.randperm(9, generator=gen)].to(torch.int32)
    table = torch.full((2, 8), -1, dtype=torch.int32)
    table[0, :3], table[1, :6] = ids[:3], ids[3:]
    for r in range(2):
        for j in range(need[r]):
            for plane in (kc, vc):
                plane[int(table[r, j])] = torch.randn(page, KVH, HD, generator=gen).half().cuda()
    T = sum(steps)
    q, k, v = (torch.randn(T, h, HD, generator=gen).half().cuda() for h in (H, KVH, KVH))
    slots = i32(torch, [int(table[r, p // page]) * page + p % page for r in range(2) for p in range(keys[r] - steps[r], keys[r])])
    pos = i32(torch, [p for r in range(2) for p in range(keys[r] - steps[r], keys[r])])
    for kernel in (0, 1):
        ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages,
                                                 max_requests=2, max_pages=8, max_tokens=T, kernel_select=kernel))
        ctx.append(k, v, kc, vc, slots)
        at = slots.long()
        assert torch.equal(kc.view(-1, KVH, HD)[at], k) and torch.equal(vc.view(-1, KVH, HD)[at], v)
        turned = torch.empty_like(q)
        ctx.norm_rope(q, k, v, pos, slots=slots, k_cache=kc, v_cache=vc, q_out=turned)
        want, size = P.rope_model(torch, k, pos, None, HD, 1, None, False, 1e-6, 1e4, 1.0)
        assert ((kc.view(-1, KVH, HD)[at].double() - want).abs() <= rope_tolerance(torch, torch.float16, size)).all()
        out = torch.empty_like(q)
        ctx.attention(turned, kc, vc, out, table.cuda(), i32(torch, [0, 1]), i32(torch, steps), i32(torch, keys), max_step=200)
        ref, tol, live = P.attend_model(torch, turned, kc, vc, table.cuda(), [0, 1], steps, keys, ctx.geometry.default_scale, page)
        assert live.all() and ((out.double() - ref).abs() <= tol).all()
        assert ctx.device_status() == 0
        ctx.close()


@pytest.mark.parametrize("steps", [[1], [70]], ids=["token", "chunk"])
def test_attention_over_a_very_long_request(hkv, cuda, steps):
    run_attention(hkv, cuda, heads=(14, 2, 64), page=16, steps=steps, keys=[200_003], dtype="bfloat16", poison=False)


def test_two_streams_take_two_contexts(hkv, cuda):
    """Two contexts at work on two streams at once, inputs made on the same streams: both give what one alone gives."""
    torch = cuda
    H, KVH, HD, page, steps, keys = 28, 4, 128, 16, [1, 1, 90], [5000, 3000, 4000]
    gen = torch.Generator().manual_seed(6)
    cols, num_pages, T = 320, 760, sum(steps)
    kc, vc, table = P.make_pages(torch, gen, keys, page, num_pages, cols, KVH, HD, torch.float16)
    q = torch.randn(T, H, HD, generator=gen).half().cuda()
    args = (table, i32(torch, [0, 1, 2]), i32(torch, steps), i32(torch, keys))
    make = lambda: hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages,
                                                      max_requests=3, max_pages=cols, max_tokens=T))
    ctxs, streams = [make(), make()], [torch.cuda.Stream(), torch.cuda.Stream()]
    want = torch.empty_like(q)
    ctxs[0].attention(q, kc, vc, want, *args, max_step=90)
    want2 = torch.empty_like(q)
    ctxs[0].attention(q * 2, kc, vc, want2, *args, max_step=90)
    torch.cuda.synchronize()
    outs = [torch.empty_like(q) for _ in range(2)]
    for _ in range(20):
        for n, (ctx, st) in enumerate(zip(ctxs, streams)):
            with torch.cuda.stream(st):
                outs[n].zero_()
                ctx.attention(q * (n + 1), kc, vc, outs[n], *args, max_step=90)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)
    for ctx, st in zip(ctxs, streams):
        with torch.cuda.stream(st):
            assert ctx.device_status() == 0
        ctx.close()


def test_out_must_not_be_q(hkv, cuda):
    torch = cuda
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=4, num_kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_requests=1,
                                             max_pages=4, max_tokens=20))
    q, kc = torch.zeros(5, 4, 64, dtype=torch.float16, device="cuda"), torch.zeros(8, 16, 2, 64, dtype=torch.float16, device="cuda")
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    with pytest.raises(hkv.HkvError) as e:
        ctx.attention(q, kc, kc, q, z(1, 4), z(1), z(1) + 5, z(1) + 5)
    assert e.value.status == 1
    ctx.close()


def test_block_tables_beyond_31_bits_of_tiles_are_not_staged(hkv, cuda):
    """4 096 requests of up to 2^31 positions: more tiles than the few-token kernel counts."""
    g = dict(num_heads=4, num_kv_heads=2, head_dim=64, page_size=64, num_pages=8, max_requests=4096, max_pages=2**25 - 1, max_tokens=8)
    with pytest.raises(hkv.HkvError) as e:
        hkv.PagedContext(hkv.PagedGeometry(**g, kernel_select=2))
    assert e.value.status == 2
    hkv.PagedContext(hkv.PagedGeometry(**g)).close()
    hkv.PagedContext(hkv.PagedGeometry(**{**g, "max_pages": 2**14}, kernel_select=2)).close()
