"""GPU tests of the paged cache at the edges of what its documentation promises: values that a mask or a vanishing weight
hides, in both types. Models and tolerances: tests/_paged.py."""
import math

import numpy as np
import pytest

import _paged as P
import test_paged_gpu as base

pytestmark = pytest.mark.gpu

DT = ["float16", "bfloat16"]
STAGED = [(28, 4, 128), (14, 2, 64), (8, 8, 96), (16, 8, 256)]


def dt(torch, name):
    return getattr(torch, name)


def i32(torch, a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32).cuda()


# ---- values that must not reach a row ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kind", ["large", "nan", "inf"])
@pytest.mark.parametrize("heads", STAGED + [(6, 2, 80)], ids=str)
@pytest.mark.parametrize("steps", [[2, 1, 2], [2, 70, 300]], ids=["tokens", "chunks"])
def test_hidden_values_of_both_types(hkv, cuda, heads, steps, kind, dtype):
    """A large finite value, NaN or infinity in each of the newest rows of a chunk in turn (16 of them: the kernels treat the
    columns of a tile in patterns of up to 16) and in a row that only its first queries' window reaches. A finite one leaves every row that does not look at it bit for bit as it was (its weight is zero, not small);
    the others send the item to be done again, so those rows are held against the 64-bit model."""
    torch = cuda
    H, KVH, HD = heads
    D = dt(torch, dtype)
    value = {"nan": math.nan, "inf": math.inf, "large": 1e30 if dtype == "bfloat16" else 6e4}[kind]
    gen = torch.Generator().manual_seed(13)
    keys, page, window = [40, 333, 700], 16, 150
    kc, vc, table = P.make_pages(torch, gen, keys, page, 70, 50, KVH, HD, D)
    q = torch.randn(sum(steps), H, HD, generator=gen).to(D).cuda()
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=70, max_requests=3,
                                             max_pages=50, max_tokens=sum(steps), window_size=window, dtype=dtype))
    starts = np.concatenate([[0], np.cumsum(steps)])
    args = (table, i32(torch, starts), i32(torch, steps), i32(torch, keys))
    clean, got = torch.empty_like(q), torch.empty_like(q)
    ctx.attention(q, kc, vc, clean, *args, max_step=max(steps))
    ref, tol, live = P.attend_model(torch, q, kc, vc, table, starts, steps, keys, ctx.geometry.default_scale, page, window)
    assert live.all()
    for r in range(3):
        newest = range(keys[r] - min(16, steps[r]), keys[r])
        for j in {*newest, max(0, keys[r] - steps[r] + 1 - window)}:
            for plane in (vc, kc):
                pg, row = int(table[r, j // page]), j % page
                old = plane[pg, row].clone()
                plane[pg, row, 0, 3] = value
                ctx.attention(q, kc, vc, got, *args, max_step=max(steps))
                plane[pg, row] = old
                pos = keys[r] - steps[r] + torch.arange(steps[r], device="cuda")
                blind = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
                blind[starts[r]:starts[r] + steps[r]] = (pos < j) | (pos >= j + window)
                if kind == "large":
                    assert torch.equal(got[blind], clean[blind]), f"{int((got[blind] != clean[blind]).sum())} elements moved"
                else:
                    assert ((got[blind].double() - ref[blind]).abs() <= tol[blind]).all()
    assert ctx.device_status() == 0
    ctx.close()


@pytest.mark.parametrize("heads", STAGED + [(6, 2, 80)], ids=str)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
def test_vanishing_weights_are_zero(hkv, cuda, heads, causal):
    """One key's score stands 640 above all others (weights of 2^-923, which is zero in 32 bits), the others' values are
    1e30: every row is that key's value. Tolerance: half a step for its weight, half a step for the result, and 2e-4 for the
    error of exp2 in weight and sum."""
    torch = cuda
    H, KVH, HD = heads
    G = H // KVH
    gen = torch.Generator().manual_seed(17)
    steps, keys, page = [1, 200, 3], [300, 500, 77], 16
    kc, vc, table = P.make_pages(torch, gen, keys, page, 70, 40, KVH, HD, torch.bfloat16)
    kc, vc = torch.zeros_like(kc), torch.full_like(vc, 1e30)
    want = []
    for r in range(3):
        at = int(table[r, 0])
        kc[at, 0, :, 0] = 40.0
        vc[at, 0] = torch.randn(KVH, HD, generator=gen).bfloat16().cuda()
        want.append(vc[at, 0].double().repeat_interleave(G, 0).expand(steps[r], H, HD))
    want = torch.cat(want)
    T = sum(steps)
    q = torch.zeros(T, H, HD, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 16.0
    out = torch.empty_like(q)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=70, max_requests=3,
                                             max_pages=40, max_tokens=T, dtype="bfloat16"))
    call = ctx.attention if causal else ctx.cross_attention
    call(q, kc, vc, out, table, i32(torch, [0, 1, 201]), i32(torch, steps), i32(torch, keys), max_step=200, scale=1.0)
    off = (out.double() - want).abs()
    assert (off <= (2 * P.unit(torch, torch.bfloat16) + 2e-4) * want.abs()).all(), f"{off.max().item():.3e}"
    assert ctx.device_status() == 0
    ctx.close()


# ---- tensors whose tokens lie on top of each other ----------------------------------------------------------------------
def test_broadcast_rows_are_refused(hkv, cuda):
    """expand()ed rows have a token stride of 0, which the library reads as dense: refused in every place they can come in."""
    torch = cuda
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=4, num_kv_heads=2, head_dim=64, page_size=16, num_pages=8, max_requests=3,
                                             max_pages=4, max_tokens=20))
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    q, k, v, out, kc, vc = h(5, 4, 64), h(5, 2, 64), h(5, 2, 64), h(5, 4, 64), h(8, 16, 2, 64), h(8, 16, 2, 64)
    wide_q, wide_k = h(1, 4, 64).expand(5, 4, 64), h(1, 2, 64).expand(5, 2, 64)
    att = lambda **o: ctx.attention(o.get("q", q), kc, vc, o.get("out", out), z(3, 4), z(4), z(3), z(3), max_step=1)
    cross = lambda **o: ctx.cross_attention(o.get("q", q), kc, vc, o.get("out", out), z(3, 4), z(4), z(3), z(3), max_step=1)
    rope = lambda **o: ctx.norm_rope(o.get("q", q), o.get("k", k), None, z(5), q_out=o.get("q_out"), k_out=o.get("k_out"))
    paged = lambda **o: ctx.norm_rope(q, o.get("k", k), o.get("v", v), z(5), slots=z(5) - 1, k_cache=kc, v_cache=vc)
    for call in (lambda: att(q=wide_q), lambda: att(out=wide_q), lambda: cross(q=wide_q), lambda: cross(out=wide_q),
                 lambda: ctx.append(wide_k, wide_k, kc, vc, z(5) - 1), lambda: ctx.append(k, wide_k, kc, vc, z(5) - 1),
                 lambda: rope(q=wide_q), lambda: rope(k=wide_k), lambda: rope(q_out=wide_q), lambda: rope(k_out=wide_k),
                 lambda: paged(k=wide_k), lambda: paged(v=wide_k)):
        with pytest.raises(hkv.HkvError) as e:
            call()
        assert e.value.status == 2, e.value
    att(), cross(), rope(), paged()
    assert ctx.device_status() == 0
    ctx.close()


# ---- arrays that no plan writes -------------------------------------------------------------------------------------------
def test_overlapping_requests_beyond_the_work_table(hkv, cuda):
    """4 096 requests that all claim the same 16 384 rows (starts left at zero): more work than the prompt kernel's table
    counts. The call leaves the rows alone and sets bit 2; the next call of the context is right."""
    torch = cuda
    H, KVH, HD, page, R, T, cols = 32, 8, 64, 16, 4096, 16384, 8192
    kc, vc = (torch.zeros(4, page, KVH, HD, dtype=torch.float16, device="cuda") for _ in range(2))
    vc += 1
    table = torch.zeros(R, cols, dtype=torch.int32, device="cuda")
    q = torch.zeros(T, H, HD, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 77.0)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=4, max_requests=R,
                                             max_pages=cols, max_tokens=T))
    z = torch.zeros(R, dtype=torch.int32, device="cuda")
    ctx.attention(q, kc, vc, out, table, z, z + T, z + cols * page)
    assert ctx.device_status() == 2
    assert (out == 77.0).all()
    step = z.clone()
    step[7] = 300
    ctx.attention(q, kc, vc, out, table, z, step, step, max_step=300)
    assert ctx.device_status() == 0
    assert (out[:300] == 1.0).all() and (out[300:] == 77.0).all()
    ctx.close()


# ---- streams ----------------------------------------------------------------------------------------------------------------
def test_a_context_is_ready_for_any_stream(hkv, cuda):
    """A context created (and its status read) while the default stream is busy, used at once on a stream that does not wait
    for the default one: its words were cleared before, so the bit that the first call sets is still there."""
    torch = cuda
    g = hkv.PagedGeometry(num_heads=2, head_dim=64, page_size=16, num_pages=4, max_requests=1, max_pages=4, max_tokens=4)
    hkv.PagedContext(g).close()                          # (modules loaded)
    k = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    bad = torch.full((4,), 64, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)                       # a tenth of a second
    ctx = hkv.PagedContext(g)
    with torch.cuda.stream(side):
        for _ in range(3):
            ctx.append(k, k, kc, vc, bad)                # a slot behind the planes
            assert ctx.device_status() == 2
        assert ctx.device_status() == 0
    torch.cuda._sleep(200_000_000)
    with torch.cuda.stream(side):
        ctx.append(k, k, kc, vc, bad)
    assert ctx.device_status(side) == 2                  # not the current stream
    with torch.cuda.stream(side):
        ctx.append(k, k, kc, vc, bad)
        side.synchronize()
        assert ctx.device_status() == 2
    torch.cuda.synchronize()
    ctx.close()


# ---- starts that only ascend --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kernel", [0, 1], ids=["staged", "generic"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
def test_empty_requests_may_start_anywhere_in_order(hkv, cuda, kernel, causal):
    """q_start ascends, and an empty request's start may lie on or inside the rows of the one before it; gaps and padded rows
    belong to nobody."""
    torch = cuda
    H, KVH, HD, page = 8, 2, 64, 16
    starts, steps, keys = [0, 0, 2, 4, 9, 9, 9, 50, 50] + [50] * 40, [4, 0, 0, 3, 40, 0, 0, 0, 1] + [0] * 40, [9, 3, 0, 30, 77, 5, 0, 8, 20] + [1] * 40
    gen = torch.Generator().manual_seed(19)
    kc, vc, table = P.make_pages(torch, gen, keys, page, 70, 6, KVH, HD, torch.float16)
    T = 60
    q = torch.randn(T, H, HD, generator=gen).half().cuda()
    out = torch.full_like(q, 77.0)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=70,
                                             max_requests=len(keys), max_pages=6, max_tokens=T, kernel_select=kernel))
    call = ctx.attention if causal else ctx.cross_attention
    call(q, kc, vc, out, table, i32(torch, starts), i32(torch, steps), i32(torch, keys), max_step=40)
    ref, tol, live = P.attend_model(torch, q, kc, vc, table, starts, steps, keys, ctx.geometry.default_scale, page, 0, causal)
    assert int(live.sum()) == sum(steps) and (out[~live] == 77.0).all()
    assert ((out.double() - ref).abs() <= tol)[live].all()
    assert ctx.device_status() == 0
    ctx.close()


# ---- one rounding, every pass ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("case", base.ROPES, ids=lambda c: f"T{c[0]}h{c[1]}x{c[3]}r{c[4]}a{c[5]}")
def test_norm_rope_rounds_once(hkv, cuda, case, dtype):
    """The result is rounded to the type once: half a step of the RESULT, beside the 24 roundings of 32 bits that
    test_paged_gpu.rope_tolerance counts, of the products' size (a second rounding, of the normalised row, would be half a
    step of the operands) — 25 with the half step of that error itself. 2^-25: half a step of fp16 below 2^-14."""
    torch = cuda
    T, H, KVH, HD, rot, axes, sections, inter, norm = case
    D, page = dt(torch, dtype), 16
    num_pages = -(-T // page) + 2
    gen = torch.Generator().manual_seed(T * HD + rot + 1)
    q, k, v = (torch.randn(T, h, HD, generator=gen).to(D).cuda() for h in (H, KVH, KVH))
    pos = torch.randint(-3, 1_000_000, (axes, T), generator=gen, dtype=torch.int32).cuda()
    qw, kw = ((1 + 0.2 * torch.randn(HD, generator=gen)).to(D).cuda() for _ in range(2))
    kc, vc = (torch.zeros(num_pages, page, KVH, HD, dtype=D, device="cuda") for _ in range(2))
    slots = torch.randperm(num_pages * page, generator=gen)[:T].to(torch.int32).cuda()
    q_out = torch.empty_like(q)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages,
                                             max_requests=1, max_pages=1, max_tokens=T, dtype=dtype, flags=hkv.FLAG_APPEND_ONLY))
    ctx.norm_rope(q, k, v, pos, slots=slots, k_cache=kc, v_cache=vc, q_out=q_out, sections=sections, interleaved=inter, rotary_dim=rot,
                  eps=1e-6, theta=1e6, scaling_factor=2.5, **(dict(q_norm_w=qw, k_norm_w=kw) if norm else {}))
    for x, w, got in ((q, qw, q_out), (k, kw, kc.view(-1, KVH, HD)[slots.long()])):
        ref, size = P.rope_model(torch, x, pos, w if norm else None, rot, axes, sections, inter, 1e-6, 1e6, 2.5)
        off = (got.double() - ref).abs() - (P.unit(torch, D) * ref.abs() + 25 * 2.0 ** -24 * size + 2.0 ** -25)
        assert off.max() <= 0, f"{off.max().item():.3e} over"
    assert ctx.device_status() == 0
    ctx.close()


@pytest.mark.parametrize("heads", [(16, 8, 256), (28, 4, 128), (14, 2, 64)], ids=str)
def test_every_pass_of_both_contexts_gives_the_same_bits(hkv, cuda, heads):
    """Hundreds of passes over a ragged windowed batch, from two contexts in turn: each of them is compared."""
    torch = cuda
    H, KVH, HD = heads
    gen = torch.Generator().manual_seed(23)
    page, steps = 32, [1, 1, 400, 1, 1, 1, 1, 250] * 4
    keys = [int(x) for x in torch.randint(2000, 6000, (len(steps),), generator=gen)]
    cols = max(-(-k // page) for k in keys)
    num_pages = sum(-(-k // page) for k in keys)
    kc, vc, table = P.make_pages(torch, gen, keys, page, num_pages, cols, KVH, HD, torch.float16)
    T = sum(steps)
    q = torch.randn(T, H, HD, generator=gen).half().cuda()
    args = (table, i32(torch, np.concatenate([[0], np.cumsum(steps)])), i32(torch, steps), i32(torch, keys))
    ctxs = [hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=page, num_pages=num_pages,
                                               max_requests=len(steps), max_pages=cols, max_tokens=T, window_size=1024)) for _ in range(2)]
    first, out = torch.empty_like(q), torch.empty_like(q)
    ctxs[0].attention(q, kc, vc, first, *args, max_step=400)
    differ = torch.zeros(2, dtype=torch.int64, device="cuda")
    for it in range(300):
        out.fill_(55.0)
        ctxs[it % 2].attention(q, kc, vc, out, *args, max_step=400)
        differ[it % 2] += (out != first).sum()
    assert [c.device_status() for c in ctxs] == [0, 0]
    assert differ.tolist() == [0, 0]
    for c in ctxs:
        c.close()


# ---- the largest batches and groups -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads", [(128, 1, 64), (65, 1, 128), (254, 2, 96), (100, 1, 256), (128, 1, 256)], ids=str)
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "cross"])
def test_large_groups(hkv, cuda, heads, causal):
    """Groups up to the 128 that one query tile holds: one or two queries per item, all of them chunks."""
    base.run_attention(hkv, cuda, heads=heads, page=16, steps=[1, 7, 0, 40], keys=[300, 7, 20, 555], causal=causal, dtype="bfloat16")
    base.run_attention(hkv, cuda, heads=heads, page=64, steps=[1, 1], keys=[64, 2100], causal=causal)


@pytest.mark.parametrize("heads", [(28, 4, 128), (4, 2, 256), (8, 8, 64), (6, 2, 80)], ids=str)
def test_4096_requests(hkv, cuda, heads):
    """The largest batch a context takes: tokens and chunks of a few rows, short requests, empty ones among them."""
    rng = np.random.default_rng(29)
    steps = rng.choice([0, 1, 1, 1, 2, 9], 4096)
    keys = np.maximum(steps, rng.integers(1, 90, 4096))
    base.run_attention(hkv, cuda, heads=heads, page=16, steps=[int(n) for n in steps], keys=[int(k) for k in keys])


def test_staged_kernels_required(hkv, cuda):
    """A context that requires the staged kernels never takes the any-geometry kernel instead: chunks with a scale that is not
    positive are refused, single tokens and AUTO contexts answer."""
    torch = cuda
    steps, keys = [40, 3], [90, 70]
    for heads in ((8, 2, 64), (4, 2, 256)):
        base.run_attention(hkv, torch, heads=heads, page=16, steps=[1, 1], keys=keys, scale=-0.1, kernel=2)
        base.run_attention(hkv, torch, heads=heads, page=16, steps=steps, keys=keys, scale=-0.1)
        for scale in (-0.1, 0.0):
            with pytest.raises(hkv.HkvError) as e:
                base.run_attention(hkv, torch, heads=heads, page=16, steps=steps, keys=keys, scale=scale, kernel=2)
            assert e.value.status == 2, e.value


# ---- scaling factors that 32 bits do not hold -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("scaling", [1.1, 0.3, 3.7])
def test_far_positions_with_any_scaling_factor(hkv, cuda, scaling, dtype):
    """Positions of a million over a factor that is no 32-bit number: rounding it alone would turn the first pairs by a
    hundredth of a radian. Tolerance as in test_norm_rope_rounds_once, without a norm."""
    torch = cuda
    T, H, KVH, HD = 70, 4, 2, 128
    D = dt(torch, dtype)
    gen = torch.Generator().manual_seed(37)
    q, k = (torch.randn(T, h, HD, generator=gen).to(D).cuda() for h in (H, KVH))
    pos = torch.randint(900_000, 1_000_000, (1, T), generator=gen, dtype=torch.int32).cuda()
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    ctx = hkv.PagedContext(hkv.PagedGeometry(num_heads=H, num_kv_heads=KVH, head_dim=HD, page_size=16, num_pages=1, max_requests=1,
                                             max_pages=1, max_tokens=T, dtype=dtype, flags=hkv.FLAG_APPEND_ONLY))
    ctx.norm_rope(q, k, None, pos, q_out=q_out, k_out=k_out, theta=1e4, scaling_factor=scaling)
    for x, got in ((q, q_out), (k, k_out)):
        ref, size = P.rope_model(torch, x, pos, None, HD, 1, None, False, 1e-6, 1e4, scaling)
        off = (got.double() - ref).abs() - (P.unit(torch, D) * ref.abs() + 25 * 2.0 ** -24 * size + 2.0 ** -25)
        assert off.max() <= 0, f"{off.max().item():.3e} over"
    ctx.close()
