"""Plain 64-bit models of the paged cache's operators and the tolerances that follow from the kernels' roundings."""
import math

import numpy as np


def unit(torch, dtype):
    """Largest relative error of one rounding to `dtype` (half a step)."""
    return torch.finfo(dtype).eps / 2


def plan_model(past, new, table, free, count, page, tokens):
    """One step's tables, request by request. Returns a dict; `table` is copied."""
    R, cols = table.shape
    table = table.copy()
    q_start, step, total = [0], [], []
    slots, positions = np.full(tokens, -1, np.int64), np.full(tokens, -1, np.int64)
    at, wanted, used = 0, 0, 0
    for r in range(R):
        p, n = int(past[r]), int(new[r])
        end = at + max(n, 0)
        fits = p >= 0 and n >= 0 and p + n <= cols * page and end <= tokens
        j0, j1 = (-(-p // page), -(-(p + n) // page)) if fits else (0, 0)
        ok = fits and (j1 == j0 or wanted + j1 - j0 <= count)
        if ok:
            for j in range(j0, j1):
                table[r, j] = free[count - 1 - wanted - (j - j0)]
            for i in range(n):
                slots[at + i] = table[r, (p + i) // page] * page + (p + i) % page
                positions[at + i] = p + i
            used += j1 - j0
        wanted += j1 - j0
        step.append(n if ok else 0)
        total.append(p + step[-1])
        at = end
        q_start.append(min(at, tokens))
    return dict(table=table, q_start=np.array(q_start), step_len=np.array(step), total_len=np.array(total), slots=slots,
                positions=positions, free_left=count - used)


def axis_of(i, axes, sections, interleaved):
    if axes == 1:
        return 0
    if interleaved:
        a = i % axes
        return a if a and i < axes * sections[a] else 0
    return next(a for a in range(axes) if i < sum(sections[:a + 1]))


def rope_model(torch, x, pos, w, rot, axes, sections, interleaved, eps, theta, scaling):
    """[T, heads, HD] in 64 bits, and the size sum |.| of the two products behind each element."""
    half = rot // 2
    y = x.double()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    pos = pos.double().view(axes, -1)
    if half == 0:
        return y, y.abs()
    ang = torch.stack([pos[axis_of(i, axes, sections, interleaved)] / scaling * theta ** (-2.0 * i / rot) for i in range(half)], -1)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b, rest = y[..., :half], y[..., half:rot], y[..., rot:]
    out = torch.cat([a * c - b * s, a * s + b * c, rest], -1)
    size = torch.cat([(a * c).abs() + (b * s).abs() + a.abs() + b.abs(), (a * s).abs() + (b * c).abs() + a.abs() + b.abs(), rest.abs()], -1)
    return out, size


def attend_model(torch, q, k_plane, v_plane, table, q_start, step, keys, scale, page, window=0, causal=True, max_step=None):
    """(out, tolerance, live) of ragged attention over pages in 64 bits; `live` marks the rows that belong to a query.

    Tolerance, per element, u = half a step of the type: u |ref| for the rounding of the result; (u + 2 e + 2 d) A for the
    rounding of the probabilities to the type before the second product, the error e = 1e-4 of exp2 (measured against
    2^x, at most 7.5e-5 for its polynomial) and of the scores — d = (HD + 8) 2^-24 max_j sum|q k| scale for sums of HD
    products in 32 bits — where A = sum p |v| / sum p; fp16 probabilities below 2^-14 lie on a grid of 2^-24, so up to
    2^-25 max|v| per key beside sum p >= 1; 32-bit sums over n keys: n 2^-24 A."""
    H, HD = q.shape[1], q.shape[2]
    KVH = k_plane.shape[2]
    G = H // KVH
    u = unit(torch, q.dtype)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    live = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    cap = table.shape[1] * page
    for r in range(len(keys)):
        n, L, at0 = int(step[r]), min(int(keys[r]), cap), int(q_start[r])
        m = n if max_step is None else min(n, max_step)
        if m <= 0:
            continue
        live[at0:at0 + m] = True
        if L <= 0:
            continue
        j = torch.arange(L, device=q.device)
        pg = table[r].long()[j // page]
        K, V = k_plane[pg, j % page].double(), v_plane[pg, j % page].double()      # [L, KVH, HD]
        K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
        x = q[at0:at0 + m].double()
        pos = L - n + torch.arange(m, device=q.device)
        seen = torch.ones(m, L, dtype=torch.bool, device=q.device)
        if causal:
            seen = j[None] <= pos[:, None]
            if window:
                seen &= j[None] > pos[:, None] - window
        s = torch.einsum("ihd,jhd->hij", x, K) * scale
        sabs = torch.einsum("ihd,jhd->hij", x.abs(), K.abs()) * abs(scale)
        s = s.masked_fill(~seen[None], -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(seen[None], torch.exp(s - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
        l = p.sum(-1, keepdim=True)
        some = l > 0
        o = torch.where(some, torch.einsum("hij,jhd->hid", p, V) / l.clamp(min=1e-300), 0.0)
        A = torch.where(some, torch.einsum("hij,jhd->hid", p, V.abs()) / l.clamp(min=1e-300), 0.0)
        d = (HD + 8) * 2.0 ** -24 * sabs.masked_fill(~seen[None], 0.0).amax(-1, keepdim=True)
        low = seen.sum(-1)[None, :, None] * 2.0 ** -25 * V.abs().amax() / l.clamp(min=1.0) if q.dtype == torch.float16 else 0.0
        t = u * o.abs() + (u + 2e-4 + 2 * d + L * 2.0 ** -24) * A + low
        out[at0:at0 + m] = o.permute(1, 0, 2)
        tol[at0:at0 + m] = (t + 2.0 ** -24).permute(1, 0, 2)
    return out, tol, live


def make_pages(torch, gen, keys, page, num_pages, cols, KVH, HD, dtype, poison=True):
    """Planes, and a block table of randomly dealt pages. Rows beyond a request's keys, unassigned pages and the
    table's unused entries hold what must never be read as data: NaN, infinities, page numbers far outside."""
    need = [-(-k // page) for k in keys]
    assert sum(need) <= num_pages
    ids = torch.randperm(num_pages, generator=gen)
    k = torch.full((num_pages, page, KVH, HD), float("nan") if poison else 0.0).to(dtype)
    v = torch.full((num_pages, page, KVH, HD), float("inf") if poison else 0.0).to(dtype)
    table = torch.full((len(keys), cols), 0x7fffff00, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        mine = ids[at:at + n]
        at += n
        table[r, :n] = mine.to(torch.int32)
        if keys[r] > 0:
            j = torch.arange(keys[r])
            k[mine[j // page], j % page] = torch.randn(keys[r], KVH, HD, generator=gen).to(dtype)
            v[mine[j // page], j % page] = torch.randn(keys[r], KVH, HD, generator=gen).to(dtype)
    return k.cuda(), v.cuda(), table.cuda()
