"""CPU tests of the paged cache: geometry checks come before any device work, calls without a context are refused, and
the plan model the GPU tests compare with keeps every page exactly once."""
import ctypes as C

import numpy as np
import pytest

import _paged as P


@pytest.mark.parametrize("kw,status", [
    (dict(num_heads=14, num_kv_heads=3), 2), (dict(head_dim=513), 2), (dict(head_dim=0), 2), (dict(page_size=0), 1),
    (dict(num_pages=0), 1), (dict(max_requests=0), 1), (dict(max_requests=4097), 7), (dict(max_pages=0), 1), (dict(max_tokens=0), 1),
    (dict(window_size=-1), 1), (dict(kernel_select=3), 1), (dict(flags=1), 1), (dict(page_size=1 << 16, num_pages=1 << 15), 7),
    (dict(page_size=1 << 16, max_pages=1 << 15), 7), (dict(dtype="float32"), 1)], ids=str)
def test_geometry_is_checked_before_the_device(hkv, kw, status):
    good = dict(num_heads=28, num_kv_heads=4, head_dim=128, page_size=16, num_pages=64, max_requests=8, max_pages=8, max_tokens=64)
    with pytest.raises(hkv.HkvError) as e:
        hkv.PagedContext(hkv.PagedGeometry(**{**good, **kw}))
    assert e.value.status == status, e.value


def test_no_cpu_fallback(hkv):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(hkv.HkvError) as e:
        hkv.PagedContext(hkv.PagedGeometry(num_pages=4, max_pages=2))
    assert e.value.status in (4, 5)


def test_calls_without_a_context_are_refused(hkv):
    lib = hkv._capi.load()
    assert lib.hkv_paged_create(None, None) == 1
    handle = C.c_void_p()
    assert lib.hkv_paged_create(C.byref(handle), None) == 1 and b"null" in lib.hkv_paged_last_error(handle)
    for h in (None, handle):
        assert lib.hkv_paged_plan(h, 1, 1, *[None] * 12) == 1
        assert lib.hkv_paged_release(h, 1, *[None] * 6) == 1
        assert lib.hkv_paged_append(h, None, None, 0, None, None, None, 1, None) == 1
        assert lib.hkv_paged_norm_rope(h, None, None) == 1
        assert lib.hkv_paged_attention(h, None, 0, None, None, None, None, None, None, None, 1, 1, 1, 1.0, None) == 1
        assert lib.hkv_paged_cross_attention(h, None, 0, None, None, None, None, None, None, None, 1, 1, 1, 1.0, None) == 1
        assert lib.hkv_paged_device_status(h, None, None) == 1
    assert lib.hkv_paged_destroy(handle) == 0 and lib.hkv_paged_destroy(None) == 0
    assert lib.hkv_paged_workspace_bytes(None) == 0


def test_plan_model_keeps_every_page_once():
    rng = np.random.default_rng(1)
    R, page, cols, num_pages = 9, 4, 10, 60
    past, table = np.zeros(R, np.int64), np.full((R, cols), -1, np.int64)
    free, count = np.arange(num_pages), num_pages
    for _ in range(30):
        out = P.plan_model(past, rng.integers(0, 9, R), table, free, count, page, 50)
        past, table, count = out["total_len"], out["table"], out["free_left"]
        held = [table[r, j] for r in range(R) for j in range(-(-int(past[r]) // page))]
        assert sorted(held + list(free[:count])) == list(range(num_pages))
        live = out["slots"][out["slots"] >= 0]
        assert len(set(live)) == len(live)


def rows_of(hkv, heads, head_dim, dtype):
    """PagedContext's check of [tokens, heads, head_dim] tensors without a device: the context of a CPU tensor's device index."""
    import torch
    ctx = object.__new__(hkv.PagedContext)
    ctx._h, ctx._hd, ctx._dtype, ctx._index = None, head_dim, getattr(torch, dtype), torch.zeros(0).get_device()
    return lambda t, tokens: ctx._rows("x", t, heads, tokens)


@pytest.mark.parametrize("heads,head_dim", [(4, 64), (1, 64), (3, 1), (1, 1)])
def test_token_strides_that_are_passed_on(hkv, heads, head_dim):
    """0 means dense in the library, so a broadcast token (stride 0) must never get there, nor tokens that overlap."""
    import torch
    rows, row = rows_of(hkv, heads, head_dim, "float16"), heads * head_dim
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)
    assert rows(h(5, heads, head_dim), 5)[1] == 0
    assert rows(h(5, row + 8)[:, :row].unflatten(1, (heads, head_dim)), 5)[1] == row + 8
    assert rows(h(1, heads, head_dim).expand(1, heads, head_dim), 1)[1] == 0
    assert rows(h(0, heads, head_dim), 0)[1] == 0
    one = h(1, heads, head_dim)
    for t in (one.expand(5, heads, head_dim), torch.as_strided(h(5 * row + 8), (2, heads, head_dim), (0, head_dim, 1)),
              *([torch.as_strided(h(5 * row), (5, heads, head_dim), (row - 1, head_dim, 1))] if row > 1 else [])):
        with pytest.raises(hkv.HkvError) as e:
            rows(t, t.shape[0])
        assert e.value.status == 2, e.value


def test_schedule_arithmetic():
    """tests/cpp/hkv_paged_schedule_tests.cu: the kernels' host-callable schedule arithmetic, run on the CPU."""
    import importlib
    import subprocess
    binary = importlib.import_module("hector-engine_b200.build").build_schedule_tests()
    res = subprocess.run([binary], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert res.stdout.count("PASS:") == 4 and "ALL PASSED" in res.stdout
