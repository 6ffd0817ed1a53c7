"""CPU-side checks of the paged cache (include/urb_cache.h) and of beam search's selection: exports,
bindings and the refusals that come before any GPU work."""

import ctypes
import shutil
import subprocess

import pytest

from urbilateria_amd import native as N

from .test_library_cpu import _declared, _prototypes

_SCALARS = {"uint32_t": ctypes.c_uint32}


def test_library_exports_every_declared_symbol():
    lib = ctypes.CDLL(N.MOE_LIB)
    declared = _declared("urb_cache.h")
    assert set(N.CACHE_EXPORTS) == set(declared)
    for name in declared:
        assert hasattr(lib, name), name


def test_bindings_match_the_header_prototypes():
    lib = N.moe_lib()
    protos = _prototypes("urb_cache.h")
    assert set(protos) == set(N.CACHE_EXPORTS)
    for name, params in protos.items():
        at = getattr(lib, name).argtypes
        assert at is not None and len(at) == len(params), name
        for p, t in zip(params, at):
            if "*" in p:
                assert t is ctypes.c_void_p or issubclass(t, ctypes._Pointer), (name, p, t)
            else:
                assert t is _SCALARS[p.rsplit(" ", 1)[0].strip()], (name, p, t)


AT = 0x1000   # never read: every call below is refused first
PTR = ctypes.c_void_p(AT)


def _struct(kind, defaults, change):
    d = dict(defaults)
    d.update(change)
    return kind(**{f: d[f] for f, _ in kind._fields_ if f in d})


CACHE = dict(k=AT, v=AT, k_scales=None, v_scales=None, dtype=0, pages=8, heads=2, page_size=16,
             head_dim=64, page_stride=2048, head_stride=1024, token_stride=64)
ROWS = dict(k=AT, v=AT, dtype=0, k_token_stride=128, k_head_stride=64, v_token_stride=128,
            v_head_stride=64)


def _append(cache=(), rows=(), slots=PTR, tokens=3):
    c, r = _struct(N.KvCache, CACHE, dict(cache)), _struct(N.KvRows, ROWS, dict(rows))
    return N.moe_lib().urb_kv_append(ctypes.byref(c), ctypes.byref(r), slots, tokens, None)


@pytest.mark.parametrize("change,status", [
    (dict(k=None), N.ERR_ARGUMENT), (dict(v=None), N.ERR_ARGUMENT), (dict(dtype=2), N.ERR_ARGUMENT),
    (dict(dtype=3), N.ERR_ARGUMENT), (dict(dtype=3, k_scales=AT), N.ERR_ARGUMENT),
    (dict(k_scales=AT), N.ERR_ARGUMENT), (dict(v_scales=AT), N.ERR_ARGUMENT),
    (dict(k=AT + 2), N.ERR_ARGUMENT), (dict(v=AT + 8), N.ERR_ARGUMENT),
    (dict(token_stride=68, head_stride=2048, page_stride=4096), N.ERR_ARGUMENT),
    (dict(page_stride=2052), N.ERR_ARGUMENT), (dict(head_stride=1028, page_stride=4096), N.ERR_ARGUMENT),
    (dict(pages=0), N.ERR_SHAPE), (dict(pages=(1 << 24) + 1), N.ERR_SHAPE), (dict(heads=0), N.ERR_SHAPE),
    (dict(heads=1025), N.ERR_SHAPE), (dict(page_size=0), N.ERR_SHAPE), (dict(page_size=1025), N.ERR_SHAPE),
    (dict(head_dim=0), N.ERR_SHAPE), (dict(head_dim=8), N.ERR_SHAPE), (dict(head_dim=72), N.ERR_SHAPE),
    (dict(head_dim=272), N.ERR_SHAPE),
    (dict(token_stride=56), N.ERR_SHAPE), (dict(head_stride=1016), N.ERR_SHAPE),
    (dict(page_stride=2040), N.ERR_SHAPE), (dict(page_stride=0), N.ERR_SHAPE),
    (dict(head_stride=64, token_stride=64), N.ERR_SHAPE),
    (dict(page_stride=1 << 33), N.ERR_SHAPE), (dict(page_stride=1 << 62), N.ERR_SHAPE),
])
def test_caches_are_refused(change, status):
    assert _append(cache=change) == status


@pytest.mark.parametrize("change,status", [
    (dict(k=None), N.ERR_ARGUMENT), (dict(v=None), N.ERR_ARGUMENT), (dict(dtype=1), N.ERR_ARGUMENT),
    (dict(dtype=3), N.ERR_ARGUMENT), (dict(k=AT + 8), N.ERR_ARGUMENT), (dict(v=AT + 4), N.ERR_ARGUMENT),
    (dict(k_token_stride=132), N.ERR_ARGUMENT), (dict(v_head_stride=65), N.ERR_ARGUMENT),
    (dict(dtype=2, k_head_stride=66), N.ERR_ARGUMENT),
])
def test_rows_are_refused(change, status):
    assert _append(rows=change) == status


def test_appends_are_refused():
    assert _append(slots=None) == N.ERR_ARGUMENT
    assert _append(tokens=0) == N.ERR_SHAPE
    assert _append(tokens=1 << 24) == N.ERR_SHAPE
    assert N.moe_lib().urb_kv_append(None, None, PTR, 1, None) == N.ERR_ARGUMENT


@pytest.mark.parametrize("change", [
    dict(pages=0), dict(pages=(1 << 24) + 1), dict(page_size=0), dict(page_size=1025), dict(max_rows=0),
    dict(max_rows=(1 << 20) + 1), dict(max_blocks=0), dict(max_blocks=(1 << 20) + 1),
    dict(max_tokens=1 << 30), dict(max_rows=1 << 16, max_blocks=1 << 15),
    dict(max_blocks=1 << 20, page_size=1024),
])
def test_pagers_are_refused(change):
    desc = _struct(N.PagerDesc, dict(pages=8, page_size=16, max_rows=4, max_blocks=4, max_tokens=8), change)
    out = ctypes.c_void_p()
    assert N.moe_lib().urb_pager_create(ctypes.byref(desc), ctypes.byref(out)) == N.ERR_SHAPE
    assert out.value is None


@pytest.mark.parametrize("change,status", [
    (dict(dtype=1), N.ERR_ARGUMENT), (dict(dtype=3), N.ERR_ARGUMENT), (dict(cache_dtype=2), N.ERR_ARGUMENT),
    (dict(q_heads=0), N.ERR_SHAPE), (dict(q_heads=9), N.ERR_SHAPE), (dict(q_heads=8194), N.ERR_SHAPE),
    (dict(heads=0), N.ERR_SHAPE), (dict(heads=1025), N.ERR_SHAPE), (dict(head_dim=24), N.ERR_SHAPE),
    (dict(head_dim=512), N.ERR_SHAPE), (dict(page_size=0), N.ERR_SHAPE), (dict(queries=0), N.ERR_SHAPE),
    (dict(queries=17), N.ERR_SHAPE), (dict(max_rows=0), N.ERR_SHAPE), (dict(max_rows=1 << 21), N.ERR_SHAPE),
    (dict(max_length=0), N.ERR_SHAPE), (dict(max_length=(1 << 27) + 1), N.ERR_SHAPE),
    (dict(scale=0.0), N.ERR_INVALID_GEOMETRY), (dict(scale=-1.0), N.ERR_INVALID_GEOMETRY),
    (dict(scale=float("nan")), N.ERR_INVALID_GEOMETRY), (dict(scale=float("inf")), N.ERR_INVALID_GEOMETRY),
    (dict(scale=2.0 ** 127.5), N.ERR_INVALID_GEOMETRY),
])
def test_attentions_are_refused(change, status):
    desc = _struct(N.AttentionDesc, dict(q_heads=8, heads=2, head_dim=64, page_size=16, dtype=0, cache_dtype=0,
                                         queries=1, window=0, scale=0.1, max_rows=4, max_length=100), change)
    out = ctypes.c_void_p()
    assert N.moe_lib().urb_attention_create(ctypes.byref(desc), ctypes.byref(out)) == status
    assert out.value is None


@pytest.mark.parametrize("change", [
    dict(max_length=(1 << 24) + 1), dict(max_rows=(1 << 20) + 1), dict(page_size=1025), dict(q_heads=8196, heads=4),
    dict(head_dim=0), dict(head_dim=272)])
def test_attentions_just_past_their_limits_are_refused(change):
    desc = _struct(N.AttentionDesc, dict(q_heads=8, heads=2, head_dim=64, page_size=16, dtype=0, cache_dtype=0,
                                         queries=1, window=0, scale=0.1, max_rows=4, max_length=100), change)
    out = ctypes.c_void_p()
    assert N.moe_lib().urb_attention_create(ctypes.byref(desc), ctypes.byref(out)) == N.ERR_SHAPE
    assert out.value is None


@pytest.mark.parametrize("change,status", [
    (dict(vocab=0), N.ERR_SHAPE), (dict(vocab=(1 << 18) + 1), N.ERR_SHAPE), (dict(width=0), N.ERR_SHAPE),
    (dict(width=33), N.ERR_SHAPE), (dict(picks=0), N.ERR_SHAPE), (dict(picks=65), N.ERR_SHAPE),
    (dict(max_requests=0), N.ERR_SHAPE), (dict(max_requests=65536), N.ERR_SHAPE),
    (dict(dtype=1), N.ERR_ARGUMENT), (dict(dtype=3), N.ERR_ARGUMENT),
])
def test_beams_are_refused(change, status):
    desc = _struct(N.BeamsDesc, dict(vocab=100, width=4, picks=4, max_requests=2, dtype=2), change)
    out = ctypes.c_void_p()
    assert N.moe_lib().urb_beams_create(ctypes.byref(desc), ctypes.byref(out)) == status
    assert out.value is None


def test_no_call_allocates_an_array():
    # contexts and plans are single objects; only a call would need an array that may be missing
    if shutil.which("nm") is None:
        pytest.skip("nm not available")
    r = subprocess.run(["nm", "-D", "--undefined-only", N.MOE_LIB], capture_output=True, text=True, check=True)
    assert "_ZnwmRKSt9nothrow_t" in r.stdout
    assert "_ZnamRKSt9nothrow_t" not in r.stdout


def test_null_arguments_are_refused():
    lib, out = N.moe_lib(), ctypes.c_void_p()
    for create in (lib.urb_pager_create, lib.urb_attention_create, lib.urb_beams_create):
        assert create(None, ctypes.byref(out)) == N.ERR_ARGUMENT
    assert lib.urb_pager_plan(None, None, None) == N.ERR_ARGUMENT
    assert lib.urb_pager_fork(None, None, None) == N.ERR_ARGUMENT
    assert lib.urb_attend(None, None, None, None) == N.ERR_ARGUMENT
    assert lib.urb_beams_select(None, None, None) == N.ERR_ARGUMENT
    for sync in (lib.urb_pager_sync, lib.urb_attention_sync, lib.urb_beams_sync):
        assert sync(None, None) == N.ERR_ARGUMENT
    for destroy in (lib.urb_pager_destroy, lib.urb_attention_destroy, lib.urb_beams_destroy):
        destroy(None)


def test_tensors_elsewhere_are_refused():
    torch = pytest.importorskip("torch")
    from urbilateria_amd import cache
    page = lambda **kw: torch.zeros((2, 1, 4, 16), dtype=torch.bfloat16, **kw)
    with pytest.raises(ValueError, match="on a GPU"):
        cache.PagedCache(page(), page())
    with pytest.raises(ValueError, match="on a GPU"):
        cache.PagedCache(page()[0], page()[0])
    with pytest.raises(ValueError, match="contiguous"):
        cache._table(torch.zeros((2, 3), dtype=torch.int64), "tables", 2, -1)
    with pytest.raises(ValueError, match="contiguous"):
        cache._table(torch.zeros((3, 2), dtype=torch.int32).T, "tables", 2, -1)
    with pytest.raises(ValueError, match="values of a head"):
        cache._strides(torch.zeros((2, 16, 4)).transpose(1, 2), "k", (2, 4, 16), torch.float32, -1)
