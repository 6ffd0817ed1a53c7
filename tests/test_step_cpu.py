"""CPU-side checks of the decoder steps (include/urb_step.h): exports, bindings and the refusals that
come before any GPU work."""

import ctypes

import pytest

from urbilateria_amd import native as N

from .test_library_cpu import _declared, _prototypes

_SCALARS = {"uint32_t": ctypes.c_uint32, "uint64_t": ctypes.c_uint64,
            "urb_weight_source": ctypes.c_int}


def test_library_exports_every_declared_symbol():
    lib = ctypes.CDLL(N.MOE_LIB)
    declared = _declared("urb_step.h")
    assert set(N.STEP_EXPORTS) == set(declared)
    for name in declared:
        assert hasattr(lib, name), name


def test_bindings_match_the_header_prototypes():
    lib = N.moe_lib()
    protos = _prototypes("urb_step.h")
    assert set(protos) == set(N.STEP_EXPORTS)
    for name, params in protos.items():
        at = getattr(lib, name).argtypes
        assert at is not None and len(at) == len(params), name
        for p, t in zip(params, at):
            if "*" in p:
                assert t is ctypes.c_void_p or issubclass(t, ctypes._Pointer), (name, p, t)
            else:
                assert t is _SCALARS[p.rsplit(" ", 1)[0].strip()], (name, p, t)


PTR = ctypes.c_void_p(0x1000)   # never read: every call below is refused first


def _create(weight=None, source=N.SOURCE_DEVICE_COPY, **change):
    d = dict(rows=64, cols=128, format=0, x_dtype=2, y_dtype=2, max_tokens=4, adapter_slots=2,
             max_rank=8)
    d.update(change)
    desc = N.ProjDesc(*(d[f] for f, _ in N.ProjDesc._fields_))
    out = ctypes.c_void_p()
    w = weight or N.Matrix(0x1000, 0x1000)
    st = N.moe_lib().urb_proj_create(ctypes.byref(desc), ctypes.byref(w), source,
                                     ctypes.byref(out))
    assert out.value is None
    return st


@pytest.mark.parametrize("change,status", [
    (dict(rows=0), N.ERR_SHAPE), (dict(rows=72), N.ERR_SHAPE), (dict(rows=(1 << 20) + 16), N.ERR_SHAPE),
    (dict(cols=0), N.ERR_SHAPE), (dict(cols=192), N.ERR_SHAPE), (dict(cols=32896), N.ERR_SHAPE),
    (dict(max_tokens=0), N.ERR_SHAPE), (dict(adapter_slots=0), N.ERR_SHAPE),
    (dict(max_rank=0), N.ERR_SHAPE), (dict(max_rank=257), N.ERR_SHAPE),
    (dict(adapter_slots=4097), N.ERR_SHAPE),
    (dict(format=3), N.ERR_ARGUMENT), (dict(x_dtype=1), N.ERR_ARGUMENT),
    (dict(y_dtype=3), N.ERR_ARGUMENT), (dict(source=3), N.ERR_ARGUMENT),
    (dict(weight=N.Matrix(None, None)), N.ERR_ARGUMENT),
    (dict(format=1, weight=N.Matrix(0x1000, None)), N.ERR_ARGUMENT),
])
def test_projection_refuses(change, status):
    assert _create(**change) == status


def test_null_arguments_are_refused():
    lib = N.moe_lib()
    out = ctypes.c_void_p()
    assert lib.urb_proj_create(None, None, 0, ctypes.byref(out)) == N.ERR_ARGUMENT
    assert lib.urb_proj_forward(None, PTR, 128, None, 1, PTR, 64, None) == N.ERR_ARGUMENT
    assert lib.urb_proj_set_adapter(None, 0, None, 0, None) == N.ERR_ARGUMENT
    assert lib.urb_proj_sync(None, None) == N.ERR_ARGUMENT
    assert lib.urb_proj_memory(None, None, None, None) == N.ERR_ARGUMENT
    assert lib.urb_sampler_create(None, ctypes.byref(out)) == N.ERR_ARGUMENT
    assert lib.urb_sample(None, PTR, 1, 1, None, PTR, PTR, None, None) == N.ERR_ARGUMENT
    assert lib.urb_sampler_sync(None, None) == N.ERR_ARGUMENT
    lib.urb_proj_destroy(None)
    lib.urb_sampler_destroy(None)


@pytest.mark.parametrize("vocab,rows,dtype,status", [
    (0, 1, 2, N.ERR_SHAPE), ((1 << 20) + 1, 1, 2, N.ERR_SHAPE), (10, 0, 2, N.ERR_SHAPE),
    (10, 1, 1, N.ERR_ARGUMENT)])
def test_sampler_refuses(vocab, rows, dtype, status):
    desc, out = N.SamplerDesc(vocab, rows, dtype), ctypes.c_void_p()
    assert N.moe_lib().urb_sampler_create(ctypes.byref(desc), ctypes.byref(out)) == status
    assert out.value is None


def _rotate(tokens=2, q=PTR, k=PTR, weight=PTR, positions=PTR, freq=PTR, **change):
    d = dict(dtype=2, q_heads=4, k_heads=1, head_dim=64, rotary_dim=32, interleaved=0,
             zero_centered=0, eps=1e-6)
    d.update(change)
    desc = N.QkDesc(*(d.get(f, 64) for f, _ in N.QkDesc._fields_))
    return N.moe_lib().urb_qk_norm_rope(ctypes.byref(desc), q, k, weight, weight, positions, freq,
                                        tokens, q, k, None)


@pytest.mark.parametrize("change,status", [
    (dict(tokens=0), N.ERR_SHAPE), (dict(q_heads=0), N.ERR_SHAPE), (dict(k_heads=65535), N.ERR_SHAPE),
    (dict(q_heads=65535, k_heads=0, tokens=1 << 16), N.ERR_SHAPE),
    (dict(head_dim=0), N.ERR_SHAPE), (dict(head_dim=63), N.ERR_SHAPE),
    (dict(head_dim=1026), N.ERR_SHAPE), (dict(rotary_dim=31), N.ERR_SHAPE),
    (dict(rotary_dim=66), N.ERR_SHAPE),
    (dict(eps=0.0), N.ERR_INVALID_GEOMETRY), (dict(eps=float("nan")), N.ERR_INVALID_GEOMETRY),
    (dict(eps=float("inf")), N.ERR_INVALID_GEOMETRY),
    (dict(dtype=1), N.ERR_ARGUMENT), (dict(q=None), N.ERR_ARGUMENT), (dict(k=None), N.ERR_ARGUMENT),
    (dict(weight=None), N.ERR_ARGUMENT), (dict(positions=None), N.ERR_ARGUMENT),
    (dict(freq=None), N.ERR_ARGUMENT), (dict(q=ctypes.c_void_p(0x1002)), N.ERR_ARGUMENT),
])
def test_rotation_refuses(change, status):
    assert _rotate(**change) == status


@pytest.mark.parametrize("change", [
    dict(), dict(q_out_token_stride=255), dict(q_out_token_stride=256, q_out_head_stride=63),
    dict(q_out_token_stride=256, k_out_token_stride=0), dict(q_out_token_stride=64, q_out_head_stride=127),
    dict(q_out_token_stride=0, q_out_head_stride=1 << 40),
    dict(q_out_token_stride=1 << 63, q_out_head_stride=1 << 63),
])
def test_rotation_refuses_outputs_that_overlap_themselves(change):
    assert _rotate(**change) == N.ERR_SHAPE


# ---- the wrapper's own refusals, before any call of the library ----

def _wrapper():
    import numpy as np
    torch = pytest.importorskip("torch")
    from urbilateria_amd import configs as C
    from urbilateria_amd import step
    return np, torch, C, step


def test_matrices_of_another_type_are_refused():
    np, torch, C, step = _wrapper()
    make = lambda fmt, data, scales=None: step.AdaptedProjection(data, scales, fmt, 16, 128, 4)
    scales = torch.full((16, 4), 127, dtype=torch.uint8)
    for fmt, data, s in (
            (C.FMT_BF16, torch.zeros(16, 128, dtype=torch.float16), None),
            (C.FMT_BF16, np.zeros((16, 128), np.float16), None),
            (C.FMT_BF16, torch.zeros(16, 64, dtype=torch.float32), None),
            (C.FMT_BF16, torch.zeros(16, 32, dtype=torch.complex64), None),
            (C.FMT_MXFP8, torch.zeros(16, 128, dtype=torch.uint8).view(torch.float8_e5m2), scales),
            (C.FMT_MXFP8, torch.zeros(16, 128, dtype=torch.uint8).view(torch.float8_e4m3fnuz), scales),
            (C.FMT_MXFP8, torch.zeros(16, 128, dtype=torch.uint8), scales.view(torch.float8_e4m3fn)),
            (C.FMT_MXFP4, torch.zeros(16, 32, dtype=torch.float16), scales),
            (C.FMT_MXFP4, torch.zeros(16, 64, dtype=torch.bool), scales)):
        with pytest.raises(ValueError, match="holding its bits"):
            make(fmt, data, s)


def test_adapters_of_another_type_are_refused():
    np, torch, C, step = _wrapper()
    p = step.AdaptedProjection.__new__(step.AdaptedProjection)
    p.rows, p.cols, p.device, p._ctx = 16, 128, 0, None
    half = lambda *shape: torch.zeros(shape, dtype=torch.float16)
    good = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16)
    for a, b in ((half(4, 128), half(16, 4)), (good(4, 128), half(16, 4)), (half(4, 128), good(16, 4)),
                 (np.zeros((4, 128), np.float16), np.zeros((16, 4), np.float16))):
        with pytest.raises(ValueError, match="holding its bits"):
            p.set_adapter(0, a, b)


def test_payloads_of_their_own_type_or_bits_are_taken():
    np, torch, C, step = _wrapper()
    for t, own in ((torch.zeros(2, dtype=torch.bfloat16), "bfloat16"), (torch.zeros(2, dtype=torch.int16), "bfloat16"),
                   (torch.zeros(2, dtype=torch.uint16), "bfloat16"), (torch.zeros(4, dtype=torch.uint8), "bfloat16"),
                   (np.zeros(2, np.uint16), "bfloat16"), (np.zeros(2, np.int16), "bfloat16"),
                   (torch.zeros(2, dtype=torch.uint8).view(torch.float8_e4m3fn), step._VALUES[C.FMT_MXFP8]),
                   (torch.zeros(2, dtype=torch.uint8), step._VALUES[C.FMT_MXFP4]),
                   (torch.zeros(2, dtype=torch.uint8).view(torch.float8_e8m0fnu), step._SCALES)):
        step._payload(t, "t", own, None)


def test_payloads_elsewhere_are_refused():
    np, torch, C, step = _wrapper()
    away = torch.zeros(4, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="cuda:1"):
        step._payload(away, "a", "bfloat16", 1)
    p = step.AdaptedProjection.__new__(step.AdaptedProjection)
    p.rows, p.cols, p.device, p._ctx = 16, 128, 0, None
    make = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="cuda:0"):
        p.set_adapter(0, make(4, 128), make(16, 4))
