"""Refusals of the gated linear recurrence (no GPU needed): Python checks raise
before any launch, and the C entries' own checks come before any device work."""

import ctypes

import pytest
import torch

import gdn_b200

X = dict(dtype=torch.bfloat16)


def tensors(shape=(2, 5, 3, 8), dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype), torch.zeros(shape)


def test_cpu_tensors_rejected():
    x, g = tensors()
    with pytest.raises(ValueError, match="CUDA"):
        gdn_b200.gated_scan(x, g)
    with pytest.raises(ValueError, match="CUDA"):
        gdn_b200.gated_scan_step(x[:, 0], g[:, 0], torch.zeros(2, 3, 8))


def test_shapes_and_types_rejected():
    x, g = tensors()
    with pytest.raises(ValueError, match="x must be"):
        gdn_b200.gated_scan(x[0], g[0])
    with pytest.raises(ValueError, match="g shape"):
        gdn_b200.gated_scan(x, g[..., :1])
    with pytest.raises(ValueError, match="empty"):
        gdn_b200.gated_scan(x[:, :0], g[:, :0])
    with pytest.raises(ValueError, match="initial_state"):
        gdn_b200.gated_scan(x, g, torch.zeros(2, 3, 7))
    with pytest.raises(NotImplementedError, match="fp16"):
        gdn_b200.gated_scan(x.double(), g)
    with pytest.raises(ValueError, match="output_dtype"):
        gdn_b200.gated_scan(x, g, output_dtype=torch.float16)
    with pytest.raises(ValueError, match="contiguous last"):
        gdn_b200.gated_scan(x.transpose(2, 3), g.transpose(2, 3))
    with pytest.raises(TypeError):
        gdn_b200.gated_scan(x, g.numpy())
    with pytest.raises(TypeError):
        gdn_b200.gated_scan_step(x[:, 0], g[:, 0], None)


@pytest.fixture(scope="module")
def lib():
    from gdn_b200 import _build, _lib
    _build.build()
    return _lib.load()


def c_args(**kw):
    from gdn_b200 import _lib
    a = _lib.GatedScanArgs()
    a.abi_version = _lib.ABI_VERSION
    a.B, a.T, a.H, a.D = 1, 4, 2, 8
    a.x_dtype = a.o_dtype = _lib.DTYPE_BF16
    a.g_dtype = _lib.DTYPE_F32
    for n in ("x", "g", "o", "states", "dx", "dg"):
        setattr(a, n, 0x10000)  # never dereferenced: a check fails or no device is found first
    for n in ("x", "g", "o", "dx", "dg"):
        setattr(a, n + "_stride", (64, 16, 8))
    for key, val in kw.items():
        setattr(a, key, val)
    return a


@pytest.mark.parametrize("field,value,expected", [
    ("abi_version", 1, 1),
    ("B", 0, 1),
    ("T", 0, 1),
    ("D", -1, 1),
    ("T", 0x7fffffff, 2),
    ("x_dtype", 3, 1),
    ("g_dtype", 1, 2),        # fp16 gates with bf16 x
    ("o_dtype", 1, 2),
    ("flags", 1, 1),
    ("x", None, 1),
    ("x", 0x10001, 3),
    ("h0", 0x10002, 3),
    ("x_stride", (64, -16, 8), 1),
])
def test_c_entries_reject_before_device_work(lib, field, value, expected):
    a = c_args(**{field: value})
    assert lib.gdn_gated_scan_fwd_sm100(ctypes.byref(a), None) == expected
    assert lib.gdn_gated_scan_bwd_sm100(ctypes.byref(a), None) == expected


def test_backward_needs_its_buffers(lib):
    for n in ("states", "dx", "dg"):
        assert lib.gdn_gated_scan_bwd_sm100(ctypes.byref(c_args(**{n: None})), None) == 1
    assert lib.gdn_gated_scan_fwd_sm100(ctypes.byref(c_args(o=None)), None) == 1
    assert lib.gdn_gated_scan_fwd_sm100(None, None) == 1


def test_states_bytes(lib):
    # one fp32 row per tile: 128 rows of 16-bit x, 64 rows of fp32 x
    assert lib.gdn_gated_scan_states_bytes(ctypes.byref(c_args(B=3, T=129))) == 3 * 2 * 16 * 4
    assert lib.gdn_gated_scan_states_bytes(ctypes.byref(c_args(B=3, T=129, x_dtype=0))) == 3 * 3 * 16 * 4
    assert lib.gdn_gated_scan_states_bytes(ctypes.byref(c_args(T=0))) == 0
