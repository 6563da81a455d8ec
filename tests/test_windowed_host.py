"""Refusals of the windowed attention and of gdn_step (no GPU needed), and the C
entries' own checks, which come before any device work."""

import ctypes

import pytest
import torch

import gdn_b200

BF = torch.bfloat16


def qkv(B=1, T=4, S=8, H=4, HK=2, D=64, dt=BF):
    return torch.zeros(B, T, H, D, dtype=dt), torch.zeros(B, S, HK, D, dtype=dt), torch.zeros(B, S, HK, D, dtype=dt)


def step_args(B=1, H=4, HK=2, D=64, cap=16, dt=BF):
    z = lambda *s: torch.zeros(*s, dtype=dt)
    return [z(B, H, D), z(B, HK, D), z(B, HK, D), z(B, cap, HK, D), z(B, cap, HK, D), torch.zeros(B, dtype=torch.int32)]


def test_window_attention_refusals():
    f = gdn_b200.window_attention
    q, k, v = qkv()
    with pytest.raises(ValueError, match="CUDA"):
        f(q, k, v, 4)
    with pytest.raises(ValueError, match="q must be"):
        f(q[0], k, v, 4)
    with pytest.raises(ValueError, match="k and v"):
        f(q, k, v[:, :4], 4)
    with pytest.raises(ValueError, match="fewer keys"):
        f(q, k[:, :3], v[:, :3], 4)
    with pytest.raises(ValueError, match="multiple"):
        f(q[:, :, :3], k, v, 4)
    with pytest.raises(ValueError, match="window"):
        f(q, k, v, 0)
    with pytest.raises(ValueError, match="window"):
        f(q, k, v, 4, -1)
    with pytest.raises(ValueError, match="scale"):
        f(q, k, v, 4, scale=0.0)
    with pytest.raises(ValueError, match="scale"):
        f(q, k, v, 4, scale=float("nan"))
    with pytest.raises(ValueError, match="dtype"):
        f(q, k.half(), v, 4)
    with pytest.raises(NotImplementedError, match="fp16"):
        f(*[t.float() for t in (q, k, v)], 4)
    with pytest.raises(NotImplementedError, match="head size"):
        f(*qkv(D=32), 4)
    with pytest.raises(ValueError, match="lengths"):
        f(q, k, v, 4, lengths=torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="empty"):
        f(q[:, :0], k, v, 4)
    with pytest.raises(TypeError):
        f(q, None, v, 4)
    with pytest.raises(NotImplementedError, match="backward"):
        f(q.requires_grad_(), k, v, 4)


def test_window_step_refusals():
    f = gdn_b200.window_attention_step
    a = step_args()
    with pytest.raises(ValueError, match="CUDA"):
        f(*a, 8, 4)
    with pytest.raises(ValueError, match="capacity"):
        f(*a, 13, 4)
    with pytest.raises(ValueError, match="positions"):
        f(*a[:5], a[5].long(), 8)
    with pytest.raises(ValueError, match="caches"):
        f(*a[:4], a[4][:, :8], a[5], 8)
    with pytest.raises(ValueError, match="expanded"):
        f(*a[:3], a[3][:, :1].expand(-1, 16, -1, -1), a[4], a[5], 8)
    with pytest.raises(NotImplementedError, match="head size"):
        f(*step_args(D=96), 8)
    with pytest.raises(NotImplementedError, match="backward"):
        f(a[0].requires_grad_(), *a[1:], 8)


def test_gdn_step_refusals():
    f = gdn_b200.gdn_step
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)
    a = [z(2, 3, 128), z(2, 3, 128), z(2, 3, 128), z(2, 3), z(2, 3), z(2, 3, 128, 128, dt=torch.float32)]
    with pytest.raises(ValueError, match="CUDA"):
        f(*a)
    with pytest.raises(ValueError, match="k shape"):
        f(a[0], a[1][:1], *a[2:])
    with pytest.raises(ValueError, match="state shape"):
        f(*a[:5], a[5][:1])
    with pytest.raises(ValueError, match="in place"):
        f(*a[:5], a[5].double())
    with pytest.raises(ValueError, match="in place"):
        f(*a[:5], a[5].transpose(2, 3))
    with pytest.raises(ValueError, match="share a dtype"):
        f(a[0].half(), *a[1:])
    with pytest.raises(NotImplementedError):
        f(*[t.float() for t in a[:3]], *a[3:])
    with pytest.raises(ValueError, match="g_activation"):
        f(*a[:4], None, a[5], g_activation="logsigmoid")
    with pytest.raises(TypeError):
        f(*a[:5], None)
    with pytest.raises(NotImplementedError, match="backward"):
        f(*a[:5], a[5].requires_grad_())


@pytest.fixture(scope="module")
def lib():
    from gdn_b200 import _build, _lib
    _build.build()
    return _lib.load()


def attn_struct(**kw):
    from gdn_b200 import _lib
    a = _lib.WindowAttnArgs()
    a.abi_version, a.dtype = _lib.ABI_VERSION, _lib.DTYPE_BF16
    a.B, a.T, a.S, a.H, a.HK, a.D, a.window, a.sinks, a.scale = 2, 4, 8, 4, 2, 64, 4, 1, 1.0
    for n in ("q", "k", "v", "o"):
        setattr(a, n, 0x10000)  # never dereferenced: a check fails or no device is found first
        setattr(a, n + "_stride", (8 * 256, 256, 64))
    for key, val in kw.items():
        setattr(a, key, val)
    return a


@pytest.mark.parametrize("field,value,expected", [
    ("abi_version", 1, 1), ("B", 0, 1), ("T", 9, 1), ("H", 3, 1), ("window", 0, 1), ("sinks", -1, 1), ("dtype", 0, 2),
    ("dtype", 9, 1), ("D", 96, 2), ("scale", 0.0, 1), ("scale", float("inf"), 1), ("q", None, 1), ("k", 0x10008, 3),
    ("k_stride", (8 * 256, 256, 60), 3), ("o_stride", (0, 256, 64), 3), ("B", 70000, 2), ("lengths", 0x10002, 3),
])
def test_window_attn_entry_rejects(lib, field, value, expected):
    assert lib.gdn_window_attn_sm100(ctypes.byref(attn_struct(**{field: value})), None) == expected
    assert lib.gdn_window_attn_sm100(None, None) == 1


def step_struct(**kw):
    from gdn_b200 import _lib
    a = _lib.WindowStepArgs()
    a.abi_version, a.dtype = _lib.ABI_VERSION, _lib.DTYPE_BF16
    a.B, a.H, a.HK, a.D, a.capacity, a.window, a.sinks, a.scale = 2, 4, 2, 64, 16, 8, 4, 1.0
    for n in ("q", "k", "v", "o"):
        setattr(a, n, 0x10000)
        setattr(a, n + "_stride", (256, 64))
    for n in ("k", "v"):
        setattr(a, n + "_cache", 0x10000)
        setattr(a, n + "c_stride", (16 * 128, 128, 64))
    a.positions = 0x10000
    for key, val in kw.items():
        setattr(a, key, val)
    return a


@pytest.mark.parametrize("field,value,expected", [
    ("abi_version", 1, 1), ("H", 5, 1), ("capacity", 11, 1), ("window", 0, 1), ("dtype", 0, 2), ("D", 32, 2),
    ("scale", -1.0, 1), ("positions", None, 1), ("positions", 0x10001, 3), ("k_cache", None, 1),
    ("kc_stride", (16 * 128, 4, 64), 3), ("q_stride", (-256, 64), 3),
])
def test_window_step_entry_rejects(lib, field, value, expected):
    assert lib.gdn_window_step_sm100(ctypes.byref(step_struct(**{field: value})), None) == expected
    assert lib.gdn_window_step_sm100(None, None) == 1


def gdn_struct(**kw):
    from gdn_b200 import _lib
    a = _lib.StepArgs()
    a.abi_version, a.in_dtype, a.out_dtype = _lib.ABI_VERSION, _lib.DTYPE_BF16, _lib.DTYPE_BF16
    a.B, a.H, a.K, a.V, a.scale = 2, 4, 128, 128, 1.0
    for n in ("q", "k", "v", "beta", "g", "o"):
        setattr(a, n, 0x10000)
        setattr(a, n + "_stride", (512, 128))
    a.state = 0x10000
    for key, val in kw.items():
        setattr(a, key, val)
    return a


@pytest.mark.parametrize("field,value,expected", [
    ("abi_version", 1, 1), ("B", 0, 1), ("K", 64, 2), ("V", 64, 2), ("in_dtype", 0, 2), ("out_dtype", 5, 1),
    ("flags", 8, 1), ("scale", float("nan"), 1), ("state", None, 1), ("state", 0x10004, 3), ("beta", None, 1),
    ("k", 0x10002, 3), ("q_stride", (512, 126), 3), ("o_stride", (-512, 128), 1),
])
def test_gdn_step_entry_rejects(lib, field, value, expected):
    assert lib.gdn_step_sm100(ctypes.byref(gdn_struct(**{field: value})), None) == expected
    assert lib.gdn_step_sm100(None, None) == 1


def test_packed_argument_formats_match_the_structs():
    """The struct formats that the calls pack have the C structs' sizes and field offsets."""
    from gdn_b200 import _lib
    for fmt, cls in ((_lib.GATED_SCAN_ARGS, _lib.GatedScanArgs), (_lib.WINDOW_ATTN_ARGS, _lib.WindowAttnArgs),
                     (_lib.WINDOW_STEP_ARGS, _lib.WindowStepArgs), (_lib.STEP_ARGS, _lib.StepArgs)):
        assert fmt.size == ctypes.sizeof(cls)
        n = sum(f[1]._length_ if hasattr(f[1], "_length_") else 1 for f in cls._fields_)
        vals = list(range(1, n + 1))
        back = cls.from_buffer_copy(fmt.pack(*vals))
        flat = []
        for name, _ in cls._fields_:
            x = getattr(back, name)
            flat += list(x) if hasattr(x, "__len__") else [x]
        assert flat == vals
