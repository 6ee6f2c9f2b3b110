"""C ABI of libartemis_ops.so without a GPU: the header's symbols are exported and bound, constants agree, and the
host-side validation refuses before any HIP call."""
import ctypes
import math
import os
import re

import pytest

from artemis_amd import _lib, build

HEADER = os.path.join(build.INCLUDE, "artemis_ops.h")


def header():
    return open(HEADER).read()


def error():
    return _lib.load_ops().artemis_ops_last_error().decode()


def test_every_declared_symbol_is_exported_and_bound():
    text = re.sub(r"/\*.*?\*/", "", header(), flags=re.S)
    names = sorted(set(re.findall(r"\b(artemis_ops_\w+)\s*\(", text)))
    lib = ctypes.CDLL(build.OPS_LIB_PATH)
    assert all(hasattr(lib, n) for n in names)
    assert sorted(_lib.OPS_SIGNATURES) == names


def test_constants_and_structures():
    get = lambda n: int(re.search(r"#define ARTEMIS_OPS_%s (\d+)" % n, header()).group(1))
    assert (get("F32"), get("BF16"), get("F16")) == (_lib.OPS_F32, _lib.OPS_BF16, _lib.OPS_F16)
    assert get("ABI_VERSION") == _lib.OPS_ABI_VERSION
    assert _lib.load_ops().artemis_ops_version().decode().startswith("artemis_ops abi %d gfx950" % _lib.OPS_ABI_VERSION)
    for name, struct in (("artemis_ops_window", _lib.WindowDesc), ("artemis_ops_tensor", _lib.TensorDesc)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, header(), re.S).group(1)
        fields = [f for decl in body.split(";") for f in re.findall(r"\*?(\w+)(?=\s*(?:,|$))", decl.strip())]
        assert fields == [f[0] for f in struct._fields_]


def test_layer_norm_validation():
    lib = _lib.load_ops()
    f, b = lib.artemis_ops_layer_norm_forward, lib.artemis_ops_layer_norm_backward
    assert f(None, None, None, None, None, None, 4, 8, 1e-5, 0, None) == 1 and "NULL" in error()
    assert f(16, None, None, 16, 16, None, 4, 8, 1e-5, 0, None) == 1 and "together" in error()
    assert f(16, None, None, 16, None, None, 4, 8, -1.0, 0, None) == 1 and "eps" in error()
    assert f(16, None, None, 16, None, None, 4, 8, math.nan, 0, None) == 1
    assert f(16, None, None, 16, None, None, 4, 8, 1e-5, 3, None) == 1 and "dtype" in error()
    assert f(16, None, None, 16, None, None, -1, 8, 1e-5, 0, None) == 1
    assert f(16, None, None, 16, None, None, 1 << 31, 8, 1e-5, 0, None) == 1
    assert f(16, None, None, 16, None, None, 4, 0, 1e-5, 0, None) == 1
    assert f(None, None, None, None, None, None, 0, 8, 1e-5, 0, None) == 0
    assert b(16, 16, None, 16, 16, 16, 16, None, 4, 8, 0, None, 0, None) == 1 and "workspace" in error()
    need = lib.artemis_ops_layer_norm_workspace_bytes(4, 8, 0)
    assert need > 0
    assert b(16, 16, None, 16, 16, 16, 16, None, 4, 8, 0, 16, need - 1, None) == 1 and "workspace" in error()
    assert b(16, 16, None, None, None, 16, None, None, 4, 8, 0, None, 0, None) == 1 and "NULL" in error()
    assert b(None, None, None, None, None, None, None, None, 4, 8, 0, None, 0, None) == 0   # nothing asked for


def desc(**kw):
    d = dict(B=1, D=2, H=8, W=8, heads=2, head_dim=32, wd=1, wh=8, ww=8, shift_d=0, shift_h=0, shift_w=0, label_maps=0,
             dtype=0, scale=0.2, outside=-100.0)
    d.update(kw)
    return _lib.WindowDesc(*[d[n] for n, _ in _lib.WindowDesc._fields_])


@pytest.mark.parametrize("kw,needle", [
    (dict(B=-1), "negative"), (dict(dtype=7), "dtype"), (dict(heads=0), "heads"), (dict(heads=2000), "heads"),
    (dict(head_dim=30), "head_dim"), (dict(head_dim=132), "head_dim"), (dict(wh=0), "window"),
    (dict(H=128, W=64, wh=128, ww=64), "window"), (dict(wh=5), "multiple"), (dict(shift_h=8), "shift"),
    (dict(shift_w=-1), "shift"), (dict(label_maps=3), "label_maps"), (dict(outside=1.0), "outside"),
    (dict(outside=math.nan), "outside"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(B=1 << 20, H=64, W=64), "too many"), (dict(B=1 << 14, H=16, W=16, wh=16, ww=16, heads=1024), "too many")])
def test_window_validation(kw, needle):
    lib = _lib.load_ops()
    w = ctypes.byref(desc(**kw))
    assert lib.artemis_ops_window_attention_forward(w, 16, None, None, 16, None, None, 0, None) == 1
    assert needle in error()
    assert lib.artemis_ops_window_attention_backward(w, 16, None, None, 16, None, 16, 16, None, None, 0, None) == 1
    assert needle in error()
    assert lib.artemis_ops_window_attention_workspace_bytes(w, 1, 1) == 0
    assert lib.artemis_ops_window_attention_lse_count(w) == 0


def test_window_pointers_and_workspace():
    lib = _lib.load_ops()
    f, b = lib.artemis_ops_window_attention_forward, lib.artemis_ops_window_attention_backward
    w = ctypes.byref(desc())
    assert f(w, None, None, None, 16, None, None, 0, None) == 1 and "NULL" in error()
    assert f(w, 16, None, 16, 16, None, None, 0, None) == 1 and "label" in error()
    assert f(w, 20, None, None, 16, None, None, 0, None) == 1 and "aligned" in error()
    assert f(ctypes.byref(desc(label_maps=1)), 16, None, None, 16, None, None, 0, None) == 1 and "label" in error()
    assert b(w, 16, 16, None, None, None, 16, 16, 16, None, 0, None) == 1 and "workspace" in error()
    long = ctypes.byref(desc(H=16, W=16, wh=16, ww=16))
    assert lib.artemis_ops_window_attention_lse_count(w) == 0
    assert lib.artemis_ops_window_attention_lse_count(long) == 2 * 2 * 256   # whole tiles of 64 tokens
    assert f(long, 16, 16, None, 16, None, None, 0, None) == 1 and "workspace" in error()
    assert b(long, 16, None, None, 16, None, 16, 16, None, None, 0, None) == 1 and "NULL" in error()
    assert f(ctypes.byref(desc(B=0)), None, None, None, None, None, None, 0, None) == 0


def test_adamw_validation():
    lib = _lib.load_ops()
    one = (_lib.TensorDesc * 1)(_lib.TensorDesc(16, 16, 16, 16, 16, 16, 10))

    def call(array=one, n=1, dtype=0, bits=32, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1):
        return lib.artemis_ops_adamw(array, n, dtype, bits, lr, b1, b2, eps, wd, step, 0, None)

    for kw in (dict(dtype=5), dict(bits=16), dict(lr=-1.0), dict(lr=math.nan), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0),
               dict(wd=-1.0), dict(step=0), dict(n=-1), dict(array=None)):
        assert call(**kw) == 1, kw
    assert call(n=0, array=None) == 0
    hole = (_lib.TensorDesc * 1)(_lib.TensorDesc(16, None, 16, 16, None, None, 10))
    assert call(array=hole) == 1 and "NULL" in error()
    hole = (_lib.TensorDesc * 1)(_lib.TensorDesc(16, 16, 16, 16, None, 16, 10))
    assert call(array=hole, bits=8) == 1 and "NULL" in error()
    assert lib.artemis_ops_moments_from_8bit(hole, 1, 1, None) == 1 and "NULL" in error()
    big = (_lib.TensorDesc * 1)(_lib.TensorDesc(16, 16, 16, 16, 16, 16, (1 << 34) + 1))
    assert call(array=big) == 1 and "elements" in error()
    two = (_lib.TensorDesc * 2)(*[_lib.TensorDesc(16, 16, 16, 16, 16, 16, 1 << 32)] * 2)
    assert call(array=two, n=2, bits=8) == 1 and "2^32" in error()
    empty = (_lib.TensorDesc * 1)(_lib.TensorDesc(None, None, None, None, None, None, 0))
    assert call(array=empty) == 0


def test_missing_library_fails_loudly(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "OPS_HOST_PATH", str(tmp_path / "nope.so"))
    monkeypatch.setattr(_lib, "_ops_host", None)
    with pytest.raises(_lib.SynthLibraryError, match="no fallback"):
        _lib.load_ops_host()
    monkeypatch.setattr(build, "OPS_LIB_PATH", str(tmp_path / "nope.so"))
    monkeypatch.setattr(_lib, "_ops", None)
    with pytest.raises(_lib.SynthLibraryError, match="no fallback"):
        _lib.load_ops_host()
