"""Window attention without a GPU: the descriptor's layout and what the functions and C entries refuse."""
import ctypes
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

from densecore_amd import _lib, functional  # noqa: E402

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
P = ctypes.c_void_p(4096)  # never dereferenced: every call here is refused before a launch


def test_descriptor_layout_matches_header(tmp_path):
    fields = [n for n, _ in _lib.WindowDesc._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "dc_window.h"\nint main(void){'
                   'printf("%zu\\n", sizeof(dc_window_desc));'
                   + "".join(f'printf("%zu\\n", offsetof(dc_window_desc, {n}));' for n in fields)
                   + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", INCLUDE, str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [ctypes.sizeof(_lib.WindowDesc)] + [getattr(_lib.WindowDesc, n).offset for n in fields]


@pytest.mark.parametrize("args,kw,error", [
    ((0,), {}, ValueError), ((-5,), {}, ValueError), ((4, -1), {}, ValueError), ((4,), dict(offset=-1), ValueError),
    ((2.0,), {}, TypeError), ((True,), {}, TypeError), ((4, 1.5), {}, TypeError), ((4,), dict(offset=0.0), TypeError),
    ((4,), dict(scale="x"), TypeError), ((4,), dict(scale=float("nan")), ValueError),
    ((4,), dict(scale=float("inf")), ValueError), ((4,), {}, ValueError),  # the last: not on the GPU
])
def test_functions_refuse(args, kw, error):
    x = torch.zeros(1, 2, 3, 8)
    with pytest.raises(error):
        functional.window_attention(x, x, x, *args, **kw)
    with pytest.raises(TypeError):
        functional.window_attention(x, x, x.numpy(), 4)
    with pytest.raises(TypeError):
        functional.window_decode(x, x, x, 4, lengths=[3])


def _desc(**kw):
    d = dict(batch=1, heads=4, kv_heads=2, q_len=1, kv_len=9, head_dim=8, offset=0, window=4, sinks=1, dtype=0,
             has_scale=0, scale=0.0)
    d.update(kw)
    r = _lib.WindowDesc()
    for n, v in d.items():
        setattr(r, n, v)
    return r


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), _lib.DC_INVALID_ARGUMENT), (dict(kv_heads=0), _lib.DC_INVALID_ARGUMENT),
    (dict(kv_heads=3), _lib.DC_INVALID_ARGUMENT), (dict(dtype=5), _lib.DC_INVALID_ARGUMENT),
    (dict(window=0), _lib.DC_INVALID_ARGUMENT), (dict(sinks=-1), _lib.DC_INVALID_ARGUMENT),
    (dict(offset=-1), _lib.DC_INVALID_ARGUMENT), (dict(has_scale=1, scale=float("nan")), _lib.DC_INVALID_ARGUMENT),
    (dict(has_scale=1, scale=1e300), _lib.DC_INVALID_ARGUMENT), (dict(head_dim=257), _lib.DC_UNSUPPORTED),
    (dict(kv_len=2 ** 31), _lib.DC_UNSUPPORTED), (dict(batch=2 ** 29, heads=8), _lib.DC_UNSUPPORTED),
])
def test_c_entries_refuse(kw, status):
    L, d = _lib.lib(), _desc(**kw)
    assert L.dc_window_fwd(d, P, P, P, P, None, P, None, 0, None) == status
    assert L.dc_window_bwd(d, *[P] * 11, 1 << 40, None) == status
    assert L.dc_window_decode(d, P, P, P, None, 0, P, P, P, 1 << 40, None) == status
    assert L.dc_last_error()


def test_c_entries_refuse_pointers_and_workspaces():
    L, bad = _lib.lib(), _lib.DC_INVALID_ARGUMENT
    assert L.dc_window_fwd(None, P, P, P, P, None, P, None, 0, None) == bad
    assert L.dc_window_fwd(_desc(), P, None, P, P, None, P, None, 0, None) == bad
    assert L.dc_window_fwd(_desc(), P, P, P, P, None, None, None, 0, None) == bad
    assert L.dc_window_fwd(_desc(head_dim=129), P, P, P, P, None, P, None, 0, None) == _lib.DC_UNSUPPORTED
    size = L.dc_window_bwd_workspace_size(_desc())
    assert size > 0
    assert L.dc_window_bwd(_desc(), *[P] * 10, None, size, None) == bad
    assert L.dc_window_bwd(_desc(), *[P] * 11, size - 1, None) == bad
    assert L.dc_window_decode(_desc(q_len=2), P, P, P, None, 0, P, P, P, 1 << 40, None) == bad
    assert L.dc_window_decode(_desc(), P, P, P, P, 2, P, P, P, 1 << 40, None) == bad
    assert L.dc_window_decode(_desc(), P, P, P, None, 8, P, P, P, 1 << 40, None) == bad
    # Nothing to compute: no pointer is looked at.
    assert L.dc_window_fwd(_desc(batch=0), *[None] * 7, 0, None) == _lib.DC_OK
    assert L.dc_window_decode(_desc(batch=0), None, None, None, None, 0, None, None, None, 0, None) == _lib.DC_OK


def test_numbers_past_the_kernels_range_are_refused():
    """A scale that is finite until it is taken in base 2, packed rows past 2^30."""
    L = _lib.lib()
    assert L.dc_window_fwd(_desc(has_scale=1, scale=3e38), P, P, P, P, None, P, None, 0, None) == _lib.DC_INVALID_ARGUMENT
    many = _desc(heads=2 ** 28, kv_heads=1, q_len=32, head_dim=1)
    assert L.dc_window_fwd(many, P, P, P, P, None, P, None, 0, None) == _lib.DC_UNSUPPORTED
    assert L.dc_window_bwd(many, *[P] * 11, 1 << 40, None) == _lib.DC_UNSUPPORTED
