"""Rotation and norm without a GPU: the frequencies against their formulas, the descriptor's layout,
and what the functions and the C entries refuse."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from densecore_amd import _lib, functional  # noqa: E402

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")


def test_descriptor_layout_matches_header(tmp_path):
    fields = [n for n, _ in _lib.RotaryDesc._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "dc_rotary.h"\nint main(void){'
                   'printf("%zu\\n", sizeof(dc_rotary_desc));'
                   + "".join(f'printf("%zu\\n", offsetof(dc_rotary_desc, {n}));' for n in fields)
                   + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", INCLUDE, str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()))
    assert got == [ctypes.sizeof(_lib.RotaryDesc)] + [getattr(_lib.RotaryDesc, n).offset for n in fields]


def test_plain_linear_and_ntk_frequencies():
    R, base, s = 64, 10000.0, 8.0
    i = np.arange(R // 2)
    plain, m = functional.rotary_frequencies(R, base)
    assert m == 1.0 and plain.dtype == torch.float64
    np.testing.assert_allclose(plain.numpy(), base ** (-2 * i / R), rtol=1e-14)
    linear, _ = functional.rotary_frequencies(R, base, "linear", s)
    np.testing.assert_allclose(linear.numpy(), plain.numpy() / s, rtol=1e-14)
    ntk, _ = functional.rotary_frequencies(R, base, "ntk", s)
    # The fastest pair is kept, the slowest divided by the factor.
    np.testing.assert_allclose([ntk[0], ntk[-1]], [1.0, plain[-1] / s], rtol=1e-13)
    assert functional.rotary_frequencies(0)[0].shape == (0,)
    assert functional.rotary_frequencies(2, base, "ntk", s)[0].tolist() == [1.0]


def test_yarn_frequencies():
    R, base, s, trained = 128, 10000.0, 4.0, 2048
    plain = functional.rotary_frequencies(R, base)[0].numpy()
    yarn, m = functional.rotary_frequencies(R, base, "yarn", s, trained)
    yarn = yarn.numpy()
    assert m == pytest.approx(0.1 * math.log(s) + 1)
    turns = trained * plain / (2 * math.pi)
    # One pair of slack: the ramp starts and ends at whole pairs.
    step = base ** (2 / R)
    assert np.allclose(yarn[turns > 32 * step], plain[turns > 32 * step], rtol=1e-14)
    assert np.allclose(yarn[turns < 1 / step], plain[turns < 1 / step] / s, rtol=1e-14)
    assert (np.diff(plain / yarn) >= -1e-12).all()


@pytest.mark.parametrize("kw", [
    dict(rotary_dim=3), dict(rotary_dim=-2), dict(rotary_dim=4, base=1.0), dict(rotary_dim=4, factor=0.5),
    dict(rotary_dim=4, scaling="other"), dict(rotary_dim=4, scaling="yarn", factor=2.0),
    dict(rotary_dim=4, scaling="yarn", original_length=64, beta_fast=1.0, beta_slow=2.0),
])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        functional.rotary_frequencies(**kw)


def test_functions_refuse():
    x, f = torch.zeros(1, 2, 3, 4), torch.zeros(2, dtype=torch.float64)
    with pytest.raises(TypeError):
        functional.rotary_embedding(x.numpy(), x, f)
    with pytest.raises(TypeError):
        functional.rotary_embedding(x, x, f, offset=1.5)
    with pytest.raises(TypeError):
        functional.rotary_embedding(x, x, f, interleaved=1)
    with pytest.raises(TypeError):
        functional.qk_norm_rotary(x, x, None, None, f, eps="1")
    with pytest.raises(ValueError, match="negative"):
        functional.qk_norm_rotary(x, x, None, None, f, eps=-1.0)
    with pytest.raises(ValueError, match="GPU"):
        functional.rotary_embedding(x, x, f)
    with pytest.raises(ValueError, match=r"\(B, H, L, E\)"):
        functional.rotary_embedding(x[0], x[0], f)
    with pytest.raises(ValueError, match="do not match"):
        functional.rotary_embedding(x, x[:, :, :2], f)


def _desc(**kw):
    d = dict(batch=1, heads=2, kv_heads=2, q_len=3, head_dim=8, rotary_dim=8, dtype=0, weight_dtype=0,
             interleaved=0, norm=0, pos_bytes=0, reserved=0, offset=0, pos_stride_b=0, pos_stride_l=0,
             magnitude=1.0, eps=0.0)
    d.update(kw)
    r = _lib.RotaryDesc()
    for n, v in d.items():
        setattr(r, n, v)
    return r


P = ctypes.c_void_p(4096)  # never dereferenced: every call here is refused before a launch


@pytest.mark.parametrize("kw,status", [
    (dict(batch=-1), _lib.DC_INVALID_ARGUMENT), (dict(rotary_dim=3), _lib.DC_INVALID_ARGUMENT),
    (dict(rotary_dim=10), _lib.DC_INVALID_ARGUMENT), (dict(dtype=7), _lib.DC_INVALID_ARGUMENT),
    (dict(weight_dtype=2), _lib.DC_INVALID_ARGUMENT), (dict(pos_bytes=2), _lib.DC_INVALID_ARGUMENT),
    (dict(reserved=1), _lib.DC_INVALID_ARGUMENT), (dict(head_dim=513), _lib.DC_UNSUPPORTED),
    (dict(q_len=2 ** 31), _lib.DC_UNSUPPORTED),
])
def test_c_entries_refuse(kw, status):
    L, d = _lib.lib(), _desc(**kw)
    assert L.dc_rotary_fwd(d, P, P, None, None, P, P, P, P, None) == status
    assert L.dc_last_error()
    assert L.dc_rotary_bwd(d, P, P, P, P, None, None, P, P, P, P, None, None, None, 0, None) == status


def test_c_entries_refuse_pointers():
    L, bad = _lib.lib(), _lib.DC_INVALID_ARGUMENT
    assert L.dc_rotary_fwd(None, P, P, None, None, P, P, P, P, None) == bad
    assert L.dc_rotary_fwd(_desc(), None, P, None, None, P, P, P, P, None) == bad
    assert L.dc_rotary_fwd(_desc(), P, P, None, None, None, P, P, P, None) == bad
    assert L.dc_rotary_fwd(_desc(pos_bytes=8), P, P, None, None, P, None, P, P, None) == bad
    assert L.dc_rotary_fwd(_desc(), P, P, P, None, P, P, P, P, None) == bad  # a weight without norm
    n = _desc(norm=1)
    size = L.dc_rotary_bwd_workspace_size(n)
    assert size > 0 and L.dc_rotary_bwd_workspace_size(_desc()) == 0
    assert L.dc_rotary_bwd(n, P, P, P, P, P, P, P, P, P, P, P, P, P, size - 1, None) == bad
    assert L.dc_rotary_bwd(n, P, P, None, P, P, P, P, P, P, P, P, P, P, size, None) == bad
    # No tokens: nothing to do.
    assert L.dc_rotary_fwd(_desc(batch=0), None, None, None, None, None, None, None, None, None) == _lib.DC_OK


@pytest.mark.parametrize("offset", [2 ** 53 + 1, -2 ** 53 - 1, 2 ** 62])
def test_offsets_that_float64_does_not_hold_are_refused(offset):
    L, d = _lib.lib(), _desc(offset=offset)
    assert L.dc_rotary_fwd(d, P, P, None, None, P, P, P, P, None) == _lib.DC_UNSUPPORTED
    assert L.dc_rotary_bwd(d, P, P, P, P, None, None, P, P, P, P, None, None, None, 0, None) == _lib.DC_UNSUPPORTED


def test_frequencies_have_no_gradient():
    x, f = torch.zeros(1, 2, 3, 4), torch.zeros(2, dtype=torch.float64, requires_grad=True)
    with pytest.raises(NotImplementedError, match="gradient"):
        functional.rotary_embedding(x, x, f)
    with pytest.raises(NotImplementedError, match="gradient"):
        functional.qk_norm_rotary(x, x, None, None, f)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        functional.rotary_embedding(x, x, f)
