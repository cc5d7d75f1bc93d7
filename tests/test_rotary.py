"""Rotary positions without a GPU: frequencies, and what the entry points refuse."""
import math

import pytest

torch = pytest.importorskip("torch")

import jaxmodules_amd as jm


def test_plain_frequencies():
    f, scale = jm.rotary_frequencies(8, 100.0)
    assert f.dtype == torch.float64 and scale == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)


def test_linear_divides_every_pair():
    f, scale = jm.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.equal(f, jm.rotary_frequencies(64)[0] / 4) and scale == 1.0


def test_ntk_keeps_the_fastest_and_divides_the_slowest():
    f, g = jm.rotary_frequencies(64, scaling="ntk", factor=4.0)[0], jm.rotary_frequencies(64)[0]
    assert f[0] == g[0] == 1.0
    assert abs(f[-1] * 4 / g[-1] - 1) < 1e-12


def test_parts():
    f, scale = jm.rotary_frequencies(128, scaling="parts", factor=8.0, context=4096)
    g = jm.rotary_frequencies(128)[0]
    turns = 4096 * g / (2 * math.pi)
    assert torch.equal(f[turns > 32], g[turns > 32])
    assert torch.allclose(f[turns < 1], g[turns < 1] / 8, rtol=1e-15)
    assert (f[1:] < f[:-1]).all() and (f <= g).all() and (f >= g / 8).all()
    assert scale == 0.1 * math.log(8.0) + 1.0
    assert jm.rotary_frequencies(128, scaling="parts", factor=1.0, context=64)[1] == 1.0


@pytest.mark.parametrize("kw", [dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=-1.0, scaling="linear"),
                                dict(dim=8, scaling="cubic"), dict(dim=8, scaling="parts"), dict(dim=2, scaling="ntk"),
                                dict(dim=8, scaling="parts", context=64, fast=1.0, slow=2.0)])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        jm.rotary_frequencies(**kw)


def _x(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


F = torch.ones(4, dtype=torch.float64)

REFUSED = {
    "cpu tensors": (RuntimeError, dict(q=_x(1, 2, 3, 8))),
    "two dimensions": (ValueError, dict(q=_x(2, 8))),
    "mixed ranks": (ValueError, dict(q=_x(1, 2, 3, 8), k=_x(2, 3, 8))),
    "lengths": (ValueError, dict(q=_x(1, 2, 3, 8), k=_x(1, 3, 3, 8))),
    "head dimensions": (ValueError, dict(q=_x(1, 2, 3, 8), k=_x(1, 2, 3, 16))),
    "dtypes": (TypeError, dict(q=_x(1, 2, 3, 8), k=_x(1, 2, 3, 8, dtype=torch.float16))),
    "float64": (TypeError, dict(q=_x(1, 2, 3, 8, dtype=torch.float64))),
    "wide heads": (NotImplementedError, dict(q=_x(1, 2, 3, 520))),
    "layout": (ValueError, dict(q=_x(1, 2, 3, 8), layout="quarter")),
    "scale": (ValueError, dict(q=_x(1, 2, 3, 8), scale=math.inf)),
    "float32 frequencies": (TypeError, dict(q=_x(1, 2, 3, 8), inv_freq=F.float())),
    "too many pairs": (ValueError, dict(q=_x(1, 2, 3, 6))),
    "float positions": (TypeError, dict(q=_x(1, 2, 3, 8), positions=torch.zeros(2))),
    "positions' shape": (ValueError, dict(q=_x(2, 2, 3, 8), positions=torch.zeros((1, 2), dtype=torch.int32))),
}


@pytest.mark.parametrize("what", REFUSED)
def test_rotary_refuses(what):
    error, kw = REFUSED[what]
    kw = {"inv_freq": F, **kw}
    with pytest.raises(error):
        jm.rotary(kw.pop("q"), kw.pop("k", None), **kw)


def test_norm_refuses():
    q = _x(1, 2, 3, 8)
    with pytest.raises(ValueError, match="weights"):
        jm.norm_rotary(q, None, _x(4))
    with pytest.raises(ValueError, match="eps"):
        jm.norm_rotary(q, eps=-1.0)
    with pytest.raises(RuntimeError, match="GPU only"):
        jm.norm_rotary(q)


def test_c_entries_refuse():
    """The library's own checks, on the host: nothing is launched."""
    import ctypes

    from jaxmodules_amd import _lib

    lib = _lib.load()

    def call(norm=0, bwd=False, **kw):
        p = _lib.MattnRotary(B=1, L=2, D=64, dim=64, n=1, dtype=_lib.MATTN_BF16, norm=norm, inv_freq=64, scale=1.0)
        p.H[0] = 2
        p.x[0] = p.y[0] = p.g[0] = 1 << 20
        for k, v in kw.items():
            if isinstance(v, tuple):
                getattr(p, k)[v[0]] = v[1]
            else:
                setattr(p, k, v)
        if bwd:
            return lib.mattn_norm_rotary_bwd(ctypes.byref(p), None, None, None, 0, None)
        return lib.mattn_rotary_fwd(ctypes.byref(p), None)

    assert lib.mattn_rotary_fwd(None, None) == -1
    assert call(n=3) == -2 and call(n=2) == -2 and call(B=0) == -2 and call(D=513) == -2
    assert call(dim=63) == -2 and call(dim=66) == -2 and call(layout=2) == -2
    assert call(dtype=5) == -4 and call(pos_bytes=2) == -4
    assert call(inv_freq=None) == -1 and call(pos_bytes=4) == -1 and call(x=(0, None)) == -1
    assert call(norm=1, eps=-1.0) == -2 and call(norm=1, inverse=1) == -2
    assert call(bwd=True, g=(0, None)) == -1 and call(bwd=True) == -1  # no workspace
    p = _lib.MattnRotary()
    assert lib.mattn_norm_rotary_bwd_workspace_bytes(ctypes.byref(p)) == 0
