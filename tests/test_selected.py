"""What block means, block selection and attention over selected blocks refuse (no GPU)."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

import jaxmodules_amd as jm
from jaxmodules_amd import _lib


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


K, Q, M = _t(2, 40, 2, 64), _t(2, 5, 4, 64), _t(2, 3, 2, 64)
I2 = torch.zeros(2, dtype=torch.int32)
BLK = torch.zeros((2, 5, 2, 3), dtype=torch.int32)


@pytest.mark.parametrize("error,args,kw", [
    (RuntimeError, (K, 16), {}), (ValueError, (K, 0), {}), (ValueError, (K, 24), {}), (ValueError, (K, 16.0), {}),
    (ValueError, (K[0], 16), {}), (TypeError, (K.double(), 16), {}), (NotImplementedError, (_t(1, 4, 1, 136), 16), {}),
    (TypeError, (K, 16, I2.long()), {}), (TypeError, (K, 16, I2[:1]), {}), (ValueError, (K, 16), dict(new=1)),
    (ValueError, (K, 16), dict(out=M)), (ValueError, (K, 16), dict(out=M, new=41)), (ValueError, (K, 16), dict(out=M, new=-1)),
    (ValueError, (K, 16), dict(out=_t(2, 4, 2, 64), new=1)), (ValueError, (K, 16), dict(out=M.half(), new=1)),
    (ValueError, (K, 16), dict(out=_t(2, 3, 64, 2).transpose(2, 3), new=1)),
])
def test_means_refuse(error, args, kw):
    with pytest.raises(error):
        jm.block_means(*args, **kw)


@pytest.mark.parametrize("error,args,kw", [
    (RuntimeError, (Q, M, 16, 3), {}), (ValueError, (Q, M, 8, 3), {}), (ValueError, (Q[:1], M, 16, 3), {}),
    (ValueError, (Q[:, :, :3], M, 16, 3), {}), (TypeError, (Q, M.half(), 16, 3), {}), (ValueError, (Q, M[..., :32], 16, 3), {}),
    (ValueError, (Q, M, 16, 0), {}), (ValueError, (Q, M, 16, 1025), {}), (ValueError, (Q, M, 16, 3), dict(first=2, last=2)),
    (ValueError, (Q, M, 16, 3), dict(first=-1)), (ValueError, (Q, M, 16, True), {}), (TypeError, (Q, M, 16, 3), dict(starts=I2.float())),
    (TypeError, (Q, M, 16, 3), dict(lengths=torch.zeros(3, dtype=torch.int32))), (ValueError, (Q, M[:, :, :0], 16, 3), {}),
])
def test_selection_refuses(error, args, kw):
    with pytest.raises(error):
        jm.select_blocks(*args, **kw)


@pytest.mark.parametrize("error,args,kw", [
    (RuntimeError, (Q, K, K, BLK, 16), {}), (ValueError, (Q, K, K, BLK, 15), {}), (TypeError, (Q, K.half(), K, BLK, 16), {}),
    (TypeError, (Q.double(), K, K, BLK, 16), {}), (ValueError, (Q, K, K[:, :30], BLK, 16), {}), (ValueError, (Q[:1], K, K, BLK, 16), {}),
    (ValueError, (Q[:, :, :3], K, K, BLK, 16), {}), (TypeError, (Q, K, K, BLK.long(), 16), {}), (TypeError, (Q, K, K, BLK[:, :4], 16), {}),
    (NotImplementedError, (Q, K, K, torch.zeros((2, 5, 2, 1025), dtype=torch.int32), 16), {}),
    (NotImplementedError, (_t(1, 5, 1, 136), _t(1, 5, 1, 136), _t(1, 5, 1, 136), BLK, 16), {}),
    (ValueError, (Q, K, K, BLK, 16), dict(scale=math.inf)), (ValueError, (Q, K, K, BLK, 16), dict(scale=math.nan)),
    (ValueError, (Q, K, K, BLK, 16), dict(scale=1e39)), (TypeError, (Q, K, K, BLK, 16), dict(lengths=I2.long())),
])
def test_attention_refuses(error, args, kw):
    with pytest.raises(error):
        jm.selected_attention(*args, **kw)


def _struct(**kw):
    p = _lib.MattnSelected(B=2, Lq=100, Lk=100, Hq=4, Hkv=2, D=64, dtype=_lib.MATTN_BF16, block_size=64, count=4,
                           scale=0.125, blocks=64)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return ctypes.byref(p)


def test_c_entries_refuse():
    lib = _lib.load()
    check = lambda **kw: lib.mattn_selected_validate(_struct(**kw))  # noqa: E731
    assert check() == 0 and lib.mattn_selected_validate(None) == -1
    assert check(Hkv=3) == -2 and check(B=0) == -2 and check(block_size=24) == -2 and check(count=1025) == -2
    assert check(D=60) == -3 and check(D=136) == -3 and check(dtype=3) == -4 and check(blocks=None) == -1
    assert check(scale=math.inf) == -2 and check(scale=math.nan) == -2
    assert check(q_stride=(4, 8, 8)) == -5 and check(dv_stride=(-8, 8, 8)) == -5
    assert check(Lq=1 << 30) == -8 and check(Lk=(1 << 31) - 1) == -8
    a = 1 << 20
    fwd = lambda ws, n, q=a, **kw: lib.mattn_selected_fwd(_struct(**kw), q, a, a, a, None, None, None, ws, n, None)  # noqa: E731
    need = lib.mattn_selected_fwd_workspace_bytes(_struct())
    assert need > 0 and fwd(a, need - 1) == -11 and fwd(None, need) == -1 and fwd(a + 16, need) == -5
    assert fwd(a, need, q=None) == -1 and fwd(a, need, q=a + 2) == -5 and fwd(a, need, count=0) == -2
    # a forward for a backward needs all it keeps
    assert lib.mattn_selected_fwd(_struct(), a, a, a, a, None, None, a, a, need, None) == -1
    n = lib.mattn_selected_bwd_workspace_bytes(_struct())
    bwd = lambda n, dk=a: lib.mattn_selected_bwd(_struct(), a, a, a, a, a, a, a, a, n, a, dk, a, None)  # noqa: E731
    assert n > 0 and bwd(n - 1) == -11 and bwd(n, dk=None) == -1 and bwd(n, dk=a + 4) == -5
    s = _lib.MattnSelect(B=1, L=1, nblk=4, Hq=2, Hkv=1, D=64, dtype=0, block_size=16, count=2, first=1, last=1, q=a, means=a, blocks=a)
    n = lib.mattn_select_workspace_bytes(ctypes.byref(s))
    assert n >= 16 and lib.mattn_select_blocks(ctypes.byref(s), None, n, None) == -1 and lib.mattn_select_blocks(ctypes.byref(s), a, n - 1, None) == -11
    for field, bad, code in (("first", 2, -2), ("D", 12, -3), ("dtype", 9, -4), ("means", None, -1), ("q", a + 2, -5), ("Hkv", 3, -2)):
        was = getattr(s, field)
        setattr(s, field, bad)
        assert lib.mattn_select_blocks(ctypes.byref(s), a, 1 << 20, None) == code, field
        setattr(s, field, was)
    m = _lib.MattnMeans(B=1, L=4, H=1, D=8, dtype=0, block_size=16, k=a, means=a)
    for field, bad, code in (("L", 0, -2), ("new_keys", 5, -2), ("dtype", 4, -4), ("k", None, -1), ("B", 65536, -8)):
        was = getattr(m, field)
        setattr(m, field, bad)
        assert lib.mattn_block_means(ctypes.byref(m), None) == code, field
        setattr(m, field, was)


def test_a_scale_that_is_no_float32_times_log2_e_is_refused():
    with pytest.raises(ValueError, match="scale"):
        jm.selected_attention(Q, K, K, BLK, 16, scale=3e38)
    assert _lib.load().mattn_selected_validate(_struct(scale=3e38)) == -2
    assert _lib.load().mattn_selected_validate(_struct(scale=-2e38)) == 0


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess

    structs = {"mattn_rotary": _lib.MattnRotary, "mattn_means": _lib.MattnMeans, "mattn_select": _lib.MattnSelect,
               "mattn_selected": _lib.MattnSelected}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mattn.h"', "int main(void){"]
    for c, cls in structs.items():
        lines.append(f'printf("{c} sizeof %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "p.c", tmp_path / "p"
    src.write_text("\n".join([*lines, "return 0;}"]))
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-I", inc, str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        c, f, v = line.split()
        cls = structs[c]
        assert int(v) == (ctypes.sizeof(cls) if f == "sizeof" else getattr(cls, f).offset), (c, f)
