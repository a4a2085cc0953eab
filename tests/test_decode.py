"""Decoder-side entry points on a machine without a GPU: refusals before any device is touched, and the layout
of the structure that crosses the C ABI."""

import ctypes as C
import math
import shutil
import subprocess
from pathlib import Path

import pytest

from ripvec_b200 import _lib as L

HEADER = Path(__file__).resolve().parents[1] / "include" / "ripvec_b200.h"


def test_null_steps_are_refused():
    lib = L.lib()
    assert lib.rv_step_last_error(None) == b"null step"
    assert lib.rv_step_tokens(None) == 0
    assert lib.rv_step_plan(None, 0, None, None, None, 0, None, None, None, 0, 1, None) == L.RV_E_INVALID
    rows = (None, 0, 0)
    assert lib.rv_step_append(None, None, *rows, *rows, *rows, *rows, None, None, 0, 0, 0, None) == L.RV_E_INVALID
    assert lib.rv_step_attend(None, None, *rows, *rows, None, 1.0, None) == L.RV_E_INVALID
    lib.rv_step_destroy(None)
    assert lib.rv_step_create(0, 8, 2, 128, 16, None) == L.RV_E_INVALID


@pytest.mark.parametrize("shape", [(0, 1, 64, 16), (8, 3, 64, 16), (8, 0, 64, 16), (8, 2, 96, 16), (8, 2, 32, 16),
                                   (8, 2, 128, 8), (8, 2, 128, 48), (8, 2, 128, 512), (2048, 1, 64, 16)])
def test_step_shapes_are_refused(shape):
    h = C.c_void_p(1)
    assert L.lib().rv_step_create(0, *shape, C.byref(h)) == L.RV_E_INVALID
    assert not h.value


def norm(act=L.RV_DTYPE_BF16, x=16, xs=64, r=16, rs=64, w=16, ro=16, ros=64, out=16, os=64, odt=None, scales=None,
         group=0, rows=2, hidden=64, eps=1e-5):
    return L.lib().rv_rms_norm(act, x, xs, r, rs, w, ro, ros, out, os, act if odt is None else odt, scales, group, rows,
                               hidden, eps, None)


@pytest.mark.parametrize("kw", [dict(act=L.RV_DTYPE_F32), dict(odt=L.RV_DTYPE_F16), dict(x=None), dict(w=None), dict(out=None),
                                dict(rows=-1), dict(hidden=0), dict(hidden=65537), dict(eps=-1.0), dict(eps=math.nan),
                                dict(eps=math.inf), dict(xs=-1), dict(rs=-1), dict(os=63), dict(ros=63), dict(group=32),
                                dict(odt=L.RV_DTYPE_E4M3), dict(odt=L.RV_DTYPE_E4M3, scales=16, group=48),
                                dict(odt=L.RV_DTYPE_E4M3, scales=16, group=128), dict(scales=16)])
def test_norm_arguments_are_refused(kw):
    assert norm(**kw) == L.RV_E_INVALID


def test_norm_of_no_rows_needs_no_device():
    assert norm(rows=0) == L.RV_OK


def test_python_checks_before_the_library():
    import torch

    from ripvec_b200.decode import PagedCache, rms_norm

    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):  # not on a CUDA device
        PagedCache(pool, pool)
    with pytest.raises(ValueError):
        rms_norm(torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(64))
    with pytest.raises(ValueError):
        rms_norm(torch.zeros(2, 64), torch.ones(64))


def test_cache_layout_matches_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "layout.c"
    fields = [f for f, _ in L.KvCache._fields_]
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "ripvec_b200.h"\nint main(void){printf("%zu", sizeof(rv_kv_cache));'
                   + "".join(f'printf(" %zu", offsetof(rv_kv_cache, {f}));' for f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run([cc, f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    got = list(map(int, subprocess.run([str(exe)], capture_output=True, text=True).stdout.split()))
    assert got == [C.sizeof(L.KvCache)] + [getattr(L.KvCache, f).offset for f in fields]
