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


RECORDS = {
    "append": ("rv_step_append_args", "_append_args",
               "cache q q_token_stride q_head_stride k k_token_stride k_head_stride v v_token_stride v_head_stride q_out "
               "q_out_token_stride q_out_head_stride cos sin positions rot interleaved stream"),
    "attend": ("rv_step_attend_args", "_attend_args",
               "cache q q_token_stride q_head_stride out out_token_stride out_head_stride lse scale stream"),
    "norm": ("rv_rms_norm_args", "_norm_args",
             "x x_stride residual residual_stride weight residual_out residual_out_stride out out_stride scales rows hidden "
             "act_dtype out_dtype group eps device stream"),
}


@pytest.mark.parametrize("kind", RECORDS)
def test_records_match_header(tmp_path, kind):
    """What Python packs is what C reads, field by field."""
    import ripvec_b200.decode as D

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    record, pack, fields = RECORDS[kind]
    fields = fields.split()
    data = getattr(D, pack)(*range(1, len(fields) + 1))
    src = tmp_path / "record.c"
    src.write_text('#include <stdio.h>\n#include "ripvec_b200.h"\n'
                   f'int main(void){{{record} r; if (fread(&r, 1, sizeof r, stdin) != sizeof r || getchar() != EOF) return 1;'
                   + "".join(f'printf("%lld ", (long long)r.{f});' for f in fields) + "return 0;}\n")
    exe = tmp_path / "record"
    subprocess.run([cc, f"-I{HEADER.parent}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], input=data, capture_output=True, check=True).stdout
    assert list(map(int, out.split())) == list(range(1, len(fields) + 1))


def test_null_and_bad_records_are_refused():
    import ripvec_b200.decode as D

    lib = L.lib()
    assert lib.rv_step_append_record(None, None) == L.RV_E_INVALID
    assert lib.rv_step_attend_record(None, None) == L.RV_E_INVALID
    assert lib.rv_step_append_record(None, D._append_args(*[0] * 19)) == L.RV_E_INVALID
    assert lib.rv_step_attend_record(None, D._attend_args(*[0] * 10)) == L.RV_E_INVALID
    assert lib.rv_rms_norm_record(None) == L.RV_E_INVALID

    def norm_record(eps, rows=2):
        return lib.rv_rms_norm_record(D._norm_args(16, 64, 0, 0, 16, 0, 0, 16, 64, 0, rows, 64, L.RV_DTYPE_BF16,
                                                   L.RV_DTYPE_BF16, 0, eps, -1, 0))

    assert norm_record(1e-5, rows=0) == L.RV_OK
    for eps in (-1.0, math.nan, math.inf, 1e300, -1e300):
        assert norm_record(eps) == L.RV_E_INVALID


class OnDevice:
    """As much of a CUDA tensor as the checks look at."""

    def __init__(self, shape, dtype, device):
        import torch

        self.shape, self.dtype, self.ndim, self.device = torch.Size(shape), dtype, len(shape), f"cuda:{device}"
        self._device = device

    def get_device(self):
        return self._device

    def stride(self):
        out, n = [], 1
        for d in reversed(self.shape):
            out.append(n)
            n *= d
        return tuple(reversed(out))

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 4096


@pytest.mark.parametrize("cache_device,step_device", [(1, 0), (0, 1)])
def test_a_cache_of_another_device_is_refused(monkeypatch, cache_device, step_device):
    """Nothing reaches the library: it would launch on the step's device with the other one's addresses."""
    from types import SimpleNamespace

    import torch

    import ripvec_b200.decode as D

    calls = []
    fake = SimpleNamespace(rv_step_append_record=lambda *a: calls.append(a) or 0,
                           rv_step_attend_record=lambda *a: calls.append(a) or 0, rv_step_destroy=lambda h: None)
    monkeypatch.setattr(D, "_current_stream", lambda device: 0)
    step = object.__new__(D.DecodeStep)
    step._lib, step._h, step.tokens = fake, 1, 2
    step.q_heads, step.kv_heads, step.head_dim, step.page_size = 8, 2, 64, 16
    step.device = torch.device("cuda", step_device)
    for device, refused in ((step_device, False), (cache_device, True)):
        cache = SimpleNamespace(dtype=torch.bfloat16, device=f"cuda:{device}", device_index=device, _ref=4096)
        q, out = (OnDevice((2, 8, 64), torch.bfloat16, device) for _ in range(2))
        k = OnDevice((2, 2, 64), torch.bfloat16, device)
        cos = OnDevice((9, 32), torch.float32, device)
        for run in (lambda: step.append(cache, q, k, k, cos, cos, q_out=out), lambda: step.attend(cache, q, out=out)):
            if refused:
                with pytest.raises(ValueError, match="device"):
                    run()
            else:
                run()
        assert len(calls) == 2
