"""The products' C ABI and Python entry points on the CPU: the library exports what the header
declares, and every bad argument is refused before anything reaches a GPU."""

from __future__ import annotations

import ctypes
import json
import re
import subprocess
from pathlib import Path

import pytest
import torch

from vibe_megakernel_amd import _lib, products
from vibe_megakernel_amd import build as pkg_build

HEADER = Path(__file__).resolve().parent.parent / "include" / "megamoe_products.h"
FAKE = 4096  # a pointer that is never followed: the checks answer first


def test_library_exports_every_declared_function():
    declared = set(re.findall(r"^int (megamoe_[a-z_0-9]+)\s*\(", HEADER.read_text(), flags=re.M))
    assert declared == set(_lib.PRODUCT_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", str(_lib.LIBRARY)], capture_output=True, text=True,
                         check=True).stdout
    assert declared <= set(re.findall(r"\bT (megamoe_[a-z_0-9]+)$", out, flags=re.M))
    assert _lib.load().megamoe_products_version() == _lib.PRODUCTS_VERSION


def _product(**change):
    p = dict(rows=8, groups=4, n=64, k=32, dtype=_lib.BF16, transposed=0, fill_rest=1, ldx=32, ldy=64)
    p.update(change)
    return _lib.Product(**p)


GEOMETRY = [
    (dict(rows=-1), _lib.ERR_SHAPE), (dict(groups=0), _lib.ERR_SHAPE), (dict(n=-1), _lib.ERR_SHAPE),
    (dict(k=-8), _lib.ERR_SHAPE), (dict(ldx=31), _lib.ERR_SHAPE), (dict(ldy=63), _lib.ERR_SHAPE),
    (dict(dtype=-1), _lib.ERR_SHAPE), (dict(dtype=3), _lib.ERR_SHAPE),
    (dict(groups=1025), _lib.ERR_UNSUPPORTED), (dict(rows=(1 << 30) + 1), _lib.ERR_UNSUPPORTED),
    (dict(ldx=(4 << 20) + 1), _lib.ERR_UNSUPPORTED), (dict(ldy=(1 << 20) + 1), _lib.ERR_UNSUPPORTED),
]


@pytest.mark.parametrize("change,status", GEOMETRY)
def test_geometry_is_checked_by_every_product(change, status):
    lib, p = _lib.load(), ctypes.byref(_product(**change))
    assert lib.megamoe_grouped_mm(p, FAKE, FAKE, FAKE, FAKE, None) == status
    assert lib.megamoe_grouped_mm_wgrad(p, FAKE, FAKE, FAKE, FAKE, None) == status
    assert lib.megamoe_int8_mm(p, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == status


def test_types_limits_and_pointers_are_checked():
    lib, bad = _lib.load(), _lib.ERR_INVALID_ARGUMENT
    P = ctypes.byref
    for fn, pointers in ((lib.megamoe_grouped_mm, 4), (lib.megamoe_grouped_mm_wgrad, 4), (lib.megamoe_int8_mm, 6)):
        args = [FAKE] * pointers
        assert fn(None, *args, None) == bad
        for i in range(pointers):
            if fn is lib.megamoe_int8_mm and i == 4:
                continue  # counts may be NULL there
            assert fn(P(_product()), *(None if j == i else FAKE for j in range(pointers)), None) == bad, i
        aligned = range(pointers) if fn is not lib.megamoe_int8_mm else (1, 3, 4, 5)
        for i in aligned:
            assert fn(P(_product()), *(FAKE + 1 if j == i else FAKE for j in range(pointers)), None) == bad, i
    # fp32 results and a NULL counts are the int8 product's alone; it has no transposed form.
    assert lib.megamoe_grouped_mm(P(_product(dtype=_lib.FP32)), FAKE, FAKE, FAKE, FAKE, None) == _lib.ERR_SHAPE
    int8 = lib.megamoe_int8_mm
    assert int8(P(_product()), FAKE, FAKE, FAKE, FAKE, None, FAKE, None) == _lib.ERR_SHAPE  # one group only
    assert int8(P(_product(transposed=1)), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == _lib.ERR_SHAPE
    long = _product(k=131072, ldx=131072)
    assert int8(P(long), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == _lib.ERR_UNSUPPORTED
    assert int8(P(_product(dtype=_lib.FP32)), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE + 2, None) == bad
    # Nothing to compute: no pointer is needed.
    for empty in (dict(rows=0), dict(n=0)):
        assert lib.megamoe_grouped_mm(P(_product(**empty)), None, None, None, None, None) == _lib.OK
        assert int8(P(_product(**empty)), None, None, None, None, FAKE, None, None) == _lib.OK
    for empty in (dict(k=0), dict(n=0)):
        assert lib.megamoe_grouped_mm_wgrad(P(_product(**empty)), None, None, None, None, None) == _lib.OK


def test_quantize_rows_int8_checks():
    q = _lib.load().megamoe_quantize_rows_int8
    assert q(-1, 64, 64, _lib.BF16, FAKE, FAKE, FAKE, None) == _lib.ERR_SHAPE
    assert q(4, -1, 64, _lib.BF16, FAKE, FAKE, FAKE, None) == _lib.ERR_SHAPE
    assert q(4, 64, 63, _lib.BF16, FAKE, FAKE, FAKE, None) == _lib.ERR_SHAPE
    assert q(4, 64, 64, 3, FAKE, FAKE, FAKE, None) == _lib.ERR_SHAPE
    for pointers in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None), (FAKE + 1, FAKE, FAKE),
                     (FAKE, FAKE, FAKE + 2)):
        assert q(4, 64, 64, _lib.BF16, *pointers, None) == _lib.ERR_INVALID_ARGUMENT
    assert q(4, 64, 64, _lib.FP32, FAKE + 2, FAKE, FAKE, None) == _lib.ERR_INVALID_ARGUMENT
    assert q(0, 64, 64, _lib.BF16, None, None, None, None) == _lib.OK


def test_python_entry_points_refuse_tensors_off_the_gpu():
    x, w, c = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(2, 6, 8, dtype=torch.bfloat16), torch.zeros(2).long()
    with pytest.raises(RuntimeError):
        products.grouped_mm(x, w, c)
    with pytest.raises(RuntimeError):
        products.grouped_mm(x.clone().requires_grad_(), w, c)
    with pytest.raises(RuntimeError):
        products.grouped_mm_wgrad(x, x, c)
    with pytest.raises(RuntimeError):
        products.int8_mm(x.char(), torch.ones(4), w[0].char(), torch.ones(6))
    with pytest.raises(RuntimeError):
        products.grouped_int8_mm(x.char(), torch.ones(4), w.char(), torch.ones(2, 6), c)
    with pytest.raises(RuntimeError):
        products.quantize_rows_int8(x)
    for call in (lambda: products.grouped_mm(None, w, c), lambda: products.quantize_rows_int8([1.0]),
                 lambda: products.int8_mm(None, None, None, None)):
        with pytest.raises(ValueError):
            call()


def test_row_strides():
    t = torch.zeros(6, 10)
    assert products._stride(t) == 10 and products._stride(t[:, :4]) == 10 and products._stride(t[::2]) == 20
    assert products._stride(t[:1, :4]) == 4 and products._stride(t[:, :1]) == 10
    assert products._stride(t.t()) is None and products._stride(t[:1].expand(6, 10)) is None
    a, b = products._extent(t[1:3, 2:5])
    assert a == t.data_ptr() + 4 * 12 and b == t.data_ptr() + 4 * 25


def test_no_kernel_spills():
    """The compiler's report of the built library: registers of the products that go to memory cost more than the
    results show, and the four wavefronts of the 256x256 tiles hold 256 AGPRs each without one to spare."""
    if not pkg_build.REPORT.exists():
        pytest.skip("no resource report: the library has not been built here")
    report = json.loads(pkg_build.REPORT.read_text())
    names = [n for n in report if re.search(r"k_(tiles|strips|product_any|wgrad_any|quantize_int8)", n)]
    assert len(names) >= 60
    for n in names:
        assert report[n]["scratch_bytes"] == 0 and report[n]["vgpr_spills"] == 0, (n, report[n])
        assert report[n]["lds_bytes"] <= 160 * 1024, (n, report[n])
