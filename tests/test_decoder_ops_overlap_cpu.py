"""CPU: results whose rows share memory are refused before anything reaches a GPU."""
import ctypes as C

import pytest

from test_decoder_ops_cpu import FAKE, _attend, _batch, _cache, _write


def _read(pkg, c, b, dtype=0, k=FAKE, v=FAKE, rs=128, hs=64):
    return pkg.lib().mw_kv_read_device(0, None, C.byref(c), C.byref(b), dtype, k, v, rs, hs)


@pytest.mark.parametrize("field,value,why", [("page_stride", 0, "rows overlap"), ("head_stride", 48, "rows overlap"), ("row_stride", 0, "rows overlap"),
                                             ("scale_page_stride", 0, "scales overlap"), ("scale_head_stride", 0, "scales overlap"),
                                             ("scale_row_stride", 0, "scales overlap")])
def test_caches_that_cannot_be_written(pkg, field, value, why):
    assert _write(pkg, _cache(pkg, **{field: value}), _batch(pkg)) == -100 and why in pkg.last_error()


def test_results_that_overlap(pkg):
    c, b = _cache(pkg), _batch(pkg)
    for kw in (dict(rs=0), dict(hs=0), dict(rs=60), dict(hs=32)):
        assert _read(pkg, c, b, **kw) == -100 and "overlap" in pkg.last_error(), kw
    for kw in (dict(rs=0), dict(hs=0), dict(hs=56)):
        assert _attend(pkg, c, b, **kw) == -100 and "overlap" in pkg.last_error(), kw
