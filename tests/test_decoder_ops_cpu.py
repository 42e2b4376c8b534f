"""CPU: the decoder operators' structures, and what they refuse before anything reaches a GPU."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20  # an aligned address that is never followed: every refused call ends on the host


def _cache(pkg, **kw):
    c = pkg._KvCache(FAKE, FAKE, FAKE, FAKE, pkg.ELEM_E4M3, 4, 16, 2, 64, 2048, 1024, 64, 32, 16, 1)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _batch(pkg, **kw):
    b = pkg._KvBatch(1, 3, FAKE, FAKE, FAKE, 4, 4, 3, 64)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def _write(pkg, c, b, dtype=1, k=FAKE, v=FAKE, rs=128, hs=64):
    return pkg.lib().mw_kv_write_device(0, None, C.byref(c), C.byref(b), dtype, k, v, rs, hs)


def _attend(pkg, c, b, heads=4, q=FAKE, out=FAKE, rs=256, hs=64, scale=0.125, window=0, sinks=0, ws=FAKE, ws_bytes=1 << 30):
    return pkg.lib().mw_kv_attend_device(0, None, C.byref(c), C.byref(b), heads, q, rs, hs, out, rs, hs, scale, window, sinks, ws, ws_bytes)


def test_structs_match_the_header(pkg):
    probe = r'''
#include <stdio.h>
#include <stddef.h>
#include "mi355_whisper.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu %zu\n", sizeof(struct mw_kv_cache), sizeof(struct mw_kv_batch), offsetof(struct mw_kv_cache, dtype),
         offsetof(struct mw_kv_cache, page_stride), offsetof(struct mw_kv_cache, scale_row_stride), offsetof(struct mw_kv_batch, table_stride),
         offsetof(struct mw_kv_batch, max_kv));
  return 0; }'''
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "p.c"), os.path.join(d, "p")
        open(src, "w").write(probe)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe])
        got = [int(x) for x in subprocess.check_output([exe]).split()]
    K, B = pkg._KvCache, pkg._KvBatch
    assert got == [C.sizeof(K), C.sizeof(B), K.dtype.offset, K.page_stride.offset, K.scale_row_stride.offset, B.table_stride.offset, B.max_kv.offset]


@pytest.mark.parametrize("field,value,why", [
    ("k", None, "null pages"), ("dtype", 0, "element type"), ("dtype", 4, "element type"), ("head_dim", 96, "head_dim"), ("n_pages", 0, "page / head"),
    ("n_kv_heads", 0, "page / head"), ("page_size", 0, "power of two"), ("page_size", 24, "power of two"), ("page_size", 65536, "power of two"),
    ("row_stride", 72, "16 bytes"), ("head_stride", -16, "16 bytes"), ("page_stride", 8, "16 bytes"), ("v", FAKE + 8, "16 bytes"),
    ("k_scale", None, "scales"), ("v_scale", FAKE + 2, "scales"), ("scale_row_stride", -1, "scales")])
def test_caches_that_are_refused(pkg, field, value, why):
    c, b = _cache(pkg, **{field: value}), _batch(pkg)
    for call in (_write, _attend):
        assert call(pkg, c, b) == -100
        assert why in pkg.last_error()
    assert pkg.lib().mw_kv_attend_workspace(0, C.byref(c), C.byref(b), 4, 0, 0) == 0


@pytest.mark.parametrize("field,value,why", [
    ("n_seqs", -1, "sequence / row"), ("n_rows", -1, "sequence / row"), ("cu_rows", None, "null cu_rows"), ("kv_len", None, "null cu_rows"),
    ("block_table", None, "null cu_rows"), ("table_cols", -1, "table_stride"), ("table_stride", 3, "table_stride"), ("max_rows", -1, "expected"),
    ("max_kv", -1, "expected")])
def test_batches_that_are_refused(pkg, field, value, why):
    c, b = _cache(pkg), _batch(pkg, **{field: value})
    for call in (_write, _attend):
        assert call(pkg, c, b) == -100
        assert why in pkg.last_error()


def test_arguments_that_are_refused(pkg):
    c, b = _cache(pkg), _batch(pkg)
    L = pkg.lib()
    assert L.mw_kv_write_device(0, None, None, C.byref(b), 1, FAKE, FAKE, 128, 64) == -1
    assert L.mw_kv_attend_device(0, None, C.byref(c), None, 4, FAKE, 256, 64, FAKE, 256, 64, 0.1, 0, 0, None, 0) == -1
    for kw, why in ((dict(dtype=2), "f32 or bf16"), (dict(k=None), "16 bytes"), (dict(v=FAKE + 8), "16 bytes"), (dict(rs=100), "16 bytes"), (dict(hs=-64), "16 bytes")):
        assert _write(pkg, c, b, **kw) == -100 and why in pkg.last_error()
    for kw, why in ((dict(heads=3), "multiple of n_kv_heads"), (dict(heads=0), "multiple"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(window=-1), "window"), (dict(sinks=-1), "window"),
                    (dict(q=None), "16 bytes"), (dict(out=FAKE + 4), "16 bytes"), (dict(rs=130), "16 bytes"), (dict(heads=1 << 26), "too many")):
        assert _attend(pkg, c, b, **kw) == -100 and why in pkg.last_error(), kw
    assert _write(pkg, c, _batch(pkg, n_rows=1 << 28)) == -100 and "too many" in pkg.last_error()

    def sample(logits=FAKE, dtype=0, rows=2, vocab=100, stride=100, t=None, k=None, p=None, m=None, u=FAKE, ids=FAKE, lp=FAKE):
        return L.mw_sample_device(0, None, logits, dtype, rows, vocab, stride, t, k, p, m, u, ids, lp)

    for kw, why in ((dict(dtype=2), "f32 or bf16"), (dict(rows=-1), "row count"), (dict(rows=1 << 22), "row count"), (dict(vocab=0), "vocabulary"),
                    (dict(vocab=(1 << 20) + 1), "vocabulary"), (dict(logits=None), "null"), (dict(u=None), "null"), (dict(ids=None), "null"),
                    (dict(logits=FAKE + 2), "unaligned"), (dict(u=FAKE + 4), "unaligned"), (dict(t=FAKE + 2), "unaligned"), (dict(stride=-1), "stride")):
        assert sample(**kw) == -100 and why in pkg.last_error(), kw
    assert sample(rows=0) == 0  # nothing to do


def test_tensors_that_are_refused(pkg):
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="one GPU"):
        pkg.KvCache(k, k)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="one GPU"):
        pkg.KvBatch(i, i[:1], i[None])
    with pytest.raises(ValueError, match="one GPU"):
        pkg.sample_logits(torch.zeros(1, 8), torch.zeros(1, dtype=torch.float64))


def test_gradients_are_refused_while_they_are_recorded(pkg):
    pkg._load_torch()
    with pytest.raises(RuntimeError, match="it has no gradient"):
        pkg._no_gradient("it")
    with torch.no_grad():
        pkg._no_gradient("it")
