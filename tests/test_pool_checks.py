"""Refusals of the serving operators over a caller-owned page pool: every check of arguments runs before the
context is used, so a null context shows them without a device (kg_last_error(NULL) has the message)."""
import ctypes
import os
import re

import pytest

A16 = 1 << 20  # a 16-byte aligned address that nothing dereferences
INVALID, UNSUPPORTED = -1, -6


def _pool(kg, **kw):
    a = dict(k_ptr=A16, v_ptr=A16 + 4096, n_pages=8, page_size=16, n_kv_head=2, head_dim=64, dtype="bf16")
    a.update(kw)
    return kg.page_pool(**a)


def _refused(kg, rc, code, text):
    msg = kg.lib().kg_last_error(None).decode()
    assert rc == code and text in msg, (rc, msg)


POOLS = [
    (dict(dtype="f32"), UNSUPPORTED, "dtype"),
    (dict(head_dim=96), UNSUPPORTED, "head_dim"),
    (dict(page_size=8), UNSUPPORTED, "page_size"),
    (dict(page_size=24), UNSUPPORTED, "page_size"),
    (dict(page_size=256), UNSUPPORTED, "page_size"),
    (dict(n_pages=0), INVALID, "positive"),
    (dict(n_kv_head=0), INVALID, "positive"),
    (dict(n_pages=1 << 27), INVALID, "2^31"),
    (dict(k_ptr=0), INVALID, "two device pointers"),
    (dict(v_ptr=A16), INVALID, "two device pointers"),
    (dict(k_ptr=A16 + 8), INVALID, "aligned"),
    (dict(row_stride=132), INVALID, "multiples of 8"),
    (dict(row_stride=120), INVALID, "overlap"),
    (dict(head_stride=56), INVALID, "overlap"),
    (dict(page_stride=128), INVALID, "overlap"),
    (dict(page_stride=-4096), INVALID, "overlap"),
    (dict(page_stride=1 << 61), INVALID, "overlap"),
]


@pytest.mark.parametrize("kw,code,text", POOLS)
def test_pool_refusals(kg, kw, code, text):
    pool = _pool(kg, **kw)
    L = kg.lib()
    _refused(kg, L.kg_pool_store_dev(None, pool, 1, A16, kg.KG_DT_F32, A16, A16, 128, 64, None), code, text)
    _refused(kg, L.kg_pool_attend_bytes(pool, 1, 2, 1), code, text)


def test_null_pool_and_context(kg):
    L = kg.lib()
    _refused(kg, L.kg_pool_store_dev(None, None, 1, A16, 0, A16, A16, 128, 64, None), INVALID, "null pool")
    _refused(kg, L.kg_pool_attend_bytes(None, 1, 2, 1), INVALID, "null pool")
    _refused(kg, L.kg_pool_status(None), INVALID, "null context")
    pool = _pool(kg)
    _refused(kg, L.kg_pool_store_dev(None, pool, 1, A16, 0, A16, A16, 128, 64, None), INVALID, "null context")
    _refused(kg, L.kg_pool_store_dev(None, pool, 0, None, 0, None, None, 0, 0, None), INVALID, "null context")
    # pools that pass: head-major pages, separate K and V, one page
    for kw in (dict(row_stride=64, head_stride=1024), dict(v_ptr=1 << 30, page_stride=2048), dict(n_pages=1, page_stride=0)):
        _refused(kg, L.kg_pool_store_dev(None, _pool(kg, **kw), 1, A16, 0, A16, A16, 128, 64, None), INVALID, "null context")


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_rows=-1), INVALID, "negative"),
    (dict(src=3), UNSUPPORTED, "src_dtype"),
    (dict(slots=None), INVALID, "null pointer"),
    (dict(k=None), INVALID, "null pointer"),
    (dict(v=None), INVALID, "null pointer"),
    (dict(k=A16 + 4), INVALID, "aligned"),
    (dict(rs=130), INVALID, "aligned"),
    (dict(src=1, rs=132), INVALID, "aligned"),
    (dict(hs=-64), INVALID, "aligned"),
    (dict(n_rows=2**31 - 1, pool=dict(n_kv_head=1024, row_stride=1024 * 64, page_stride=1 << 21)), UNSUPPORTED, "too many rows"),
])
def test_store_refusals(kg, kw, code, text):
    a = dict(n_rows=4, slots=A16, src=0, k=A16, v=A16, rs=128, hs=64, pool={})
    a.update(kw)
    rc = kg.lib().kg_pool_store_dev(None, _pool(kg, **a["pool"]), a["n_rows"], a["slots"], a["src"], a["k"], a["v"], a["rs"], a["hs"], None)
    _refused(kg, rc, code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(page=20), UNSUPPORTED, "page_size"),
    (dict(n_pages=0), INVALID, "n_pages"),
    (dict(n_pages=1 << 30), INVALID, "n_pages"),
    (dict(n_req=-1), INVALID, "negative"),
    (dict(n_req=16385), UNSUPPORTED, "16384"),
    (dict(width=0), INVALID, "table_width"),
    (dict(max_tokens=-1), INVALID, "negative"),
    (dict(cached=None), INVALID, "null pointer"),
    (dict(new=None), INVALID, "null pointer"),
    (dict(table=None), INVALID, "null pointer"),
    (dict(free=None), INVALID, "null pointer"),
    (dict(n_free=None), INVALID, "null pointer"),
    (dict(status=None), INVALID, "null pointer"),
    (dict(slots=None), INVALID, "null pointer"),
    (dict(), INVALID, "null context"),
    (dict(n_req=0, cached=None, new=None, table=None, kv=None), INVALID, "null context"),
    (dict(max_tokens=0, slots=None), INVALID, "null context"),
])
def test_plan_refusals(kg, kw, code, text):
    a = dict(page=16, n_pages=64, n_req=4, cached=A16, new=A16, table=A16, width=8, free=A16, n_free=A16, left=A16, max_tokens=10,
             cu=A16, kv=A16, slots=A16, req=A16, pos=A16, status=A16)
    a.update(kw)
    _refused(kg, kg.lib().kg_pool_plan_dev(None, *a.values(), None), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_req=-1), INVALID, "negative"),
    (dict(total_q=-1), INVALID, "negative"),
    (dict(n_req=16385), UNSUPPORTED, "16384"),
    (dict(n_head=0), INVALID, "multiple"),
    (dict(n_head=3), INVALID, "multiple"),
    (dict(n_head=130), UNSUPPORTED, "64 query heads"),
    (dict(total_q=1 << 30), UNSUPPORTED, "2^31"),
    (dict(width=0), INVALID, "table_width"),
    (dict(cu=None), INVALID, "null pointer"),
    (dict(kv=None), INVALID, "null pointer"),
    (dict(table=None), INVALID, "null pointer"),
    (dict(q=None), INVALID, "null pointer"),
    (dict(out=None), INVALID, "null pointer"),
    (dict(ws=None), INVALID, "null pointer"),
    (dict(out=A16), INVALID, "overlap"),
    (dict(q=A16 + 2), INVALID, "aligned"),
    (dict(ws=A16 + 8), INVALID, "aligned"),
    (dict(qrs=260), INVALID, "multiples of 8"),
    (dict(ors=248), INVALID, "overlap"),
    (dict(ohs=0), INVALID, "overlap"),
    (dict(qhs=-64), INVALID, "overlap"),
    (dict(wsb=0), INVALID, "workspace"),
    (dict(scale=float("inf")), INVALID, "scale"),
    (dict(scale=float("nan")), INVALID, "scale"),
    (dict(scale=-0.125), INVALID, "scale"),
    (dict(), INVALID, "null context"),
    (dict(qrs=64, qhs=64 * 12, ors=64, ohs=64 * 12), INVALID, "null context"),  # head-major
    (dict(n_req=0, cu=None, kv=None, table=None, q=None, out=None, ws=None), INVALID, "null context"),
])
def test_attend_refusals(kg, kw, code, text):
    a = dict(n_req=2, n_head=4, total_q=12, cu=A16, kv=A16, table=A16, width=4, q=A16, qrs=256, qhs=64, out=A16 << 1, ors=256, ohs=64,
             scale=0.125, causal=1, ws=A16, wsb=1 << 40)
    a.update(kw)
    _refused(kg, kg.lib().kg_pool_attend_dev(None, _pool(kg), *a.values(), None), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_rows=-1), INVALID, "negative"),
    (dict(vocab=0), INVALID, "positive"),
    (dict(vocab=262145, ld=262145), UNSUPPORTED, "262144"),
    (dict(dtype=3), UNSUPPORTED, "dtype"),
    (dict(logits=None), INVALID, "null pointer"),
    (dict(u=None), INVALID, "null pointer"),
    (dict(out=None), INVALID, "null pointer"),
    (dict(ld=99), INVALID, "overlap"),
    (dict(logits=A16 + 2), INVALID, "aligned"),
    (dict(logits=A16 + 1, dtype=1), INVALID, "aligned"),
    (dict(), INVALID, "null context"),
    (dict(logits=A16 + 2, dtype=2, t=None, k=None, p=None, m=None), INVALID, "null context"),
    (dict(n_rows=1, ld=0), INVALID, "null context"),
])
def test_sample_refusals(kg, kw, code, text):
    a = dict(n_rows=3, vocab=100, dtype=0, logits=A16, ld=100, t=A16, k=A16, p=A16, m=A16, u=A16, out=A16)
    a.update(kw)
    _refused(kg, kg.lib().kg_sample_logits_dev(None, *a.values(), None), code, text)


def test_pool_mirrors_have_the_headers_fields(kg):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    header = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "kg_abi.h")).read(), flags=re.S)
    fields = re.findall(r"\b(\w+)\s*;", re.search(r"typedef struct \{([^}]*)\}\s*kg_pool;", header).group(1))
    assert fields == [f for f, _ in kg.KgPool._fields_]
    rust = re.search(r"pub struct KgPool \{([^}]*)\}", open(os.path.join(root, "INTEGRATION.md")).read()).group(1)
    assert re.findall(r"pub (\w+):", rust) == fields


def test_attend_bytes_raises_in_python(kg):
    with pytest.raises(kg.KgError, match="head_dim"):
        kg.CudaBackend.pool_attend_bytes(_pool(kg, head_dim=32), 1, 2, 1)
    assert kg.CudaBackend.pool_attend_bytes(_pool(kg), 1, 2, 1) > 0
    assert ctypes.sizeof(kg.KgPool) == 64
