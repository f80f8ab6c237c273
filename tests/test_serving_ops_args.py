"""Refusals of the 8-bit projection and paged-cache entry points: every wrong
argument is a status and a message before anything is launched.  No GPU needed
(the pointers are never followed)."""
import ctypes as C

import pytest

import xl_capi as X

P = 1 << 20  # a 16-byte aligned address that nothing reads
BAD = 1      # XL_ERR_ARG


def refused(rc, word):
    assert rc == BAD
    assert word in X.lib().xl_last_error().decode(), X.lib().xl_last_error()


def with_(base, **over):
    a = dict(base)
    a.update(over)
    return list(a.values())


QUANT = dict(dtype=0, x=P, ldx=256, q=P, ldq=256, scale=P, n=4, k=256, rows=1, stream=None)
NORM = dict(dtype=0, delta=P, residual=P, out=P + 4096, gamma=P, q=P, ldq=256, scale=P, n=4, k=256, stream=None)
LINEAR = dict(mode=0, dtype=0, xq=P, ldx=256, xs=P, wq=P, ldw=256, ws=P, bias=None, y=P, n=4, m=128, k=256, stream=None)


@pytest.mark.parametrize("over,word", [
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"), (dict(dtype=3), "dtype"),
    (dict(dtype=-1), "dtype"), (dict(n=0), "positive"), (dict(k=-1), "positive"), (dict(rows=2), "rows_per_scale"),
    (dict(ldx=255), "ldx"), (dict(ldq=255), "multiple"), (dict(ldq=264), "multiple"), (dict(ldq=240), "multiple"),
    (dict(q=P + 8), "aligned"), (dict(x=P + 2), "aligned"), (dict(scale=P + 1), "aligned"),
    (dict(n=2147483647), "groups"),
])
def test_quantize_refusals(built, over, word):
    refused(X.lib().xl_op_quantize_fp8(*with_(QUANT, **over)), word)


@pytest.mark.parametrize("over,word", [
    (dict(residual=None), "null"), (dict(gamma=None), "null"), (dict(q=None), "null"), (dict(scale=None), "null"),
    (dict(out=None), "residual_out"), (dict(out=P), "delta"), (dict(dtype=7), "dtype"), (dict(n=0), "positive"),
    (dict(k=32769, ldq=32784), "32768"), (dict(k=0), "32768"), (dict(ldq=100), "multiple"), (dict(q=P + 1), "aligned"),
    (dict(residual=P + 8), "aligned"), (dict(delta=P + 4), "aligned"), (dict(gamma=P + 4), "aligned"),
])
def test_norm_refusals(built, over, word):
    refused(X.lib().xl_op_add_rmsnorm_fp8(*with_(NORM, **over)), word)


@pytest.mark.parametrize("over,word", [
    (dict(xq=None), "null"), (dict(xs=None), "null"), (dict(wq=None), "null"), (dict(ws=None), "null"),
    (dict(y=None), "null"), (dict(mode=3), "mode"), (dict(mode=-1), "mode"), (dict(dtype=9), "dtype"),
    (dict(n=0), "positive"), (dict(m=0), "positive"), (dict(k=0), "positive"), (dict(mode=1, m=127), "even"),
    (dict(ldx=272 + 8), "multiple"), (dict(ldw=240), "multiple"), (dict(xq=P + 8), "aligned"),
    (dict(wq=P + 4), "aligned"), (dict(y=P + 8), "aligned"), (dict(bias=P + 2), "aligned"),
])
def test_linear_refusals(built, over, word):
    refused(X.lib().xl_op_linear_fp8(*with_(LINEAR, **over)), word)


CACHE = dict(k=P, v=P, page_table=P, dtype=0, batch=2, kv_heads=2, head_dim=64, page_size=16, max_pages=4, num_pages=8)
CACHE_FAULTS = [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(page_table=None), "null"), (dict(dtype=4), "dtype"),
    (dict(batch=0), "positive"), (dict(kv_heads=0), "positive"), (dict(page_size=0), "positive"),
    (dict(max_pages=0), "positive"), (dict(num_pages=-2), "positive"), (dict(head_dim=96), "head_dim"),
    (dict(kv_heads=3), "multiple"), (dict(page_size=1 << 16, max_pages=1 << 16), "2^31"), (dict(page_size=1 << 10, max_pages=(1 << 21) - 1), "2^31"),
    (dict(batch=1 << 30), "2^30"), (dict(k=P + 8), "aligned"), (dict(num_pages=1 << 30), "2^32"),
]


def attend(described=CACHE, **over):
    base = dict(cache=C.byref(X.PagedKV(**described)), dtype=0, qkv=P, rope=P, rope_len=64, pos=P, out=P, heads=4, ws=P,
                ws_bytes=1 << 30, stream=None)
    return X.lib().xl_op_attn_decode_paged(*with_(base, **over))


def append(described=CACHE, **over):
    base = dict(cache=C.byref(X.PagedKV(**described)), dtype=0, qkv=P, rope=P, rope_len=64, seq=P, pos=P, rows=3, heads=4,
                stream=None)
    return X.lib().xl_op_kv_append_paged(*with_(base, **over))


@pytest.mark.parametrize("over,word", CACHE_FAULTS)
def test_cache_refusals(built, over, word):
    refused(attend(dict(CACHE, **over)), word)
    refused(append(dict(CACHE, **over)), word)
    assert X.lib().xl_op_attn_decode_paged_workspace_bytes(C.byref(X.PagedKV(**dict(CACHE, **over))), 4) == 0


@pytest.mark.parametrize("over,word", [
    (dict(cache=None), "null"), (dict(qkv=None), "null"), (dict(pos=None), "null"), (dict(out=None), "null"),
    (dict(ws=None), "null"), (dict(dtype=5), "dtype"), (dict(rope_len=0), "rope_len"), (dict(heads=0), "positive"),
    (dict(heads=3), "multiple"), (dict(qkv=P + 4), "aligned"), (dict(out=P + 8), "aligned"), (dict(rope=P + 8), "aligned"),
    (dict(ws=P + 8), "aligned"), (dict(ws_bytes=16), "workspace"),
])
def test_attend_refusals(built, over, word):
    refused(attend(**over), word)


@pytest.mark.parametrize("over,word", [
    (dict(cache=None), "null"), (dict(qkv=None), "null"), (dict(seq=None), "null"), (dict(pos=None), "null"),
    (dict(dtype=5), "dtype"), (dict(rope_len=-1), "rope_len"), (dict(rows=0), "positive"), (dict(heads=5), "multiple"),
    (dict(qkv=P + 4), "aligned"),
])
def test_append_refusals(built, over, word):
    refused(append(**over), word)


def test_arguments_in_order_reach_the_device_check(built):
    """With nothing wrong but the pointers themselves the call ends in the
    check of their memory (no device here, or not a device's address)."""
    want = {BAD, 5}  # XL_ERR_ARG, XL_ERR_CUDA
    assert X.lib().xl_op_quantize_fp8(*QUANT.values()) in want
    assert X.lib().xl_op_add_rmsnorm_fp8(*NORM.values()) in want
    assert X.lib().xl_op_linear_fp8(*LINEAR.values()) in want
    assert attend() in want and append() in want
    assert X.lib().xl_last_error()
