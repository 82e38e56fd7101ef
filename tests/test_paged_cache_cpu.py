"""Argument checks of the paged cache operators that need no device."""
import ctypes

import pytest
import torch


class Cache(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("k", "v", "page_table")]
                + [(n, ctypes.c_int64) for n in ("page_table_stride", "page_stride", "head_stride", "token_stride")]
                + [(n, ctypes.c_void_p) for n in ("k_scale", "v_scale")]
                + [(n, ctypes.c_int) for n in ("sequences", "max_pages", "pages", "page_size", "kv_heads", "head_dim")])


def cache(**kw):
    """A cache that passes every check; the addresses are never used."""
    c = Cache(256, 256, 256, 4, 2 * 16 * 128, 16 * 128, 128, None, None, 3, 4, 12, 16, 2, 128)
    for name, value in kw.items():
        setattr(c, name, value)
    return ctypes.byref(c)


BAD = [
    (dict(k=None), b"null buffer"), (dict(page_table=None), b"null buffer"), (dict(k_scale=256), b"go together"),
    (dict(sequences=0), b"positive"), (dict(pages=0), b"positive"), (dict(page_size=0), b"positive"), (dict(kv_heads=-1), b"positive"),
    (dict(page_table_stride=3), b"cover max_pages"), (dict(page_stride=-128), b"negative"), (dict(k=264), b"multiples of 16"),
    (dict(head_stride=129), b"multiples of 16"), (dict(token_stride=4), b"multiples of 16"),
    (dict(k_scale=256, v_scale=256, token_stride=136), b"multiples of 16"),
]


@pytest.mark.parametrize("change,message", BAD)
def test_caches_that_are_refused(change, message):
    from sharq_b200 import _lib

    L = _lib.lib()
    one = ctypes.c_void_p(256)
    assert L.sharq_paged_attention(one, 512, 128, 4, cache(**change), one, 0.1, one, one, 1 << 30, None, None) != 0
    assert message in L.sharq_last_error()
    assert L.sharq_rope_append_paged(one, 1024, 2, 4, one, one, 64, one, None, cache(**change), one, None, None, None) != 0
    assert message in L.sharq_last_error()


def test_other_arguments_that_are_refused():
    from sharq_b200 import _lib

    L = _lib.lib()
    one, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)
    # a table of few tokens needs no scratch, one of many does, arguments that are refused have none
    long = dict(max_pages=10000, page_table_stride=10000)
    need = L.sharq_paged_attention_workspace_bytes(4, cache(**long))
    assert need > 0 and L.sharq_paged_attention_workspace_bytes(4, cache()) == 0
    assert L.sharq_paged_attention_workspace_bytes(0, cache(**long)) == 0 and L.sharq_paged_attention_workspace_bytes(3, cache(**long)) == 0

    def attend(message, q=one, q_row=512, q_head=128, heads=4, c=None, ws=need):
        assert L.sharq_paged_attention(q, q_row, q_head, heads, c or cache(), one, 0.1, one, one, ws, None, None) != 0
        assert message in L.sharq_last_error()

    attend(b"null buffer", q=None)
    attend(b"64 or 128", c=cache(head_dim=96))
    attend(b"multiple of kv_heads", heads=3)
    attend(b"too many sequences", c=cache(sequences=2 ** 30))
    attend(b"multiples of 8", q_row=516)
    attend(b"16-byte aligned", q=odd)
    attend(b"workspace too small", ws=need - 1, c=cache(**long))

    def append(message, qkv=one, stride=1024, rows=2, heads=4, table=64, c=None):
        assert L.sharq_rope_append_paged(qkv, stride, rows, heads, one, one, table, one, None, c or cache(), one, None, None, None) != 0
        assert message in L.sharq_last_error()

    append(b"null buffer", qkv=None)
    append(b"rows must be", rows=-1)
    append(b"rows must be", table=0)
    append(b"multiple of 16, at most 256", c=cache(head_dim=264))
    append(b"row_stride", stride=1016)
    append(b"row_stride", stride=1028)
    append(b"16-byte aligned", qkv=odd)
    append(b"65536 heads", heads=70000)


def test_ops_refuse_cpu_tensors():
    from sharq_b200 import ops

    k = torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_attention(torch.zeros(1, 4, 128, dtype=torch.bfloat16), k, k, table, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rope_append_paged(torch.zeros(1, 1024, dtype=torch.bfloat16), 4, 2, 128, k[0, 0], k[0, 0], n, table, k, k)


def test_weight_only_arguments_that_are_refused():
    from sharq_b200 import _lib, ops

    L = _lib.lib()
    one, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)

    def refuse(message, x=one, x_row=256, m=2, n=128, k=256, qw=one):
        assert L.sharq_weight_only_linear(x, x_row, m, n, k, qw, one, None, 1.0, None, one, None, None) != 0
        assert message in L.sharq_last_error()

    refuse(b"null buffer", x=None)
    refuse(b"1 to 16 rows", m=0)
    refuse(b"1 to 16 rows", m=17)
    refuse(b"N must be", n=0)
    refuse(b"N must be", n=65535 * 128 + 1)
    refuse(b"multiple of 64", k=96)
    refuse(b"must not overlap", x_row=128)
    refuse(b"must not overlap", x_row=260)
    refuse(b"16-byte aligned", qw=odd)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.weight_only_linear(torch.zeros(1, 64, dtype=torch.bfloat16), torch.zeros(4, 32, dtype=torch.uint8),
                               torch.zeros(512, dtype=torch.uint8), 1.0)


@pytest.mark.parametrize("change", [dict(page_stride=0), dict(head_stride=0), dict(token_stride=0), dict(token_stride=64)])
def test_caches_whose_elements_overlap_are_refused(change):
    from sharq_b200 import _lib

    L = _lib.lib()
    one = ctypes.c_void_p(256)
    assert L.sharq_paged_attention(one, 512, 128, 4, cache(**change), one, 0.1, one, one, 1 << 30, None, None) != 0
    assert b"must not overlap" in L.sharq_last_error()
    assert L.sharq_rope_append_paged(one, 1024, 2, 4, one, one, 64, one, None, cache(**change), one, None, None, None) != 0
    assert b"must not overlap" in L.sharq_last_error()


def test_a_weight_whose_rows_are_too_long_is_refused():
    from sharq_b200 import _lib

    L = _lib.lib()
    one = ctypes.c_void_p(256)
    assert L.sharq_weight_only_linear(one, 2 ** 31 - 64, 1, 1, 2 ** 31 - 64, one, one, None, 1.0, None, one, None, None) != 0
    assert b"K up to" in L.sharq_last_error()
