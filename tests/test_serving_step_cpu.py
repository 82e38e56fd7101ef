"""What the operators of a server's step refuse before any launch, and the host's part of a cache whose pages are handed out on the device."""
import ctypes
import re

import pytest
import torch

from sharq_b200 import _lib
from sharq_b200._build import CSRC
from sharq_b200.decoder import DecoderConfig, _attention, rope_tables
from sharq_b200.kv_cache import PagedKVCache
from sharq_b200.logit_rules import LogitRules
from tests.test_dependent_launch_cpu import _block, _code

ONE, ODD = ctypes.c_void_p(256), ctypes.c_void_p(264)  # any addresses: the checks below fail before they are used


def refused(name, args, said):
    lib = _lib.lib()
    assert getattr(lib, name)(*args) != 0
    assert said in lib.sharq_last_error().decode()


def test_prompt_attention_refuses():
    good = dict(q=ONE, q_row=128, q_head=64, k=ONE, k_row=64, k_head=64, v=ONE, v_row=64, v_head=64, rows=10, k_rows=10, heads=2, kv_heads=1, head_dim=64,
                offsets=ONE, k_offsets=None, sequences=1, window=0, sinks=0, scale=1.0, out=ONE, fill=0, workspace=None, workspace_bytes=0, flag=None, stream=None)
    for changes, said in [(dict(q=None), "null"), (dict(offsets=None), "null"), (dict(head_dim=96), "64 or 128"), (dict(rows=0), "rows"), (dict(k_rows=0), "rows"),
                          (dict(rows=2 ** 30 + 1), "2^30"), (dict(heads=3, kv_heads=2), "multiple"), (dict(kv_heads=0), "multiple"), (dict(sequences=0), "sequences"),
                          (dict(window=-1), "negative"), (dict(sinks=-1), "negative"), (dict(k_rows=11), "key for every query"), (dict(q_row=0), "strides"),
                          (dict(k_head=60), "strides"), (dict(v_row=-64), "strides"), (dict(q=ODD), "16-byte"), (dict(out=ODD), "16-byte"),
                          (dict(rows=10, k_rows=90000, k_offsets=ONE), "workspace")]:
        refused("sharq_prompt_attention", {**good, **changes}.values(), said)
    size = _lib.lib().sharq_prompt_attention_workspace_bytes
    assert size(10, 90000, 2, 1, 64, 1, 0, 0) > size(10, 10, 2, 1, 64, 1, 0, 0) == 0 == size(10, 90000, 2, 1, 64, 0, 0, 0)


def test_plan_and_rules_refuse():
    good = dict(table=ONE, stride=4, sequences=3, max_pages=4, page_size=16, max_tokens=0, lengths=ONE, counts=ONE, released=None, free=ONE, size=9, count=ONE,
                rows=5, offsets=ONE, positions=ONE, row_sequences=ONE, flag=None, stream=None)
    for changes, said in [(dict(table=None), "null"), (dict(count=None), "null"), (dict(offsets=None), "null"), (dict(sequences=0), "positive"), (dict(page_size=0), "positive"),
                          (dict(max_tokens=-1), "max_tokens"), (dict(stride=3), "stride"), (dict(free=None), "room"), (dict(size=2 ** 30 + 1), "2^30"),
                          (dict(positions=None), "rows"), (dict(rows=-1), "rows")]:
        refused("sharq_plan_paged_step", {**good, **changes}.values(), said)

    class Rules(ctypes.Structure):
        _fields_ = [("tokens", ctypes.c_void_p), ("tokens_stride", ctypes.c_int64), ("width", ctypes.c_int), ("wide", ctypes.c_int), ("lengths", ctypes.c_void_p),
                    ("prompt_lengths", ctypes.c_void_p), ("repetition", ctypes.c_void_p), ("presence", ctypes.c_void_p), ("frequency", ctypes.c_void_p),
                    ("bias_offsets", ctypes.c_void_p), ("bias_ids", ctypes.c_void_p), ("bias_values", ctypes.c_void_p), ("biases", ctypes.c_int),
                    ("mask", ctypes.c_void_p), ("mask_stride", ctypes.c_int64)]

    def call(said, rows=2, vocab=9, stride=9, logits=ONE, **kw):
        rules = Rules(**kw)
        refused("sharq_adjust_logits", (logits, stride, ONE, 9, rows, vocab, 0, ctypes.byref(rules), None, None), said)

    call("null", logits=None)
    call("rows must be", rows=0)
    call("rows must be", rows=65536)
    call("overlap", stride=8)
    call("together", tokens=256)
    call("together", lengths=256, width=3)
    call("need tokens", repetition=256)
    call("biases go", biases=3)
    call("biases go", bias_offsets=256, biases=3)
    call("mask", mask=256, mask_stride=-1)


def test_windowed_attention_refuses():
    class Cache(ctypes.Structure):
        _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("page_table", ctypes.c_void_p), ("page_table_stride", ctypes.c_int64),
                    ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64), ("k_scale", ctypes.c_void_p),
                    ("v_scale", ctypes.c_void_p), ("sequences", ctypes.c_int), ("max_pages", ctypes.c_int), ("pages", ctypes.c_int),
                    ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int)]

    cache = Cache(256, 256, 256, 4, 16 * 64, 16 * 64, 64, None, None, 1, 4, 9, 16, 1, 64)
    for window, sinks in ((-1, 0), (5, -1)):
        refused("sharq_paged_attention_windowed", (ONE, 64, 64, 1, ctypes.byref(cache), ONE, 1.0, window, sinks, ONE, None, 0, None, None), "negative")


def test_a_cache_whose_pages_are_handed_out_on_the_device():
    cos, sin = rope_tables(40, 64, 1e4, torch.device("cpu"))
    cache = PagedKVCache(1, 2, 64, 3, 40, cos, sin, 8, pages=7, on_device=True)
    assert cache.lengths is None and cache.free_pages.tolist() == [6, 5, 4, 3, 2, 1, 0] and cache.free_count.tolist() == [7]
    assert cache.held_table().shape == (3, 5)
    for call in (lambda: cache.reserve([1, 0, 0]), lambda: cache.advance([1, 0, 0]), lambda: cache.prompt_step(2)):
        with pytest.raises(RuntimeError, match="device"):
            call()
    with pytest.raises(RuntimeError, match="CUDA"):  # the kernel does it, and there is no other way
        cache.plan(torch.ones(3, dtype=torch.int32), 3)
    with pytest.raises(IndexError):
        cache.free(3)
    with pytest.raises(RuntimeError, match="host"):
        PagedKVCache(1, 2, 64, 3, 40, cos, sin, 8).plan(torch.ones(3, dtype=torch.int32), 3)


def test_rules_without_a_history():
    for rules in (LogitRules(), LogitRules(tokens=torch.zeros(2, 0, dtype=torch.int64), lengths=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="no history"):
            rules.append_(torch.zeros(2, dtype=torch.int64))
    rules = LogitRules(tokens=torch.zeros(2, 3, dtype=torch.int64), lengths=torch.tensor([1, 3], dtype=torch.int32))
    rules.append_(torch.tensor([7, 8]))
    assert rules.tokens.tolist() == [[0, 7, 0], [0, 0, 8]] and rules.lengths.tolist() == [2, 4]


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (100, 1)])
def test_the_window_of_the_library_composition(window, sinks):
    cfg = DecoderConfig(heads=4, kv_heads=2, head_dim=16)
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(2 * 9, 8 * 16, generator=g)
    cos, sin = (x.float() for x in rope_tables(9, 16, 1e4, torch.device("cpu")))
    got = _attention(qkv, 2, 9, 4, 2, 16, cos, sin, False, None, window, sinks).view(2, 9, 4, 16)
    turned = lambda x: x * cos[:, None] + torch.cat((-x[..., 8:], x[..., :8]), -1) * sin[:, None]  # noqa: E731
    for b in range(2):
        x = qkv.view(2, 9, 8, 16)[b]
        q, k, v = turned(x[:, :4]), turned(x[:, 4:6]), x[:, 6:]
        for p in range(9):
            j = [i for i in range(p + 1) if p - i < window or i < sinks]
            for h in range(cfg.heads):
                w = torch.softmax(k[j, h // 2] @ q[p, h] / 4, 0)
                assert torch.allclose(got[b, p, h], w @ v[j, h // 2], atol=1e-5)


def test_waits_of_the_prompt_attention_are_bounded():
    """Every wait ends by itself: a phase, another's abort, or the limit; and what is on its way when one gave up is waited for, with a limit."""
    code = _code(CSRC / "prompt_attention.cu")
    wait = _block(code, code.index("bool wait_for("))
    assert "clock64() - start > ptx::kWaitLimitCycles" in wait and "*abort_flag != 0" in wait
    assert "mbar_wait(" not in code and len(re.findall(r"while \(", code.replace(wait, ""))) <= 1  # the loader's loop over its stretch
    assert code.count("ptx::mbar_drain(") == 3
    # a warp that waits leaves its loops together
    assert all("__all_sync" in code[m.end():m.end() + 220] for m in re.finditer(r"if \(!wait_for\((s_full|v_ok|o_full)", code))
