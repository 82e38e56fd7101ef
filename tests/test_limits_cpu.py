"""The largest sizes of the serving step's operators, refused before any launch."""
import ctypes

from tests.test_serving_step_cpu import ONE, refused


def test_sequences_of_prompt_attention():
    """More than the walk through their offsets gets through before the waits of the other warps run out."""
    good = dict(q=ONE, q_row=128, q_head=64, k=ONE, k_row=64, k_head=64, v=ONE, v_row=64, v_head=64, rows=10, k_rows=10, heads=2, kv_heads=1, head_dim=64,
                offsets=ONE, k_offsets=None, sequences=1, window=0, sinks=0, scale=1.0, out=ONE, fill=0, workspace=None, workspace_bytes=0, flag=None, stream=None)
    for sequences in (2 ** 24 + 1, 2 ** 28, 2 ** 31 - 1):
        refused("sharq_prompt_attention", {**good, "sequences": sequences}.values(), "2^24")


class Rules(ctypes.Structure):
    _fields_ = [("tokens", ctypes.c_void_p), ("tokens_stride", ctypes.c_int64), ("width", ctypes.c_int), ("wide", ctypes.c_int), ("lengths", ctypes.c_void_p),
                ("prompt_lengths", ctypes.c_void_p), ("repetition", ctypes.c_void_p), ("presence", ctypes.c_void_p), ("frequency", ctypes.c_void_p),
                ("bias_offsets", ctypes.c_void_p), ("bias_ids", ctypes.c_void_p), ("bias_values", ctypes.c_void_p), ("biases", ctypes.c_int),
                ("mask", ctypes.c_void_p), ("mask_stride", ctypes.c_int64)]


def test_histories_and_biases_of_adjust_logits():
    """A thread's index runs some thousands beyond the last token or bias, which must not pass 2^31."""
    for n in (2 ** 30 + 1, 2 ** 31 - 4096, 2 ** 31 - 1):
        for said, kw in (("width", dict(tokens=256, lengths=256, width=n)), ("biases", dict(bias_offsets=256, bias_ids=256, bias_values=256, biases=n))):
            refused("sharq_adjust_logits", (ONE, 9, ONE, 9, 2, 9, 0, ctypes.byref(Rules(**kw)), None, None), said)
