"""The largest sizes of the serving step's operators, refused before any launch."""
from tests.test_serving_step_cpu import ONE, refused


def test_sequences_of_prompt_attention():
    """More than the walk through their offsets gets through before the waits of the other warps run out."""
    good = dict(q=ONE, q_row=128, q_head=64, k=ONE, k_row=64, k_head=64, v=ONE, v_row=64, v_head=64, rows=10, k_rows=10, heads=2, kv_heads=1, head_dim=64,
                offsets=ONE, k_offsets=None, sequences=1, window=0, sinks=0, scale=1.0, out=ONE, fill=0, workspace=None, workspace_bytes=0, flag=None, stream=None)
    for sequences in (2 ** 24 + 1, 2 ** 28, 2 ** 31 - 1):
        refused("sharq_prompt_attention", {**good, "sequences": sequences}.values(), "2^24")
