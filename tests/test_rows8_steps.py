"""How a step over a cache held in 8 bits is laid out for the prompt kernel, and which heads such a cache is offered for (no GPU)."""
import numpy as np

from llmi_b200.ops.kernels import _prompt8_pages, prompt8_parts


def test_pages_that_a_block_sees():
    """Against every block of a message of ``q`` tokens behind ``h`` positions: never fewer than it sees, and reached."""
    rng = np.random.default_rng(3)
    for _ in range(300):
        group, q, window = int(rng.integers(1, 41)), int(rng.integers(1, 400)), int(rng.choice([1, 2, 63, 64, 65, 66, 200, 512, 5000]))
        table, most = 500, 0
        for h in range(6000, 6064):
            for row0 in range(0, q * group, 256):
                first, last = h + row0 // group, h + min(row0 + 255, q * group - 1) // group
                most = max(most, last // 64 - max(0, first - window + 1) // 64 + 1)
        assert most <= _prompt8_pages(table, window, group, q) <= most + 1
    assert _prompt8_pages(500, 0, 4, 300) == 500 and _prompt8_pages(7, 4000, 4, 300) == 7


def test_parts_follow_the_window():
    """300 tokens of 32 heads by 8 of 128, 500 pages in the table: many parts, but none under a window of eight pages."""
    assert prompt8_parts(1200, 8, 128, 1, _prompt8_pages(500, 0, 4, 300), 300, 148) > 4
    assert prompt8_parts(1200, 8, 128, 1, _prompt8_pages(500, 512, 4, 300), 300, 148) == 1


def test_attention_plans_with_the_window(monkeypatch):
    """What attention8 asks prompt8_parts for is what a block sees under the call's window."""
    import types

    import torch

    from llmi_b200.ops import kernels as k
    asked = []

    class Stop(Exception):
        pass

    def parts(*a):
        asked.append(a)
        raise Stop
    monkeypatch.setattr(k, "_check8", lambda *a: 0)
    monkeypatch.setattr(k, "prompt8_parts", parts)
    monkeypatch.setattr(k, "sm_count", lambda: 148)
    rows = k.Rows8(torch.zeros((1, 8, 64, 128), dtype=torch.int8), torch.zeros((1, 8, 64)))
    i = torch.zeros(2, dtype=torch.int32)
    ctx = types.SimpleNamespace(tok_seq=i, tok_pos=i, seq_q_start=i, seq_kv_len=i, n_tokens=300, decode=False, short_message=0)
    q = torch.zeros((300, 32 * 128), dtype=torch.bfloat16)
    for window in (0, 512):
        try:
            k.attention8(q, torch.zeros_like(q), rows, rows, ctx, torch.zeros((1, 500), dtype=torch.int32), 32, 8, 128, 0.1, window, kernel="prompt")
        except Stop:
            pass
    assert [a[4] for a in asked] == [500, _prompt8_pages(500, 512, 4, 300)]


def test_heads_that_the_kernels_do_not_take_get_no_such_cache():
    """Refused where the cache is made, not in its first step."""
    import types

    from llmi_b200.parts.attention import GQAttention
    position = types.SimpleNamespace(fused_rotation=lambda: (None, 0))
    assert [GQAttention.holds_8bit.fget(types.SimpleNamespace(position=position, head_dim=d)) for d in (64, 256, 257, 320)] == [True, True, False, False]
