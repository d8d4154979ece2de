"""Attention over a cache held in 8 bits by the kernel for few rows: steps of several prompts, long histories (GPU)."""
import pytest
import torch

from test_rows8_gpu import DT, Batch, K, check

pytestmark = pytest.mark.gpu


def by_rows(b, H, q, dtype):
    out = torch.full((b.T, H * b.D), 7.0, dtype=DT[dtype], device="cuda")
    K().attention8(q, out, b.k, b.v, b.ctx, b.table, H, b.G, b.D, b.D ** -0.5, kernel="rows")
    K().check_device_errors("cuda:0")
    return out


PROMPTS = {  # (new tokens, positions held)
    "equal": [(512, 512)] * 8,
    "a prompt among single tokens": [(1, 5 + 3 * i) for i in range(40)] + [(700, 700)] + [(1, 70 + i) for i in range(40)],
    "messages and padding": [(0, 0), (3, 40), (0, 0), (66, 66), (2, 300), (65, 200), (0, 0)],
}


@pytest.mark.parametrize("dtype,H,G,D", [("float32", 4, 1, 64), ("float32", 4, 1, 128), ("float32", 3, 3, 64), ("bfloat16", 10, 2, 64), ("bfloat16", 8, 1, 128)])
@pytest.mark.parametrize("step", PROMPTS)
def test_steps_of_several_prompts(dtype, H, G, D, step):
    """Row tiles are counted over the whole step: a prompt beside many sequences, or several prompts, are taken."""
    b = Batch(PROMPTS[step], G, D, "int8", seed=6, pad_tokens=3)
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, H * D)) * 1.5).to(DT[dtype]).cuda()
    check(b, H, q, by_rows(b, H, q, dtype), dtype)


@pytest.mark.parametrize("dtype,H,G,D,step", [("bfloat16", 16, 1, 64, [(1, 100001)]), ("bfloat16", 4, 1, 128, [(3, 20011)]), ("float32", 6, 1, 64, [(1, 100001)]),
                                              ("float32", 4, 2, 128, [(1, 30000), (2, 100)]), ("bfloat16", 9, 3, 64, [(1, 60001), (1, 7), (2, 30000)])])
@pytest.mark.parametrize("size", [1.0, 12.0])
def test_long_histories(dtype, H, G, D, step, size):
    """A (sequence, kv head) in up to 200 parts, which are joined 32 and 8 at a time; with scores of ordinary size, and of 12 times that:
    parts whose maxima are far apart."""
    b = Batch(step, G, D, "int8", seed=8)
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, H * D)) * size).to(DT[dtype]).cuda()
    check(b, H, q, by_rows(b, H, q, dtype), dtype)
