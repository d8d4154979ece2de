"""Attention over a cache held in 8 bits by the kernel for few rows: steps of several prompts (GPU)."""
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
