"""Attention over a cache held in 8 bits where numbers are far apart or small: factors of a page's scores that underflow,
queries far below 1 and with one entry far above the others (GPU)."""
import numpy as np
import pytest
import torch

from test_rows8_gpu import DT, STEPS, Batch, K, attend_by, check

pytestmark = pytest.mark.gpu


def times_keys(b, f, since=0):
    """Every key from its sequence's position ``since`` on (below 0: from that many pages ahead of its last one) f times as large;
    f = 0: with codes of zero, as the append leaves them."""
    for i, (n, h) in enumerate(b.lens):
        if h:
            p = np.arange(max(0, (h - 1) // 64 + 1 + since) * 64 if since < 0 else since, h)
            page, row = torch.tensor(b.table_np[i][p // 64]).long().cuda(), torch.tensor(p % 64).cuda()
            b.k.scales[page, :, row] *= f
            if f == 0.0:
                b.k.codes.view(torch.uint8)[page, :, row] = 0
            b.kx[i][p] *= f


@pytest.mark.parametrize("kernel", ["rows", "prompt", "any"])
@pytest.mark.parametrize("H,G,D,step", [(4, 2, 64, "prompts"), (8, 2, 128, "messages")])
@pytest.mark.parametrize("queries,keys,scale", [(2.0 ** -60, 0.0, None), (2.0 ** -70, 2.0 ** -80, None), (1.0, 0.0, 0.0), (1.0, 0.0, 1e-30),
                                                (1.0, 2.0 ** -60, 1e-30), (0.0, 0.0, -0.2)])
def test_scores_whose_factor_is_tiny(kernel, H, G, D, step, queries, keys, scale):
    """Queries, keys and softmax scales whose product is 0 in 32 bits: a mean of what is seen, not NaN, in the page that is partly masked."""
    b = Batch(STEPS[step], G, D, "int8", seed=3)
    b.fill()
    times_keys(b, keys, since=-1)
    q = torch.tensor(b.rng.normal(size=(b.T, H * D)) * queries).to(torch.bfloat16).cuda()
    scale = D ** -0.5 if scale is None else scale
    check(b, H, q, attend_by(kernel, b, H, q, 0, scale), "bfloat16", 0, scale)


@pytest.mark.parametrize("kernel,dtype", [("rows", "bfloat16"), ("prompt", "bfloat16"), ("any", "bfloat16"), ("rows", "float32")])
@pytest.mark.parametrize("H,G,D,step", [(4, 2, 64, "prompts"), (8, 2, 128, "messages")])
def test_queries_far_below_one(kernel, dtype, H, G, D, step):
    """Queries around 2^-100 and keys around 2^100: scores of ordinary size."""
    b = Batch(STEPS[step], G, D, "int8", seed=3)
    b.fill()
    times_keys(b, 2.0 ** 100)
    q = torch.tensor(b.rng.normal(size=(b.T, H * D)) * 2.0 ** -100).to(DT[dtype]).cuda()
    out = torch.full((b.T, H * D), 7.0, dtype=DT[dtype], device="cuda")
    K().attention8(q, out, b.k, b.v, b.ctx, b.table, H, G, D, D ** -0.5, kernel=kernel)
    K().check_device_errors("cuda:0")
    check(b, H, q, out, dtype)


@pytest.mark.parametrize("kernel,dtype,ratio", [("rows", "bfloat16", 22), ("prompt", "bfloat16", 22), ("any", "bfloat16", 22), ("rows", "float32", 14)])
@pytest.mark.parametrize("H,G,D,step", [(4, 2, 64, "prompts"), (8, 2, 128, "messages")])
def test_queries_with_one_entry_far_above_the_others(kernel, dtype, ratio, H, G, D, step):
    """The entry that sticks out meets zeros in every key: the scores are those of the others, 2^-ratio as large."""
    b = Batch(STEPS[step], G, D, "int8", seed=3)
    b.fill()
    b.k.codes[..., 5] = 0
    for x in b.kx:
        x[..., 5] = 0.0
    q = b.rng.normal(size=(b.T, H, D)) * 1.5
    q[..., 5] = 2.0 ** ratio
    q = torch.tensor(q.reshape(b.T, H * D)).to(DT[dtype]).cuda()
    out = torch.full((b.T, H * D), 7.0, dtype=DT[dtype], device="cuda")
    K().attention8(q, out, b.k, b.v, b.ctx, b.table, H, G, D, D ** -0.5, kernel=kernel)
    K().check_device_errors("cuda:0")
    check(b, H, q, out, dtype)
