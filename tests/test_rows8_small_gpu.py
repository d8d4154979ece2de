"""Attention over a cache held in 8 bits where numbers are far apart or small: factors of a page's scores that underflow,
queries far below 1 and with one entry far above the others, a weight far above many,
queries that are no numbers (GPU)."""
import numpy as np
import pytest
import torch

from test_rows8_gpu import DT, HELD, STEPS, Batch, K, attend_by, check

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


def one_above(S, G, D, n, held, nats):
    """S sequences of n positions: position 5 scores ``nats`` for a query whose first entry is 1, all others 0; its value is 1 in the
    first dim, the others' are 1 in all dims but that."""
    k = K()
    P = -(-n // 64)
    table = torch.randperm(S * P).to(torch.int32).view(S, P).cuda()
    kk, vv = (k.Rows8(torch.zeros((S * P, G, 64, D), dtype=torch.uint8, device="cuda").view(HELD[held]), torch.ones((S * P, G, 64), device="cuda"))
              for _ in range(2))
    one = 1 if held == "int8" else 0x38           # the code of 1
    first = table[:, 0].long()
    kk.codes.view(torch.uint8)[first, :, 5, 0] = one
    kk.scales[first, :, 5] = nats
    values = vv.codes.view(torch.uint8)
    values.fill_(one)
    values[..., 0] = 0
    values[first, :, 5] = 0
    values[first, :, 5, 0] = one
    return table, kk, vv


def of_the_last(kernel, dtype, table, k, v, H, n, new):
    """Attention of the last ``new`` of n tokens of every sequence, with queries whose first entry is 1 and softmax scale 1."""
    from llmi_b200.engine.batch import StepContext, short_message
    S, G, D = table.shape[0], k.codes.shape[1], k.codes.shape[3]
    cu = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    c = StepContext()
    c.tok_seq, c.tok_pos = cu([s for s in range(S) for _ in range(new)]), cu([p for s in range(S) for p in range(n - new, n)])
    c.seq_q_start, c.seq_kv_len = cu([s * new for s in range(S + 1)]), cu([n] * S)
    c.n_tokens, c.n_seqs, c.max_q_len, c.decode = S * new, S, new, new == 1
    c.short_message = 0 if c.decode else short_message(new)
    q = torch.zeros(S * new, H, D, dtype=DT[dtype], device="cuda")
    q[..., 0] = 1.0
    out = torch.full((S * new, H * D), 7.0, dtype=DT[dtype], device="cuda")
    K().attention8(q.view(S * new, -1), out, k, v, c, table, H, G, D, 1.0, kernel=kernel)
    K().check_device_errors("cuda:0")
    return out


@pytest.mark.parametrize("kernel,dtype,S,G,H,D,n,new", [
    # (a block for each sequence and kv head, and many blocks for one)
    ("rows", "float32", 3, 32, 32, 64, 32000, 1), ("rows", "float32", 6, 16, 16, 128, 16000, 1), ("rows", "float32", 1, 1, 1, 64, 100000, 1),
    ("rows", "bfloat16", 6, 32, 32, 64, 32000, 1), ("rows", "bfloat16", 12, 16, 16, 128, 16000, 1), ("rows", "bfloat16", 1, 1, 1, 64, 100000, 1),
    ("prompt", "bfloat16", 3, 32, 32, 64, 32000, 3), ("prompt", "bfloat16", 6, 16, 32, 128, 16000, 20), ("prompt", "bfloat16", 1, 1, 1, 64, 100000, 200),
    ("any", "float32", 1, 1, 1, 64, 100000, 3)])
@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
def test_one_key_far_above_many(kernel, dtype, S, G, H, D, n, new, held):
    """One key 17.5 nats above tens of thousands, whose weights count together.

    Tolerances: 2^-17 as elsewhere; a sum of n weights is n / 64 additions a thread or fewer, each rounded by 2^-24 of it; bf16: weights
    and values are off by 2^-11 each, a weight far below the largest by 2^-32 of that, and the output by 2^-8."""
    nats = 17.5
    table, k, v = one_above(S, G, D, n, held, nats)
    out = of_the_last(kernel, dtype, table, k, v, H, n, new)
    others = torch.arange(n - new, n, dtype=torch.float64) * np.exp(-nats)
    want = (others / (others + 1.0)).repeat(S)[:, None, None].repeat(1, H, D)
    want[..., 0] = 1.0 - want[..., 0]
    off = (out.double().cpu().view(-1, H, D) - want).abs()
    tol = 2.0 ** -17 + n / 64 * 2.0 ** -24 * want + (2.0 ** -24 * want if dtype == "float32" else (2.0 ** -10 + 2.0 ** -8) * want + n * 2.0 ** -32)
    assert bool((off <= tol).all()), (float((off / tol).max()), float(off[..., 0].max()), float(off[..., 1:].max()))


@pytest.mark.parametrize("kernel,dtype", [("rows", "float32"), ("rows", "bfloat16"), ("prompt", "bfloat16"), ("any", "float32")])
@pytest.mark.parametrize("D", [64, 128])
def test_many_values_near_the_least_that_there_are(kernel, dtype, D):
    """100,000 values of 127 * 2^-107, next to what counts as zero, and weights that grow late by less than moves a running maximum: the sum
    of weights relative to it stays a number of 32 bits.  All values are equal, so the output is that value; it is off by 2^-11 for each
    of weights and values, 2^-8 or 2^-24 for the output, and n / 64 additions."""
    k, n, G = K(), 100000, 2
    P = -(-n // 64)
    table = torch.randperm(P).to(torch.int32).view(1, P).cuda()
    kk, vv = (k.Rows8(torch.full((P, G, 64, D), c, dtype=torch.int8, device="cuda"), torch.full((P, G, 64), s, device="cuda"))
              for c, s in ((1, 0.0), (127, 2.0 ** -107)))
    kk.scales[table[0, 1:].long()] = 7.9 * float(np.log(2.0))          # scores of 0 on the first page, 7.9 (to base 2) on the others
    out = of_the_last(kernel, dtype, table, kk, vv, 2 * G, n, 40 if kernel == "prompt" else 1).double().cpu()
    want = 127 * 2.0 ** -107
    tol = (2.0 ** -10 + 2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -17) + n / 64 * 2.0 ** -24
    assert bool(((out - want).abs() <= tol * want).all()), (float(out.min() / want), float(out.max() / want))


@pytest.mark.parametrize("kernel,dtype", [("rows", "bfloat16"), ("prompt", "bfloat16"), ("any", "bfloat16"), ("rows", "float32")])
@pytest.mark.parametrize("H,G,D,step", [(4, 2, 64, "prompts"), (8, 2, 128, "messages"), (4, 4, 128, "single tokens")])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_queries_that_are_not_finite_reach_only_their_rows(kernel, dtype, H, G, D, step, bad):
    """They are NaN, as a softmax over infinite scores is; with -infinity and keys above zero all of a row's scores are that."""
    b = Batch(STEPS[step], G, D, "int8", seed=3)
    b.fill()
    b.k.codes[..., 7] = 5
    q = torch.tensor(b.rng.normal(size=(b.T, H, D))).to(DT[dtype]).cuda()
    hit = torch.zeros(b.T, H, dtype=torch.bool, device="cuda")
    hit[::3, 1] = hit[1, 2] = True
    outs = []
    for x in (q, torch.where(hit[..., None] & (torch.arange(D, device="cuda") == 7), bad, q)):
        out = torch.full((b.T, H * D), 7.0, dtype=DT[dtype], device="cuda")
        K().attention8(x.view(b.T, -1), out, b.k, b.v, b.ctx, b.table, H, G, D, D ** -0.5, kernel=kernel)
        K().check_device_errors("cuda:0")
        outs.append(out.view(b.T, H, D))
    assert bool(outs[1][hit].isnan().all())
    off = (outs[1][~hit].double() - outs[0][~hit].double()).abs()
    # (the other rows' maxima may move on other pages: two roundings of the output)
    assert bool((off <= 2.0 ** -7 * outs[0][~hit].double().abs() + 2.0 ** -9).all())
