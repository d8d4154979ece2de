"""The append to and the attention over a cache held in 8 bits, against plain 64-bit statements (plain_rows8.py), and models that
keep such a cache against the plain decoder with the same held rows (GPU).

Tolerances.  A code may be off by half its step beyond what the arithmetic before it is off (fp32 products of the rotation: 2^-20 of
the row's largest number covers them).  An attention output is a mean of values with softmax weights: scores that are off by d change
it by at most 2 d of the largest value (each weight by a factor within exp(+-d), their sum too); d is at most (2^-11 + 2^-18) of sum
|q_d k_d| * scale where keys are made fp16 numbers (half a step of fp16 is 2^-11), 2^-18 of it in fp32.  Weights and values made fp16
add 2^-11 each, fp32 sums over thousands of keys 2^-17; the result is rounded once to the output's type (bf16: 2^-8 of it).
"""

import numpy as np
import pytest
import torch

import plain_llama as P
import plain_rows8 as R

pytestmark = pytest.mark.gpu

DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
HELD = {"int8": torch.int8, "float8_e4m3": torch.float8_e4m3fn}
POISON = {"int8": 0x80, "float8_e4m3": 0x7F}          # -128 is no code of a row, 0x7f is a NaN


def K():
    from llmi_b200.ops import kernels
    return kernels


def pool(held, n_pages, G, D):
    """Pages that are all poison: codes that no row has, scales that are NaN."""
    K_ = K()
    make = lambda: K_.Rows8(torch.full((n_pages, G, 64, D), POISON[held], dtype=torch.uint8, device="cuda").view(HELD[held]),  # noqa: E731
                            torch.full((n_pages, G, 64), float("nan"), device="cuda"))
    return make(), make()


def codes_of(rows):
    return rows.codes.double().cpu().numpy() if rows.codes.dtype != torch.int8 else rows.codes.cpu().numpy().astype(np.float64)


class Batch:
    """A step over paged sequences: ``lens`` = [(new tokens, positions held behind the step)]; (0, 0): a padding sequence.
    ``pad_tokens``: token rows of no sequence at the end."""

    def __init__(self, lens, G, D, held, seed=0, pad_tokens=0, extra_pages=3, table_extra=1):
        rng = np.random.default_rng(seed)
        self.lens, self.G, self.D, self.held, self.rng = lens, G, D, held, rng
        n_pages = [-(-h // 64) for _, h in lens]
        self.n_pool = sum(n_pages) + extra_pages
        ids = rng.permutation(self.n_pool)
        table = np.full((len(lens), max(n_pages + [1]) + table_extra), -1, dtype=np.int32)
        at = 0
        for i, n in enumerate(n_pages):
            table[i, :n] = ids[at:at + n]
            at += n
        self.table_np = table
        seq, pos, start = [], [], [0]
        for i, (n, h) in enumerate(lens):
            seq += [i] * n
            pos += list(range(h - n, h))
            start.append(start[-1] + n)
        self.n_real = len(seq)
        seq += [-1] * pad_tokens
        pos += [0] * pad_tokens
        cu = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        self.seq, self.pos = np.array(seq), np.array(pos)
        self.table = cu(table)
        self.T = len(seq)
        most = max(n for n, _ in lens)
        from llmi_b200.engine.batch import StepContext, short_message
        c = self.ctx = StepContext()
        c.tok_seq, c.tok_pos, c.seq_q_start, c.seq_kv_len = cu(seq), cu(pos), cu(start), cu([h for _, h in lens])
        c.n_tokens, c.n_seqs, c.max_q_len, c.decode = self.T, len(lens), most, most <= 1
        c.short_message = 0 if c.decode else short_message(most)
        self.k, self.v = pool(held, self.n_pool, G, D)

    def fill(self, size=1.0, only_seen=0):
        """Random rows at every position that a sequence holds (under a window of ``only_seen`` positions only those its tokens see);
        everything else stays poison.  Keeps what they stand for: self.kx, self.vx [sequence][N, G, D]."""
        self.kx, self.vx = [], []
        for i, (n, h) in enumerate(self.lens):
            both = []
            for rows in (self.k, self.v):
                x = self.rng.normal(size=(h, self.G, self.D)) * size * np.exp(0.5 * self.rng.normal(size=(h, self.G, 1)))
                codes, scale = R.held(x, self.held)
                scale = scale.astype(np.float32).astype(np.float64)
                lo = max(0, h - n - only_seen + 1) if only_seen else 0
                p = np.arange(lo, h)
                page, row = torch.tensor(self.table_np[i][p // 64]).long().cuda(), torch.tensor(p % 64).cuda()
                c = torch.tensor(codes[lo:]).to(HELD[self.held]).cuda()
                rows.codes.view(torch.uint8)[page, :, row] = c.view(torch.uint8)
                rows.scales[page, :, row] = torch.tensor(scale[lo:], dtype=torch.float32).cuda()
                both.append(codes * scale[..., None])
            self.kx.append(both[0])
            self.vx.append(both[1])

    def plain(self, q, scale, window=0):
        """q [T, H, D] float64 -> (out, sums, most) over all real tokens."""
        parts, at = [], 0
        for i, (n, h) in enumerate(self.lens):
            if n:
                parts.append(R.attention(q[at:at + n], self.kx[i], self.vx[i], np.arange(h - n, h), scale, window))
            at += n
        return tuple(np.concatenate([p[j] for p in parts]) for j in range(3))


def tolerance(out, sums, most, dtype):
    d = (2.0 ** -18 + (2.0 ** -11 if dtype == "bfloat16" else 0.0)) * sums
    rest = 2.0 ** -17 + (2.0 ** -10 if dtype == "bfloat16" else 0.0)
    return (2.0 ** -8 * np.abs(out) if dtype == "bfloat16" else 2.0 ** -24 * np.abs(out)) + ((2 * d + rest) * most)[..., None]


# ----------------------------------------------------------------------------- the append

APPENDS = [  # (heads, kv heads, head size, rotary size)
    (9, 3, 64, 64), (32, 8, 128, 128), (3, 3, 12, 12), (5, 1, 24, 16), (2, 2, 256, 256), (4, 2, 96, 0), (1, 1, 1, 0), (4, 4, 64, 32),
    (4, 2, 32, 32), (3, 1, 100, 100)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("H,G,D,rot", APPENDS)
def test_append(dtype, held, H, G, D, rot):
    b = Batch([(1, 1), (70, 200), (0, 0), (2, 65), (1, 100001)], G, D, held, seed=H * D, pad_tokens=3)
    qkv = torch.tensor(b.rng.normal(size=(b.T, (H + 2 * G) * D))).to(DT[dtype]).cuda()
    rows = qkv.view(b.T, H + 2 * G, D)
    rows[1, H:] = 0.0                                   # zeros, tiny and huge rows, rows that are not finite
    rows[2, H:] *= 2.0 ** -110
    rows[3, H:] *= 1e30
    rows[4, H, D // 2] = float("inf")
    rows[5, H + G, 0] = float("nan")
    rows[6, H:] *= 2.0 ** -90
    before = qkv.clone()
    wide = torch.full((b.T, H * D + 8), 7.0, dtype=DT[dtype], device="cuda")          # (strided rows)
    q_out = wide[:, :H * D]
    inv = torch.tensor([10000.0 ** (-2.0 * i / max(rot, 1)) for i in range(rot // 2)], dtype=torch.float32, device="cuda")
    K().rope_store8(qkv, q_out, inv if rot else None, rot, b.ctx.tok_seq, b.ctx.tok_pos, b.table, b.k, b.v, H, G, D)
    assert torch.equal(qkv.view(torch.uint8), before.view(torch.uint8))
    x = before.double().cpu().numpy().reshape(b.T, H + 2 * G, D)
    turned = x.copy()
    if rot:
        with np.errstate(invalid="ignore"):
            turned[:, :H + G, :rot] = P.rope(x[:, :H + G, :rot], b.pos, inv.cpu().numpy())
    got_q = q_out.double().cpu().numpy().reshape(b.T, H, D)
    n = b.n_real
    u = 2.0 ** -8 if dtype == "bfloat16" else 0.0
    assert (np.abs(got_q[:n] - turned[:n, :H]) <= u * np.abs(turned[:n, :H]) + 2.0 ** -21 * np.abs(x[:n, :H]).max(-1, keepdims=True)).all()
    assert (got_q[n:] == 7.0).all() and (wide[:, H * D:] == 7.0).all()
    page, row = b.table_np[b.seq[:n], b.pos[:n] // 64], b.pos[:n] % 64
    for cache, want in ((b.k, turned[:n, H:H + G]), (b.v, x[:n, H + G:])):
        codes, scales = codes_of(cache)[page, :, row], cache.scales.double().cpu().numpy()[page, :, row]
        ref_codes, ref_scale = R.held(want, held)
        assert np.array_equal(np.isnan(scales), np.isnan(ref_scale))
        fine = ~np.isnan(ref_scale)
        assert (codes[~fine] == 0).all() and (codes[ref_scale == 0] == 0).all() and (scales[ref_scale == 0] == 0).all()
        assert (np.abs(scales - ref_scale)[fine] <= 2.0 ** -20 * ref_scale[fine]).all()
        fine &= ref_scale > 0                 # (rows below 2^-100 are zeros by definition, as was asserted)
        most = ref_scale * R.MOST[held]
        off = np.abs(codes * scales[..., None] - want)[fine]
        assert (off <= (R.half_step(codes, scales, held) * (1 + 2.0 ** -20) + 2.0 ** -20 * most[..., None])[fine]).all()
        assert (np.abs(codes).max(-1)[fine] == R.MOST[held]).all()
        # nothing else was written
        touched = np.zeros(cache.scales.shape, dtype=bool)
        touched[page, :, row] = True
        raw = cache.codes.view(torch.uint8).cpu().numpy()
        assert (raw[~touched] == POISON[held]).all() and torch.isnan(cache.scales.cpu()[torch.from_numpy(~touched)]).all()


@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("D", [64, 128, 40])
def test_append_without_rotation_gives_the_formula_s_codes(held, D):
    """fp32 rows, nothing turned: scale and codes are the formula's fp32 numbers, bit for bit."""
    G = 4
    b = Batch([(300, 300)], G, D, held)
    qkv = torch.randn(b.T, 6 * G * D // 2, device="cuda")
    q_out = torch.empty(b.T, G * D, device="cuda")
    K().rope_store8(qkv, q_out, None, 0, b.ctx.tok_seq, b.ctx.tok_pos, b.table, b.k, b.v, G, G, D)
    assert torch.equal(q_out, qkv[:, :G * D])
    page, row = torch.tensor(b.table_np[0][b.pos // 64]).long().cuda(), torch.tensor(b.pos % 64).cuda()
    for cache, x in ((b.k, qkv[:, G * D:2 * G * D]), (b.v, qkv[:, 2 * G * D:])):
        x = x.reshape(b.T, G, D).cpu()        # (the CPU divides; torch's division by a number on the GPU is a product with its reciprocal)
        scale = x.abs().amax(-1) / torch.full((), R.MOST[held])
        y = x * (torch.ones(()) / scale)[..., None]
        want = torch.round(y).clamp(-127, 127).to(torch.int8) if held == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)
        assert torch.equal(cache.scales[page, :, row].cpu(), scale)
        assert torch.equal(cache.codes[page, :, row].view(torch.uint8).cpu(), want.view(torch.uint8))


def test_append_in_place_and_of_queries_only():
    H, G, D = 6, 2, 64
    b = Batch([(3, 70), (1, 5)], G, D, "int8")
    qkv = torch.randn(b.T, (H + 2 * G) * D, device="cuda").bfloat16()
    inv = torch.tensor([100.0 ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float32, device="cuda")
    apart = torch.empty(b.T, H * D, device="cuda", dtype=torch.bfloat16)
    K().rope_store8(qkv, apart, inv, D, b.ctx.tok_seq, b.ctx.tok_pos, b.table, b.k, b.v, H, G, D, write_kv=False)
    assert (b.k.codes.view(torch.uint8) == POISON["int8"]).all() and torch.isnan(b.v.scales).all()
    whole = torch.empty(b.T, H * D, device="cuda")           # fp32: the same queries before they are rounded
    K().rope_store8(qkv, whole, inv, D, b.ctx.tok_seq, b.ctx.tok_pos, b.table, b.k, b.v, H, G, D, write_kv=False)
    assert torch.equal(whole.bfloat16(), apart)
    K().rope_store8(qkv, qkv[:, :H * D], inv, D, b.ctx.tok_seq, b.ctx.tok_pos, b.table, b.k, b.v, H, G, D)
    assert torch.equal(qkv[:, :H * D], apart)


# ----------------------------------------------------------------------------- attention

SHAPES = [  # (heads, kv heads, head size)
    (9, 3, 64), (4, 4, 64), (32, 8, 128), (16, 1, 64), (40, 1, 128), (3, 3, 12), (5, 1, 24), (4, 2, 96), (2, 1, 256), (6, 2, 32)]
STEPS = {  # (new tokens, positions held)
    "one token": [(1, 1)],
    "single tokens": [(1, 1), (1, 64), (1, 65), (1, 1000), (1, 63), (1, 128), (1, 333)],
    "single tokens and padding": [(1, 70), (0, 0), (1, 3), (0, 0)],
    "messages": [(5, 5), (3, 130), (1, 64), (7, 700)],
    "a message on a long history": [(12, 3100)],
    "prompts": [(100, 100), (1, 50), (65, 190), (33, 33)],
    "a long prompt": [(517, 517)],
    "a portion": [(130, 1500)],
}


def attend(b, H, q, dtype, window=0, scale=None, rt=None):
    scale = b.D ** -0.5 if scale is None else scale
    out = torch.full((b.T, H * b.D), 7.0, dtype=DT[dtype], device="cuda")
    K().attention8(q, out, b.k, b.v, b.ctx, b.table, H, b.G, b.D, scale, window, rt=rt)
    K().check_device_errors("cuda:0")
    return out


def check(b, H, q, out, dtype, window=0, scale=None):
    scale = b.D ** -0.5 if scale is None else scale
    n = b.n_real
    got = out.double().cpu().numpy().reshape(b.T, H, b.D)
    ref, sums, most = b.plain(q[:n].double().cpu().numpy()[:, :H * b.D].reshape(n, H, b.D), scale, window)
    assert (got[n:] == 7.0).all()
    assert np.array_equal(np.isnan(got[:n]), np.isnan(ref))
    off = np.abs(got[:n] - ref)
    tol = tolerance(ref, sums, most, dtype)
    ok = (off <= tol) | np.isnan(ref)
    assert ok.all(), (float(np.nanmax(off / tol)), np.argwhere(~ok)[:5].tolist())


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("H,G,D", SHAPES)
@pytest.mark.parametrize("dtype,held", [("bfloat16", "int8"), ("bfloat16", "float8_e4m3"), ("float32", "int8"), ("float32", "float8_e4m3")])
def test_attention(dtype, held, H, G, D, step):
    b = Batch(STEPS[step], G, D, held, seed=H + D, pad_tokens=0 if step != "single tokens and padding" else 2)
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, H * D + 8)) * 1.5).to(DT[dtype]).cuda()
    check(b, H, q, attend(b, H, q, dtype), dtype)


@pytest.mark.parametrize("kernel", ["rows", "prompt", "any"])
@pytest.mark.parametrize("H,G,D,step", [(9, 3, 64, "one token"), (9, 3, 64, "a long prompt"), (8, 2, 128, "single tokens and padding"),
                                        (32, 1, 128, "messages"), (4, 4, 64, "a portion"), (6, 2, 64, "a message on a long history"),
                                        (16, 16, 128, "single tokens")])
@pytest.mark.parametrize("window", [0, 90])
def test_a_kernel_named(kernel, H, G, D, step, window):
    """Each kernel takes what the others are chosen for."""
    b = Batch(STEPS[step], G, D, "int8")
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, H * D)) * 1.5).to(torch.bfloat16).cuda()
    out = torch.full((b.T, H * D), 7.0, dtype=torch.bfloat16, device="cuda")
    K().attention8(q, out, b.k, b.v, b.ctx, b.table, H, G, D, D ** -0.5, window, kernel=kernel)
    K().check_device_errors("cuda:0")
    check(b, H, q, out, "bfloat16", window)


def attend_by(kernel, b, H, q, window=0, scale=None, table=None):
    out = torch.full((b.T, H * b.D), 7.0, dtype=torch.bfloat16, device="cuda")
    K().attention8(q, out, b.k, b.v, b.ctx, b.table if table is None else table, H, b.G, b.D, b.D ** -0.5 if scale is None else scale, window, kernel=kernel)
    K().check_device_errors("cuda:0")
    return out


@pytest.mark.parametrize("kernel", ["rows", "prompt", "any"])
@pytest.mark.parametrize("wrong", ["a table too short", "no page", "a page past the pool"])
def test_pages_that_are_not_there_reach_only_who_sees_them(kernel, wrong):
    """A sequence's rows that see such a page are NaN; nothing is read, and its neighbours and its own earlier rows stay as they are."""
    b = Batch([(3, 40), (70, 150), (1, 64)], 2, 64, "int8")
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, 4 * 64))).to(torch.bfloat16).cuda()
    want = attend_by(kernel, b, 4, q)
    table = b.table.clone()
    if wrong == "a table too short":
        table = table[:, :2].contiguous()
    else:
        table[1, 2] = -1 if wrong == "no page" else b.n_pool
    got = attend_by(kernel, b, 4, q, table=table)
    sees = torch.tensor((b.seq == 1) & (b.pos >= 128)).cuda()
    assert bool(got[sees].isnan().all()) and int(sees.sum()) == 22
    rest = got[~sees].double() - want[~sees].double()
    # (the other rows' sums may be cut otherwise: two roundings of the output)
    assert bool((rest.abs() <= 2.0 ** -7 * want[~sees].double().abs() + 2.0 ** -9).all())


@pytest.mark.parametrize("kernel", ["rows", "prompt", "any"])
def test_sequences_far_longer_than_their_table_end(kernel):
    """Lengths that no table holds: as many pages are walked as the table has."""
    b = Batch([(3, 100), (2, 60)], 2, 64, "int8")
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, 4 * 64))).to(torch.bfloat16).cuda()
    want = attend_by(kernel, b, 4, q)
    b.ctx.seq_kv_len = torch.tensor([2 ** 31 - 64, 60], dtype=torch.int32, device="cuda")
    b.ctx.tok_pos = torch.tensor([2 ** 31 - 67, 2 ** 31 - 66, 2 ** 31 - 65, 58, 59], dtype=torch.int32, device="cuda")
    got = attend_by(kernel, b, 4, q)
    assert bool(got[:3].isnan().all())
    assert bool(((got[3:].double() - want[3:].double()).abs() <= 2.0 ** -7 * want[3:].double().abs() + 2.0 ** -9).all())


@pytest.mark.parametrize("kernel", ["rows", "prompt", "any"])
@pytest.mark.parametrize("scale,window", [(0.0, 0), (-0.2, 0), (1e-30, 0), (0.125, 2 ** 31 - 1), (3.0, 2 ** 31 - 1)])
@pytest.mark.parametrize("step", ["one token", "single tokens", "messages"])
def test_scales_and_windows_at_their_ends(kernel, scale, window, step):
    b = Batch(STEPS[step], 2, 64, "int8")
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, 4 * 64))).to(torch.bfloat16).cuda()
    check(b, 4, q, attend_by(kernel, b, 4, q, window, scale), "bfloat16", 0, scale)


def test_more_sequences_than_the_kernel_for_few_rows_takes():
    b = Batch([(1, 1 + i % 5) for i in range(4200)], 1, 64, "int8")
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, 2 * 64))).to(torch.bfloat16).cuda()
    check(b, 2, q, attend(b, 2, q, "bfloat16"), "bfloat16")
    with pytest.raises(K().KernelError, match="rows"):
        attend_by("rows", b, 2, q)


@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
def test_offsets_past_32_bits(held):
    """A pool of more than 2^32 codes: its last pages give the bits that its first ones give, append and attention."""
    k = K()
    G, D, H = 8, 128, 16
    n_pool = 2 ** 32 // (G * 64 * D) + 40
    near, far = Batch([(3, 130), (1, 200), (40, 90)], G, D, held), Batch([(3, 130), (1, 200), (40, 90)], G, D, held)
    far.k, far.v = (k.Rows8(torch.empty((n_pool, G, 64, D), dtype=HELD[held], device="cuda"),
                            torch.empty((n_pool, G, 64), dtype=torch.float32, device="cuda")) for _ in range(2))
    near.fill()
    there = torch.tensor(sorted(set(near.table_np[near.table_np >= 0].tolist()))).cuda()
    for a, z in ((near.k, far.k), (near.v, far.v)):
        z.codes.view(torch.uint8)[there + n_pool - near.n_pool] = a.codes.view(torch.uint8)[there]
        z.scales[there + n_pool - near.n_pool] = a.scales[there]
    far.table = torch.where(near.table >= 0, near.table + (n_pool - near.n_pool), near.table).to(torch.int32)
    assert int(far.table.max()) * G * 64 * D > 2 ** 32
    rows = torch.tensor(near.rng.normal(size=(near.T, (H + 2 * G) * D))).to(torch.bfloat16).cuda()
    inv = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().cuda()
    for kernel in ("rows", "prompt", "any"):
        outs = []
        for b in (near, far):
            out = torch.zeros(b.T, H * D, dtype=torch.bfloat16, device="cuda")
            k.attention8(rows, out, b.k, b.v, b.ctx, b.table, H, G, D, D ** -0.5, rope=(inv, D, True), kernel=kernel)
            outs.append(out)
        k.check_device_errors("cuda:0")
        assert torch.equal(outs[0], outs[1]) and not bool(outs[0].isnan().any())
    assert torch.equal(far.k.codes.view(torch.uint8)[there + n_pool - near.n_pool], near.k.codes.view(torch.uint8)[there])
    assert torch.equal(far.v.scales[there + n_pool - near.n_pool].nan_to_num(-1.0), near.v.scales[there].nan_to_num(-1.0))


@pytest.mark.parametrize("kernel,D,dtype", [("rows", 40, "bfloat16"), ("prompt", 32, "bfloat16"), ("prompt", 64, "float32"), ("columns", 64, "bfloat16")])
def test_a_kernel_named_that_does_not_take_the_call(kernel, D, dtype):
    b = Batch([(3, 10)], 2, D, "int8")
    b.fill()
    q = torch.zeros(3, 4 * D, dtype=DT[dtype], device="cuda")
    with pytest.raises(K().KernelError, match=kernel):
        K().attention8(q, torch.zeros_like(q), b.k, b.v, b.ctx, b.table, 4, 2, D, 0.1, kernel=kernel)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200])
@pytest.mark.parametrize("H,G,D,step", [(9, 3, 64, "single tokens"), (9, 3, 64, "messages"), (8, 2, 128, "prompts"), (4, 4, 64, "a portion"),
                                        (4, 2, 32, "messages"), (32, 8, 128, "single tokens")])
@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
def test_attention_under_a_window(held, H, G, D, step, window):
    """What lies before the window of a sequence's first token is poison (its pages may be another sequence's by now)."""
    b = Batch(STEPS[step], G, D, held, seed=window)
    b.fill(only_seen=window)
    for i, (n, h) in enumerate(b.lens):
        b.table[i, :max(0, h - n - window + 1) // 64] = -1
    q = torch.tensor(b.rng.normal(size=(b.T, H * D)) * 1.5).to(torch.bfloat16).cuda()
    check(b, H, q, attend(b, H, q, "bfloat16", window), "bfloat16", window)


@pytest.mark.parametrize("H,G,D,step", [(9, 3, 64, "single tokens"), (8, 2, 128, "messages"), (4, 2, 64, "prompts"), (4, 2, 32, "messages")])
@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_rows_that_are_not_finite_reach_only_who_sees_them(dtype, held, H, G, D, step):
    b = Batch(STEPS[step], G, D, held, seed=5)
    b.fill()
    for i, (n, h) in enumerate(b.lens):       # key head 0 of one position, value head 0 of another
        for rows, x, p in ((b.k, b.kx[i], h - 1 - n // 2), (b.v, b.vx[i], h - 1 - n // 3)):
            if i % 2 == 1:
                rows.scales[b.table_np[i][p // 64], 0, p % 64] = float("nan")
                rows.codes.view(torch.uint8)[b.table_np[i][p // 64], 0, p % 64] = 0
                x[p, 0] = np.nan
    q = torch.tensor(b.rng.normal(size=(b.T, H * D))).to(DT[dtype]).cuda()
    check(b, H, q, attend(b, H, q, dtype), dtype)


@pytest.mark.parametrize("H,G,D,step", [(9, 3, 64, "single tokens"), (8, 2, 128, "messages"), (4, 2, 64, "prompts"), (4, 2, 32, "messages")])
@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("size", [1e-20, 1e-6, 1.0, 1e4, 1e12])
def test_sizes_of_values_and_of_queries(held, H, G, D, step, size):
    """Rows of very different sizes, zeros among them; queries whose product with the keys stays that of ordinary ones."""
    b = Batch(STEPS[step], G, D, held, seed=9)
    b.fill(size)
    for i, (n, h) in enumerate(b.lens):
        for rows, x in ((b.k, b.kx[i]), (b.v, b.vx[i])):
            for p in range(0, h, 3):          # every third row zero, every fifth 2^-40 as large
                f = 0.0 if p % 2 else 2.0 ** -40
                rows.scales[b.table_np[i][p // 64], :, p % 64] *= f
                x[p] *= f
    q = torch.tensor(b.rng.normal(size=(b.T, H * D)) / size).to(torch.bfloat16).cuda()
    check(b, H, q, attend(b, H, q, "bfloat16"), "bfloat16")


@pytest.mark.parametrize("H,G,D,step", [(9, 3, 64, "single tokens"), (8, 2, 128, "messages"), (4, 2, 64, "prompts"), (4, 2, 32, "messages")])
def test_peaked_and_growing_scores(H, G, D, step):
    """Scores of hundreds, whose largest comes last: the running maximum moves all along."""
    b = Batch(STEPS[step], G, D, "int8", seed=2)
    b.fill()
    for i, (n, h) in enumerate(b.lens):
        ramp = np.linspace(0.01, 1.0, h).astype(np.float32)
        for p in range(h):
            b.k.scales[b.table_np[i][p // 64], :, p % 64] *= float(ramp[p])
        f = ramp.astype(np.float64)[:, None, None]
        b.kx[i] = b.kx[i] * f
    q = torch.tensor(b.rng.normal(size=(b.T, H * D)) * 30).to(torch.bfloat16).cuda()
    check(b, H, q, attend(b, H, q, "bfloat16"), "bfloat16")


@pytest.mark.parametrize("H,G,D,step", [(9, 3, 64, "single tokens"), (32, 32, 64, "single tokens"), (8, 2, 128, "messages"), (4, 2, 64, "prompts")])
def test_the_same_call_gives_the_same_bits(H, G, D, step):
    b = Batch(STEPS[step], G, D, "float8_e4m3", seed=1)
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, H * D))).to(torch.bfloat16).cuda()
    first = attend(b, H, q, "bfloat16")
    for _ in range(20):
        assert torch.equal(attend(b, H, q, "bfloat16").view(torch.uint8), first.view(torch.uint8))


@pytest.mark.parametrize("H,G,D,step", [(9, 3, 64, "single tokens"), (32, 8, 128, "single tokens"), (8, 2, 128, "messages"), (4, 2, 64, "prompts"),
                                        (4, 2, 32, "single tokens"), (9, 3, 64, "single tokens and padding")])
@pytest.mark.parametrize("dtype,held", [("bfloat16", "int8"), ("bfloat16", "float8_e4m3"), ("float32", "int8")])
@pytest.mark.parametrize("window", [0, 100])
def test_append_and_attend_together(dtype, held, H, G, D, step, window):
    """attention8 with ``rope``: the rows it appends are rope_store8's, bit for bit; the output is that of attention over them."""
    b = Batch(STEPS[step], G, D, held, seed=4, pad_tokens=2 if step != "single tokens" else 0)
    b.fill()
    qkv = torch.tensor(b.rng.normal(size=(b.T, (H + 2 * G) * D))).to(DT[dtype]).cuda()
    before = qkv.clone()
    inv = torch.tensor([1000.0 ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float32, device="cuda")
    k, v = (K().Rows8(r.codes.clone(), r.scales.clone()) for r in (b.k, b.v))
    q = torch.empty(b.T, H * D, dtype=DT[dtype], device="cuda")
    K().rope_store8(qkv, q, inv, D, b.ctx.tok_seq, b.ctx.tok_pos, b.table, k, v, H, G, D)
    out = torch.full((b.T, H * D), 7.0, dtype=DT[dtype], device="cuda")
    K().attention8(qkv, out, b.k, b.v, b.ctx, b.table, H, G, D, D ** -0.5, window, rope=(inv, D, True))
    K().check_device_errors("cuda:0")
    assert torch.equal(qkv, before)
    for x, y in ((k, b.k), (v, b.v)):
        assert torch.equal(x.codes.view(torch.uint8), y.codes.view(torch.uint8))
        assert torch.equal(torch.nan_to_num(x.scales, nan=-1.0), torch.nan_to_num(y.scales, nan=-1.0))
    for i, (n, h) in enumerate(b.lens):       # what the new rows stand for
        p = np.arange(h - n, h)
        page, row = b.table_np[i][p // 64], p % 64
        for rows, x in ((k, b.kx[i]), (v, b.vx[i])):
            x[p] = codes_of(rows)[page, :, row] * rows.scales.double().cpu().numpy()[page, :, row][..., None]
    xq = before[:, :H * D].double().cpu().numpy().reshape(b.T, H, D)
    exact_q = P.rope(xq, b.pos, inv.cpu().numpy())[:b.n_real]
    ref, sums, most = b.plain(exact_q, D ** -0.5, window)
    got = out.double().cpu().numpy().reshape(b.T, H, D)
    assert (got[b.n_real:] == 7.0).all()
    # (the rotation's fp32 arithmetic; the rotated q is not rounded in between)
    tol = tolerance(ref, sums, most, dtype) + (2 * 2.0 ** -20 * sums * most)[..., None]
    assert (np.abs(got[:b.n_real] - ref) <= tol).all()


def test_captured_and_replayed_on_two_streams_at_once():
    """Two captured calls with no workspace of their own, replayed on two streams at once, on inputs that change in between."""
    cases = []
    for seed, (H, G, D) in enumerate(((9, 3, 64), (32, 8, 128))):
        b = Batch([(1, 3000), (1, 5), (1, 900)], G, D, "int8", seed=seed)
        b.fill()
        q = torch.tensor(b.rng.normal(size=(b.T, H * D))).to(torch.bfloat16).cuda()
        out = torch.zeros(b.T, H * D, dtype=torch.bfloat16, device="cuda")
        call = lambda b=b, H=H, q=q, out=out: K().attention8(q, out, b.k, b.v, b.ctx, b.table, H, b.G, b.D, b.D ** -0.5)  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        cases.append((b, H, q, out, graph, torch.cuda.Stream()))
    for turn in range(5):
        for b, H, q, out, graph, stream in cases:
            q.copy_(torch.tensor(b.rng.normal(size=(b.T, H * b.D))).to(torch.bfloat16))
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(10):
            for b, H, q, out, graph, stream in cases:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for b, H, q, out, graph, stream in cases:
            check(b, H, q, out, "bfloat16")


def test_a_side_stream():
    b = Batch(STEPS["single tokens"], 3, 64, "int8")
    b.fill()
    q = torch.tensor(b.rng.normal(size=(b.T, 9 * 64))).to(torch.bfloat16).cuda()
    want = attend(b, 9, q, "bfloat16")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(q)
        out = attend(b, 9, late, "bfloat16")
    side.synchronize()
    assert torch.equal(out, want)


def test_refusals():
    k = K()
    b = Batch([(1, 10)], 2, 64, "int8")
    b.fill()
    q, out = torch.zeros(1, 8 * 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device="cuda")
    call = lambda q=q, out=out, kk=b.k, vv=b.v, table=b.table, H=4, G=2, D=64, window=0: k.attention8(q, out, kk, vv, b.ctx, table, H, G, D, 0.1, window)  # noqa: E731
    call()
    other = k.Rows8(b.k.codes.view(torch.float8_e4m3fn), b.k.scales)
    for wrong in (dict(vv=other), dict(H=3), dict(D=32), dict(G=4, H=8), dict(window=-1), dict(q=q.half()), dict(out=out.float()), dict(out=out[:, ::2]),
                  dict(table=b.table.long()), dict(kk=k.Rows8(b.k.codes, b.k.scales.half())), dict(kk=k.Rows8(b.k.codes.transpose(0, 1), b.k.scales)),
                  dict(kk=k.Rows8(b.k.codes.cpu(), b.k.scales)), dict(q=q[:, :100])):
        with pytest.raises(k.KernelError):
            call(**wrong)
    i = b.ctx.tok_seq
    store = lambda qkv=q, qo=out, inv=None, rot=0, seq=i, H=4: k.rope_store8(qkv, qo, inv, rot, seq, b.ctx.tok_pos, b.table, b.k, b.v, H, 2, 64)  # noqa: E731
    store()
    for wrong in (dict(rot=64), dict(rot=3), dict(rot=66, inv=torch.zeros(64, device="cuda")), dict(seq=i.long()), dict(qo=out.half()), dict(qkv=q[:, :-1]),
                  dict(rot=64, inv=torch.zeros(16, device="cuda"))):
        with pytest.raises(k.KernelError):
            store(**wrong)


# ----------------------------------------------------------------------------- models

MODEL_TOL = {("float32", "int8"): 1e-3, ("float32", "float8_e4m3"): 4e-3, ("bfloat16", "int8"): 2.5e-2, ("bfloat16", "float8_e4m3"): 4e-2}
WIDE = {"architectures": ["LlamaForCausalLM"], "num_hidden_layers": 2, "hidden_size": 192, "num_attention_heads": 6, "num_key_value_heads": 2,
        "head_dim": 64, "intermediate_size": 256, "vocab_size": 320, "rope_theta": 10000.0, "rms_norm_eps": 1e-5, "tie_word_embeddings": True,
        "max_position_embeddings": 1024, "hidden_act": "silu"}


def plain_logits(cfg, w, tokens, held, monkeypatch):
    whole = P.attention
    with monkeypatch.context() as m:
        m.setattr(P, "attention", lambda q, k, v: whole(q, R.stands_for(k, held), R.stands_for(v, held)))
        return P.forward(cfg, w, tokens)


@pytest.mark.parametrize("name", ["A", "B", "C", "wide"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
def test_models_over_such_a_cache(model_dirs, tmp_path, monkeypatch, name, dtype, held):
    """Whole prompts, portions and single tokens of a batch: the logits are those of the plain decoder whose keys and values are
    held rows.  (Where the compute type's rounding crosses the border between two codes, the code differs: a step of one number of
    one row, which is what the tolerances leave room for.)"""
    import llmi_b200 as L
    if name == "wide":
        d = str(tmp_path)
        L.write_random_model(d, WIDE, 3, torch.float32)
    else:
        d = model_dirs(name)
    cfg, w = P.read_model(d)
    model = L.load(d, dtype)
    cache = model.new_cache(64 * 12, kv_type=held)
    for g in cache.kv_groups:
        assert g.k.dtype == HELD[held]
        g.k.view(torch.uint8).fill_(POISON[held])
        g.v.view(torch.uint8).fill_(POISON[held])
        g.k_scale.fill_(float("nan"))
        g.v_scale.fill_(float("nan"))
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, cfg["vocab_size"], n).tolist() for n in (90, 3, 70)]
    slots = [cache.alloc_slot() for _ in prompts]
    rows = [[] for _ in prompts]

    def step(parts):
        out = model.step(cache, [L.SequenceStep(slots[i], t, list(range(len(t)))) for i, t in parts]).cpu().numpy()
        at = 0
        for i, t in parts:
            rows[i].append(out[at:at + len(t)])
            at += len(t)
    step([(0, prompts[0][:40]), (1, prompts[1][:1])])
    step([(0, prompts[0][40:45]), (1, prompts[1][1:2]), (2, prompts[2][:66])])
    step([(0, prompts[0][45:87]), (2, prompts[2][66:68])])
    for t in range(2):
        step([(0, prompts[0][87 + t:88 + t]), (2, prompts[2][68 + t:69 + t])])
    step([(0, prompts[0][89:]), (1, prompts[1][2:])])
    for i, p in enumerate(prompts):
        ref = plain_logits(cfg, w, p, held, monkeypatch)
        got = np.concatenate(rows[i])
        err = np.abs(got - ref).max(axis=1) / np.abs(ref).max()
        assert float(err.max()) < MODEL_TOL[dtype, held], (i, float(err.max()))


@pytest.mark.parametrize("held", ["int8", "float8_e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_recorded_and_launch_by_launch(tmp_path, dtype, held):
    """generate() with kv_type: the recorded steps choose the same tokens as steps launched one by one."""
    import llmi_b200 as L
    L.write_random_model(str(tmp_path), WIDE, 11, torch.float32)
    model = L.load(str(tmp_path), dtype)
    prompts = [[5, 9, 1, 30, 7], list(range(100, 170)), [3]]
    out = L.generate(model, prompts, max_new=80, ignore_eos=True, kv_type=held)
    again = L.generate(model, prompts, max_new=80, ignore_eos=True, kv_type=held, use_graphs=False)
    assert out == again and all(len(o) == 80 for o in out)


def test_a_model_whose_mixers_do_not_read_such_a_cache():
    import fusazen_models as FM
    import llmi_b200 as L
    import tempfile
    with tempfile.TemporaryDirectory() as d:
        cfg = FM.CONFIGS["wide"]
        FM.write_model(d, cfg, FM.make_weights(cfg, 1), "F32")
        model = L.load(d, "float32")
        with pytest.raises(RuntimeError, match="8 bits"):
            model.new_cache(128, kv_type="int8")
        model.new_cache(128)


def test_trace_replay(tmp_path):
    """bin/trace_run's replayer over such a cache gives the step function's logits."""
    import llmi_b200 as L
    from llmi_b200.engine.trace import TraceReplayer
    L.write_random_model(str(tmp_path), WIDE, 2, torch.float32)
    model = L.load(str(tmp_path), "float32")
    rp = TraceReplayer(model, 200, kv_type="int8")
    assert rp.cache.kv_groups[0].k.dtype == torch.int8
    toks = list(range(3, 80))
    a = rp.run_step({"step": 0, "entries": [{"id": "x", "tokens": toks, "want": [76]}], "end": ["x"]})
    cache = model.new_cache(128, kv_type="int8")
    b = model.step(cache, [L.SequenceStep(cache.alloc_slot(), toks, [76])]).cpu().numpy()
    assert np.array_equal(a, b)
