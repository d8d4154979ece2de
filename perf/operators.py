"""A paged cache of keys and values held in 8 bits: what appends to it and what reads it.

Three kinds of pass, of one layer each.

* ``append``: a step's rows [q | k | v] are rotated by position; q goes to rows of its own, k and v to their sequences' pages, each
  row of a head as 8-bit codes (``int8`` or ``float8_e4m3fn``) with one fp32 scale.
* ``step``: the same rows, appended and attended over at once, as a layer of a decode step does it.
* ``attend``: attention of rotated queries over what the pages hold: single tokens, short messages and prompts behind what is there.

A row of D numbers x (a key after its rotation, a value) is held as codes and a scale: a = max|x|; scale = a / 127 (int8) or a / 448
(e4m3); code = x / scale rounded to the nearest (ties to even); it stands for code * scale.  The angle of pair i at position p is the
fp32 product p * inv_freq[i].  Query head h reads kv head h // (heads / kv_heads); the query at position p sees the positions
max(0, p - window + 1) .. p of its sequence (window 0: all up to p).

A page holds 64 positions; a sequence's pages lie anywhere in the pool.  Rows of a page behind a sequence's last position hold what an
earlier sequence left there.
"""
import math
import random

import torch

own = False
DEVICE = "cuda:0"
PAGE = 64
MOST = {"int8": 127.0, "float8_e4m3fn": 448.0}


# ----------------------------------------------------------------------------- the cases

def _case(kind, held, type, seqs, heads, kv_heads, dim, new, least, most, window=0, order=1):
    """``new``: most tokens that a sequence brings (each brings between half of them and all); ``least``, ``most``: positions that
    the sequences hold after the pass, spread evenly in their logarithm, shuffled by ``order``."""
    return {"kind": kind, "held": held, "type": type, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "new": new,
            "least": least, "most": most, "window": window, "order": order}


def listed():
    return [
        # a decode step of a few conversations on the smallest model: all launch and latency
        dict(_case("append", "int8", "bfloat16", 4, 9, 3, 64, 1, 40, 300), name="append 4 tokens int8"),
        # one long prompt of a model with ungrouped heads
        dict(_case("append", "float8_e4m3fn", "bfloat16", 1, 32, 32, 64, 8192, 8192, 8192), name="append 8192 e4m3"),
        # prompts of a batch, unequal, some behind earlier turns; 32-bit model
        dict(_case("append", "int8", "float32", 9, 15, 5, 64, 700, 700, 2500), name="append ragged int8 fp32"),
        # one conversation on the smallest model: a decode layer's attention, bound by latency
        dict(_case("step", "float8_e4m3fn", "bfloat16", 1, 9, 3, 64, 1, 1000, 1000), name="step 1 x 1000 e4m3"),
        # the decode benchmark's batch at its longest context
        dict(_case("step", "float8_e4m3fn", "bfloat16", 8, 32, 32, 64, 1, 4096, 4096), name="step 8 x 4096 e4m3"),
        # a full server of grouped heads of 128, unequal conversations
        dict(_case("attend", "int8", "bfloat16", 64, 32, 8, 128, 1, 200, 4400), name="attend 64 ragged int8"),
        # few conversations over very long documents
        dict(_case("attend", "int8", "bfloat16", 3, 15, 5, 64, 1, 60001, 131071), name="attend 3 x 100k int8"),
        # the 32-bit path's decode step
        dict(_case("attend", "float8_e4m3fn", "float32", 16, 9, 3, 64, 1, 100, 1500), name="attend 16 fp32 e4m3"),
        # short messages (a few tokens each) under a sliding window
        dict(_case("attend", "float8_e4m3fn", "bfloat16", 24, 9, 3, 64, 7, 900, 4000, 512), name="attend messages e4m3"),
        # messages of chats that go on
        dict(_case("attend", "int8", "bfloat16", 4, 32, 8, 128, 45, 500, 2000), name="attend chat turns int8"),
        # the prefill benchmark's prompt
        dict(_case("attend", "float8_e4m3fn", "bfloat16", 1, 32, 32, 64, 2048, 2048, 2048), name="attend prompt 2048 e4m3"),
        # portions of two long documents, behind what is there
        dict(_case("attend", "int8", "bfloat16", 2, 32, 8, 128, 600, 20011, 31001), name="attend portions int8"),
    ]


LAYOUTS = ((9, 3, 64), (15, 5, 64), (32, 32, 64), (32, 8, 128), (16, 16, 128), (16, 1, 64), (24, 3, 128), (12, 12, 64))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    while True:
        kind = rng.choice(("append", "step", "attend", "attend", "attend"))
        heads, kv_heads, dim = rng.choice(LAYOUTS)
        held, seqs, order = rng.choice(sorted(MOST)), _log(rng, 1, 64), rng.randrange(1 << 20)
        if kind == "step":
            held = "float8_e4m3fn"
        kind_of_new = rng.choice(("one", "message", "prompt"))
        new = 1 if kind == "step" or kind_of_new == "one" else _log(rng, 2, 64) if kind_of_new == "message" else _log(rng, 65, 6000)
        least = max(new, _log(rng, 1, 60000))
        most = max(least, _log(rng, least, 4 * least))
        window = _log(rng, 16, 4096) if kind != "append" and rng.random() < 0.2 else 0
        type = "float32" if (kind == "append" or (new == 1 and kv_heads == 3)) and rng.random() < 0.25 else "bfloat16"
        case = _case(kind, held, type, seqs, heads, kv_heads, dim, new, least, most, window, order)
        scores = seqs * heads * new * most
        if seqs * most * kv_heads * dim <= 1.5e8 and scores <= (1.2e9 if new > 1 else 1.5e8) and (type == "bfloat16" or scores <= 5e6 or kind == "append") \
                and seqs * new * (heads + 2 * kv_heads) * dim <= 5e7:
            return case


def _lengths(case):
    """(tokens that each sequence brings, positions that it holds behind them)."""
    r, n = random.Random(case["order"]), case["seqs"]
    lo, hi = math.log(case["least"]), math.log(case["most"])
    holds = [max(case["least"], min(case["most"], int(round(math.exp(lo + (hi - lo) * (i + 0.5) / n))))) for i in range(n)]
    r.shuffle(holds)
    brings = [min(h, r.randint((case["new"] + 1) // 2, case["new"])) for h in holds]
    brings[0] = min(holds[0], case["new"])
    return brings, holds


# ----------------------------------------------------------------------------- inputs

def _rows(gen, *shape):
    """Random rows as projections make them: a few entries of a head are larger for every token, and tokens differ in size."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    big = 1.0 + 3.0 * (torch.rand(shape[-1], generator=gen, device=DEVICE) > 0.93)
    return x * big * torch.exp(0.3 * torch.randn((*shape[:-1], 1), generator=gen, device=DEVICE))


def _held(x, held):
    """fp32 rows [..., D] -> (codes, fp32 scales [...])."""
    scale = x.abs().amax(dim=-1) / MOST[held]
    y = x * (1.0 / torch.where(scale > 0, scale, torch.ones_like(scale)))[..., None]
    y = y.clamp(-MOST[held], MOST[held])
    return (torch.round(y).to(torch.int8) if held == "int8" else y.to(torch.float8_e4m3fn)), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    type = getattr(torch, case["type"])
    brings, holds = _lengths(case)
    n_pages = [-(-h // PAGE) for h in holds]
    pool, widest = sum(n_pages), max(n_pages)
    order = torch.randperm(pool, generator=gen, device=DEVICE).to(torch.int32)
    starts = torch.tensor([0] + n_pages, device=DEVICE).cumsum(0)[:-1]
    place = torch.arange(widest, device=DEVICE)
    inside = place[None, :] < torch.tensor(n_pages, device=DEVICE)[:, None]
    table = torch.where(inside, order[(starts[:, None] + place[None, :]).clamp(max=pool - 1)], -1).to(torch.int32).contiguous()
    k_codes, k_scales = _held(_rows(gen, pool, G, PAGE, D), case["held"])
    v_codes, v_scales = _held(_rows(gen, pool, G, PAGE, D), case["held"])
    T = sum(brings)
    n = torch.tensor(brings, device=DEVICE)
    kv_len = torch.tensor(holds, dtype=torch.int32, device=DEVICE)
    q_start = torch.tensor([0] + brings, device=DEVICE).cumsum(0).to(torch.int32)
    tok_seq = torch.repeat_interleave(torch.arange(len(brings), device=DEVICE), n).to(torch.int32)
    local = torch.arange(T, device=DEVICE) - q_start[tok_seq.long()]
    state = {"case": case, "type": type, "table": table, "kv_len": kv_len, "q_start": q_start, "tok_seq": tok_seq,
             "tok_pos": (kv_len[tok_seq.long()] - n[tok_seq.long()] + local).to(torch.int32), "local": local,
             "k_codes": k_codes, "k_scales": k_scales, "v_codes": v_codes, "v_scales": v_scales, "brings": brings,
             "most_new": max(brings), "inv_freq": torch.tensor([10000.0 ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float32, device=DEVICE),
             "out": torch.zeros((T, H * D), dtype=type, device=DEVICE)}
    if case["kind"] == "attend":
        state["q"] = (1.5 * torch.randn((T, H * D), generator=gen, device=DEVICE)).to(type)
    else:
        state["qkv"] = torch.cat([1.5 * torch.randn((T, H * D), generator=gen, device=DEVICE), _rows(gen, T, 2 * G, D).reshape(T, -1)], dim=1).to(type)
    return state


# ----------------------------------------------------------------------------- the plain form

def _turned(x, pos, inv_freq):
    """x [T, heads, D] fp32: the pairs (i, i + D/2) turned by the angle of the token's position."""
    angle = (pos.float()[:, None] * inv_freq[None, :]).double()
    c, s = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _plain_append(st):
    c = st["case"]
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    x = st["qkv"].float().view(-1, H + 2 * G, D)
    qk = _turned(x[:, :H + G], st["tok_pos"], st["inv_freq"])
    page = st["table"][st["tok_seq"].long(), st["tok_pos"].long() // PAGE].long()
    row = st["tok_pos"].long() % PAGE
    codes, scales = _held(qk[:, H:], c["held"])
    st["k_codes"].view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
    st["k_scales"][page, :, row] = scales
    codes, scales = _held(x[:, H + G:], c["held"])
    st["v_codes"].view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
    st["v_scales"][page, :, row] = scales
    return qk[:, :H].reshape(-1, H * D)


def _plain_attention(st, q):
    c = st["case"]
    H, G, D, S = c["heads"], c["kv_heads"], c["dim"], c["seqs"]
    table = st["table"].long().clamp(min=0)
    L = table.shape[1] * PAGE
    k = (st["k_codes"][table].float() * st["k_scales"][table][..., None]).permute(0, 2, 1, 3, 4).reshape(S, G, L, D)
    v = (st["v_codes"][table].float() * st["v_scales"][table][..., None]).permute(0, 2, 1, 3, 4).reshape(S, G, L, D)
    Q, seq = st["most_new"], st["tok_seq"].long()
    rows = torch.zeros((S, Q, H, D), dtype=torch.float32, device=q.device)
    rows[seq, st["local"]] = q.float().view(-1, H, D)
    rows = rows.view(S, Q, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(S, G, -1, D)
    n = st["q_start"][1:] - st["q_start"][:-1]
    pos = (st["kv_len"] - n).long()[:, None] + torch.arange(Q, device=q.device)[None, :]
    key = torch.arange(L, device=q.device)
    hidden = key[None, None, :] > pos[:, :, None]
    if c["window"] > 0:
        hidden |= key[None, None, :] <= pos[:, :, None] - c["window"]
    s = (rows @ k.transpose(-1, -2)).mul_(D ** -0.5).view(S, G, H // G, Q, L).masked_fill_(hidden[:, None, None], -math.inf)
    s = torch.exp_(s.sub_(s.amax(dim=-1, keepdim=True)))
    total = s.sum(dim=-1, keepdim=True)
    o = (s.view(S, G, -1, L) @ v).view(S, G, H // G, Q, D) / total
    return o.permute(0, 3, 1, 2, 4)[seq, st["local"]].reshape(-1, H * D).to(st["type"])


# ----------------------------------------------------------------------------- a pass

def _cache(st):
    """What a pass leaves in the cache: 8-bit floats as they are, int8 codes as the values that they stand for."""
    if st["case"]["held"] == "int8":
        return {"k": (st["k_codes"] * st["k_scales"][..., None]).to(torch.bfloat16), "v": (st["v_codes"] * st["v_scales"][..., None]).to(torch.bfloat16),
                "k_scales": st["k_scales"], "v_scales": st["v_scales"]}
    return {"k": st["k_codes"], "v": st["v_codes"], "k_scales": st["k_scales"], "v_scales": st["v_scales"]}


def _own(st):
    from llmi_b200.engine.batch import StepContext, short_message
    from llmi_b200.ops import kernels
    c = st["case"]
    k, v = kernels.Rows8(st["k_codes"], st["k_scales"]), kernels.Rows8(st["v_codes"], st["v_scales"])
    sizes = (c["heads"], c["kv_heads"], c["dim"])
    if c["kind"] == "append":
        kernels.rope_store8(st["qkv"], st["out"], st["inv_freq"], c["dim"], st["tok_seq"], st["tok_pos"], st["table"], k, v, *sizes)
        return {"q": st["out"], **_cache(st)}
    ctx = StepContext()
    ctx.n_tokens, ctx.n_seqs, ctx.max_q_len = st["out"].shape[0], c["seqs"], st["most_new"]
    ctx.decode, ctx.short_message = st["most_new"] == 1, short_message(st["most_new"])
    ctx.tok_seq, ctx.tok_pos, ctx.seq_q_start, ctx.seq_kv_len = st["tok_seq"], st["tok_pos"], st["q_start"], st["kv_len"]
    if c["kind"] == "step":
        kernels.attention8(st["qkv"], st["out"], k, v, ctx, st["table"], *sizes, c["dim"] ** -0.5, c["window"], rope=(st["inv_freq"], c["dim"], True))
        return {"out": st["out"], **_cache(st)}
    kernels.attention8(st["q"], st["out"], k, v, ctx, st["table"], *sizes, c["dim"] ** -0.5, c["window"])
    return {"out": st["out"]}


def run(state):
    if own:
        return _own(state)
    if state["case"]["kind"] == "append":
        return {"q": _plain_append(state).to(state["type"]), **_cache(state)}
    if state["case"]["kind"] == "step":
        return {"out": _plain_attention(state, _plain_append(state)), **_cache(state)}
    return {"out": _plain_attention(state, state["q"])}


def work(case):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    e = 4 if case["type"] == "float32" else 2
    brings, holds = _lengths(case)
    T, row = sum(brings), 2 * G * (D + 4)
    if case["kind"] == "append":
        return {"bytes": T * (2 * H + 2 * G) * D * e + T * row, "flops": T * 6 * (H + 2 * G) * D}
    w = case["window"]
    read = sum(h - max(0, h - n - w + 1) if w else h for n, h in zip(brings, holds))
    pairs = sum(sum(min(p + 1, w) if w else p + 1 for p in range(h - n, h)) for n, h in zip(brings, holds))
    return {"bytes": read * row + T * 2 * H * D * e + (T * 2 * G * D * e if case["kind"] == "step" else 0), "flops": 4 * D * H * pairs}


# ----------------------------------------------------------------------------- the same in 64 bits

def _exact_e4m3(y):
    """The e4m3 number next to y (3 bits behind the leading one, least normal 2^-6, steps of 2^-9 below), ties to even."""
    _, exponent = torch.frexp(y)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=y.device), (exponent - 1).clamp(min=-6).double() - 3.0)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exact_held(x, held):
    scale = x.abs().max(dim=-1).values / MOST[held]
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale)).unsqueeze(-1)
    return (torch.round(y) if held == "int8" else _exact_e4m3(y)), scale


def exact(case, seed):
    st = prepare(case, seed)
    H, G, D, held = case["heads"], case["kv_heads"], case["dim"], case["held"]
    brings, holds = _lengths(case)
    codes = {"k": st["k_codes"].double(), "v": st["v_codes"].double()}
    scales = {"k": st["k_scales"].double(), "v": st["v_scales"].double()}
    queries = st["q"].double() if case["kind"] == "attend" else None
    if queries is None:
        x = st["qkv"].double().view(-1, H + 2 * G, D)
        angle = (st["tok_pos"].float().unsqueeze(1) * st["inv_freq"]).double()
        turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
        z = torch.complex(x[:, :H + G, :D // 2], x[:, :H + G, D // 2:]) * turn
        x = torch.cat([torch.cat([z.real, z.imag], dim=-1), x[:, H + G:]], dim=1)
        queries, at = x[:, :H].reshape(-1, H * D), 0
        new = {"k": _exact_held(x[:, H:H + G], held), "v": _exact_held(x[:, H + G:], held)}
        for i, (n, h) in enumerate(zip(brings, holds)):
            p = torch.arange(h - n, h, device=DEVICE)
            page = st["table"][i].long()[p // PAGE]
            for name in ("k", "v"):
                codes[name][page, :, p % PAGE] = new[name][0][at:at + n]
                scales[name][page, :, p % PAGE] = new[name][1][at:at + n]
            at += n
    state = {}
    if case["kind"] != "attend":
        state = {name: codes[name] * scales[name].unsqueeze(-1) if held == "int8" else codes[name] for name in ("k", "v")}
        state.update({name + "_scales": scales[name] for name in ("k", "v")})
    if case["kind"] == "append":
        return {"q": queries, **state}
    out = torch.zeros((sum(brings), H, D), dtype=torch.float64, device=DEVICE)
    at = 0
    for i, (n, h) in enumerate(zip(brings, holds)):
        pages = st["table"][i].long()[:-(-h // PAGE)]
        pos = torch.arange(h - n, h, device=DEVICE).unsqueeze(1)
        key = torch.arange(h, device=DEVICE).unsqueeze(0)
        seen = (key <= pos) & ((key > pos - case["window"]) if case["window"] else (key >= 0))
        for g in range(G):
            k, v = ((codes[m][pages, g] * scales[m][pages, g].unsqueeze(-1)).reshape(-1, D)[:h] for m in ("k", "v"))
            for j in range(g * (H // G), (g + 1) * (H // G)):
                s = queries[at:at + n].view(n, H, D)[:, j] @ k.T / math.sqrt(D)
                out[at:at + n, j] = torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf)), dim=-1) @ v
        at += n
    return {"out": out.view(-1, H * D), **state}
