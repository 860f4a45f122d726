"""Workloads of the ragged-generation operators: block tables and slot maps
(page_tables), the paged 4-bit k/v history's writer (kv4_write) and the AFT
decode step that reads it (aft_decode4), penalties, biases and masks on
logits (logits_controls), and the greedy pick with a position per row
(greedy_embed_rows).

``run`` computes a case in plain torch operations, or, with ``own`` set,
through ``dart_cuda_b200.ops``; ``exact`` is the definition in 64 bits.

Layout of the 4-bit history: pages [n_pages, D/W, page_size, 5W/4] bytes, W
the largest of 256, 128, 64, 32 that divides D.  The record of W channels at
one position holds, for every 8 channels, 4 bytes of k codes then 4 of v
codes (channel j in bits 4j..4j+3), then for every 32 channels four bf16: k
step, k low, v step, v low.  A code c stands for low + step * c.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of the greedy-decode benchmark's batch: 64 requests
        # of at most 512 positions get the page and slot of one new token
        {"name": "tables-step", "op": "tables", "B": 64, "page": 16, "cap": 512, "start": 511, "new": 1, "padded": 0},
        # a prefill wave: 500 new prompts of up to 2047 tokens, packed slots
        {"name": "tables-prefill", "op": "tables", "B": 500, "page": 32, "cap": 2048, "start": 0, "new": 2047,
         "padded": 0},
        # prompts of the greedy-decode benchmark (64 x 256 positions, d = 512)
        # into the history, padded rows skipped, values back for the forward
        {"name": "write-prompts", "op": "write", "n": 16384, "D": 512, "page": 16, "dtype": "f32", "skip": 0.25},
        # long prompts of a wide layer, bf16 activations
        {"name": "write-wide-bf16", "op": "write", "n": 65521, "D": 2048, "page": 64, "dtype": "bf16", "skip": 0.0},
        # the smallest step: the tests' two-head decoder, three requests
        {"name": "decode-tiny", "op": "decode", "B": 3, "H": 2, "hs": 16, "T": 16, "low": 0, "page": 8, "dtype": "f32"},
        # the greedy-decode benchmark's step in the second half of its context
        {"name": "decode-512", "op": "decode", "B": 64, "H": 4, "hs": 128, "T": 512, "low": 256, "page": 16,
         "dtype": "f32"},
        # long ragged contexts of a wide layer, bf16 activations
        {"name": "decode-long-bf16", "op": "decode", "B": 32, "H": 16, "hs": 128, "T": 8192, "low": 0, "page": 64,
         "dtype": "bf16"},
        # one request of the character model: 65 logits, repetition penalty
        {"name": "logits-char", "op": "logits", "B": 1, "V": 65, "T": 256, "dtype": "f32", "pens": 1, "bias": 0,
         "mask": 0},
        # the greedy-decode benchmark's logits, every control, one bias and
        # one grammar for the batch
        {"name": "logits-8192", "op": "logits", "B": 64, "V": 8192, "T": 512, "dtype": "f32", "pens": 3, "bias": 1,
         "mask": 1},
        # a large batch over an odd vocabulary, bf16, a bias and a mask a row
        {"name": "logits-50257-bf16", "op": "logits", "B": 512, "V": 50257, "T": 4096, "dtype": "bf16", "pens": 3,
         "bias": 2, "mask": 2},
        # the pick that ends a decode step of the greedy-decode benchmark
        {"name": "pick-8192", "op": "pick", "B": 64, "V": 8192, "D": 512, "T": 512, "dtype": "f32"},
        # the same for the large batch, odd vocabulary
        {"name": "pick-50257-bf16", "op": "pick", "B": 512, "V": 50257, "D": 768, "T": 2048, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("tables", "write", "decode", "decode", "logits", "logits", "pick"))
    if op == "tables":
        B, page = _log(rng, 1, 1500), rng.choice((8, 16, 32, 64, 128, 256))
        new = _log(rng, 1, max(1, min(8000, 1000000 // B)))
        start = rng.choice((0, _log(rng, 1, 8000)))
        return {"op": op, "B": B, "page": page, "cap": page * (-(-(start + new) // page)), "start": start, "new": new,
                "padded": rng.randrange(2)}
    if op == "write":
        D, dtype = 32 * _log(rng, 1, 64), rng.choice(("f32", "bf16"))
        most = int(1.2e9 / (D * (4 * SIZE[dtype] + 1.25)))
        return {"op": op, "n": _log(rng, 1, min(200000, most)), "D": D, "page": rng.choice((8, 16, 32, 64)),
                "dtype": dtype, "skip": rng.choice((0.0, 0.3))}
    if op == "decode":
        D = 32 * _log(rng, 1, 64)
        H = rng.choice([h for h in range(1, 33) if D % (8 * h) == 0])
        T = min(_log(rng, 2, 8192), int(math.sqrt(1.0e9 / H)))  # the positional bias [H, T, T]
        B = _log(rng, 1, max(1, min(256, 32 * 8192 * 2048 // (T * D))))
        return {"op": op, "B": B, "H": H, "hs": D // H, "T": T, "low": rng.choice((0, T // 2, T - 1)),
                "page": rng.choice((8, 16, 32, 64, 128)), "dtype": rng.choice(("f32", "bf16"))}
    V = _log(rng, 2, 150000)
    B = _log(rng, 1, max(1, min(512, 512 * 50257 // (2 * V))))
    if op == "logits":
        return {"op": op, "B": B, "V": V, "T": _log(rng, 1, 4096), "dtype": rng.choice(("f32", "bf16")),
                "pens": rng.randrange(4), "bias": rng.randrange(3), "mask": rng.randrange(3)}
    D = _log(rng, 1, 2048)
    D = min(D, 100000000 // V)  # the embedding table [V, D]
    return {"op": op, "B": B, "V": V, "D": D, "T": _log(rng, 2, 2048), "dtype": rng.choice(("f32", "bf16"))}


def _slab(D):
    return next(w for w in (256, 128, 64, 32) if D % w == 0)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _ints(g, lo, hi, *shape):
    """Whole numbers of lo..hi, int32."""
    return torch.randint(int(lo), int(hi) + 1, shape, generator=g, device=DEV, dtype=torch.int32)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _empty_pages(n_pages, page, D):
    W = _slab(D)
    return torch.zeros(n_pages, D // W, page, W * 5 // 4, dtype=torch.uint8, device=DEV)


def _block_table(g, lens, page, width):
    """A table that gives every request the pages of its first lens tokens,
    scattered over a pool of width pages a request."""
    need = (lens.long() + page - 1) // page
    first = need.cumsum(0) - need
    pool = torch.randperm(lens.numel() * width, generator=g, device=DEV)
    cols = torch.arange(width, device=DEV)[None]
    at = (first[:, None] + cols).clamp(max=pool.numel() - 1)
    return torch.where(cols < need[:, None], pool[at], -1).int().contiguous()


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"op": op}
    if op == "tables":
        B, page, new = case["B"], case["page"], case["new"]
        width = case["cap"] // page
        start = _ints(g, 0, case["start"], B)
        count = _ints(g, 1, new, B)
        s["table"] = _block_table(g, start, page, width)
        s["free"] = s["table"].numel() + torch.randperm(B * (new // page + 2), generator=g, device=DEV).int()
        s["head"] = torch.full((1,), 3, dtype=torch.int32, device=DEV)
        s.update(page=page, start=start, count=count, ld=new if case["padded"] else 0,
                 slots=torch.full((B * new,), -1, dtype=torch.int32, device=DEV),
                 row_start=torch.zeros(B + 1, dtype=torch.int32, device=DEV), head_out=torch.zeros_like(s["head"]))
    elif op == "write":
        n, D, page = case["n"], case["D"], case["page"]
        n_pages = -(-n // page) + 3
        s["pages"] = _empty_pages(n_pages, page, D)
        # a fused projection row: q | k | v, the channels with means of their own
        qkv = _normal(g, n, 3 * D) + _normal(g, 3 * D)
        s["qkv"] = qkv.to(DTYPES[case["dtype"]])
        slots = torch.randperm(n_pages, generator=g, device=DEV)[:, None] * page + torch.arange(page, device=DEV)
        slots = slots.reshape(-1)[:n].int()
        s["slots"] = torch.where(torch.rand(n, generator=g, device=DEV) < case["skip"], -1, slots).int()
        s["D"] = D
        s["values"] = torch.zeros(n, 2 * D, dtype=s["qkv"].dtype, device=DEV)
    elif op == "decode":
        B, H, hs, T, page = (case[k] for k in ("B", "H", "hs", "T", "page"))
        D = H * hs
        pos = _ints(g, case["low"], T - 1, B)
        table = _block_table(g, pos + 1, page, -(-T // page))
        pages = _empty_pages(table.numel(), page, D)
        mean = _normal(g, 2, D)
        slots = torch.arange(table.numel() * page, device=DEV)
        step = max(1, (1 << 25) // D)
        for a in range(0, slots.numel(), step):
            at = slots[a: a + step]
            _plain_store(pages, _normal(g, at.numel(), D) + mean[0], _normal(g, at.numel(), D) + mean[1], at)
        dt = DTYPES[case["dtype"]]
        qkv = _normal(g, B, 3, D)
        qkv[:, 1:] += mean
        s.update(B=B, H=H, hs=hs, D=D, T=T, page=page, pos=pos, table=table, pages=pages,
                 qkv=qkv.reshape(B, 3 * D).to(dt), w=0.3 * _normal(g, H, T, T), z=torch.zeros(B, D, dtype=dt, device=DEV))
        if own:
            from dart_cuda_b200 import ops
            s["workspace"] = ops.aft_decode4_workspace(B, D)
    else:
        B, V, T = case["B"], case["V"], case["T"]
        dt = DTYPES[case["dtype"]]
        s["V"] = V
        s["logits"] = (3.0 * _normal(g, B, V)).to(dt)
        s["tokens"] = _ints(g, 0, V - 1, B, T + 1)
        if op == "logits":
            s["pos"] = _ints(g, 0, T - 1, B)
            s["prompt"] = (s["pos"].float() * torch.rand(B, generator=g, device=DEV)).int() + 1
            # text repeats itself: half of the tokens come from a few of the vocabulary
            few = _ints(g, 0, min(V - 1, 40), B, T + 1)
            s["tokens"] = torch.where(torch.rand(B, T + 1, generator=g, device=DEV) < 0.5, few, s["tokens"])
            rows = lambda lo, hi: lo + (hi - lo) * torch.rand(B, generator=g, device=DEV)  # noqa: E731
            s["repetition"] = rows(1.0, 1.5) if case["pens"] & 1 else None
            s["presence"] = rows(0.0, 1.0) if case["pens"] & 2 else None
            s["frequency"] = rows(0.0, 0.5) if case["pens"] & 2 else None
            s["bias"] = s["mask"] = None
            if case["bias"]:
                bias = 2.0 * _normal(g, *((V,) if case["bias"] == 1 else (B, V)))
                s["bias"] = bias * (torch.rand(bias.shape, generator=g, device=DEV) < 0.1)
            if case["mask"]:
                words = (V + 31) // 32
                shape = (words,) if case["mask"] == 1 else (B, words)
                s["mask"] = torch.randint(-2**31, 2**31, shape, generator=g, device=DEV, dtype=torch.int64).int()
            s["out"] = torch.empty_like(s["logits"])
        else:
            D = case["D"]
            s["pos"] = _ints(g, 0, T - 1, B)
            # a grammar has masked half of the vocabulary
            s["logits"].masked_fill_(torch.rand(B, V, generator=g, device=DEV) < 0.5, -math.inf)
            s["wte"], s["wpe"] = 0.5 * _normal(g, V, D), 0.5 * _normal(g, T + 1, D)
            s["x"] = torch.zeros(B, D, device=DEV)
            s["pos_out"] = torch.zeros_like(s["pos"])
    return s


# ------------------------------------------------------------------ passes
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from dart_cuda_b200 import ops

    op = s["op"]
    if op == "tables":
        ops.page_tables(s["start"], s["count"], s["free"], s["head"], s["table"], s["page"], slots=s["slots"],
                        ld_slots=s["ld"], row_start=s["row_start"], head_out=s["head_out"])
        return {k: s[k] for k in ("table", "slots", "row_start", "head_out")}
    if op == "write":
        D, x, v = s["D"], s["qkv"], s["values"]
        ops.kv4_write(x[:, D: 2 * D], x[:, 2 * D:], s["slots"], s["pages"], values=(v[:, :D], v[:, D:]))
        return {"values": v, "pages": s["pages"]}
    if op == "decode":
        ops.aft_decode4(s["qkv"], s["w"], s["pages"], s["table"], s["pos"], out=s["z"], workspace=s["workspace"])
        return {"z": s["z"], "pages": s["pages"]}
    if op == "logits":
        return ops.logits_controls(s["logits"], s["tokens"], s["pos"], prompt_len=s["prompt"], repetition=s["repetition"],
                                   presence=s["presence"], frequency=s["frequency"], bias=s["bias"], mask=s["mask"],
                                   out=s["out"])
    ops.greedy_embed_rows(s["logits"], s["tokens"], s["pos"], wte=s["wte"], wpe=s["wpe"], x=s["x"], pos_out=s["pos_out"])
    return {k: s[k] for k in ("tokens", "x", "pos_out")}


def _run_plain(s):
    return {"tables": _plain_tables, "write": _plain_write, "decode": _plain_decode, "logits": _plain_logits,
            "pick": _plain_pick}[s["op"]](s)


def _plain_tables(s):
    page, table, free = s["page"], s["table"], s["free"]
    width = table.shape[1]
    start, count = s["start"].long(), s["count"].long()
    have = (start + page - 1) // page
    last = ((start + count + page - 1) // page).clamp(max=width)
    need = (last - have).clamp(min=0)
    first = s["head"].long() + need.cumsum(0) - need
    cols = torch.arange(width, device=table.device)[None]
    at = first[:, None] + cols - have[:, None]
    page_of = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table = torch.where((cols >= have[:, None]) & (cols < last[:, None]), page_of, table)
    row_start = torch.cat([torch.zeros_like(count[:1]), count.cumsum(0)])
    i = torch.arange(s["slots"].numel(), device=table.device)
    if s["ld"]:
        b, j = i // s["ld"], i % s["ld"]
    else:
        b = torch.searchsorted(row_start[1:].contiguous(), i, right=True).clamp(max=start.numel() - 1)
        j = i - row_start[b]
    p = start[b] + j
    there = table[b, (p // page).clamp(max=width - 1)].long()
    ok = (j < count[b]) & (p // page < width) & (there >= 0)
    slots = torch.where(ok, there * page + p % page, -1)
    head = (s["head"].long() + need.sum()).clamp(max=free.numel())
    return {"table": table, "slots": slots.int(), "row_start": row_start.int(), "head_out": head.int()}


def _plain_quantise(x):
    """codes, step and low (in 64 bits, where values lie next to a border) of
    x [n, D] in groups of 32: low is the bf16 at or below the smallest value,
    step the bf16 at or above (largest - low) / 15."""
    x = x.float().reshape(x.shape[0], -1, 32)
    lo = x.amin(-1) + 0.0
    cut = lo.view(torch.int32) >> 16 << 16
    lo = torch.where(cut.view(torch.float32) > lo, cut + 0x10000, cut).view(torch.float32)
    step = (x.amax(-1).double() - lo.double()) / 15
    up = step.float()
    up = torch.where(up.double() < step, up.view(torch.int32) + 1, up.view(torch.int32))
    step = ((up + 0xFFFF) >> 16 << 16).view(torch.float32)
    q = (x.double() - lo.double()[..., None]) / step.double()[..., None]
    codes = torch.where(step[..., None] > 0, (q + 0.5).floor(), 0.0).clamp(0, 15)
    return codes, step, lo


def _plain_pack(k, v):
    """The records [n, D/W, 5W/4] of rows k, v [n, D], and the values that
    the codes stand for."""
    n, D = k.shape
    W = _slab(D)
    codes, params, values = [], [], []
    for x in (k, v):
        c, step, lo = _plain_quantise(x)
        values.append((lo.double()[..., None] + step.double()[..., None] * c).reshape(n, D))
        b = c.to(torch.uint8).reshape(n, D // W, W // 8, 4, 2)
        codes.append(b[..., 0] | b[..., 1] << 4)
        params.append(torch.stack([step, lo], -1).bfloat16().reshape(n, D // W, W // 32, 2))
    codes = torch.stack(codes, 3).reshape(n, D // W, W)
    params = torch.stack(params, 3).reshape(n, D // W, W // 8).contiguous().view(torch.uint8).reshape(n, D // W, W // 4)
    return torch.cat([codes, params], -1), values


def _plain_store(pages, k, v, slots):
    page = pages.shape[2]
    rec, values = _plain_pack(k, v)
    pages[slots // page, :, slots % page] = rec
    return values


def _plain_write(s):
    D, x, slots = s["D"], s["qkv"], s["slots"].long()
    keep = (slots >= 0).nonzero()[:, 0]
    k, v = _plain_store(s["pages"], x[keep, D: 2 * D], x[keep, 2 * D:], slots[keep])
    s["values"][keep] = torch.cat([k, v], 1).float().to(x.dtype)
    return {"values": s["values"], "pages": s["pages"]}


def _plain_load(pages, slots):
    """k and v [..., D] (float32) at the given slots."""
    page, nslab = pages.shape[2], pages.shape[1]
    W = pages.shape[3] * 4 // 5
    rec = pages[slots // page, :, slots % page]  # [..., nslab, 5W/4]
    codes = rec[..., :W].unflatten(-1, (W // 8, 2, 4))
    par = rec[..., W:].contiguous().view(torch.bfloat16).unflatten(-1, (W // 32, 2, 2)).float()
    out = []
    for j in (0, 1):
        b = codes[..., j, :]
        c = torch.stack([b & 15, b >> 4], -1).flatten(-3).unflatten(-1, (W // 32, 32))
        out.append((par[..., j, 1, None] + par[..., j, 0, None] * c.float()).reshape(*slots.shape, nslab * W))
    return out


def _plain_decode(s):
    B, H, hs, D, T, page = (s[k] for k in ("B", "H", "hs", "D", "T", "page"))
    table, pos, x = s["table"].long(), s["pos"].long(), s["qkv"]
    _plain_store(s["pages"], x[:, D: 2 * D], x[:, 2 * D:],
                 table.gather(1, pos[:, None] // page)[:, 0] * page + pos % page)
    i = torch.arange(T, device=table.device)
    seen = i[None] <= pos[:, None]  # [B, T]
    slots = torch.where(seen, table[:, i // page] * page + i % page, 0)
    k, v = _plain_load(s["pages"], slots)  # [B, T, D]
    w = s["w"][:, pos].permute(1, 2, 0)  # [B, T, H]
    k = (k.unflatten(-1, (H, hs)) + w[..., None]).masked_fill_(~seen[..., None, None], -math.inf)
    k = (k - k.amax(1, keepdim=True)).exp_()
    r = (k * v.unflatten(-1, (H, hs))).sum(1) / k.sum(1)
    z = torch.sigmoid(x[:, :D].float()) * r.reshape(B, D)
    return {"z": z.to(x.dtype), "pages": s["pages"]}


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    tokens = s["tokens"].long()
    i = torch.arange(tokens.shape[1], device=x.device)[None]
    known = i <= s["pos"][:, None]
    made = known & (i >= s["prompt"][:, None])
    seen = torch.zeros(B, V, device=x.device).scatter_add_(1, tokens, known.float()) > 0
    count = torch.zeros(B, V, device=x.device).scatter_add_(1, tokens, made.float())
    if s["repetition"] is not None:
        r = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    if s["frequency"] is not None:
        x = x - s["frequency"][:, None] * count
    if s["presence"] is not None:
        x = x - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        v = torch.arange(V, device=x.device)
        x = x.masked_fill((s["mask"][..., v // 32] >> (v % 32) & 1) == 0, -math.inf)
    return x.to(s["logits"].dtype)


def _plain_pick(s):
    x, pos = s["logits"], s["pos"].long()
    v = torch.arange(x.shape[1], device=x.device)
    token = torch.where(x == x.amax(1, keepdim=True), v, x.shape[1]).amin(1)
    s["tokens"].scatter_(1, pos[:, None] + 1, token[:, None].int())
    return {"tokens": s["tokens"], "x": s["wte"][token] + s["wpe"][pos + 1], "pos_out": s["pos"] + 1}


# ------------------------------------------------------------------ 64 bits
def _exact_values(x):
    """What the 4-bit codes of x [n, D] stand for, by counting the borders
    between codes that lie at or below each value."""
    x = x.double().reshape(x.shape[0], -1, 32)

    def grid(y):  # spacing of the bf16 numbers around y
        return torch.ldexp(torch.ones_like(y), torch.frexp(y)[1] - 8)

    lo = x.min(-1).values
    lo = torch.where(lo == 0, lo, torch.floor(lo / grid(lo)) * grid(lo))
    st = (x.max(-1).values - lo) / 15
    st = torch.where(st == 0, st, torch.ceil(st / grid(st)) * grid(st))
    lo, st = lo[..., None], st[..., None]
    c = torch.zeros_like(x)
    for k in range(15):
        c += (x >= lo + st * (k + 0.5)) & (st > 0)
    return (lo + st * c).reshape(x.shape[0], -1)


def exact(case, seed):
    op = case["op"]
    if op == "tables":
        return None  # whole numbers only
    s = prepare(case, seed)
    if op == "write":
        D = s["D"]
        x = _exact_values(s["qkv"][:, D:])
        return {"values": torch.where(s["slots"][:, None] >= 0, x, 0.0), "pages": None}
    if op == "decode":
        B, H, hs, D, page = (s[k] for k in ("B", "H", "hs", "D", "page"))
        W, z = _slab(D), []
        new = _exact_values(s["qkv"][:, D:])
        for b in range(B):
            t = int(s["pos"][b])
            ids = s["table"][b, : t // page + 1].long()
            rec = s["pages"][ids].transpose(1, 2).flatten(0, 1)[: t + 1]  # [t+1, D/W, 5W/4]
            code = rec[..., :W].to(torch.int16)
            code = torch.stack([code % 16, code // 16], -1).reshape(t + 1, D // W, W // 8, 2, 8).double()
            par = rec[..., W:].contiguous().view(torch.bfloat16).double().reshape(t + 1, D // W, W // 32, 1, 4)
            par = par.expand(-1, -1, -1, 4, -1).reshape(t + 1, D // W, W // 8, 4)
            k = (par[..., 1:2] + par[..., 0:1] * code[..., 0, :]).reshape(t + 1, D)
            v = (par[..., 3:4] + par[..., 2:3] * code[..., 1, :]).reshape(t + 1, D)
            k[t], v[t] = new[b, :D], new[b, D:]
            a = torch.softmax(k + s["w"][:, t, : t + 1].double().T.repeat_interleave(hs, 1), 0)
            z.append(torch.sigmoid(s["qkv"][b, :D].double()) * (a * v).sum(0))
        return {"z": torch.stack(z), "pages": None}
    if op == "logits":
        x = s["logits"].double()
        B, V = x.shape
        hist = torch.zeros(2, B, V, dtype=torch.float64, device=x.device)
        i = torch.arange(s["tokens"].shape[1], device=x.device)
        for part, first in ((0, torch.zeros_like(s["prompt"])), (1, s["prompt"])):
            at = ((i >= first[:, None]) & (i <= s["pos"][:, None])).nonzero()
            hist[part].index_put_((at[:, 0], s["tokens"][at[:, 0], at[:, 1]].long()),
                                  torch.ones_like(at[:, 0], dtype=torch.float64), accumulate=True)
        if s["repetition"] is not None:
            r = s["repetition"].double()[:, None]
            x = x * torch.where(hist[0] == 0, 1.0, torch.where(x > 0, 1 / r, r))
        if s["presence"] is not None:
            x = x - (hist[1] * s["frequency"].double()[:, None] + hist[1].clamp(max=1) * s["presence"].double()[:, None])
        if s["bias"] is not None:
            x = x + s["bias"].double()
        if s["mask"] is not None:
            m = s["mask"].long().reshape(-1, (V + 31) // 32, 1).bitwise_and(2 ** torch.arange(32, device=x.device))
            x = torch.where(m.flatten(1)[:, :V] != 0, x, -math.inf)
        return x
    token = s["logits"].double().cpu().numpy().argmax(1)  # the first of equal ones
    at = s["pos"].long() + 1
    x = s["wte"].double()[torch.from_numpy(token).to(DEV)] + s["wpe"].double()[at]
    return {"tokens": None, "x": x, "pos_out": None}


# ------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op == "tables":
        B, n = case["B"], case["B"] * (case["new"] + 1) / 2
        pages = n / case["page"] + B
        return {"bytes": 8 * B + 8 * pages + 4 * (B + 1) + 4 * B * case["new"], "flops": 0}
    if op == "write":
        n, e = case["n"] * (1 - case["skip"]), SIZE[case["dtype"]]
        return {"bytes": n * case["D"] * (4 * e + 1.25) + 4 * case["n"], "flops": n * case["D"] * 8}
    if op == "decode":
        D, e = case["H"] * case["hs"], SIZE[case["dtype"]]
        rows = case["B"] * ((case["low"] + case["T"] - 1) / 2 + 1)
        return {"bytes": rows * (1.25 * D + 4 * case["H"]) + case["B"] * D * (4 * e + 1.25), "flops": rows * D * 8}
    n, e = case["B"] * case["V"], SIZE[case["dtype"]]
    if op == "logits":
        extra = (0, 4 * case["V"], 4 * n)[case["bias"]] + (0, case["V"] / 8, n / 8)[case["mask"]]
        return {"bytes": 2 * n * e + extra + 2 * case["B"] * case["T"], "flops": 4 * n}
    return {"bytes": n * e + case["B"] * (12 * case["D"] + 12), "flops": n}
