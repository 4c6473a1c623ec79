"""The 8-bit paged KV cache's operators as workloads: writing tokens into the cache (quantised a
block of 64 tokens and head at a time), reading them back, attending to them, and the decode step
that writes one token per sequence and attends.

Cache (one attention layer): pages ``[n_pages, Hkv, 64, D]`` of 8-bit codes for K and for V, scales
``[n_pages, Hkv, 2]`` float32 (K, V), ``page_table [B, max_blocks]`` int32, and a ring of the newest
tokens ``[B, Hkv, 128, D]`` in the cache's type: position p at slot p % 128.  Complete blocks
(64 tokens) are held as codes, the tokens behind them in the ring.  A block's scale is its largest
magnitude over the largest code (448 for e4m3, 127 for int8), at least 2^-126; its codes are its
values times the scale's reciprocal, rounded to nearest even.

``run`` is the plain form in elementary torch operations, or, where ``own`` is set, the calls that
a user makes of ``Kv8Cache``.  ``exact`` restates the results in 64 bits.
"""
import importlib
import math
import random

import torch

own = False

DEV = "cuda"
BLOCK, RING = 64, 128
TOP = {"e4m3": 448.0, "int8": 127.0}
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------- cases
def _case(kind, batch, heads, kv_heads, dim, dtype, codes, lo, hi, tokens=1, window=0, ragged=1):
    """lo..hi: the sequences' lengths before the call (log-uniform, drawn from ``ragged``);
    tokens: new tokens a sequence (append, step), query tokens (attend) or tokens read (read);
    window: sink + window attention with 4 sink tokens, 0 for all tokens."""
    return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "codes": codes, "lo": lo, "hi": hi, "tokens": tokens, "window": window, "ragged": ragged}


def listed():
    return [
        # one user's chat turn: the latency of a step over a short cache
        {"name": "step_b1_l500", **_case("step", 1, 64, 8, 128, "fp16", "e4m3", 500, 500)},
        # the package's decode batch at 8192 tokens: bound by reading the cache
        {"name": "step_b32_l8191", **_case("step", 32, 64, 8, 128, "fp16", "e4m3", 8191, 8191)},
        # a wide serving batch of short ragged chats; some of its sequences complete a block in the step
        {"name": "step_b256_ragged", **_case("step", 256, 32, 8, 128, "bf16", "e4m3", 1, 700, ragged=7)},
        # few sequences of the package's longest context: work split along the sequence
        {"name": "attend_b4_l163840", **_case("attend", 4, 64, 8, 128, "fp16", "e4m3", 163840, 163840)},
        # a mixed serving batch, three decades of lengths, int8 codes, four query heads a KV head
        {"name": "attend_b48_ragged_int8", **_case("attend", 48, 32, 8, 128, "bf16", "int8", 20, 20000, ragged=3)},
        # verification of four drafted tokens a sequence: causal among themselves, 32 query rows a KV head
        {"name": "attend_b16_drafts4", **_case("attend", 16, 64, 8, 128, "bf16", "e4m3", 4000, 9000, tokens=4, ragged=5)},
        # sink + window attention over a long cache: most of it is not read
        {"name": "attend_b16_window4096", **_case("attend", 16, 64, 8, 128, "fp16", "e4m3", 20000, 33000, window=4096, ragged=9)},
        # a small model: 64-wide heads without grouping
        {"name": "attend_b64_d64_mha", **_case("attend", 64, 16, 16, 64, "fp16", "int8", 1, 4097, ragged=11)},
        # prompts written into an empty cache
        {"name": "append_b16_prompt8000", **_case("append", 16, 64, 8, 128, "bf16", "e4m3", 0, 0, tokens=8000)},
        # a decode batch's new tokens, written alone
        {"name": "append_b256_token", **_case("append", 256, 64, 8, 128, "fp16", "e4m3", 1, 3000, ragged=13)},
        # contexts read back at 16 bits (for a prompt's attention, or to move a sequence)
        {"name": "read_b8_n16000", **_case("read", 8, 64, 8, 128, "bf16", "e4m3", 16001, 17000, tokens=16000, ragged=15)},
        # a prompt's chunk written at int8 and read back; odd sizes, 64-wide heads
        {"name": "append_read_b24_n333_int8", **_case("append_read", 24, 16, 4, 64, "fp16", "int8", 64, 64, tokens=333)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "step", "attend", "attend", "attend", "append", "read", "append_read"])
    dim = rng.choice([128, 128, 64])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    group = rng.choice([1, 2, 4, 6, 7, 8, 8, 16])
    dtype = rng.choice(["fp16", "bf16"])
    batch = _log(rng, 1, 200)
    room = 2 ** 30 // (2 * dim * kv * batch)  # tokens a sequence: a gigabyte of codes at most
    if kind in ("step", "attend"):
        hi = max(2, min(_log(rng, 30, 130000), room))
        lo = max(1, rng.choice([hi, hi // 2, hi // 50]))
        tokens = rng.choice([1, 1, 2, 3, 5, 8]) if kind == "attend" else 1
        tokens = max(1, min(tokens, 32 // group))
        window = rng.choice([0, 0, 0, _log(rng, 16, 6000)]) if kind == "attend" else 0
        codes = rng.choice(["e4m3", "int8"]) if kind == "attend" else "e4m3"
        return _case(kind, batch, kv * group, kv, dim, dtype, codes, lo, hi, tokens, window, rng.randrange(1 << 20))
    if kind == "append" and rng.random() < 0.4:  # a decode batch's tokens
        hi = max(2, min(_log(rng, 2, 4000), room))
        return _case(kind, batch, kv * group, kv, dim, dtype, "e4m3", 1, hi, 1, 0, rng.randrange(1 << 20))
    n = max(1, min(_log(rng, 2, 20000), room // 4))
    lo = 0 if kind != "read" else n + rng.randrange(200)
    if kind == "read":
        return _case(kind, batch, kv * group, kv, dim, dtype, rng.choice(["e4m3", "int8"]), lo, lo + rng.randrange(300), n, 0,
                     rng.randrange(1 << 20))
    lo = BLOCK * rng.randrange(4)
    return _case(kind, batch, kv * group, kv, dim, dtype, "e4m3" if kind == "append" else "int8", lo, lo, n, 0,
                 rng.randrange(1 << 20))


def _lens(case):
    """The sequences' lengths before the call: part of the case, not of the seed."""
    r, lo, hi = random.Random(case["ragged"]), case["lo"], case["hi"]
    return [lo if lo == hi else max(lo, min(hi, _log(r, max(lo, 1), hi))) for _ in range(case["batch"])]


def _blocks(case):
    """Blocks a sequence has room for."""
    grow = case["tokens"] if case["kind"] in ("step", "append", "append_read") else 0
    return (max(_lens(case)) + grow + BLOCK - 1) // BLOCK


# ---------------------------------------------------------------------------------------- inputs
def _tokens(g, shape, dtype, outliers):
    """Keys or values of random directions; keys with a few channels far above the rest, as in trained models."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    if outliers:
        x[..., torch.randperm(shape[-1], generator=g, device=DEV)[: shape[-1] // 32]] *= 8.0
    return x.to(dtype)


def _code(x, codes):
    """x [..., 64, D] -> (codes as float32, scales [...]): the operator's definition, in 32 bits."""
    x = x.float()
    amax = x.abs().amax((-2, -1))
    scale = (amax / torch.full_like(amax, TOP[codes])).clamp_min(2.0 ** -126)  # (a Python divisor would be a multiplication)
    y = x * (1.0 / scale)[..., None, None]
    y = y.clamp(-TOP[codes], TOP[codes])
    return (y.to(torch.float8_e4m3fn) if codes == "e4m3" else torch.round(y).to(torch.int8)), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, b, h, d, t = case["kind"], case["batch"], case["kv_heads"], case["dim"], case["tokens"]
    dtype, codes = TYPES[case["dtype"]], case["codes"]
    lens, m = _lens(case), _blocks(case)
    table = torch.randperm(b * m, generator=g, device=DEV).to(torch.int32).view(b, m)
    form = torch.float8_e4m3fn if codes == "e4m3" else torch.int8
    s = {"kind": kind, "codes": codes, "window": case["window"], "tokens": t, "dtype": dtype, "table": table,
         "lens": torch.tensor(lens, dtype=torch.int64, device=DEV), "scales": torch.zeros(b * m, h, 2, device=DEV)}
    for k in ("k", "v"):
        s[k + "_codes"] = torch.zeros(b * m, h, BLOCK, d, dtype=form, device=DEV)
        s[k + "_ring"] = torch.zeros(b, h, RING, d, dtype=dtype, device=DEV)
        for i, n in enumerate(lens):  # the tokens that are in the cache already
            full = n // BLOCK
            if full:
                x = _tokens(g, (full, h, BLOCK, d), dtype, k == "k")
                c, sc = _code(x, codes)
                at = table[i, :full].long()
                s[k + "_codes"].view(torch.uint8)[at] = c.view(torch.uint8)
                s["scales"][at, :, 0 if k == "k" else 1] = sc
            if n % BLOCK:
                slots = torch.arange(BLOCK * full, n, device=DEV) % RING
                s[k + "_ring"][i, :, slots] = _tokens(g, (h, n % BLOCK, d), dtype, k == "k")
    if kind in ("step", "append", "append_read"):  # as a projection leaves them: token-major
        s["new_k"], s["new_v"] = (_tokens(g, (b, t, h, d), dtype, o).transpose(1, 2) for o in (True, False))
    if kind in ("step", "attend"):
        q = torch.randn(b, t, case["heads"], d, generator=g, device=DEV).to(dtype).transpose(1, 2)
        s["q"] = q if kind == "attend" and t > 1 else q[:, :, 0]
    if kind == "step":
        s["new_k"], s["new_v"] = s["new_k"][:, :, 0], s["new_v"][:, :, 0]
    if own:  # the handle that a user's program keeps, holding the same tokens
        c = importlib.import_module("numerics-and-sparse-attn_b200").Kv8Cache(b, h, m * BLOCK, head_dim=d, dtype=dtype, codes=codes, device=DEV)
        for mine, its in (("k_codes", c.k_codes), ("v_codes", c.v_codes), ("scales", c.scales), ("k_ring", c.k_ring),
                          ("v_ring", c.v_ring), ("table", c.page_table), ("lens", c.lens)):
            its.copy_(s.pop(mine) if mine != "lens" else s[mine])
        s["cache"] = c
    return s


# ---------------------------------------------------------------------------------------- plain forms
def _rows(s, which, pos, lens):
    """Positions pos [B, n] of the cache as float32 [B, Hkv, n, D]: codes times scale from complete blocks, else the ring."""
    b, h = s["lens"].shape[0], s["k_ring"].shape[1]
    codes, ring = s[which + "_codes"], s[which + "_ring"]
    seq = torch.arange(b, device=DEV)[:, None]
    pos = pos.clamp_min(0)
    page = s["table"][seq, (pos // BLOCK).clamp_max(s["table"].shape[1] - 1)].long()
    x = codes.view(torch.uint8)[page, :, pos % BLOCK].view(codes.dtype).float()  # [B, n, Hkv, D]
    x = x * s["scales"][page][..., 0 if which == "k" else 1][..., None]
    in_ring = pos >= (lens // BLOCK * BLOCK)[:, None]
    x = torch.where(in_ring[..., None, None], ring[seq, :, pos % RING].float(), x)
    return x.transpose(1, 2)


def _append(s, new_k, new_v):
    """new_k, new_v [B, Hkv, T, D] at positions lens .. lens + T - 1.  Returns the new lengths."""
    b, h, t, d = new_k.shape
    start, end = s["lens"], s["lens"] + t
    first = start // BLOCK
    m = (BLOCK - 1 + t) // BLOCK  # blocks that the call can complete
    pos = (first * BLOCK)[:, None] + torch.arange(m * BLOCK, device=DEV)
    seq = torch.arange(b, device=DEV)[:, None]
    done = (first[:, None] + 1 + torch.arange(m, device=DEV)) * BLOCK <= end[:, None]
    page = s["table"][seq, (pos[:, ::BLOCK] // BLOCK).clamp_max(s["table"].shape[1] - 1)].long()
    for i, (which, new) in enumerate((("k", new_k), ("v", new_v))):
        codes, ring, rows = s[which + "_codes"], s[which + "_ring"], new.transpose(1, 2)
        old = ring[seq, :, pos % RING]
        x = torch.where((pos < start[:, None])[..., None, None], old, rows[seq, (pos - start[:, None]).clamp(0, t - 1)])
        c, scale = _code(x.view(b, m, BLOCK, h, d).transpose(2, 3), s["codes"])
        raw = codes.view(torch.uint8)
        raw[page] = torch.where(done[..., None, None, None], c.view(torch.uint8), raw[page])
        s["scales"][..., i][page] = torch.where(done[..., None], scale, s["scales"][..., i][page])
        n = min(t, RING)  # the newest tokens; those of the last two blocks stay in the ring
        last = end[:, None] - n + torch.arange(n, device=DEV)
        keep = last >= ((end // BLOCK - 1) * BLOCK)[:, None]
        ring[seq, :, last % RING] = torch.where(keep[..., None, None], rows[:, t - n:], ring[seq, :, last % RING])
    return end


def _attend(s, q, lens):
    """q [B, H, T, D], its tokens the last T of the sequences: softmax attention in 32 bits, rounded once."""
    b, h, t, d = q.shape
    hkv, w, dtype = s["k_ring"].shape[1], s["window"], q.dtype
    if w:  # four sink tokens and what any query token's window holds
        near = lens[:, None] - (w + t - 1) + torch.arange(w + t - 1, device=DEV)
        pos = torch.cat([torch.arange(4, device=DEV).expand(b, 4), torch.where(near < 4, -1, near)], 1)
    else:
        pos = torch.arange(s["table"].shape[1] * BLOCK, device=DEV).expand(b, -1)
    limit = lens[:, None] - t + 1 + torch.arange(t, device=DEV)  # a query token sees positions below its limit
    seen = (pos[:, None] >= 0) & (pos[:, None] < limit[..., None])
    if w:
        seen &= (pos[:, None] < 4) | (pos[:, None] >= limit[..., None] - w)
    k, v = _rows(s, "k", pos, lens), _rows(s, "v", pos, lens)
    qf = q.float().reshape(b, hkv, h // hkv * t, d)
    score = torch.matmul(qf, k.transpose(2, 3)).view(b, hkv, h // hkv, t, -1) * d ** -0.5
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, h // hkv * t, -1), v).view(b, hkv, h // hkv, t, d)
    return torch.where(total > 0, o / total, 0.0).view(b, h, t, d).to(dtype)


def run(s):
    """One pass.  Appends and steps start at the same lengths every time, so a pass can be repeated."""
    kind, t = s["kind"], s["tokens"]
    if own:
        c = s["cache"]
        if kind == "attend":
            return c.attend(s["q"], window=s["window"] or None)
        if kind == "read":
            return c.read(t)
        if kind == "append_read":
            c.append(s["new_k"], s["new_v"], starts=s["lens"])
            return c.read(t, starts=s["lens"])
        out = {}
        if kind == "step":
            out["o"] = c.decode_step(s["q"], s["new_k"], s["new_v"], starts=s["lens"])
        else:
            c.append(s["new_k"], s["new_v"], starts=s["lens"])
        return {**out, "lens": c.lens, "k_codes": c.k_codes, "v_codes": c.v_codes, "scales": c.scales, "k_ring": c.k_ring,
                "v_ring": c.v_ring}
    if kind == "attend":
        q = s["q"]
        return _attend(s, q if q.dim() == 4 else q[:, :, None], s["lens"]).view(q.shape)
    b = s["lens"].shape[0]
    if kind == "read":
        pos = torch.arange(t, device=DEV).expand(b, t)
        return tuple(_rows(s, k, pos, s["lens"]).to(s["dtype"]) for k in ("k", "v"))
    if kind == "step":
        lens = _append(s, s["new_k"][:, :, None], s["new_v"][:, :, None])
        out = {"o": _attend(s, s["q"][:, :, None], lens)[:, :, 0]}
    else:
        lens, out = _append(s, s["new_k"], s["new_v"]), {}
    if kind == "append_read":
        pos = s["lens"][:, None] + torch.arange(t, device=DEV)
        return tuple(_rows(s, k, pos, lens).to(s["dtype"]) for k in ("k", "v"))
    return {**out, "lens": lens, **{k: s[k] for k in ("k_codes", "v_codes", "scales", "k_ring", "v_ring")}}


# ---------------------------------------------------------------------------------------- what a pass needs
def work(case):
    """Each input read once, each output written once."""
    kind, h, hkv, d, t, w = (case[k] for k in ("kind", "heads", "kv_heads", "dim", "tokens", "window"))
    nbytes = flops = 0
    row = 2 * hkv * d  # elements of one token's K and V
    for n in _lens(case):
        if kind in ("step", "attend"):
            new = 1 if kind == "step" else 0
            m = n + new
            full, tail = m // BLOCK * BLOCK, m % BLOCK
            if w and m > w + 4:
                tail = min(tail, w + t - 1)
                full = min(full, w + t - 1 - tail + 4)
            nbytes += row * (full + 2 * (tail - (new if tail else 0))) + full // BLOCK * (8 * hkv + 4)
            nbytes += 2 * h * t * d * 2 + 8 + new * (2 * row + 8)  # q, o, length; the new token
            flops += sum(4 * h * d * min(m - t + 1 + i, w + 4 if w else m) for i in range(t) if m - t + 1 + i > 0)
            if new:
                nbytes += 2 * row + (row * BLOCK + 8 * hkv if m % BLOCK == 0 else 0)  # its ring row, a completed block
        elif kind in ("append", "append_read"):
            done = (n + t) // BLOCK - n // BLOCK
            old = n % BLOCK if done else 0
            stay = min(t, n + t - max(0, (n + t) // BLOCK - 1) * BLOCK)
            nbytes += 2 * row * (t + old + stay) + done * (row * BLOCK + 8 * hkv + 4) + 16
            if kind == "append_read":
                nbytes += 2 * row * t
            flops += 2 * row * done * BLOCK
        else:
            full = min(t, n // BLOCK * BLOCK)
            nbytes += row * full + 2 * row * (t - full) + 2 * row * t + full // BLOCK * (8 * hkv + 4) + 8
            flops += row * full
    return {"bytes": float(nbytes), "flops": float(flops)}


# ---------------------------------------------------------------------------------------- 64 bits
def _exact_code(x, codes):
    """One block [Hkv, 64, D] in float64 -> (code values, scales [Hkv])."""
    x = x.double()
    scale = (x.abs().amax((1, 2)) / TOP[codes]).clamp_min(2.0 ** -126)
    y = x / scale[:, None, None]
    if codes == "int8":
        return torch.round(y), scale
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)  # e4m3: three fraction bits, least exponent -6
    return torch.round(y / step) * step, scale


def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    kind, t, codes, w = case["kind"], case["tokens"], case["codes"], case["window"]
    lens, h, hkv, d = _lens(case), case["heads"], case["kv_heads"], case["dim"]
    table, scales = s["table"].tolist(), s["scales"].double()
    if kind in ("step", "append", "append_read"):
        held = {k: s[k + "_codes"].float().to(torch.float32 if codes == "e4m3" else torch.float64) for k in ("k", "v")}
        rings = {k: s[k + "_ring"].double() for k in ("k", "v")}
        for i, n in enumerate(lens):
            e = n + t
            for c, k in enumerate(("k", "v")):
                new = s["new_" + k][i].double().view(hkv, t, d)
                block0 = n // BLOCK * BLOCK
                before = rings[k][i][:, [p % RING for p in range(block0, n)]]
                run_ = torch.cat([before, new], 1)  # positions block0 .. e - 1
                for j in range(e // BLOCK - n // BLOCK):
                    x, sc = _exact_code(run_[:, BLOCK * j:BLOCK * (j + 1)], codes)
                    page = table[i][n // BLOCK + j]
                    held[k][page], scales[page, :, c] = x.to(held[k].dtype), sc
                stay = list(range(max(n, (e // BLOCK - 1) * BLOCK), e))
                rings[k][i][:, [p % RING for p in stay]] = new[:, [p - n for p in stay]]
    else:
        held = {k: s[k + "_codes"] for k in ("k", "v")}
        rings = {k: s[k + "_ring"] for k in ("k", "v")}
    grow = t if kind in ("step", "append", "append_read") else 0

    def values(i, k, n, blocks):
        """The blocks' tokens, then the ring's, in float64 [Hkv, tokens, D]."""
        c = 0 if k == "k" else 1
        at = torch.tensor([table[i][j] for j in blocks], dtype=torch.int64, device=DEV)
        x = held[k][at].double() * scales[at][:, :, c, None, None]
        x = x.transpose(0, 1).reshape(hkv, -1, d)
        slots = [p % RING for p in range(n // BLOCK * BLOCK, n)]
        return torch.cat([x, rings[k][i][:, slots].double()], 1)

    state = {"lens": s["lens"] + grow, "k_codes": held["k"], "v_codes": held["v"], "scales": scales, "k_ring": rings["k"],
             "v_ring": rings["v"]} if grow else {}
    if kind == "append":
        return state
    if kind in ("read", "append_read"):
        out = []
        for k in ("k", "v"):
            rows = [values(i, k, n + grow, range((n + grow) // BLOCK)) for i, n in enumerate(lens)]
            out.append(torch.stack([r[:, n:n + t] if grow else r[:, :t] for r, n in zip(rows, lens)]))
        return tuple(out)
    tq = t if kind == "attend" else 1
    o = torch.zeros(case["batch"], h, tq, d, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(case["batch"], h, tq, d) if tq == 1 else s["q"].double()
    for i, n in enumerate(lens):
        n += grow
        from_ = max(0, n - w - tq + 1) // BLOCK if w else 0
        blocks = [j for j in range(n // BLOCK) if j >= from_ or (w and j == 0)]
        pos = torch.tensor([p for j in blocks for p in range(BLOCK * j, BLOCK * (j + 1))] + list(range(n // BLOCK * BLOCK, n)),
                           dtype=torch.int64, device=DEV)
        k, v = values(i, "k", n, blocks), values(i, "v", n, blocks)
        for a in range(tq):
            limit = n - tq + a + 1
            if limit <= 0:
                continue
            see = pos < limit
            if w:
                see &= (pos < 4) | (pos >= limit - w)
            score = torch.einsum("gqd,gnd->gqn", q[i, :, a].view(hkv, h // hkv, d), k[:, see]) * d ** -0.5
            o[i, :, a] = torch.einsum("gqn,gnd->gqd", torch.softmax(score, -1), v[:, see]).reshape(h, d)
    o = o if kind == "attend" and t > 1 else o[:, :, 0]
    return {"o": o, **state} if grow else o
