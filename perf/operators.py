"""What is measured of the batched serving operators: page tables from request lengths, the 8-bit K/V store,
attention over the 8-bit cache and token log probabilities.

`run` computes a case in plain torch operations, or, with `own` set, through the library's entry points on
the same device memory.
"""
import ctypes
import math
import random

import torch

own = False

BLOCK = 32                        # positions of a row that share a page
QMAX = {"i8": 127.0, "e4m3": 448.0}
FORMAT = {"i8": 0, "e4m3": 1}     # RBN_KV_I8, RBN_KV_E4M3
DEV = "cuda"


def listed():
    return [
        # one scheduling tick of 64 running sequences: every row gets one more token
        {"name": "plan tick 64", "op": "plan", "rows": 64, "running": 64, "len_lo": 20, "len_hi": 1000, "new_lo": 1,
         "new_hi": 1, "release": 0, "max_blocks": 128},
        # a busy server: 1000 rows of which most run, some are finished and hand their pages back, some are admitted with prompts
        {"name": "plan mixed 1000", "op": "plan", "rows": 1000, "running": 900, "len_lo": 1, "len_hi": 8000,
         "new_lo": 1, "new_hi": 131, "release": 100, "max_blocks": 512},
        # the K/V store of one decode step of 16 sequences, five K/V heads for twenty query heads
        {"name": "store step 16", "op": "store", "rows": 16, "heads": 20, "kv_heads": 5, "hd": 128, "fmt": "i8",
         "len_lo": 31, "len_hi": 100000, "new_lo": 1, "new_hi": 1, "theta": 10000.0},
        # four ragged prompts that go in at once, as many K/V heads as query heads
        {"name": "store prompts 4", "op": "store", "rows": 4, "heads": 20, "kv_heads": 20, "hd": 128, "fmt": "i8",
         "len_lo": 1, "len_hi": 77, "new_lo": 301, "new_hi": 1500, "theta": 10000.0},
        # one sequence, one token, a short context: latency
        {"name": "attend step 1x1000", "op": "attend", "rows": 1, "heads": 20, "kv_heads": 20, "hd": 128, "fmt": "i8",
         "len_lo": 1000, "len_hi": 1000, "new_lo": 1, "new_hi": 1},
        # 16 sequences of the decoder's own head layout in one decode step
        {"name": "attend step 16", "op": "attend", "rows": 16, "heads": 20, "kv_heads": 5, "hd": 128, "fmt": "i8",
         "len_lo": 517, "len_hi": 4000, "new_lo": 1, "new_hi": 1},
        # 64 sequences of very different lengths, e4m3 codes
        {"name": "attend step 64 ragged", "op": "attend", "rows": 64, "heads": 32, "kv_heads": 8, "hd": 128,
         "fmt": "e4m3", "len_lo": 63, "len_hi": 16000, "new_lo": 1, "new_hi": 1},
        # one very long sequence: the work has to be split along the keys
        {"name": "attend step 1x131000", "op": "attend", "rows": 1, "heads": 32, "kv_heads": 8, "hd": 128, "fmt": "i8",
         "len_lo": 131000, "len_hi": 131000, "new_lo": 1, "new_hi": 1},
        # the decoder's 512-token prompt
        {"name": "attend prompt 512", "op": "attend", "rows": 1, "heads": 20, "kv_heads": 20, "hd": 128, "fmt": "i8",
         "len_lo": 0, "len_hi": 0, "new_lo": 512, "new_hi": 512},
        # ragged prompts on top of what the rows hold already
        {"name": "attend prompts 5", "op": "attend", "rows": 5, "heads": 20, "kv_heads": 5, "hd": 128, "fmt": "i8",
         "len_lo": 1, "len_hi": 2000, "new_lo": 250, "new_hi": 1500},
        # the logits of one decode step of 16 sequences, the decoder's vocabulary
        {"name": "logprobs 16x32000", "op": "logprobs", "rows": 16, "vocab": 32000, "top": 5, "masked": 0.0},
        # scoring a prompt: a thousand positions of a large odd vocabulary, a part of it masked
        {"name": "logprobs 1000x100003", "op": "logprobs", "rows": 1000, "vocab": 100003, "top": 8, "masked": 0.3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "store", "attend", "attend", "logprobs"])
    if op == "plan":
        rows = _log_int(rng, 2, 1000)
        running = rng.randint(1, rows)
        return {"op": op, "rows": rows, "running": running, "len_lo": 1, "len_hi": _log_int(rng, 40, 8000), "new_lo": 1,
                "new_hi": _log_int(rng, 1, 130), "release": rng.randint(0, rows - running), "max_blocks": 512}
    if op == "logprobs":
        vocab = _log_int(rng, 300, 150000)
        return {"op": op, "rows": _log_int(rng, 1, max(2, min(2000, 10 ** 8 // vocab))), "vocab": vocab,
                "top": rng.randint(0, 20), "masked": rng.choice([0.0, 0.2, 0.9])}
    kv_heads = rng.choice([1, 2, 4, 5, 8, 20])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7] if kv_heads <= 8 else [1])
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "hd": rng.choice([64, 128, 128]),
         "fmt": rng.choice(["i8", "i8", "e4m3"])}
    if op == "store":
        new = _log_int(rng, 1, 1500)
        rows = _log_int(rng, 1, max(2, min(256, 6000 // new)))
        return dict(c, rows=rows, len_lo=0, len_hi=_log_int(rng, 1, 130000), new_lo=max(1, new // 3), new_hi=new,
                    theta=rng.choice([10000.0, 500000.0]))
    if rng.random() < 0.6:        # a decode step
        ctx = _log_int(rng, 2, 131000)
        rows = _log_int(rng, 1, max(2, min(128, 10 ** 6 // ctx * 8 // kv_heads)))
        rows = max(1, min(rows, 131000 * 8 // (ctx * kv_heads)))
        new = rng.choice([1, 1, 1, 3])
        return dict(c, rows=rows, len_lo=max(0, ctx // 7), len_hi=ctx, new_lo=1, new_hi=new)
    new = _log_int(rng, 5, 1500)
    ctx = _log_int(rng, 1, 2000)
    rows = max(1, min(_log_int(rng, 1, 16), 5 * 1500 * 3500 * 20 // (new * (new + ctx) * heads)))
    return dict(c, rows=rows, len_lo=0, len_hi=ctx, new_lo=max(1, new // 4), new_hi=new)


# ---- shapes: the lengths belong to the case, the values to the seed ---------------------------
def _lengths(case):
    """(tokens held before, tokens new) of every row."""
    rng = random.Random("%s" % sorted((k, v) for k, v in case.items() if k != "name"))
    held, new = [], []
    for _ in range(case["rows"]):
        lo, hi = case["len_lo"], case["len_hi"]
        held.append(_log_int(rng, lo + 1, hi + 1) - 1)
        new.append(_log_int(rng, case["new_lo"], case["new_hi"]))
    if case["op"] == "plan":
        rows = list(range(case["rows"]))
        rng.shuffle(rows)
        for r in rows[case["running"]:]:
            new[r] = 0
        for r in rows[case["running"]:case["running"] + case["release"]]:
            new[r] = -1
        for r in rows[case["running"] + case["release"]:]:   # rows that hold nothing
            held[r] = 0
    return held, new


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}
    held, new = _lengths(case)
    if op == "plan":
        t = sum(n for n in new if n > 0)
        pages = sum(_blocks(h + n) - _blocks(h) if n > 0 else _blocks(h) if n < 0 else 0 for h, n in zip(held, new))
        return {"bytes": 4 * (5 * case["rows"] + 3 * t + 3 * pages), "flops": 10 * t}
    h, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
    t = sum(new)
    if op == "store":
        touched = sum(n + m % BLOCK for m, n in zip(held, new))
        return {"bytes": 4 * t * (2 * h + 2 * kvh) * hd + 2 * touched * kvh * hd * 5, "flops": 6 * t * (h + kvh) * hd}
    keys = sum(m * n + n * (n + 1) // 2 for m, n in zip(held, new))
    cache = sum((m + n) // BLOCK * BLOCK + 2 * ((m + n) % BLOCK) for m, n in zip(held, new))
    return {"bytes": 2 * cache * kvh * hd + 8 * t * h * hd, "flops": 4 * keys * h * hd}


# ---- inputs ------------------------------------------------------------------------------------
def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _batch(held, new, pages_of, max_blocks):
    """The plan of a batch, as rbn_kv_plan writes it: tokens in row order and the blocks they touch."""
    rows = len(held)
    start, row, pos, slot, unit = [0], [], [], [], []
    table = torch.full((rows, max_blocks), -1, dtype=torch.int32)
    for r in range(rows):
        n_b = _blocks(held[r] + new[r])
        table[r, :n_b] = pages_of[r][:n_b]
        for p in range(held[r], held[r] + new[r]):
            if p == held[r] or p % BLOCK == 0:
                unit.append(len(row))
            row.append(r)
            pos.append(p)
            slot.append(int(pages_of[r][p // BLOCK]) * BLOCK + p % BLOCK)
        start.append(len(row))
    t = len(row)
    cap = -(-t // 8) * 8          # a batch padded to a multiple of eight tokens, as a captured step would be
    unit_t = torch.full((cap,), -1, dtype=torch.int32)
    unit_t[:len(unit)] = torch.tensor(unit, dtype=torch.int32)
    pad = [-1] * (cap - t)
    return {"table": table.to(DEV), "start": _i32(start), "row": _i32(row + pad), "pos": _i32(pos + pad),
            "slot": _i32(slot + pad), "unit": unit_t.to(DEV), "count": _i32([t, len(unit)]), "tokens": t,
            "units": len(unit), "max_tokens": cap, "len": _i32([h + n for h, n in zip(held, new)])}


def _page_lists(gen, counts, pages):
    perm = torch.randperm(pages, generator=gen, dtype=torch.int32)
    return list(torch.split(perm[:sum(counts)], counts))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    op = case["op"]
    if op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn(rows, vocab, device=DEV, generator=gen) * 2.5
        logits += torch.randn(rows, 1, device=DEV, generator=gen) * 5     # rows have levels of their own
        if case["masked"]:
            logits.masked_fill_(torch.rand(rows, vocab, device=DEV, generator=gen) < case["masked"], -math.inf)
        target = torch.randint(0, vocab, (rows,), device=DEV, generator=gen, dtype=torch.int32)
        top = case["top"]
        out = {"logprob": torch.zeros(rows, device=DEV), "entropy": torch.zeros(rows, device=DEV),
               "top_token": torch.zeros(rows, top, dtype=torch.int32, device=DEV),
               "top_logprob": torch.zeros(rows, top, device=DEV)}
        return {"case": case, "logits": logits, "target": target, "out": out}
    held, new = _lengths(case)
    rows = case["rows"]
    if op == "plan":
        counts = [_blocks(h) for h in held]
        spare = sum(_blocks(h + max(n, 0)) - _blocks(h) for h, n in zip(held, new)) + rows
        pages = sum(counts) + spare
        perm = torch.randperm(pages, generator=cpu, dtype=torch.int32)
        lists = torch.split(perm[:sum(counts)], counts)
        table = torch.full((rows, case["max_blocks"]), -1, dtype=torch.int32)
        for r in range(rows):
            table[r, :counts[r]] = lists[r]
        head = int(torch.randint(0, pages, (1,), generator=cpu))
        ring = torch.full((pages,), -1, dtype=torch.int32)
        ring[(head + torch.arange(spare)) % pages] = perm[sum(counts):]
        t = sum(n for n in new if n > 0)
        cap = -(-t // 8) * 8
        blank = lambda n: torch.full((n,), -1, dtype=torch.int32, device=DEV)  # noqa: E731
        return {"case": case, "pages": pages, "table": table.to(DEV), "len": _i32(held), "new": _i32(new),
                "ring": ring.to(DEV), "ring_state": _i32([head, spare]), "max_tokens": cap, "start": blank(rows + 1),
                "row": blank(cap), "pos": blank(cap), "slot": blank(cap), "unit": blank(cap), "count": blank(2),
                "len_out": blank(rows), "ring_state_out": blank(2)}
    h, kvh, hd, fmt = case["heads"], case["kv_heads"], case["hd"], case["fmt"]
    total = [a + b for a, b in zip(held, new)]
    max_blocks = _blocks(max(total)) + 1
    if op == "store":             # only the blocks that the call touches need pages here
        counts = [_blocks(n) - m // BLOCK for m, n in zip(held, total)]
        pages = sum(counts) + 3
        lists = [torch.cat([torch.full((m // BLOCK,), -1, dtype=torch.int32), p])
                 for m, p in zip(held, _page_lists(cpu, counts, pages))]
    else:
        counts = [_blocks(n) for n in total]
        pages = sum(counts) + 3
        lists = _page_lists(cpu, counts, pages)
    s = {"case": case, "pages": pages, "max_blocks": max_blocks, "rows": rows}
    s.update(_batch(held, new, lists, max_blocks))
    cap = s["max_tokens"]
    s["max_new"] = max(new)
    s["k_open"] = torch.randn(rows, kvh, BLOCK, hd, device=DEV, generator=gen).half()
    s["v_open"] = torch.randn(rows, kvh, BLOCK, hd, device=DEV, generator=gen).half()
    if op == "store":
        s["qkv"] = torch.randn(cap, (h + 2 * kvh) * hd, device=DEV, generator=gen)
        s["q"] = torch.zeros(cap, h, hd, device=DEV)
        s["k_codes"] = torch.zeros(pages, kvh, BLOCK * hd, dtype=torch.uint8, device=DEV)
        s["v_codes"] = torch.zeros(pages, kvh, BLOCK * hd, dtype=torch.uint8, device=DEV)
        s["k_scale"] = torch.zeros(pages, kvh, device=DEV)
        s["v_scale"] = torch.zeros(pages, kvh, device=DEV)
        # what is read back: every position of the blocks that the call touches
        rd, u = [], 0
        for r in range(rows):
            for b in range(held[r] // BLOCK, _blocks(total[r])):
                rd += [(r, p, u, p % BLOCK) for p in range(b * BLOCK, min(total[r], (b + 1) * BLOCK))]
                u += 1
        rd = _i32(rd)
        s["rd_row"], s["rd_pos"], s["rd_unit"], s["rd_off"] = (rd[:, i].contiguous() for i in range(4))
        s["rd_k"] = torch.zeros(len(rd), kvh, hd, dtype=torch.float16, device=DEV)
        s["rd_v"] = torch.zeros(len(rd), kvh, hd, dtype=torch.float16, device=DEV)
        return s
    s["out"] = torch.zeros(cap, h, hd, device=DEV)
    s["q"] = torch.randn(cap, h, hd, device=DEV, generator=gen) * 1.5
    for which in ("k", "v"):
        # codes as the store leaves them: each block reaches the format's largest value
        x = torch.randn(pages, kvh, BLOCK, hd, device=DEV, generator=gen)
        x *= QMAX[fmt] / x.abs().amax(dim=(2, 3), keepdim=True)
        s[which] = x.round().to(torch.int8) if fmt == "i8" else x.to(torch.float8_e4m3fn)
        del x
        s[which + "_scale"] = (4.0 * torch.exp(0.4 * torch.randn(pages, kvh, device=DEV, generator=gen))) / QMAX[fmt]
        raw = s[which].view(torch.uint8)
        if which == "k":          # the library's page layouts (include/ronn_bitnet_hip.h)
            raw = raw.view(pages, kvh, 2, 16, hd // 64, 2, 4, 8).permute(0, 1, 2, 4, 6, 3, 5, 7)
        else:
            raw = raw.view(pages, kvh, 2, 4, 4, hd // 32, 2, 16).permute(0, 1, 5, 3, 7, 6, 2, 4)
        s[which + "_codes"] = raw.contiguous().view(pages, kvh, BLOCK * hd)
    return s


# ---- the plain forms ---------------------------------------------------------------------------
def _plain_plan(s):
    c = s["case"]
    length, new, table = s["len"].long(), s["new"].long(), s["table"].clone()
    rows, cap, pages, max_tokens = c["rows"], c["max_blocks"] * BLOCK, s["pages"], s["max_tokens"]
    head, count = s["ring_state"].long()
    blocks = lambda n: (n + BLOCK - 1) // BLOCK  # noqa: E731
    release = new < 0
    n = torch.where((new > 0) & (length + new <= cap) & (new <= max_tokens), new, 0)
    need = blocks(length + n) - blocks(length)
    n = torch.where((need == 0) | (need.cumsum(0) <= count), n, 0)
    n = torch.where(n.cumsum(0) <= max_tokens, n, 0)
    need = torch.where(n > 0, blocks(length + n) - blocks(length), 0)
    end = n.cumsum(0)
    first_page = need.cumsum(0) - need
    back = torch.where(release, blocks(length), 0)
    start = torch.cat([torch.zeros_like(end[:1]), end])
    tokens = end[-1]
    i = torch.arange(max_tokens, device=DEV)
    valid = i < tokens
    row = torch.searchsorted(end, i, right=True).clamp(max=rows - 1)
    pos = length[row] + i - start[row]
    block = (pos // BLOCK).clamp(0, c["max_blocks"] - 1)
    fresh = block - blocks(length[row])
    ring = s["ring"].clone()
    page = torch.where(fresh >= 0, ring[(head + first_page[row] + fresh) % pages].long(), table[row, block].long())
    keep = lambda x, old: torch.where(valid, x, old.long()).int()  # noqa: E731
    flat = torch.cat([table.view(-1), table.new_zeros(1)])
    flat[torch.where(valid & (fresh >= 0), row * c["max_blocks"] + block, rows * c["max_blocks"])] = page.int()
    leader = valid & ((pos % BLOCK == 0) | (i == start[row]))
    unit = torch.cat([s["unit"], s["unit"].new_zeros(1)])
    unit[torch.where(leader, leader.long().cumsum(0) - 1, max_tokens)] = i.int()
    # pages of released rows go behind the free ones
    j = torch.arange(table.shape[1], device=DEV)
    gone = j[None, :] < back[:, None]
    behind = (head + count + (back.cumsum(0) - back)[:, None] + j[None, :]) % pages
    ring = torch.cat([ring, ring.new_zeros(1)])
    ring[torch.where(gone, behind, pages)] = s["table"]
    return {"start": start.int(), "row": keep(row, s["row"]), "pos": keep(pos, s["pos"]),
            "slot": keep(page * BLOCK + pos % BLOCK, s["slot"]), "unit": unit[:-1],
            "count": torch.stack([tokens, leader.sum()]).int(), "table": flat[:-1].view_as(table), "ring": ring[:-1],
            "len_out": torch.where(release, 0, length + n).int(),
            "ring_state_out": torch.stack([(head + need.sum()) % pages, count - need.sum() + back.sum()]).int()}


def _rotated(x, pos, theta):
    """Pairs (i, i + hd/2) of x [T, heads, hd] turned by pos * theta^(-2i/hd); the angle in 64 bits."""
    half = x.shape[-1] // 2
    i = torch.arange(half, device=DEV, dtype=torch.float64)
    angle = pos.double()[:, None] * theta ** (-i / half)
    cs, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cs - b * sn, b * cs + a * sn], dim=-1)


def _plain_store(s):
    c, t, rows = s["case"], s["tokens"], s["rows"]
    h, kvh, hd = c["heads"], c["kv_heads"], c["hd"]
    x = s["qkv"][:t].view(t, h + 2 * kvh, hd)
    pos, start = s["pos"][:t].long(), s["start"].long()
    q = s["q"].clone()
    q[:t] = _rotated(x[:, :h], pos, c["theta"])
    lead = s["unit"][:s["units"]].long()
    r = s["row"][lead].long()
    b = pos[lead] // BLOCK
    p = b[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)
    first = pos[start[:-1].clamp(max=t - 1)][r][:, None]
    end = first + (start[1:] - start[:-1])[r][:, None]
    full = ((b + 1) * BLOCK)[:, None] <= end
    src = torch.where((p >= first) & (p < end), start[r][:, None] + p - first, t + r[:, None] * BLOCK + p % BLOCK)
    got = {"q": q}
    # the unfinished block of a row is the last one the call touches
    last = torch.cat([r[1:] != r[:-1], r[:1] == r[:1]])
    dump = torch.where(last, r, rows)
    for which, new in (("k", _rotated(x[:, h:h + kvh], pos, c["theta"])), ("v", x[:, h + kvh:])):
        held = s[which + "_open"]
        new = torch.nan_to_num(new, nan=0.0).clamp(-65504.0, 65504.0).half()
        every = torch.cat([new, held.permute(0, 2, 1, 3).reshape(rows * BLOCK, kvh, hd)])
        v = every[src]                                     # [units, 32, kv_heads, hd]
        f = v.float()
        scale = f.abs().amax(dim=(1, 3), keepdim=True) / QMAX[c["fmt"]]
        code = torch.where(scale > 0, f / scale, torch.zeros_like(f))
        code = code.round().clamp(-127, 127) if c["fmt"] == "i8" else code.to(torch.float8_e4m3fn).float()
        value = torch.where(full[:, :, None, None], (code * scale).half(), v)
        got[which] = value[s["rd_unit"].long(), s["rd_off"].long()]
        write = ((p < end) & ~full)[:, :, None, None].permute(0, 2, 1, 3)
        more = torch.cat([held, held[:1]])
        more[dump] = torch.where(write, v.permute(0, 2, 1, 3), held[r])
        held.copy_(more[:rows])
    return got


def _plain_attend(s):
    c, t, rows = s["case"], s["tokens"], s["rows"]
    h, kvh, hd, g = c["heads"], c["kv_heads"], c["hd"], c["heads"] // c["kv_heads"]
    nb = s["max_blocks"]
    start, length = s["start"].long(), s["len"].long()
    table = s["table"].long().clamp(min=0)
    at = torch.arange(rows, device=DEV)
    kv = []
    for which in ("k", "v"):
        x = s[which][table].float() * s[which + "_scale"][table][..., None, None]
        x[at, length // BLOCK] = s[which + "_open"].float()
        kv.append(x.permute(0, 2, 1, 3, 4).reshape(rows, kvh, nb * BLOCK, hd))
        del x
    n = s["max_new"]
    tok = start[:-1, None] + torch.arange(n, device=DEV)
    valid = tok < start[1:, None]
    tok = tok.clamp(max=t - 1)
    pos = s["pos"].long()[tok]
    q = s["q"][tok].view(rows, n, kvh, g, hd).permute(0, 2, 3, 1, 4).reshape(rows, kvh, g * n, hd)
    score = torch.matmul(q, kv[0].transpose(2, 3)).view(rows, kvh, g, n, nb * BLOCK) / math.sqrt(hd)
    score.masked_fill_((torch.arange(nb * BLOCK, device=DEV) > pos[..., None])[:, None, None], -math.inf)
    score -= score.amax(dim=-1, keepdim=True)
    score.exp_()
    total = score.sum(dim=-1, keepdim=True)
    # values behind the end of a row may be anything
    kv[1].masked_fill_((torch.arange(nb * BLOCK, device=DEV) >= length[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(score.view(rows, kvh, g * n, nb * BLOCK), kv[1]).view(rows, kvh, g, n, hd) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(rows * n, h, hd)
    more = torch.cat([s["out"], s["out"][:1]])
    more[torch.where(valid, tok, s["max_tokens"]).view(-1)] = o
    return more[:-1]


def _plain_logprobs(s):
    x, top = s["logits"], s["case"]["top"]
    m = x.amax(dim=1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    norm = torch.log(total)
    entropy = norm[:, 0] - torch.where(e > 0, e * d, 0.0).sum(dim=1) / total[:, 0]
    logprob = (torch.gather(d, 1, s["target"].long()[:, None]) - norm)[:, 0]
    # one key per value orders by value and then by the lower index
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 31) + (
        (1 << 31) - 1 - torch.arange(x.shape[1], device=DEV))
    index = torch.topk(key, min(top, x.shape[1]), dim=1).indices
    return {"logprob": logprob, "entropy": entropy, "top_token": index.int(),
            "top_logprob": torch.gather(d, 1, index) - norm}


# ---- the library's calls -----------------------------------------------------------------------
_CTX = {}


def _context():
    """One context on torch's own stream, as a program that mixes torch and the library keeps."""
    if not _CTX:
        from ronn_amd.device import Context
        _CTX["ctx"] = Context(0, stream=torch.cuda.current_stream().cuda_stream)
    return _CTX["ctx"]


def _descriptors(s):
    """The library's descriptors of the state's buffers, which a program makes once beside them."""
    if "desc" not in s:
        from ronn_amd import _lib
        c, p = s["case"], lambda name: s[name].data_ptr() if name in s else None
        table = _lib.KvTable(rows=c["rows"], max_blocks=s["table"].shape[1], pages=s["pages"], d_table=p("table"),
                             d_len=p("len"), d_ring=p("ring"), d_ring_state=p("ring_state"))
        batch = _lib.KvBatch(max_tokens=s["max_tokens"], d_start=p("start"), d_row=p("row"), d_pos=p("pos"),
                             d_slot=p("slot"), d_unit=p("unit"), d_count=p("count"))
        layer = None
        if c["op"] != "plan":
            layer = ctypes.byref(_lib.KvLayer(
                format=FORMAT[c["fmt"]], kv_heads=c["kv_heads"], head_dim=c["hd"], d_k=p("k_codes"), d_v=p("v_codes"),
                d_k_scale=p("k_scale"), d_v_scale=p("v_scale"), d_k_open=p("k_open"), d_v_open=p("v_open")))
        s["desc"] = ctypes.byref(table), ctypes.byref(batch), layer
    return s["desc"]


def _own(s):
    from ronn_amd._lib import check
    c, ctx = s["case"], _context()
    lib, handle = ctx.lib, ctx.handle
    if c["op"] == "logprobs":
        o, top = s["out"], c["top"]
        check(lib.rbn_token_logprobs_f32(
            handle, s["logits"].data_ptr(), c["rows"], c["vocab"], c["vocab"], s["target"].data_ptr(), top,
            o["logprob"].data_ptr(), o["entropy"].data_ptr(), o["top_token"].data_ptr() if top else None,
            o["top_logprob"].data_ptr() if top else None))
        return o
    table, batch, layer = _descriptors(s)
    if c["op"] == "plan":
        check(lib.rbn_kv_plan(handle, table, s["new"].data_ptr(), batch, s["len_out"].data_ptr(),
                              s["ring_state_out"].data_ptr()))
        return {k: s[k] for k in ("start", "row", "pos", "slot", "unit", "count", "table", "ring", "len_out",
                                  "ring_state_out")}
    if c["op"] == "store":
        check(lib.rbn_rope_kv_store_q8(handle, s["qkv"].data_ptr(), table, batch, layer, c["heads"], c["theta"],
                                       s["q"].data_ptr()))
        check(lib.rbn_kv_read_f16(handle, table, layer, s["rd_row"].data_ptr(), s["rd_pos"].data_ptr(),
                                  s["rd_row"].numel(), s["rd_k"].data_ptr(), s["rd_v"].data_ptr()))
        return {"q": s["q"], "k": s["rd_k"], "v": s["rd_v"]}
    check(lib.rbn_attention_q8kv(handle, s["q"].data_ptr(), table, batch, layer, c["heads"], s["max_new"],
                                 s["out"].data_ptr()))
    return s["out"]


PLAIN = {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend, "logprobs": _plain_logprobs}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---- 64 bits, from the definitions, row by row ---------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None               # whole numbers only
    if op == "logprobs":
        got = {"logprob": [], "entropy": [], "top_token": None, "top_logprob": []}
        for x, y in zip(s["logits"], s["target"].tolist()):
            x = x.double()
            lp = x - torch.logsumexp(x, 0)
            got["logprob"].append(lp[y])
            p = torch.softmax(x, 0)
            got["entropy"].append(-torch.special.xlogy(p, p).sum())
            got["top_logprob"].append(torch.sort(lp, descending=True).values[:case["top"]])
        return {k: torch.stack(v) if v is not None else None for k, v in got.items()}
    held, new = _lengths(case)
    h, kvh, hd, fmt = case["heads"], case["kv_heads"], case["hd"], case["fmt"]
    first = 0
    if op == "store":
        q_all, k_all, v_all = [], [], []
        freq = torch.tensor([case["theta"] ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64, device=DEV)
        for r, (m, n) in enumerate(zip(held, new)):
            x = s["qkv"][first:first + n].double().view(n, h + 2 * kvh, hd)
            first += n
            z = torch.complex(x[..., :hd // 2], x[..., hd // 2:])
            z = z * torch.polar(torch.ones_like(freq), torch.arange(m, m + n, device=DEV).double()[:, None] * freq)[:, None]
            turned = torch.cat([z.real, z.imag], dim=-1)
            q_all.append(turned[:, :h])
            for to, vals, before in ((k_all, turned[:, h:h + kvh], s["k_open"]), (v_all, x[:, h + kvh:], s["v_open"])):
                seq = torch.cat([before[r].double().transpose(0, 1)[:m % BLOCK], vals.half().double()])
                for b in range(0, len(seq), BLOCK):
                    y = seq[b:b + BLOCK].clone()
                    if len(y) == BLOCK:
                        step = y.abs().amax(dim=(0, 2), keepdim=True) / QMAX[fmt]
                        y = y / step
                        y = (torch.round(y) if fmt == "i8" else y.float().to(torch.float8_e4m3fn).double()) * step
                    to.append(y)
        q = torch.zeros(s["max_tokens"], h, hd, dtype=torch.float64, device=DEV)
        q[:first] = torch.cat(q_all)
        return {"q": q, "k": torch.cat(k_all), "v": torch.cat(v_all)}
    out = torch.zeros(s["max_tokens"], h, hd, dtype=torch.float64, device=DEV)
    for r, (m, n) in enumerate(zip(held, new)):
        whole, rest = divmod(m + n, BLOCK)
        pages = s["table"][r, :whole].long()
        kv = []
        for which in ("k", "v"):
            x = s[which][pages].double() * s[which + "_scale"][pages].double()[:, :, None, None]
            x = x.transpose(0, 1).reshape(kvh, whole * BLOCK, hd)
            kv.append(torch.cat([x, s[which + "_open"][r][:, :rest].double()], dim=1))
        q = s["q"][first:first + n].double().view(n, kvh, h // kvh, hd)
        keys = torch.arange(m + n, device=DEV)
        hidden = keys[None, :] > (m + torch.arange(n, device=DEV))[:, None]
        for j in range(kvh):
            for i in range(h // kvh):
                score = (q[:, j, i] @ kv[0][j].T / math.sqrt(hd)).masked_fill(hidden, -math.inf)
                out[first:first + n, j * (h // kvh) + i] = torch.softmax(score, -1) @ kv[1][j]
        first += n
    return out
