"""numpy restatement of the batched serving operators: page plan, 8-bit K/V cache, attention, token log
probabilities.  Test infrastructure only; 64 bits wherever a result is rounded once at the end."""
import numpy as np

BLOCK = 32
QMAX = {"i8": 127.0, "e4m3": 448.0}


def blocks(n):
    return -(-n // BLOCK)


def e4m3_values():
    """The finite values of e4m3 (4 exponent bits, bias 7, 3 mantissa bits, no infinities), by code."""
    v = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v.append(np.nan if e == 15 and m == 7 else -x if c & 128 else x)
    return np.array(v)


_E4M3 = np.sort(np.unique(np.abs(e4m3_values()[:127])))


def round_e4m3(x):
    """Nearest e4m3 value, ties to the even mantissa; |x| <= 448."""
    x = np.asarray(x, dtype=np.float64)
    a = np.minimum(np.abs(x), 448.0)
    e = np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0)
    step = np.exp2(e - 3)
    return np.copysign(np.minimum(np.round(a / step) * step, 448.0), x)


def to_f16(x):
    x = np.where(np.isnan(x), np.float32(0), np.asarray(x, dtype=np.float32))
    return np.clip(x, -65504.0, 65504.0).astype(np.float16)


def quantise_block(x16, fmt):
    """[32, hd] f16 -> (values the codes stand for, float32 scale), codes as numbers."""
    x = x16.astype(np.float32)
    scale = np.float32(np.abs(x).max() * np.float32(1 / QMAX[fmt]))
    y = (x / scale).astype(np.float32) if scale > 0 else np.zeros_like(x)
    code = np.round(y) if fmt == "i8" else round_e4m3(y)
    return code.astype(np.float32), scale


def rope64(x, pos, theta):
    """x [n, heads, hd] rotated in 64 bits."""
    x = np.asarray(x, dtype=np.float64)
    half = x.shape[-1] // 2
    ang = np.asarray(pos, dtype=np.float64)[:, None] * float(theta) ** (-np.arange(half) / half)
    cs, sn = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * cs - b * sn, b * cs + a * sn], axis=-1)


def plan(length, new, table, ring, state, max_tokens):
    """rbn_kv_plan on numpy arrays, row by row; returns a dict like the device's arrays and the flags."""
    rows, max_blocks = table.shape
    pages = len(ring)
    head, count = int(state[0]), int(state[1])
    table, ring = table.copy(), ring.copy()
    n_of, need_sum, flags = [], 0, 0
    for r in range(rows):
        n = int(new[r])
        if n > 0:
            if length[r] + n > max_blocks * BLOCK or n > max_tokens:
                n, flags = 0, flags | 2
            else:
                need = blocks(length[r] + n) - blocks(length[r])
                need_sum += need
                if need and need_sum > count:
                    n, flags = 0, flags | 2
        n_of.append(n)
    tok = 0
    for r in range(rows):
        if n_of[r] > 0:
            tok += n_of[r]
            if tok > max_tokens:
                n_of[r], flags = 0, flags | 2
    start, row, pos, slot, unit = [0], [], [], [], []
    taken, back = 0, []
    len_out = np.array(length).copy()
    for r in range(rows):
        n = n_of[r]
        if n < 0:
            back += [int(p) for p in table[r, :blocks(length[r])]]
            len_out[r] = 0
        for p in range(length[r], length[r] + max(n, 0)):
            if p % BLOCK == 0:
                table[r, p // BLOCK] = ring[(head + taken) % pages]
                taken += 1
            if p == length[r] or p % BLOCK == 0:
                unit.append(len(row))
            row.append(r)
            pos.append(p)
            slot.append(int(table[r, p // BLOCK]) * BLOCK + p % BLOCK)
        if n > 0:
            len_out[r] += n
        start.append(len(row))
    for j, p in enumerate(back):
        ring[(head + count + j) % pages] = p
    state_out = np.array([(head + taken) % pages, count - taken + len(back)], dtype=np.int32)
    return dict(start=np.array(start), row=np.array(row, dtype=np.int32), pos=np.array(pos, dtype=np.int32),
                slot=np.array(slot, dtype=np.int32), unit=np.array(unit, dtype=np.int32), table=table, ring=ring,
                len_out=len_out, ring_state_out=state_out, flags=flags)


class Cache:
    """One layer: the f16 values of every row's tokens; what the cache holds follows from them alone."""

    def __init__(self, rows, kv_heads, hd, fmt):
        self.fmt, self.kv_heads, self.hd = fmt, kv_heads, hd
        self.x = [[np.zeros((0, kv_heads, hd), np.float16) for _ in range(2)] for _ in range(rows)]

    def append(self, row, k, v):
        """k (rotated), v [n, kv_heads, hd] float."""
        for i, y in enumerate((k, v)):
            self.x[row][i] = np.concatenate([self.x[row][i], to_f16(y)])

    def end(self, row):
        self.x[row] = [np.zeros((0, self.kv_heads, self.hd), np.float16) for _ in range(2)]

    def values(self, row):
        """K and V [len, kv_heads, hd] in 64 bits: code * scale in full blocks, f16 in the last one."""
        out = []
        for x in self.x[row]:
            v = x.astype(np.float64)
            for b in range(len(x) // BLOCK):
                for h in range(self.kv_heads):
                    code, scale = quantise_block(x[b * BLOCK:(b + 1) * BLOCK, h], self.fmt)
                    v[b * BLOCK:(b + 1) * BLOCK, h] = code.astype(np.float64) * np.float64(scale)
            out.append(v)
        return out


def attention(q, pos, k, v):
    """q [n, heads, hd], positions [n], K and V [len, kv_heads, hd]; 64 bits."""
    q = np.asarray(q, dtype=np.float64)
    n, heads, hd = q.shape
    group = heads // k.shape[1]
    out = np.zeros((n, heads, hd))
    for i in range(n):
        m = pos[i] + 1
        for h in range(heads):
            s = k[:m, h // group] @ q[i, h] / np.sqrt(hd)
            p = np.exp(s - s.max())
            out[i, h] = p @ v[:m, h // group] / p.sum()
    return out


def logprobs(x, target, top):
    """Row by row in 64 bits: (log probability of the target, entropy, top tokens, their log probabilities)."""
    rows, vocab = x.shape
    lp, ent = np.zeros(rows), np.zeros(rows)
    tok, top_lp = np.full((rows, top), -1, np.int32), np.full((rows, top), -np.inf)
    for r in range(rows):
        z = x[r].astype(np.float64)
        with np.errstate(all="ignore"):
            m = z.max()
            if m == -np.inf:
                d = np.full(vocab, -np.inf)
                ent[r] = 0.0
            else:
                d = z - m
                e = np.exp(d)
                d = d - np.log(e.sum())
                p = np.exp(d)
                ent[r] = -np.where(p > 0, p * d, np.where(p == 0, 0.0, np.nan)).sum()
        if 0 <= target[r] < vocab:
            lp[r] = d[target[r]]
        value = np.where(np.isnan(x[r]), -np.inf, x[r])
        order = np.lexsort((np.arange(vocab), -value, np.isnan(x[r])))[:top]
        tok[r, :len(order)] = order
        top_lp[r, :len(order)] = d[order]
    return lp, ent, tok, top_lp
