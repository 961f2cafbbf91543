"""The batched serving operators against tests/batch_model.py (64 bits): page plan, 8-bit K/V store, attention
over it, token log probabilities, and a run of them together.

Tolerances, u = 2^-24 (half a step of f32, relative):
  plan, V of the store, what the cache returns for V: equal bits (every step is one exactly rounded operation).
  K of the store: the rotation is computed in f32, so an f16 rounding may fall to the neighbour (one f16 step), a block's
    scale may move by one f16 step of its largest value (2^-10 relative at most), and a code by one step.
  attention: a score is off by at most (hd + 8) u sum|q k| / sqrt(hd) =: e, a weight by 2 e + 8 u relatively (both scores of its
    exponent, the exponential), sums over L keys by L u: |error| <= (2 e + (L + 16) u) max|v|; errors of independent
    sign add in squares, so the 2-norm is held to 4 u (sqrt(hd) S + sqrt(L) + 16), S = max sum|q k| / sqrt(hd).
  log probabilities: |x - m| and log sum are rounded once (u relative each), the sum of V terms by at most
    (V/1024 + 32) u in threads, waves and workgroups, exp and log by 2^-22: |error| <= u (2 |x - m| + V/1024 + 64).
"""
import ctypes as C
import itertools

import numpy as np
import pytest

import batch_model as BM
from ronn_amd import _lib
from ronn_amd._lib import check
from ronn_amd.device import Context
from ronn_amd.kvcache import PagedKVCache

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


# ---- plan ------------------------------------------------------------------------------------------
def run_plan(ctx, length, new, table, ring, state, max_tokens, in_place=False, repeats=1):
    rows, max_blocks = table.shape
    i32 = lambda x: ctx.to_device(np.asarray(x, dtype=np.int32))  # noqa: E731
    d = dict(len=i32(length), new=i32(new), table=i32(table), ring=i32(ring), state=i32(state), start=i32([-9] * (rows + 2)),
             count=i32([-9, -9]), len_out=i32([-9] * rows), state_out=i32([-9, -9]))
    for k in ("row", "pos", "slot", "unit"):
        d[k] = i32([-9] * (max_tokens + 8))
    t = _lib.KvTable(rows, max_blocks, len(ring), d["table"].ptr, d["len"].ptr, d["ring"].ptr, d["state"].ptr)
    b = _lib.KvBatch(max_tokens, *(d[k].ptr for k in ("start", "row", "pos", "slot", "unit", "count")))
    lo, so = (d["len"], d["state"]) if in_place else (d["len_out"], d["state_out"])
    for _ in range(repeats):
        check(ctx.lib.rbn_kv_plan(ctx.handle, t, d["new"].ptr, b, lo.ptr, so.ptr))
    get = lambda buf, n: buf.download(np.int32, n)  # noqa: E731
    out = dict(table=get(d["table"], rows * max_blocks).reshape(rows, max_blocks), ring=get(d["ring"], len(ring)),
               start=get(d["start"], rows + 2), count=get(d["count"], 2), len_out=get(lo, rows), ring_state_out=get(so, 2),
               flags=ctx.device_flags())
    for k in ("row", "pos", "slot", "unit"):
        out[k] = get(d[k], max_tokens + 8)
    return out


def same_plan(got, want):
    tokens, units = len(want["row"]), len(want["unit"])
    assert list(got["count"]) == [tokens, units]
    assert (got["start"][:-1] == want["start"]).all() and got["start"][-1] == -9
    for k in ("row", "pos", "slot"):
        assert (got[k][:tokens] == want[k]).all(), k
        assert (got[k][tokens:] == -9).all(), k          # behind the last token: left as they were
    assert (got["unit"][:units] == want["unit"]).all() and (got["unit"][units:] == -9).all()
    for k in ("table", "ring", "len_out", "ring_state_out"):
        assert (got[k] == want[k]).all(), k
    assert got["flags"] == want["flags"]


def plan_case(rows, max_blocks, spare, hi_len, hi_new, seed, p_idle=0.2, p_end=0.2):
    rng = np.random.default_rng(seed)
    length = rng.integers(0, hi_len + 1, rows)
    new = rng.integers(1, hi_new + 1, rows)
    what = rng.random(rows)
    new[what < p_idle] = 0
    new[(what >= p_idle) & (what < p_idle + p_end)] = -rng.integers(1, 9)
    held = sum(BM.blocks(n) for n in length)
    pages = held + spare
    perm = rng.permutation(pages).astype(np.int32)
    table = np.full((rows, max_blocks), -5, np.int32)
    at = 0
    for r in range(rows):
        n = BM.blocks(length[r])
        table[r, :n] = perm[at:at + n]
        at += n
    head = int(rng.integers(0, pages))
    ring = np.full(pages, -6, np.int32)
    ring[(head + np.arange(spare)) % pages] = perm[held:]
    return length, new, table, ring, (head, spare)


@pytest.mark.parametrize("rows,hi_len,hi_new,max_tokens", [
    (1, 0, 1, 1), (1, 31, 1, 1), (3, 100, 40, 128), (64, 1000, 1, 64), (65, 500, 33, 3000), (1000, 900, 40, 40000),
    (2048, 300, 64, 131072), (2047, 40, 1, 2048), (5, 30000, 9000, 45000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(ctx, rows, hi_len, hi_new, max_tokens, in_place):
    case = plan_case(rows, BM.blocks(hi_len + hi_new), rows * BM.blocks(hi_new + 32), hi_len, hi_new, rows + hi_new)
    want = BM.plan(*case, max_tokens)
    assert want["flags"] == 0
    # not in place the call can be repeated: the second run gives the same
    same_plan(run_plan(ctx, *case, max_tokens, in_place, repeats=1 if in_place else 3), want)


@pytest.mark.parametrize("rows,spare,max_tokens,max_blocks", [
    (40, 5, 4000, 20), (40, 0, 4000, 20), (40, 400, 700, 20), (40, 60, 900, 17), (1500, 700, 20000, 20), (7, 1, 1, 20)])
def test_plan_refuses_what_does_not_fit(ctx, rows, spare, max_tokens, max_blocks):
    length, new, table, ring, state = plan_case(rows, 20, spare, 500, 100, 7 * rows + spare, p_idle=0.1, p_end=0.05)
    length = np.minimum(length, max_blocks * 32)
    table = np.ascontiguousarray(table[:, :max_blocks])
    want = BM.plan(length, new, table, ring, state, max_tokens)
    assert want["flags"] == _lib.FLAG_KV_REFUSED and (rows == 7 or len(want["row"]))
    same_plan(run_plan(ctx, length, new, table, ring, state, max_tokens), want)


def test_plan_all_idle_and_all_ended(ctx):
    length, new, table, ring, state = plan_case(30, 10, 12, 200, 10, 5)
    same_plan(run_plan(ctx, length, 0 * new, table, ring, state, 64), BM.plan(length, 0 * new, table, ring, state, 64))
    gone = 0 * new - 1
    want = BM.plan(length, gone, table, ring, state, 64)
    got = run_plan(ctx, length, gone, table, ring, state, 64)
    same_plan(got, want)
    assert got["ring_state_out"][1] == len(ring) and sorted(got["ring"]) == list(range(len(ring)))


def test_plan_huge_requests_do_not_wrap(ctx):
    length, new, table, ring, state = plan_case(50, 10, 40, 200, 10, 6, p_idle=0, p_end=0)
    new[::3] = 2 ** 31 - 1
    new[1::7] = -2 ** 31
    want = BM.plan(length, new, table, ring, state, 512)
    same_plan(run_plan(ctx, length, new, table, ring, state, 512), want)
    assert want["flags"] == _lib.FLAG_KV_REFUSED


def test_plan_bad_state_stays_inside(ctx):
    """Lengths, ring state and pages out of range: nothing is written outside the buffers (their guards stay), the rows
    concerned are left alone, and the flag says so."""
    length, new, table, ring, state = plan_case(20, 10, 80, 200, 10, 8, p_idle=0, p_end=0.2)
    bad_len = np.array(length)
    bad_len[[0, 5]] = [-1, 321]
    got = run_plan(ctx, bad_len, new, table, ring, state, 512)
    assert got["flags"] == _lib.FLAG_KV_BAD_INDEX
    assert (got["len_out"][[0, 5]] == [-1, 321]).all()
    assert got["start"][1] == got["start"][0] and got["start"][6] == got["start"][5]
    for st in ((-1, 80), (len(ring), 80), (0, -1), (0, len(ring) + 1)):
        got = run_plan(ctx, length, new, table, ring, st, 512)
        assert got["flags"] & _lib.FLAG_KV_BAD_INDEX, st
        assert 0 <= got["ring_state_out"][0] < len(ring) and 0 <= got["ring_state_out"][1] <= len(ring)
    got = run_plan(ctx, length, new, table, ring * 0 + 2 ** 30, state, 512)     # pages that do not exist
    assert got["flags"] == _lib.FLAG_KV_BAD_INDEX
    slots = got["slot"][:got["count"][0]]
    assert ((slots == -1) | ((slots >= 0) & (slots < 32 * len(ring)))).all() and (slots == -1).any()
    # every row ends although the ring is full already: nothing goes past it
    got = run_plan(ctx, length, 0 * new - 1, table, ring, (3, len(ring)), 512)
    assert got["flags"] == _lib.FLAG_KV_BAD_INDEX and got["ring_state_out"][1] == len(ring)
    assert (got["ring"] == ring).all()


# ---- store and attention ---------------------------------------------------------------------------
class Rig:
    """A cache on the device, its model, and random calls of both."""

    def __init__(self, ctx, heads, kv_heads, hd, fmt, rows, max_len=512, pages=None, max_tokens=256, theta=10000.0, seed=0):
        self.ctx, self.heads, self.kv_heads, self.hd, self.theta = ctx, heads, kv_heads, hd, theta
        self.rng = np.random.default_rng(seed)
        pages = pages or rows * BM.blocks(max_len)
        self.cache = PagedKVCache(ctx, 1, kv_heads, hd, rows, pages, max_len, max_tokens, fmt)
        self.model = BM.Cache(rows, kv_heads, hd, fmt)
        self.rows, self.max_tokens = rows, max_tokens
        self.length = np.zeros(rows, int)
        # whatever is in the buffers before counts for nothing: NaN patterns
        for buf in self.cache.buffers[0]:
            check(ctx.lib.rbn_fill_u8(ctx.handle, buf.ptr, 0xFF, buf.nbytes))
        self.width = (heads + 2 * kv_heads) * hd
        self.d_new = ctx.alloc(4 * rows)
        self.d_q = ctx.alloc(4 * max_tokens * heads * hd)
        self.d_out = ctx.alloc(4 * max_tokens * heads * hd)

    def qkv(self, tokens):
        x = self.rng.normal(0, 1, (tokens, self.width)).astype(np.float32)
        x[:, ::7] *= 3.0
        return x

    def step(self, new, x=None):
        """Plans and stores `new` tokens per row; x: their (q | k | v) in row order."""
        new = np.asarray(new, dtype=np.int32)
        tokens = int(new[new > 0].sum())
        x = self.qkv(tokens) if x is None else x
        pad = np.full((self.max_tokens, self.width), np.nan, np.float32)     # behind the last token: never used
        pad[:tokens] = x
        self.d_new.upload(new)
        d_qkv = self.ctx.to_device(pad)
        self.cache.plan(self.d_new)
        check(self.ctx.lib.rbn_fill_u8(self.ctx.handle, self.d_q.ptr, 0xFE, self.d_q.nbytes))
        self.cache.store(0, d_qkv, self.heads, self.theta, self.d_q)
        q = self.d_q.download(np.uint32, self.max_tokens * self.heads * self.hd)
        assert (q[tokens * self.heads * self.hd:] == 0xFEFEFEFE).all()
        assert (d_qkv.download(np.uint32, pad.size) == pad.view(np.uint32).ravel()).all()
        q = q[:tokens * self.heads * self.hd].view(np.float32).reshape(tokens, self.heads, self.hd)
        self.token_row, self.token_pos = [], []
        at = 0
        want_q = np.zeros(q.shape)
        for r in range(self.rows):
            n = int(new[r])
            if n < 0:
                self.model.end(r)
                self.length[r] = 0
            if n <= 0:
                continue
            pos = np.arange(self.length[r], self.length[r] + n)
            y = x[at:at + n].reshape(n, -1, self.hd)
            with np.errstate(invalid="ignore"):
                self.model.append(r, BM.rope64(y[:, self.heads:self.heads + self.kv_heads], pos, self.theta),
                                  y[:, self.heads + self.kv_heads:])
            want_q[at:at + n] = BM.rope64(y[:, :self.heads], pos, self.theta)
            self.token_row += [r] * n
            self.token_pos += list(pos)
            self.length[r] += n
            at += n
        # each product and the sum rounded once, cos and sin to a few u
        assert np.abs(q - want_q).max(initial=0) <= 12 * U * np.abs(x[:, :self.heads * self.hd]).max(initial=0) * 2
        return q

    def check_cache(self, exact_k=False):
        assert (self.cache.lengths() == self.length).all()
        for r in range(self.rows):
            n = self.length[r]
            if n == 0:
                continue
            k, v = self.cache.read(0, np.full(n, r), np.arange(n))
            want_k, want_v = self.model.values(r)
            assert (v == want_v.astype(np.float16)).all(), r
            if exact_k:
                assert (k == want_k.astype(np.float16)).all(), r
                continue
            # one f16 step in the open block; in a full one a code may be off by one and the scale by 2^-10
            step = np.abs(want_k) * 2.0 ** -10 + 2.0 ** -24
            for b in range(n // 32):
                for h in range(self.kv_heads):
                    at = (slice(32 * b, 32 * b + 32), h)
                    m = np.abs(self.model.x[r][0][at].astype(np.float64)).max()
                    if self.model.fmt == "i8":
                        step[at] = m / 127 + np.abs(want_k[at]) * 2.0 ** -9 + 2.0 ** -24
                    else:       # one e4m3 step: 2^-3 relative at most, 2^-9 of the scale below its normal range
                        step[at] = np.abs(want_k[at]) * (2.0 ** -3 + 2.0 ** -9) + m / 448 * 2.0 ** -9 + 2.0 ** -24
            off = np.abs(k.astype(np.float64) - want_k)
            assert (off <= step * 1.001).all(), (r, off.max())
            assert (off > np.abs(want_k) * 2.0 ** -9 + 2.0 ** -24).mean() < 0.01      # and hardly any is off at all

    def device_values(self, r):
        """K and V of a row as the cache holds them, codes times scales in 64 bits."""
        n, c = self.length[r], self.cache
        table = c.d_table.download(np.int32, self.rows * c.max_blocks).reshape(self.rows, c.max_blocks)
        out = []
        for which in (0, 1):
            codes = c.buffers[0][which].download(np.uint8, c.pages * self.kv_heads * 32 * self.hd).reshape(
                c.pages, self.kv_heads, -1)
            scale = c.buffers[0][4 + which].download(np.float32, c.pages * self.kv_heads).reshape(c.pages, -1)
            opened = c.buffers[0][2 + which].download(np.float16, self.rows * self.kv_heads * 32 * self.hd).reshape(
                self.rows, self.kv_heads, 32, self.hd)
            t, d = np.meshgrid(np.arange(32), np.arange(self.hd), indexing="ij")
            if which == 0:
                at = ((t // 16 * (self.hd // 64) + d // 64) * 64 + d % 32 // 8 * 16 + t % 16) * 16 + d // 32 % 2 * 8 + d % 8
            else:
                at = (d // 32 * 64 + t % 16 // 4 * 16 + d % 16) * 16 + d // 16 % 2 * 8 + t // 16 * 4 + t % 4
            rows = []
            for b in range(BM.blocks(n)):
                if 32 * b + 32 <= n:
                    raw = codes[table[r, b]][:, at]
                    value = raw.view(np.int8).astype(np.float64) if c.fmt == "i8" else BM.e4m3_values()[raw]
                    rows.append((value * scale[table[r, b]][:, None, None].astype(np.float64)).transpose(1, 0, 2))
                else:
                    rows.append(opened[r, :, :n % 32].astype(np.float64).transpose(1, 0, 2))
            out.append(np.concatenate(rows))
        return out

    def attend(self, q, max_new):
        tokens = len(q)
        check(self.ctx.lib.rbn_fill_u8(self.ctx.handle, self.d_out.ptr, 0xFE, self.d_out.nbytes))
        self.cache.attend(0, self.d_q, self.heads, max_new, self.d_out)
        out = self.d_out.download(np.uint32, self.max_tokens * self.heads * self.hd)
        assert (out[tokens * self.heads * self.hd:] == 0xFEFEFEFE).all()
        return out[:tokens * self.heads * self.hd].view(np.float32).reshape(tokens, self.heads, self.hd)

    def check_attention(self, q, max_new, sample=40):
        out = self.attend(q, max_new)
        assert np.isfinite(out).all()
        pick = np.arange(len(q))
        if len(pick) > sample:
            pick = np.unique(np.concatenate([pick[:4], pick[-4:], self.rng.choice(pick, sample)]))
        for r in sorted({self.token_row[i] for i in pick}):
            mine = [i for i in pick if self.token_row[i] == r]
            k, v = self.device_values(r)
            close_attention(out[mine], q[mine], [self.token_pos[i] for i in mine], k, v)


def close_attention(out, q, pos, k, v):
    want = BM.attention(q, pos, k, v)
    hd, group = q.shape[2], q.shape[1] // k.shape[1]
    s = max(float((np.abs(k[:, h // group]) @ np.abs(q[:, h]).T.astype(np.float64)).max()) for h in range(q.shape[1])) / np.sqrt(hd)
    n = max(pos) + 1
    off = np.abs(out - want)
    assert off.max() <= (2 * (hd + 8) * U * s + (n + 16) * U) * np.abs(v).max(), (off.max(), s)
    assert np.linalg.norm(off) <= 4 * U * (np.sqrt(hd) * s + np.sqrt(n) + 16) * np.linalg.norm(want)


SHAPES = [(4, 4, 128, "i8"), (4, 1, 64, "e4m3"), (20, 5, 128, "e4m3"), (6, 2, 64, "i8")]


@pytest.mark.parametrize("heads,kv_heads,hd,fmt", SHAPES + [(7, 1, 128, "i8"), (34, 2, 64, "i8")])
def test_store_in_calls_of_any_size(ctx, heads, kv_heads, hd, fmt):
    rig = Rig(ctx, heads, kv_heads, hd, fmt, rows=5, seed=heads)
    for new in ([3, 0, 32, 1, 65], [1, 1, 1, 0, 1], [28, 31, 2, 64, 30], [1, 33, 0, 100, 96], [0, 0, -1, 0, 1],
                [31, 5, 70, -3, 32], [2, 40, 26, 1, 1]):
        rig.step(new)
        rig.check_cache()
    assert ctx.device_flags() == 0


@pytest.mark.parametrize("heads,kv_heads,hd,fmt", SHAPES)
def test_cache_does_not_depend_on_the_calls(ctx, heads, kv_heads, hd, fmt):
    """The same tokens in one call, token by token and in odd chunks: the same codes, scales, open block and rotated q."""
    total, bits = 101, []
    for chunks in ([101], [1] * 101, [30, 5, 31, 35], [33, 64, 4], [32, 32, 32, 5]):
        rig = Rig(ctx, heads, kv_heads, hd, fmt, rows=1, max_len=128, pages=4, max_tokens=128, seed=9)
        x, at, q = np.random.default_rng(1).normal(0, 1, (total, rig.width)).astype(np.float32), 0, []
        for n in chunks:
            q.append(rig.step([n], x[at:at + n]))
            at += n
        pages = rig.cache.d_table.download(np.int32, 4)
        got = [np.concatenate(q).view(np.uint32)]
        for which in (0, 1):
            codes = rig.cache.buffers[0][which].download(np.uint8, 4 * kv_heads * 32 * hd).reshape(4, -1)
            scale = rig.cache.buffers[0][4 + which].download(np.uint32, 4 * kv_heads).reshape(4, -1)
            opened = rig.cache.buffers[0][2 + which].download(np.uint16, kv_heads * 32 * hd).reshape(kv_heads, 32, hd)
            got += [codes[pages[:3]], scale[pages[:3]], opened[:, :total % 32]]
        bits.append(got)
    for other in bits[1:]:
        assert all((a == b).all() for a, b in zip(other, bits[0]))


def test_store_saturates_and_flags(ctx):
    rig = Rig(ctx, 2, 1, 64, "i8", rows=2, seed=4)
    x = rig.qkv(40)
    v = 3 * 64                                    # first column of v
    x[3, v + 5], x[7, v + 6], x[9, v + 1], x[39, v] = np.nan, np.inf, -1e6, 65519.0
    with np.errstate(invalid="ignore", over="ignore"):
        rig.step([40, 0], x)
    rig.check_cache()
    assert ctx.device_flags() == _lib.FLAG_KV_NONFINITE
    x = rig.qkv(33)
    x[5, v:] = 65504.0                             # the largest f16 itself, and what rounds to it, is no saturation
    x[32, v + 3] = -65519.9
    rig.step([0, 33], x)
    rig.check_cache()
    assert ctx.device_flags() == 0


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_store_of_zeros_and_tiny_values(ctx, fmt):
    rig = Rig(ctx, 1, 1, 64, fmt, rows=3, seed=5)
    x = rig.qkv(96)
    x[:32, 64:] = 0.0                              # scale 0
    x[32:64, 64:] = -0.0
    x[64:, 64:] *= 1e-7                            # below f16's normal range
    rig.step([32, 32, 32], x)
    rig.check_cache()
    q = rig.step([1, 1, 1])
    rig.check_attention(q, 1)


def test_far_positions_are_rotated_by_their_own_angle(ctx):
    """Position 2^25 - 2: the angle has 25 bits before the point, f32 would keep none behind it."""
    max_blocks = _lib.KV_MAX_BLOCKS
    pos0 = max_blocks * 32 - 2
    heads, hd = 2, 64
    i32 = lambda x: ctx.to_device(np.asarray(x, dtype=np.int32))  # noqa: E731
    table = ctx.alloc(4 * max_blocks)
    length = i32([pos0 + 2])
    arrays = [i32(x) for x in ([0, 2], [0, 0], [pos0, pos0 + 1], [64, 65], [0, -1], [2, 1])]
    t = _lib.KvTable(1, max_blocks, 4, table.ptr, length.ptr, None, None)
    b = _lib.KvBatch(2, *(a.ptr for a in arrays))
    bufs = [ctx.alloc(n) for n in (4 * 32 * hd, 4 * 32 * hd, 32 * hd * 2, 32 * hd * 2, 16, 16)]
    ctx.to_device(np.zeros(1))
    l = _lib.KvLayer(0, 1, hd, 0, *(x.ptr for x in bufs))
    check(ctx.lib.rbn_fill_u8(ctx.handle, bufs[2].ptr, 0, bufs[2].nbytes))
    check(ctx.lib.rbn_fill_u8(ctx.handle, bufs[3].ptr, 0, bufs[3].nbytes))
    x = np.random.default_rng(0).normal(0, 1, (2, (heads + 2) * hd)).astype(np.float32)
    d_q = ctx.alloc(4 * 2 * heads * hd)
    for theta in (10000.0, 500000.0):
        check(ctx.lib.rbn_rope_kv_store_q8(ctx.handle, ctx.to_device(x).ptr, t, b, l, heads, theta, d_q.ptr))
        q = d_q.download(np.float32, 2 * heads * hd).reshape(2, heads, hd)
        want = BM.rope64(x.reshape(2, -1, hd)[:, :heads], [pos0, pos0 + 1], theta)
        # theta^(-2i/hd) is off by a few 2^-53, times 2^25 turns at most: 2^-26; then as at near positions
        assert np.abs(q - want).max() <= (12 * U + 2.0 ** -25) * 2 * np.abs(x).max()


@pytest.mark.parametrize("heads,kv_heads,hd,fmt", SHAPES + [(8, 8, 64, "i8"), (16, 1, 128, "i8"), (40, 2, 128, "e4m3")])
@pytest.mark.parametrize("news", [
    ([1, 1, 1], [1, 1, 1]),                                     # the very first token of a row
    ([30, 31, 32], [1, 1, 1], [1, 1, 1], [1, 1, 1]),            # over the end of a block, token by token
    ([63, 64, 65], [2, 3, 1], [5, 0, 8]),                       # a few tokens at once
    ([200, 1, 129], [33, 70, 64], [1, 100, 2]),                 # prompts on top of what is there, mixed with single tokens
])
def test_attention(ctx, heads, kv_heads, hd, fmt, news):
    rig = Rig(ctx, heads, kv_heads, hd, fmt, rows=3, max_tokens=352, seed=len(news) + heads)
    for i, new in enumerate(news):
        q = rig.step(new)
        if i or max(new) < 40 or hd == 64:
            for hint in {max(new), 1, 1000}:                    # the hint picks kernels, not results
                rig.check_attention(q, hint)
    assert ctx.device_flags() == 0


@pytest.mark.parametrize("rows,length,kv_heads,heads,hd", [(1, 5000, 2, 8, 128), (1, 9001, 1, 1, 64), (2, 4100, 4, 4, 128),
                                                             (40, 700, 5, 10, 64)])
def test_attention_long_rows(ctx, rows, length, kv_heads, heads, hd):
    """Keys split over workgroups: the rows go in by prompts, then single tokens and a prompt on top."""
    rig = Rig(ctx, heads, kv_heads, hd, "i8", rows=rows, max_len=length + 200, max_tokens=max(1024, 64 * rows), seed=rows)
    left = length
    while left:
        n = min(left, 1024 // rows)
        q = rig.step([n] * rows)
        left -= n
    rig.check_attention(q, n, sample=6)
    for _ in range(2):
        q = rig.step([1] * rows)
        rig.check_attention(q, 1, sample=6)
    q = rig.step([40 if r % 3 == 0 else r % 3 - 1 for r in range(rows)])
    rig.check_attention(q, 40, sample=6)


def test_attention_with_dominant_and_extreme_scores(ctx):
    """One key far above the others, scores of +-1e4, and queries whose sizes lie many powers of two apart."""
    rig = Rig(ctx, 4, 2, 128, "i8", rows=2, max_tokens=256, seed=11)
    rig.step([150, 77])
    x = rig.qkv(5)
    for i, factor in enumerate((300.0, 1e-30, 1e4, 1e-6, 0.0)):
        x[i, :4 * 128] *= factor
    q = rig.step([4, 1], x)
    # the bound grows with the scores; the largest are taken apart so that the small ones keep a tight one
    out = rig.attend(q, 4)
    assert np.isfinite(out).all()
    for i in range(5):
        r, p = rig.token_row[i], rig.token_pos[i]
        k, v = rig.device_values(r)
        want = BM.attention(q[i:i + 1], [p], k, v)
        s = np.abs(q[i]).max() * np.abs(k).max() * 128 / np.sqrt(128)
        assert np.abs(out[i] - want[0]).max() <= (2 * (128 + 8) * U * s + 300 * U) * np.abs(v).max(), i


def test_attention_keeps_a_nan_query_to_itself(ctx):
    rig = Rig(ctx, 4, 2, 128, "i8", rows=2, max_tokens=256, seed=12)
    for new, hint in (([50, 40], 50), ([1, 1], 1), ([3, 3], 3)):
        x = rig.qkv(sum(new))
        x[1, 5] = np.nan                      # head 0 of the second token
        rig.step(new, np.nan_to_num(x))
        q = rig.d_q.download(np.float32, sum(new) * 512).reshape(-1, 4, 128)
        q[1, 0, 5] = np.nan
        rig.d_q.upload(q)
        out = rig.attend(q, hint)
        assert np.isnan(out[1, 0]).all()
        out[1, 0], q[1, 0, 5] = 0, 0
        assert np.isfinite(out).all()


def test_attention_without_pages(ctx):
    """Pages out of range are left out: a token that keeps some blocks attends to those, one that keeps none gets zeros."""
    rig = Rig(ctx, 2, 1, 64, "i8", rows=3, max_tokens=256, seed=13)
    rig.step([64, 70, 64])
    table = rig.cache.d_table.download(np.int32, 3 * rig.cache.max_blocks).reshape(3, -1)
    for hint, new in ((1, [1, 1, 32]), (64, [20, 1, 32])):
        q = rig.step(new)
        bad = rig.cache.d_table.download(np.int32, table.size).reshape(3, -1)
        keep = bad.copy()
        bad[0, 0], bad[2, :] = -1, 2 ** 30
        n2 = rig.length[2]
        assert n2 % 32 == 0                         # the third row has full blocks only, and none with a page
        rig.cache.d_table.upload(bad)
        out = rig.attend(q, hint)
        rig.cache.d_table.upload(keep)
        assert ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX
        for i in range(len(q)):
            r, p = rig.token_row[i], rig.token_pos[i]
            k, v = rig.device_values(r)
            if r == 2:
                assert (out[i] == 0).all()
                continue
            if r == 0:
                k, v, p = k[32:], v[32:], p - 32
            close_attention(out[i:i + 1], q[i:i + 1], [p], k, v)
    assert ctx.device_flags() == 0


def test_store_and_read_without_pages(ctx):
    rig = Rig(ctx, 2, 1, 64, "i8", rows=2, max_tokens=64, seed=14)
    rig.step([40, 20])
    before = [b.download(np.uint8, b.nbytes) for b in rig.cache.buffers[0]]
    rig.cache.d_slot.upload(np.array([-1] * 30 + [2 ** 31 - 1] * 34, dtype=np.int32))
    d_qkv = ctx.to_device(rig.qkv(64))
    rig.cache.store(0, d_qkv, 2, 1e4, rig.d_q)
    assert ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX
    for i in (0, 1, 4, 5):                         # no page and no scale was written
        assert (rig.cache.buffers[0][i].download(np.uint8, rig.cache.buffers[0][i].nbytes) == before[i]).all()
    k, v = rig.cache.read(0, [0, 0, -1, 2, 1, 1], [-1, 40, 0, 0, 20, 2 ** 31 - 1])
    assert (k == 0).all() and (v == 0).all() and ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX
    rig.cache.d_table.upload(np.full(rig.cache.max_blocks, 10 ** 6, dtype=np.int32))
    k, v = rig.cache.read(0, [0], [3])
    assert (k == 0).all() and (v == 0).all() and ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX


def test_pages_past_four_gigabytes(ctx):
    """Page numbers whose bytes lie past 2^32 in the code buffers."""
    kv_heads, hd, pages = 16, 128, 80000                     # 5.2 GB of codes each for K and V
    cache = PagedKVCache(ctx, 1, kv_heads, hd, 2, pages, 96, 128)
    ring = np.arange(pages, dtype=np.int32)[::-1].copy()     # the last pages first
    ring[:6] = [pages - 1, 0, pages - 2, 65537, 70000, 3]
    cache.d_ring.upload(ring)
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (128, 3 * kv_heads * hd)).astype(np.float32)
    d_q, d_out = ctx.alloc(4 * 128 * kv_heads * hd), ctx.alloc(4 * 128 * kv_heads * hd)
    model = BM.Cache(2, kv_heads, hd, "i8")
    d_new = ctx.to_device(np.array([64, 64], np.int32))
    cache.plan(d_new)
    cache.store(0, ctx.to_device(x), kv_heads, 1e4, d_q)
    assert (cache.d_table.download(np.int32, 6).reshape(2, 3)[:, :2] == ring[:4].reshape(2, 2)).all()
    y = x.reshape(128, 3, kv_heads, hd)
    for r in range(2):
        pos = np.arange(64)
        model.append(r, BM.rope64(y[64 * r:64 * r + 64, 1], pos, 1e4), y[64 * r:64 * r + 64, 2])
        k, v = cache.read(0, np.full(64, r), pos)
        assert (v == model.values(r)[1].astype(np.float16)).all()
    for hint in (1, 64):
        cache.attend(0, d_q, kv_heads, hint, d_out)
        out = d_out.download(np.float32, 128 * kv_heads * hd).reshape(128, kv_heads, hd)
        q = d_q.download(np.float32, 128 * kv_heads * hd).reshape(128, kv_heads, hd)
        for i in (0, 63, 64, 127):
            k, v = model.values(i // 64)
            want = BM.attention(q[i:i + 1], [i % 64], k, v)
            # K of the model may differ by a code step here and there: 2^-8 of the values
            assert np.abs(out[i] - want[0]).max() <= 2.0 ** -6 and np.linalg.norm(out[i] - want[0]) <= 0.02 * np.linalg.norm(want)
    assert ctx.device_flags() == 0


# ---- log probabilities -------------------------------------------------------------------------------
def run_logprobs(ctx, x, target, top, pitch=None, shift=0):
    rows, vocab = x.shape
    pitch = pitch or vocab
    buf = np.full(shift + rows * pitch, np.nan, np.float32)          # what lies between the rows is never looked at
    for r in range(rows):
        buf[shift + r * pitch:shift + r * pitch + vocab] = x[r]
    d_x, d_t = ctx.to_device(buf), ctx.to_device(np.asarray(target, dtype=np.int32))
    d = [ctx.to_device(np.full(n, -77, t)) for n, t in ((rows + 1, np.float32), (rows + 1, np.float32),
                                                          (rows * top + 1, np.int32), (rows * top + 1, np.float32))]
    check(ctx.lib.rbn_token_logprobs_f32(ctx.handle, d_x.ptr + 4 * shift, rows, vocab, pitch, d_t.ptr, top, d[0].ptr, d[1].ptr,
                                         d[2].ptr if top else None, d[3].ptr if top else None))
    lp, ent, tok, tlp = (b.download(t, n) for b, n, t in zip(d, (rows + 1, rows + 1, rows * top + 1, rows * top + 1),
                                                               (np.float32, np.float32, np.int32, np.float32)))
    for a in (lp, ent, tok, tlp):
        assert a[-1] == -77
    return lp[:-1], ent[:-1], tok[:-1].reshape(rows, top), tlp[:-1].reshape(rows, top)


def check_logprobs(ctx, x, target, top, **kw):
    got = run_logprobs(ctx, x, target, top, **kw)
    want = BM.logprobs(x, target, top)
    vocab = x.shape[1]
    assert (got[2] == want[2]).all()
    with np.errstate(invalid="ignore", over="ignore"):
        for g, w in ((got[0], want[0]), (got[1], want[1]), (got[3], want[3])):
            fine = np.isfinite(w.astype(np.float32))         # -6e38 is -inf as an f32
            assert (np.isnan(w) == np.isnan(g)).all() and (np.isfinite(g) == fine).all()
            assert (g[~fine & ~np.isnan(w)] == w.astype(np.float32)[~fine & ~np.isnan(w)]).all()
            bound = U * (2 * np.abs(w[fine]) + vocab / 1024 + 64)
            if w is want[1]:         # the entropy is a mean of |x - m| under p: its sums round like the others, times it
                bound = U * (np.abs(w[fine]) + 1) * (vocab / 1024 + 64)
            assert (np.abs(g[fine] - w[fine]) <= bound).all(), np.abs(g[fine] - w[fine]).max()


@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (2, 5, 8), (3, 63, 32), (1, 64, 0), (5, 1000, 20), (16, 32000, 5),
                                             (1, 32000, 32), (300, 4097, 3), (7, 100003, 20), (1, 262147, 8), (700, 2048, 1)])
def test_logprobs(ctx, rows, vocab, top):
    rng = np.random.default_rng(rows + vocab)
    x = (rng.normal(0, 3, (rows, vocab)) + rng.normal(0, 20, (rows, 1))).astype(np.float32)
    target = rng.integers(-2, vocab + 2, rows)
    check_logprobs(ctx, x, target, top)
    x[rng.random(x.shape) < 0.5] = -np.inf
    x[:, 0] = 1.0
    check_logprobs(ctx, x, target, top, pitch=vocab + 3, shift=1)        # rows at any 4-byte address


def test_logprobs_ties_take_the_lowest_index(ctx):
    rng = np.random.default_rng(1)
    for vocab in (50, 5000, 70001):
        x = rng.integers(0, 3, (4, vocab)).astype(np.float32)
        x[1] = 2.5                                                 # all equal
        x[2, :] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)     # both zeros are one value
        check_logprobs(ctx, x, [0, 1, 2, 3], 32)


def test_logprobs_sorted_rows(ctx):
    """The largest values next to each other, at the start, the end, or one stride apart: where a selection by lanes or
    stretches has most to keep."""
    for vocab in (4096, 40000, 131072):
        up = np.arange(vocab, dtype=np.float32) / vocab * 30
        rows = [up, up[::-1], np.roll(up, 777)]
        for stride in (64, 256, 1024, 4096):
            z = np.zeros(vocab, np.float32)
            z[5::stride] = 10 + np.arange(len(z[5::stride]), dtype=np.float32) / 100
            rows.append(z)
        check_logprobs(ctx, np.stack(rows), np.arange(len(rows)), 32)


def test_logprobs_special_values(ctx):
    inf, nan = np.inf, np.nan
    base = np.random.default_rng(2).normal(0, 1, 3000).astype(np.float32)
    x = np.stack([base] * 9)
    x[0, :] = -inf                       # nothing left
    x[1, :] = -inf
    x[1, 2000] = 3.0                     # one thing left
    x[2, 17] = nan
    x[3, 17] = inf
    x[4, 5:2900] = -inf
    x[5] = -3e38
    x[5, 1:3] = 3e38                     # differences beyond f32
    x[6] = np.finfo(np.float32).min      # masked by the lowest value everywhere: an even distribution
    x[7, :] = nan
    x[8, 100] = 200.0                    # everything else vanishes
    check_logprobs(ctx, x, [5, 2000, 17, 17, 2, 0, 9, 1, 100], 10)


def test_logprobs_parts_are_optional(ctx):
    x = np.random.default_rng(3).normal(0, 1, (3, 777)).astype(np.float32)
    want = BM.logprobs(x, [1, 2, 3], 4)
    d_x, d_t = ctx.to_device(x), ctx.to_device(np.array([1, 2, 3], np.int32))
    d_a, d_b, d_i = ctx.alloc(12), ctx.alloc(48), ctx.alloc(48)
    f = ctx.lib.rbn_token_logprobs_f32
    check(f(ctx.handle, d_x.ptr, 3, 777, 777, d_t.ptr, 0, d_a.ptr, None, None, None))
    assert np.allclose(d_a.download(np.float32, 3), want[0], rtol=1e-5)
    check(f(ctx.handle, d_x.ptr, 3, 777, 777, None, 0, None, d_a.ptr, None, None))
    assert np.allclose(d_a.download(np.float32, 3), want[1], rtol=1e-5)
    check(f(ctx.handle, d_x.ptr, 3, 777, 777, None, 4, None, None, d_i.ptr, d_b.ptr))
    assert (d_i.download(np.int32, 12).reshape(3, 4) == want[2]).all()


# ---- streams and graphs --------------------------------------------------------------------------------
def test_context_on_a_stream_of_the_callers(ctx):
    """A context on another context's stream is ordered with it: what one queues the other sees, without a wait."""
    hip = C.CDLL("libamdhip64.so")
    s = C.c_void_p()
    assert hip.hipStreamCreateWithFlags(C.byref(s), 1) == 0
    with Context(0, stream=s.value) as a, Context(0, stream=s.value) as b:
        x = np.random.default_rng(1).normal(0, 1, (400, 30000)).astype(np.float32)
        d_x = a.to_device(x)
        d_y = a.alloc(x.nbytes)
        d_lp, d_t = a.alloc(1600), a.to_device(np.zeros(400, np.int32))
        for _ in range(3):
            check(a.lib.rbn_fill_u8(a.handle, d_y.ptr, 0, x.nbytes))
            check(a.lib.rbn_d2d(a.handle, d_y.ptr, d_x.ptr, x.nbytes))
            check(b.lib.rbn_token_logprobs_f32(b.handle, d_y.ptr, 400, 30000, 30000, d_t.ptr, 0, d_lp.ptr, None, None, None))
        b.sync()
        want = BM.logprobs(x, [0] * 400, 0)[0]
        assert np.abs(d_lp.download(np.float32, 400) - want).max() <= 1e-4
        # it captures like any other
        a.graph_begin()
        check(a.lib.rbn_token_logprobs_f32(a.handle, d_y.ptr, 400, 30000, 30000, d_t.ptr, 0, d_lp.ptr, None, None, None))
        g = a.graph_end()
        for _ in range(2):
            check(a.lib.rbn_fill_u8(a.handle, d_lp.ptr, 0xFF, 1600))
            a.graph_launch(g)
            a.sync()
            assert np.abs(d_lp.download(np.float32, 400) - want).max() <= 1e-4
        a.graph_destroy(g)
        for d in (d_x, d_y, d_lp, d_t):
            d.free()
    assert hip.hipStreamSynchronize(s) == 0 and hip.hipStreamDestroy(s) == 0     # still the caller's
    with Context(0, stream=0) as z:                # the default stream
        d = z.to_device(np.arange(4, dtype=np.int32))
        assert (d.download(np.int32, 4) == np.arange(4)).all()
        d.free()


def test_captured_step_replays_for_other_lengths(ctx):
    """One captured step (plan, store, attend) replayed while the rows grow, end and start again, with eager calls and
    waits in between, against an eager twin: the same bits."""
    rows, heads, kv_heads, hd = 4, 8, 2, 128
    rigs = [Rig(ctx, heads, kv_heads, hd, "i8", rows=rows, max_len=256, max_tokens=64, seed=21) for _ in range(2)]
    rng = np.random.default_rng(5)
    start = rng.normal(0, 1, (60, rigs[0].width)).astype(np.float32)
    for rig in rigs:
        rig.step([30, 1, 29, 0], start)
    d_qkv = ctx.alloc(4 * 64 * rigs[0].width)
    eager, captured = rigs

    def queue(rig):
        rig.cache.plan(rig.d_new)
        rig.cache.store(0, d_qkv, heads, 1e4, rig.d_q)
        rig.cache.attend(0, rig.d_q, heads, 64, rig.d_out)

    ctx.sync()
    ctx.graph_begin()
    queue(captured)
    g = ctx.graph_end()
    n = heads * hd
    for new in ([1, 1, 1, 0], [1, 1, 1, 40], [2, -1, 30, 1], [1, 33, 1, 1], [-1, 1, 1, 1], [50, 1, 1, -1]):
        tokens = sum(v for v in new if v > 0)
        d_qkv.upload(rng.normal(0, 1, (64, eager.width)).astype(np.float32))
        for rig in rigs:
            rig.d_new.upload(np.array(new, np.int32))
        queue(eager)
        ctx.graph_launch(g)
        ctx.sync()
        assert (eager.cache.lengths() == captured.cache.lengths()).all()
        a, b = (rig.d_out.download(np.uint32, tokens * n) for rig in rigs)
        assert (a == b).all() and np.isfinite(a.view(np.float32)).all()
        a, b = (rig.d_q.download(np.uint32, tokens * n) for rig in rigs)
        assert (a == b).all()
    ctx.graph_destroy(g)
    assert ctx.device_flags() == 0
