"""The batched serving operators where their work is dealt out in other ways than in test_gpu_batch.py: more entries than one look
takes in, more items than may be shared, long shares, scales far apart, several graphs and streams at once."""
import ctypes as C

import numpy as np
import pytest

import batch_model as BM
from ronn_amd import _lib
from ronn_amd._lib import check
from ronn_amd.device import Context
from test_gpu_batch import U, Rig, check_logprobs, close_attention, plan_case, run_plan, same_plan

pytestmark = pytest.mark.gpu


# ---- plan ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,max_tokens,spare", [(2048, 4096, 900), (130, 1024, 130), (64, 1023, 64), (65, 64, 0)])
def test_plan_fits_to_the_last_token_and_page(ctx, rows, max_tokens, spare):
    """Just what the batch and the pool hold, and one more."""
    rng = np.random.default_rng(rows)
    length, _, table, ring, state = plan_case(rows, 40, spare, 600, 1, rows, p_idle=0, p_end=0)
    new = np.zeros(rows, int)
    use = rng.permutation(rows)[:min(rows, max_tokens)]
    new[use] = 1
    left = max_tokens - len(use)
    need = lambda n: sum(BM.blocks(a + b) - BM.blocks(a) for a, b in zip(length, n))  # noqa: E731
    for r in use:
        more = min(left, 31)
        new[r] += more
        left -= more
    if spare:       # lengths such that the pages come out even
        while need(new) > spare:
            new[rng.choice(np.flatnonzero(new))] = 0
    want = BM.plan(length, new, table, ring, state, max_tokens)
    same_plan(run_plan(ctx, length, new, table, ring, state, max_tokens), want)
    for extra in (int(new.sum()), max(1, int(new.sum()) - 1)):      # the batch holds them just so, then one too few
        want = BM.plan(length, new, table, ring, state, extra)
        same_plan(run_plan(ctx, length, new, table, ring, state, extra), want)
    gone = new.copy()
    gone[rng.random(rows) < 0.3] = -1                               # refusals and returned pages in one call
    want = BM.plan(length, gone, table, ring, state, max(1, max_tokens // 2))
    same_plan(run_plan(ctx, length, gone, table, ring, state, max(1, max_tokens // 2)), want)


def test_plan_returns_the_pages_of_many_long_rows(ctx):
    length, new, table, ring, state = plan_case(900, 300, 50, 9600, 1, 3, p_idle=0.1, p_end=0.6)
    for max_tokens in (900, 64):
        want = BM.plan(length, new, table, ring, state, max_tokens)
        same_plan(run_plan(ctx, length, new, table, ring, state, max_tokens), want)


# ---- store -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,hd", [(40, 1, 64), (17, 1, 128), (128, 4, 64)])
def test_store_of_single_tokens_with_many_heads(ctx, heads, kv_heads, hd):
    """More query heads than the positions that share a token's work, at every place of a block."""
    rig = Rig(ctx, heads, kv_heads, hd, "i8", rows=3, max_tokens=64, seed=heads)
    rig.step([0, 14, 29])
    for _ in range(36):
        rig.step([1, 1, 1])
    rig.check_cache()
    assert ctx.device_flags() == 0


@pytest.mark.parametrize("heads,kv_heads,hd,fmt", [(4, 4, 128, "i8"), (40, 1, 64, "e4m3"), (17, 1, 128, "i8"), (6, 2, 64, "i8")])
def test_store_of_decode_steps(ctx, heads, kv_heads, hd, fmt):
    """Calls with no more tokens than rows: single tokens at every place of a block, now and then a few of one row over the end
    of one, rows that end and start again."""
    rows = 6
    rig = Rig(ctx, heads, kv_heads, hd, fmt, rows=rows, max_len=160, max_tokens=rows, seed=heads)
    rng = np.random.default_rng(heads)
    for step in range(90):
        new = np.ones(rows, int)
        if step % 9 == 4:
            new = np.zeros(rows, int)
            new[rng.integers(rows)] = rng.integers(2, rows + 1)
        elif step % 9 == 7:
            new = rng.permutation([2, 2, 1, 1, 0, 0])
        elif step % 20 == 19:
            new[rng.integers(rows)] = -1
        q = rig.step(new)
        if step % 10 == 0:
            rig.check_attention(q, int(new.max()), sample=6)
    rig.check_cache()
    assert ctx.device_flags() == 0


def test_store_of_a_decode_step_saturates_flags_and_checks(ctx):
    rig = Rig(ctx, 2, 1, 64, "i8", rows=4, max_tokens=4, seed=3)
    rig.step([1, 1, 1, 1])
    x = rig.qkv(4)
    x[0, 2 * 64 + 64 + 3], x[1, 2 * 64 + 64 + 5], x[2, 2 * 64 + 64 + 7] = np.nan, 1e9, -np.inf      # in v
    rig.step([1, 1, 1, 1], x)
    assert ctx.device_flags() == _lib.FLAG_KV_NONFINITE
    rig.check_cache()
    # slots without a page: flagged; units that are none: left out
    before = [b.download(np.uint8, b.nbytes) for b in rig.cache.buffers[0]]
    rig.cache.plan(rig.d_new)
    d_qkv = ctx.to_device(rig.qkv(4))
    rig.cache.d_unit.upload(np.array([-1, 4, 2 ** 31 - 1, -2 ** 31], np.int32))
    rig.cache.store(0, d_qkv, 2, 1e4, rig.d_q)
    assert ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX
    for b, was in zip(rig.cache.buffers[0], before):
        assert (b.download(np.uint8, b.nbytes) == was).all()
    rig.cache.d_unit.upload(np.arange(4, dtype=np.int32))
    rig.cache.d_slot.upload(np.array([-1, 2 ** 31 - 1, -1, -1], np.int32))
    rig.cache.store(0, d_qkv, 2, 1e4, rig.d_q)
    assert ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX
    for i in (0, 1, 4, 5):                         # no page and no scale
        assert (rig.cache.buffers[0][i].download(np.uint8, rig.cache.buffers[0][i].nbytes) == before[i]).all()


def test_read_of_any_places(ctx):
    """Places in any order, the same one twice, open and full blocks and none, over several workgroups."""
    rig = Rig(ctx, 3, 3, 64, "e4m3", rows=5, max_tokens=512, seed=4)
    rig.step([70, 1, 0, 96, 200])
    rng = np.random.default_rng(0)
    row, pos = rng.integers(-1, 6, 300), rng.integers(-2, 210, 300)
    pos[::50] = [2 ** 31 - 1, -2 ** 31, 69, 70, 199, 200]
    k, v = rig.cache.read(0, row, pos)
    values = {r: [x.astype(np.float16) for x in rig.device_values(r)] for r in (0, 1, 3, 4)}
    for i, (r, p) in enumerate(zip(row, pos)):
        there = r in values and 0 <= p < rig.length[r]
        assert (k[i] == (values[r][0][p] if there else 0)).all() and (v[i] == (values[r][1][p] if there else 0)).all(), (r, p)
    assert ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX


# ---- attention -------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,heads,kv_heads,hd,longest", [
    (300, 2, 2, 64, 90),          # entries over several looks, shared ones among them
    (300, 8, 8, 64, 90),          # ... and too many items to share
    (257, 8, 8, 64, 9000)])       # ... and a row whose waves have more than 64 blocks each
def test_attention_of_many_rows(ctx, rows, heads, kv_heads, hd, longest):
    rng = np.random.default_rng(rows + heads)
    held = rng.integers(1, 60, rows)
    held[rows // 2] = longest
    pages = sum(BM.blocks(n + 80) for n in held)
    rig = Rig(ctx, heads, kv_heads, hd, "i8", rows=rows, max_len=longest + 128, pages=pages, max_tokens=8192, seed=rows)
    left = held.copy()
    while left.any():                                  # in calls that fit
        new, room = np.zeros(rows, int), rig.max_tokens
        for r in np.flatnonzero(left):
            new[r] = min(left[r], room)
            room -= new[r]
        rig.step(new)
        left -= new
    q = rig.step([1] * rows)
    for hint in (1, 5):
        rig.check_attention(q, hint, sample=20)
    new = rng.choice([0, 1, 2, 17, 40], rows, p=[0.2, 0.3, 0.2, 0.2, 0.1])
    new[rows // 2] = 35
    q = rig.step(new)
    for hint in (40, 1):
        rig.check_attention(q, hint, sample=20)
    assert ctx.device_flags() == 0


def long_row(ctx, heads, kv_heads, hd, fmt, length, extra_rows=0, seed=1):
    rig = Rig(ctx, heads, kv_heads, hd, fmt, rows=1 + extra_rows, max_len=length + 256, max_tokens=4096, seed=seed)
    left = length
    while left:
        n = min(left, 4096)
        rig.step([n] + [0] * extra_rows)
        left -= n
    return rig


def test_attention_prompt_behind_a_very_long_row(ctx):
    """Shares of more than 64 blocks: 40000 positions before a prompt, whole and without some pages."""
    rig = long_row(ctx, 2, 1, 64, "i8", 40000)
    q = rig.step([50])
    rig.check_attention(q, 50, sample=8)
    q = rig.step([3])
    rig.check_attention(q, 3, sample=3)
    table = rig.cache.d_table.download(np.int32, rig.cache.max_blocks)
    q = rig.step([40])
    k, v = rig.device_values(0)
    table = rig.cache.d_table.download(np.int32, rig.cache.max_blocks)
    bad = table.copy()
    out_of = [0, 63, 64, 65, 200, 1000, 1200]          # pages of first, last and middle blocks of shares
    bad[out_of] = [-1, 2 ** 31 - 1, -2 ** 31, rig.cache.pages, -5, -1, -1]
    keep = np.ones(len(k), bool)
    for b in out_of:
        keep[32 * b:32 * b + 32] = False
    rig.cache.d_table.upload(bad)
    for hint in (40, 1):
        out = rig.attend(q, hint)
        assert ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX
        pick = [0, 20, 39]
        close_attention(out[pick], q[pick], [rig.token_pos[i] - 32 * len(out_of) for i in pick], k[keep], v[keep])
    rig.cache.d_table.upload(table)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_with_scales_far_apart(ctx, fmt, hd):
    """Blocks whose V (and K) are many powers of two apart or all zero, in any order: every part of the output as good as if its
    unit had always been the largest."""
    rig = Rig(ctx, 4, 2, hd, fmt, rows=2, max_tokens=1024, seed=hd)
    sizes = [1e-4, 1.0, 0.0, 3e3, 1e-6, 6e4, 0.0, 0.0, 1e-2, 1.0, 2e4, 1e-7]
    n = 32 * len(sizes)
    x = rig.qkv(2 * n)
    for r, order in enumerate((sizes, sizes[::-1])):
        for b, size in enumerate(order):
            part = x[r * n + 32 * b:r * n + 32 * b + 32, 4 * hd:]
            part[:, 2 * hd:] *= size / 4                     # V
            part[:, :2 * hd] *= 0.0 if size == 0.0 else 1.0 if size < 1 else 0.05
    x = np.clip(x, -6e4, 6e4)
    q = rig.step([n, n], x)
    rig.check_attention(q, n, sample=60)
    rig.check_attention(q, 1, sample=30)
    q = rig.step([33, 7])
    for hint in (33, 1):
        rig.check_attention(q, hint)
    assert ctx.device_flags() == 0


@pytest.mark.parametrize("heads,kv_heads,hd", [(3, 1, 128), (10, 2, 64), (7, 1, 64), (33, 3, 128), (18, 1, 128)])
def test_attention_prompts_of_odd_groups(ctx, heads, kv_heads, hd):
    """Heads per K/V head that do not divide into fours: workgroups whose four pairs lie in two or more blocks of positions."""
    rig = Rig(ctx, heads, kv_heads, hd, "i8", rows=4, max_len=2048, max_tokens=1024, seed=heads)
    rig.step([5, 300, 0, 31])
    q = rig.step([97, 64, 33, 1])
    for hint in (97, 1):
        rig.check_attention(q, hint, sample=60)
    rig.step([900, 0, 0, 0])
    q = rig.step([700, 20, 0, 200])
    rig.check_attention(q, 700, sample=60)
    assert ctx.device_flags() == 0


def test_attention_leaves_out_rows_behind_their_length(ctx):
    """Lengths from before the plan, as when its new lengths stand elsewhere and were not passed on: flagged, nothing written."""
    rig = Rig(ctx, 4, 2, 64, "i8", rows=3, max_tokens=160, seed=6)
    rig.step([40, 64, 31])
    q = rig.step([1, 40, 2])
    good = rig.cache.d_len.download(np.int32, 3)
    rig.cache.d_len.upload(np.array([40, 64, good[2]], np.int32))
    for hint in (40, 1):
        out = rig.attend(q, hint)
        assert ctx.device_flags() == _lib.FLAG_KV_BAD_INDEX
        raw = out.view(np.uint32)
        # a token at a time, those that end inside the length are answered; a row at a time, none
        assert (raw[0] == 0xFEFEFEFE).all() and (raw[1:41] == 0xFEFEFEFE).all()
        k, v = rig.device_values(2)
        close_attention(out[41:], q[41:], rig.token_pos[41:], k, v)
    rig.cache.d_len.upload(good)


@pytest.mark.parametrize("heads,kv_heads", [(200, 1), (1024, 1), (256, 256)])
def test_attention_of_many_heads(ctx, heads, kv_heads):
    rig = Rig(ctx, heads, kv_heads, 64, "i8", rows=2, max_len=128, max_tokens=64, seed=heads)
    q = rig.step([40, 20])
    rig.check_attention(q, 40, sample=4)
    q = rig.step([1, 13])
    for hint in (13, 1):
        rig.check_attention(q, hint, sample=4)
    rig.check_cache()
    assert ctx.device_flags() == 0


def test_cache_checks_its_buffers(ctx):
    rig = Rig(ctx, 4, 2, 64, "i8", rows=2, max_len=128, max_tokens=32)
    small, qkv = ctx.alloc(4), ctx.alloc(4 * 32 * rig.width)
    for call in (lambda: rig.cache.plan(small), lambda: rig.cache.store(0, small, 4, 1e4, rig.d_q),
                 lambda: rig.cache.store(0, qkv, 4, 1e4, small), lambda: rig.cache.store(1, qkv, 4, 1e4, rig.d_q),
                 lambda: rig.cache.store(-1, qkv, 4, 1e4, rig.d_q), lambda: rig.cache.attend(0, small, 4, 1, rig.d_out),
                 lambda: rig.cache.attend(0, rig.d_q, 4, 1, small), lambda: rig.cache.attend(2, rig.d_q, 4, 1, rig.d_out),
                 lambda: rig.cache.attend(0, rig.d_q, 8, 1, rig.d_out), lambda: rig.cache.read(1, [0], [0]),
                 lambda: rig.cache.batch(33), lambda: rig.cache.batch(0)):
        with pytest.raises(ValueError):
            call()


# ---- several at once -------------------------------------------------------------------------------
def test_two_graphs_of_a_context_share_its_workspace(ctx):
    """Two captured steps with shared rows, launched in turn without a wait, against eager calls: the same bits every time."""
    shapes = [(1, 3000, 4, 4), (2, 1500, 8, 2)]
    rigs = []
    for rows, length, heads, kv in shapes:
        rig = Rig(ctx, heads, kv, 64, "i8", rows=rows, max_len=length + 64, max_tokens=4096, seed=rows)
        rig.step([length] * rows)
        rig.q = rig.step([3] * rows)
        rigs.append(rig)
    want = [[rig.attend(rig.q, hint).view(np.uint32).copy() for hint in (1, 3)] for rig in rigs]
    graphs = []
    ctx.sync()
    for rig in rigs:
        for hint in (1, 3):
            ctx.graph_begin()
            rig.cache.attend(0, rig.d_q, rig.heads, hint, rig.d_out)
            graphs.append(ctx.graph_end())
    for trial in range(3):
        for h in range(2):
            for rig in rigs:
                check(ctx.lib.rbn_fill_u8(ctx.handle, rig.d_out.ptr, 0xFE, rig.d_out.nbytes))
            for i in range(2):
                ctx.graph_launch(graphs[2 * i + h])
                ctx.graph_launch(graphs[2 * (1 - i) + 1 - h] if trial == 1 else graphs[2 * i + h])
                ctx.graph_launch(graphs[2 * i + h])
            for i, rig in enumerate(rigs):
                n = want[i][h].size
                got = rig.d_out.download(np.uint32, n).reshape(want[i][h].shape)
                last = h if not (trial == 1 and i == 0) else 1 - h      # what was launched last into this output
                assert (got == want[i][last]).all(), (trial, h, i)
            rigs[0].cache.attend(0, rigs[0].d_q, rigs[0].heads, 1, rigs[0].d_out)      # eager work in between
    for g in graphs:
        ctx.graph_destroy(g)
    assert ctx.device_flags() == 0


def test_contexts_on_streams_of_their_own_at_the_same_time(ctx):
    """Each context has its own workspace: shared rows and shared logits on two streams at once."""
    with Context(0) as other:
        rigs = [Rig(c, 4, 2, 128, "e4m3", rows=2, max_len=4200, max_tokens=4096, seed=9) for c in (ctx, other)]
        for rig in rigs:
            rig.step([2048, 1000])
            rig.step([1500, 2000])
            rig.q = rig.step([1, 1])
        want = rigs[0].attend(rigs[0].q, 1).view(np.uint32).copy()
        x = np.random.default_rng(1).normal(0, 3, (3, 60000)).astype(np.float32)
        logits = [c.to_device(x) for c in (ctx, other)]
        outs = [c.alloc(4 * 96) for c in (ctx, other)]
        toks = [c.alloc(4 * 96) for c in (ctx, other)]
        for _ in range(20):
            for rig, d_x, d_t, d_o in zip(rigs, logits, toks, outs):
                rig.cache.attend(0, rig.d_q, 4, 1, rig.d_out)
                check(rig.ctx.lib.rbn_token_logprobs_f32(rig.ctx.handle, d_x.ptr, 3, 60000, 60000, None, 32, None, None, d_t.ptr,
                                                         d_o.ptr))
        top = BM.logprobs(x, [0, 0, 0], 32)
        for rig, d_t in zip(rigs, toks):
            rig.ctx.sync()
            assert (rig.d_out.download(np.uint32, want.size).reshape(want.shape) == want).all()
            assert (d_t.download(np.int32, 96).reshape(3, 32) == top[2]).all()
        for rig in rigs[1:]:
            for d in (logits[1], outs[1], toks[1]):
                d.free()


# ---- log probabilities -----------------------------------------------------------------------------
@pytest.mark.parametrize("vocab", [8191, 8192, 8193, 8196, 16383, 16384, 16385, 16391, 24577, 65537])
@pytest.mark.parametrize("rows", [1, 3, 600])
def test_logprobs_around_whole_sweeps(ctx, vocab, rows):
    if rows == 600 and vocab > 16391:
        rows = 300
    rng = np.random.default_rng(vocab + rows)
    x = rng.normal(0, 2, (rows, vocab)).astype(np.float32)
    x[0, -1], x[-1, 0] = 30.0, 31.0                # the largest at the very ends
    check_logprobs(ctx, x, rng.integers(0, vocab, rows), 20, pitch=vocab + 1, shift=3)


def test_logprobs_of_negative_and_nearly_equal_logits(ctx):
    """Group maxima that differ in their last bits only, all negative, denormal, or the lowest value but for a few."""
    rng = np.random.default_rng(8)
    vocab = 20000
    near = (-1.0 - rng.integers(0, 64, vocab) * 2.0 ** -23).astype(np.float32)
    tiny = (rng.integers(-60, 60, vocab) * 2.0 ** -149).astype(np.float32)
    low = np.full(vocab, np.finfo(np.float32).min, np.float32)
    low[[3, 9000, 19999]] = [-1.0, -1.0, 5.0]
    lonely = np.full(vocab, -np.inf, np.float32)
    lonely[[17, 8200]] = -3e38
    mixed = np.where(rng.random(vocab) < 0.999, -np.inf, rng.normal(-50, 1, vocab)).astype(np.float32)
    x = np.stack([near, tiny, low, lonely, mixed, -np.abs(rng.normal(0, 1e30, vocab)).astype(np.float32)])
    check_logprobs(ctx, x, [0, 1, 19999, 17, 5, 6], 32)


@pytest.mark.parametrize("mask", [-np.inf, -1e9, -10000.0, float(np.finfo(np.float32).min), 0.0])
def test_logprobs_of_masked_rows(ctx, mask):
    """Nearly all logits at one value, as a constrained choice leaves them: the rest by value, then the lowest indices; also with
    smaller logits at the front, NaN among them, and fewer left than are asked for in one stretch but not in another."""
    rng = np.random.default_rng(3)
    for vocab in (9000, 50021):
        x = np.full((8, vocab), mask, np.float32)
        for r, n in enumerate((0, 1, 5, 19, 20, 300, 40, 6)):
            at = rng.choice(vocab, n, replace=False)
            x[r, at] = rng.normal(5, 2, n)
        x[6, :50] = -2e9 if np.isfinite(mask) and mask > -1e30 else mask
        x[7, [3, 4000, 8999]] = np.nan
        check_logprobs(ctx, x, rng.integers(0, vocab, 8), 20)
        check_logprobs(ctx, x[:, :vocab - 3], rng.integers(0, vocab - 3, 8), 32, pitch=vocab + 2, shift=1)


def test_rows_of_one_block(ctx):
    """A table with a single block per row: nothing to share, the block is unfinished until the very last position."""
    rig = Rig(ctx, 6, 2, 64, "e4m3", rows=20, max_len=32, max_tokens=640, seed=2)
    rng = np.random.default_rng(1)
    q = rig.step(rng.integers(1, 20, 20))
    for hint in (1, 5, 32):
        rig.check_attention(q, hint, sample=60)
    for kind in range(3):
        q = rig.step([np.ones(20, int), 32 - rig.length, np.where(np.arange(20) % 3, 0, -1)][kind])
        for hint in (1, 40):
            rig.check_attention(q, hint) if len(q) else rig.attend(q, hint)
    rig.check_cache()
    assert ctx.device_flags() == 0
